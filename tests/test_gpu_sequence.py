"""Sequence operators (genie/sequence.py) on the GPU against their 64-bit references: packed causal attention and its single-token form over a cache, linear attention
with a decay per head and its recurrence.  Bounds: tests/sequence_ref.py."""
import math

import pytest
import torch

import sequence_ref as R

pytestmark = pytest.mark.gpu


def _gf():
    from genie import functional
    return functional


def _randn(*shape, seed, scale=1.0):
    return (torch.randn(shape, generator=torch.Generator(device='cuda').manual_seed(seed), device='cuda') * scale).to(torch.bfloat16)


def _cu(lens):
    return torch.tensor([0] + list(lens), dtype=torch.int32, device='cuda').cumsum(0).to(torch.int32)


def _packed_inputs(lens, spare, hq, hkv, d, seed, lens_k=None):
    n, m = sum(lens) + spare, sum(lens if lens_k is None else lens_k) + spare
    x = [_randn(n, hq, d, seed=seed), _randn(m, hkv, d, seed=seed + 1), _randn(m, hkv, d, seed=seed + 2), _randn(n, hq, d, seed=seed + 3)]
    for t in x:                                                   # what lies behind the last sequence must not matter
        if spare:
            t[t.shape[0] - spare:] = float('nan')
    return x


def _check_packed(lens, spare, hq, hkv, d, seed, lens_k=None, scale=None, grad=True):
    q, k, v, g = _packed_inputs(lens, spare, hq, hkv, d, seed, lens_k)
    cu, cuk = _cu(lens), None if lens_k is None else _cu(lens_k)
    val, tol = R.packed_reference(q, k, v, lens, d ** -0.5 if scale is None else scale, g if grad else None, lens_k)
    gf = _gf()
    with torch.no_grad():
        plain = gf.packed_attention(q, k, v, cu, scale=scale, cu_seqlens_k=cuk)
    R.assert_within(plain, val['out'], tol['out'], 'out')
    if not grad:
        return
    for t in (q, k, v):
        t.requires_grad_(True)
    out = gf.packed_attention(q, k, v, cu, scale=scale, cu_seqlens_k=cuk)
    assert torch.equal(out, plain)
    out.backward(g)
    for name, t in (('dq', q), ('dk', k), ('dv', v)):
        R.assert_within(t.grad, val[name], tol[name], name)


PACKED_LENS = [[1], [2], [64], [65], [129], [0, 5, 0], [127, 128, 1, 300, 64, 0, 7], [700]]


@pytest.mark.parametrize('lens', PACKED_LENS, ids=str)
@pytest.mark.parametrize('d', [64, 128])
def test_packed_attention_lengths(lens, d):
    _check_packed(lens, 3, 4, 2, d, 10)


@pytest.mark.parametrize('heads', [(1, 1), (8, 8), (6, 2), (7, 1), (9, 3), (20, 1)], ids=str)
@pytest.mark.parametrize('d', [8, 24, 32, 40, 64, 72, 96, 104, 128])
def test_packed_attention_heads_and_widths(heads, d):
    _check_packed([70, 1, 133], 0, *heads, d, 20)


@pytest.mark.parametrize('lens, lens_k', [([3, 5, 64], [200, 5, 130]), ([100], [3]), ([5, 130, 2], [0, 65, 400]), ([1, 1, 1], [1, 64, 257]), ([200], [1])], ids=str)
@pytest.mark.parametrize('d', [64, 128])
def test_packed_attention_other_keys_than_queries(lens, lens_k, d):
    """Continued prompts (more keys than queries) and queries that see nothing (fewer): their rows and gradients are zero."""
    _check_packed(lens, 2, 4, 2, d, 30, lens_k=lens_k)


@pytest.mark.parametrize('scale', [1e-3, 1.0, 3.0])
def test_packed_attention_scales(scale):
    """scale 3 on unit inputs: scores of +-100, weights of a few keys, maxima that arrive late in the sequence."""
    q, k, v, _ = _packed_inputs([500], 0, 2, 1, 64, 40)
    # scores up to ~150 in size: the exponent's fp32 error (|s| log2 e 2^-24 and the score's own sum, ~2^-14) is larger than the references' SLACK assumes
    val, tol = R.packed_reference(q, k, v, [500], scale)
    big = 2.0 ** -11 if scale == 3.0 else 0.0
    R.assert_within(_gf().packed_attention(q, k, v, _cu([500]), scale=scale), val['out'], tol['out'] + big * v.double().abs().amax(), 'out')


def test_packed_attention_late_maximum():
    """Scores that grow along the keys: the running maximum moves in every tile."""
    n = 640
    q, k, v, _ = _packed_inputs([n], 0, 2, 2, 64, 41)
    k *= torch.linspace(0.05, 4.0, n, device='cuda')[:, None, None].to(torch.bfloat16)
    q[:, :, :] = k.flip(0)
    val, tol = R.packed_reference(q, k, v, [n], 0.125)
    R.assert_within(_gf().packed_attention(q, k, v, _cu([n]), scale=0.125), val['out'], tol['out'] + 2.0 ** -11 * v.double().abs().amax(), 'out')


def test_packed_attention_many_sequences():
    """More sequences than one level of the slot search holds (63), most of them shorter than a tile."""
    lens = [(i * 37) % 90 for i in range(200)]
    _check_packed(lens, 5, 2, 1, 32, 50)


def test_packed_attention_long():
    """2048 keys and more: the sums of many tiles."""
    _check_packed([2100, 31], 0, 2, 1, 64, 60)


def test_packed_attention_layouts():
    """Slices of a fused projection, transposed heads, a broadcast value, an unaligned storage offset, an expanded gradient."""
    gf, lens, d = _gf(), [70, 30], 64
    n = sum(lens)
    fused = _randn(n, 4 + 2 + 2, d, seed=70).requires_grad_(True)
    q, k, v = fused[:, :4], fused[:, 4:6], fused[:, 6:]
    out = gf.packed_attention(q, k, v, _cu(lens))
    g = torch.ones((), dtype=torch.bfloat16, device='cuda').expand(out.shape)
    out.backward(g)
    val, tol = R.packed_reference(q.detach(), k.detach(), v.detach(), lens, d ** -0.5, g)
    R.assert_within(out, val['out'], tol['out'], 'out')
    R.assert_within(fused.grad, torch.cat([val[x] for x in ('dq', 'dk', 'dv')], 1), torch.cat([tol[x] for x in ('dq', 'dk', 'dv')], 1), 'dqkv')
    with torch.no_grad():
        heads_first = fused.detach().transpose(0, 1).contiguous().transpose(0, 1)
        assert torch.equal(gf.packed_attention(heads_first[:, :4], heads_first[:, 4:6], heads_first[:, 6:], _cu(lens)), out)
        pad = torch.empty(n * 8 * d + 3, dtype=torch.bfloat16, device='cuda')
        odd = pad[3:].view(n, 8, d)
        odd.copy_(fused.detach())
        assert torch.equal(gf.packed_attention(odd[:, :4], odd[:, 4:6], odd[:, 6:], _cu(lens)), out)
        one = _randn(1, 1, d, seed=71).expand(n, 2, d)                           # every key's value the same: the output is that value
        got = gf.packed_attention(q, k, one, _cu(lens))
        R.assert_within(got, one[:, :1].expand(n, 4, d).double(), (2 * R.U + R.SLACK) * one[:, :1].expand(n, 4, d).double().abs(), 'broadcast value')
        strided = torch.zeros(n, 8, 2 * d, dtype=torch.bfloat16, device='cuda')[..., ::2]
        strided.copy_(fused.detach())
        assert torch.equal(gf.packed_attention(strided[:, :4], strided[:, 4:6], strided[:, 6:], _cu(lens)), out)


def test_packed_attention_broadcast_input_gradient():
    """A key that all heads share by expand(): autograd sums the gradients of its copies."""
    gf, n, d = _gf(), 90, 64
    q, v, g = _randn(n, 4, d, seed=72), _randn(n, 4, d, seed=73), _randn(n, 4, d, seed=74)
    k = _randn(n, 1, d, seed=75).requires_grad_(True)
    gf.packed_attention(q, k.expand(n, 4, d), v, _cu([n])).backward(g)
    val, tol = R.packed_reference(q, k.detach().expand(n, 4, d), v, [n], d ** -0.5, g)
    # the four heads' gradients are rounded one by one (in tol) and their sum once more, pairwise at worst three times
    want = val['dk'].sum(1, keepdim=True)
    R.assert_within(k.grad, want, tol['dk'].sum(1, keepdim=True) + 3 * R.U * val['dk'].abs().sum(1, keepdim=True), 'dk')


def test_packed_attention_grouped_equals_repeated_keys():
    gf, lens, d = _gf(), [200, 57], 128
    q, k, v, _ = _packed_inputs(lens, 0, 6, 2, d, 80)
    a = gf.packed_attention(q, k, v, _cu(lens))
    b = gf.packed_attention(q, k.repeat_interleave(3, 1), v.repeat_interleave(3, 1), _cu(lens))
    assert torch.equal(a, b)


def test_packed_attention_is_causal_and_separates_sequences():
    """Changing a token changes nothing in front of it and nothing in the other sequences, to the bit."""
    gf, lens, d = _gf(), [100, 150, 60], 64
    q, k, v, _ = _packed_inputs(lens, 0, 2, 2, d, 90)
    a = gf.packed_attention(q, k, v, _cu(lens))
    k2, v2 = k.clone(), v.clone()
    k2[180] += 1
    v2[180] -= 3
    b = gf.packed_attention(q, k2, v2, _cu(lens))
    assert torch.equal(a[:180], b[:180]) and torch.equal(a[250:], b[250:]) and not torch.equal(a[180:250], b[180:250])


def test_packed_attention_empty_calls():
    gf = _gf()
    z = torch.zeros(0, 4, 64, dtype=torch.bfloat16, device='cuda')
    assert gf.packed_attention(z, z, z, _cu([])).shape == (0, 4, 64)
    assert gf.packed_attention(z, z, z, _cu([0, 0])).shape == (0, 4, 64)
    x = _randn(5, 4, 64, seed=1).requires_grad_(True)
    out = gf.packed_attention(x, x, x, _cu([]))                                   # rows, but no sequence
    assert torch.equal(out, torch.zeros_like(out))
    out.backward(torch.ones_like(out))
    assert torch.equal(x.grad, torch.zeros_like(x))
    y = _randn(5, 4, 64, seed=1)
    out = gf.packed_attention(y, z, z, _cu([5]), cu_seqlens_k=_cu([0]))           # queries, but no keys
    assert torch.equal(out, torch.zeros_like(out))


def test_packed_attention_partial_gradients_and_nan():
    gf, lens, d = _gf(), [90], 64
    q, k, v, g = _packed_inputs(lens, 0, 2, 2, d, 100)
    full = torch.autograd.grad(gf.packed_attention(q.requires_grad_(), k.requires_grad_(), v.requires_grad_(), _cu(lens)), (q, k, v), g)
    only = torch.autograd.grad(gf.packed_attention(q.detach(), k.detach(), v, _cu(lens)), v, g)[0]
    assert torch.equal(only, full[2])
    bad = q.detach().clone()
    bad[50, 1, 7] = float('nan')
    out = gf.packed_attention(bad, k.detach(), v.detach(), _cu(lens))
    assert torch.isnan(out[50, 1]).all() and torch.isfinite(out[:50]).all() and torch.isfinite(out[51:]).all() and torch.isfinite(out[50, 0]).all()


# ------------------------------------------------------------------------------------------------------------------------------------
# single token against a cache
# ------------------------------------------------------------------------------------------------------------------------------------
def _cache(b, cap, hkv, d, seed, layout='bthd'):
    if layout == 'bthd':
        return _randn(b, cap, hkv, d, seed=seed)
    return _randn(b, hkv, cap, d, seed=seed).transpose(1, 2)                      # heads outside tokens


@pytest.mark.parametrize('heads', [(1, 1), (8, 2), (16, 4), (5, 1), (20, 1), (8, 8)], ids=str)
@pytest.mark.parametrize('d', [8, 40, 64, 96, 128])
def test_cached_step_heads_and_widths(heads, d):
    gf, (hq, hkv), cap = _gf(), heads, 300
    lengths = [0, 1, 31, 32, 33, 150, 299, -1]
    b = len(lengths)
    q, kn, vn = _randn(b, hq, d, seed=1), _randn(b, hkv, d, seed=2), _randn(b, hkv, d, seed=3)
    kc, vc = _cache(b, cap, hkv, d, 4), _cache(b, cap, hkv, d, 5)
    for i, n in enumerate(lengths):                                               # what the caches hold from the length on must not matter
        kc[i, max(n, 0):] = float('nan')
        vc[i, max(n, 0):] = float('nan')
    want_k, want_v = kc.clone(), vc.clone()
    for i, n in enumerate(lengths):
        if n >= 0:
            want_k[i, n], want_v[i, n] = kn[i], vn[i]
    out = gf.cached_attention_step(q, kc, vc, torch.tensor(lengths, dtype=torch.int32, device='cuda'), kn, vn)
    assert torch.equal(kc.view(torch.int16), want_k.view(torch.int16)) and torch.equal(vc.view(torch.int16), want_v.view(torch.int16))
    val, tol = R.step_reference(q, kc, vc, [n + 1 for n in lengths], d ** -0.5)
    R.assert_within(out, val, tol, 'out')
    again = gf.cached_attention_step(q, kc, vc, torch.tensor([n + 1 if n >= 0 else -1 for n in lengths], dtype=torch.int32, device='cuda'))
    R.assert_within(again, val, tol, 'without a new token')


@pytest.mark.parametrize('layout', ['bthd', 'bhtd'])
@pytest.mark.parametrize('b, cap, n', [(1, 5000, 4990), (1, 70, 64), (3, 2000, 1024), (2, 20000, 19999), (40, 129, 128)])
def test_cached_step_split_lengths(layout, b, cap, n):
    """Caches that are split over blocks: few sequences, long contexts; contexts much shorter than their cache."""
    gf, hq, hkv, d = _gf(), 8, 2, 64
    q, kn, vn = _randn(b, hq, d, seed=1), _randn(b, hkv, d, seed=2), _randn(b, hkv, d, seed=3)
    kc, vc = _cache(b, cap, hkv, d, 4, layout), _cache(b, cap, hkv, d, 5, layout)
    for m in (n, 3):
        lengths = torch.full((b,), m, dtype=torch.int32, device='cuda')
        out = gf.cached_attention_step(q, kc, vc, lengths, kn, vn)
        val, tol = R.step_reference(q, kc, vc, [m + 1] * b, d ** -0.5)
        R.assert_within(out, val, tol, f'length {m}')


def test_cached_step_full_cache_says_nan_and_writes_nothing():
    gf, d = _gf(), 64
    for cap in (40, 1000):
        q, kn, vn = _randn(3, 4, d, seed=1), _randn(3, 2, d, seed=2), _randn(3, 2, d, seed=3)
        kc, vc = _cache(3, cap, 2, d, 4), _cache(3, cap, 2, d, 5)
        before = kc.clone(), vc.clone()
        lengths = torch.tensor([cap, cap + 7, -5], dtype=torch.int32, device='cuda')
        out = gf.cached_attention_step(q, kc, vc, lengths, kn, vn)
        assert torch.isnan(out[:2]).all() and torch.equal(out[2], torch.zeros_like(out[2]))
        assert torch.equal(kc, before[0]) and torch.equal(vc, before[1])
        out = gf.cached_attention_step(q, kc, vc, lengths)                        # without a new token a full cache is just full
        assert torch.isfinite(out[0]).all() and torch.isnan(out[1]).all()


def test_cached_step_late_maximum():
    gf, d, cap = _gf(), 64, 600
    q = _randn(2, 4, d, seed=1)
    kc, vc = _cache(2, cap, 1, d, 2), _cache(2, cap, 1, d, 3)
    kc *= torch.linspace(0.05, 4.0, cap, device='cuda')[None, :, None, None].to(torch.bfloat16)
    kc[:, -40:] = q[:, :1, None].reshape(2, 1, 1, d) * 2
    val, tol = R.step_reference(q, kc, vc, [cap, cap], 0.125)
    out = gf.cached_attention_step(q, kc, vc, torch.full((2,), cap, dtype=torch.int32, device='cuda'), scale=0.125)
    R.assert_within(out, val, tol + 2.0 ** -11 * vc.double().abs().amax(), 'out')


def test_prompt_then_steps_equal_the_whole_prompt():
    """As a session uses them: a packed prompt fills the caches, tokens are appended one at a time, a continued prompt follows -- the same as one long prompt."""
    gf, hq, hkv, d = _gf(), 8, 2, 64
    lens, steps = [70, 5], 4
    total = [n + steps for n in lens]
    q, k, v, _ = _packed_inputs(total, 0, hq, hkv, d, 110)
    whole = gf.packed_attention(q, k, v, _cu(total))
    val, tol = R.packed_reference(q, k, v, total, d ** -0.5)
    R.assert_within(whole, val['out'], tol['out'], 'whole')
    kc, vc = (torch.full((2, 128, hkv, d), float('nan'), dtype=torch.bfloat16, device='cuda') for _ in range(2))
    starts = [0, total[0]]
    for i, n in enumerate(lens):
        kc[i, :n], vc[i, :n] = k[starts[i]:starts[i] + n], v[starts[i]:starts[i] + n]
    lengths = torch.tensor(lens, dtype=torch.int32, device='cuda')
    for t in range(steps):
        at = [starts[i] + lens[i] + t for i in range(2)]
        out = gf.cached_attention_step(q[at], kc, vc, lengths, k[at], v[at])
        lengths += 1
        R.assert_within(out, val['out'][at], tol['out'][at], f'step {t}')
    rows = [r for i in range(2) for r in range(starts[i] + lens[i], starts[i] + total[i])]
    cont = gf.packed_attention(q[rows], k, v, _cu([steps, steps]), cu_seqlens_k=_cu(total))
    R.assert_within(cont, val['out'][rows], tol['out'][rows], 'continued prompt')


# ------------------------------------------------------------------------------------------------------------------------------------
# linear attention with a decay per head
# ------------------------------------------------------------------------------------------------------------------------------------
def _decays(h):
    """From no memory at all over a few tokens' to a perfect one."""
    return torch.tensor([-0.05, 0.0, float('-inf'), -3.0, -1e-3, -0.5, -40.0, -0.01][:h] if h <= 8 else [-2.0 ** -(i % 12) for i in range(h)], device='cuda')


def _check_decay(lens, spare, h, dk, dv, seed, state=False, grad=True):
    gf, n = _gf(), sum(lens) + spare
    q, k, v, g = _randn(n, h, dk, seed=seed), _randn(n, h, dk, seed=seed + 1), _randn(n, h, dv, seed=seed + 2), _randn(n, h, dv, seed=seed + 3)
    for t in (q, k, v, g):
        if spare:
            t[n - spare:] = float('nan')
    ld, scale = _decays(h), dk ** -0.5
    s0 = torch.randn((len(lens), h, dk, dv), generator=torch.Generator(device='cuda').manual_seed(seed), device='cuda') if state else None
    out, last = gf.decay_attention(q, k, v, ld, _cu(lens), initial_state=s0, return_state=True)
    R.assert_within(out, *R.decay_form(q, k, v, ld, lens, scale, state=s0), 'out')
    R.assert_within(last, *R.decay_state(k, v, ld, lens, s0), 'state')
    assert last.dtype == torch.float32 and not last.requires_grad
    if not grad:
        return
    for t in (q, k, v):
        t.requires_grad_(True)
    again = gf.decay_attention(q, k, v, ld, _cu(lens), initial_state=s0)
    assert torch.equal(again, out)
    again.backward(g)
    st = None if s0 is None else s0.transpose(2, 3)
    R.assert_within(q.grad, *R.decay_form(g, v.detach(), k.detach(), ld, lens, scale, state=st), 'dq')
    R.assert_within(k.grad, *R.decay_form(v.detach(), g, q.detach(), ld, lens, scale, reverse=True), 'dk')
    R.assert_within(v.grad, *R.decay_form(k.detach(), q.detach(), g, ld, lens, scale, reverse=True), 'dv')


@pytest.mark.parametrize('lens', [[1], [31], [64], [65], [0, 5, 0], [63, 128, 1, 300, 0, 96], [257], [1000, 256, 513]], ids=str)
@pytest.mark.parametrize('state', [False, True])
@pytest.mark.parametrize('d', [64, 128])
def test_decay_attention_lengths(lens, state, d):
    """Chunks of 64 and segments of 256 that end anywhere, with and without a state in front."""
    _check_decay(lens, 3, 4, d, d, 10, state)


@pytest.mark.parametrize('dk, dv', [(8, 8), (32, 32), (24, 64), (64, 40), (96, 96), (128, 64), (80, 104)])
@pytest.mark.parametrize('h', [1, 3, 8])
def test_decay_attention_widths(dk, dv, h):
    _check_decay([70, 400], 0, h, dk, dv, 20, True)


def test_decay_attention_many_sequences():
    _check_decay([(i * 37) % 90 for i in range(150)], 5, 2, 32, 32, 30, True)


def test_decay_attention_long():
    _check_decay([3000, 17], 0, 2, 64, 64, 40, False)


@pytest.mark.parametrize('lens', [[33100], [17000, 40], [8193]], ids=str)
def test_decay_attention_many_segments(lens):
    """More segments of 256 tokens than one step of the state scan takes (32, or 128 in sequences that long)."""
    _check_decay(lens, 0, 1, 16, 16, 45, True)


def test_decay_attention_layouts():
    gf, lens, d, h = _gf(), [70, 230], 64, 4
    fused = _randn(300, 3, h, d, seed=50).requires_grad_(True)
    q, k, v = fused.unbind(1)
    ld = _decays(h)
    out = gf.decay_attention(q, k, v, ld, _cu(lens))
    g = _randn(1, 1, 1, seed=51).expand(out.shape)
    out.backward(g)
    qd, kd, vd = fused.detach().unbind(1)
    R.assert_within(out, *R.decay_form(qd, kd, vd, ld, lens, d ** -0.5), 'out')
    for i, (x, y, z, rev) in enumerate([(g, vd, kd, False), (vd, g, qd, True), (kd, qd, g, True)]):
        R.assert_within(fused.grad[:, i], *R.decay_form(x, y, z, ld, lens, d ** -0.5, reverse=rev), 'qkv'[i])
    with torch.no_grad():
        pad = torch.empty(300 * h * d + 5, dtype=torch.bfloat16, device='cuda')
        odd = pad[5:].view(300, h, d)
        odd.copy_(qd)
        assert torch.equal(gf.decay_attention(odd, kd.contiguous(), vd.transpose(0, 1).contiguous().transpose(0, 1), ld, _cu(lens)), out)


def test_decay_attention_empty_calls():
    gf = _gf()
    z, ld = torch.zeros(0, 2, 64, dtype=torch.bfloat16, device='cuda'), _decays(2)
    s0 = torch.randn(2, 2, 64, 64, device='cuda')
    out, last = gf.decay_attention(z, z, z, ld, _cu([0, 0]), initial_state=s0, return_state=True)
    assert out.shape == z.shape and torch.equal(last, s0)
    x = _randn(5, 2, 64, seed=1).requires_grad_(True)
    out = gf.decay_attention(x, x, x, ld, _cu([]))
    out.backward(torch.ones_like(out))
    assert torch.equal(out, torch.zeros_like(out)) and torch.equal(x.grad, torch.zeros_like(x))


@pytest.mark.parametrize('b, h, dk, dv', [(1, 1, 8, 8), (1, 8, 64, 64), (3, 5, 80, 96), (40, 8, 128, 128), (2, 3, 128, 24), (300, 2, 32, 64)])
def test_decay_step(b, h, dk, dv):
    gf = _gf()
    q, k, v = _randn(b, h, dk, seed=1), _randn(b, h, dk, seed=2), _randn(b, h, dv, seed=3)
    ld = _decays(h)
    s = torch.randn((b, h, dk, dv), generator=torch.Generator(device='cuda').manual_seed(4), device='cuda')
    l = torch.exp(ld.double())[None, :, None, None]
    new = torch.where(l == 0, torch.zeros_like(s).double(), l * s.double()) + k.double()[..., None] * v.double()[..., None, :]
    val = dk ** -0.5 * (q.double()[..., None, :] @ new)[..., 0, :]
    # fp32 throughout, a hardware exponential (2^-21 of the decay) and one rounding of the output
    mag = l * s.double().abs() + (k.double()[..., None] * v.double()[..., None, :]).abs()
    tol = R.U * val.abs() + 2.0 ** -18 * dk ** -0.5 * (q.double().abs()[..., None, :] @ mag)[..., 0, :]
    keep, into = s.clone(), torch.full_like(s, float('nan'))
    out = gf.decay_attention_step(q, k, v, ld, s, new_state=into)
    assert torch.equal(s, keep)
    R.assert_within(out, val, tol, 'out')
    R.assert_within(into, new, 2.0 ** -20 * mag, 'state')
    assert torch.equal(gf.decay_attention_step(q, k, v, ld, s), out) and torch.equal(s, into)


def test_decay_prompt_then_steps_equal_the_whole_prompt():
    gf, h, d, lens, steps = _gf(), 4, 64, [300, 20], 3
    total = [n + steps for n in lens]
    n = sum(total)
    q, k, v = (_randn(n, h, d, seed=60 + i) for i in range(3))
    ld = torch.tensor([-0.05, -0.5, -1e-3, -2.0], device='cuda')
    val, tol = R.decay_form(q, k, v, ld, total, d ** -0.5)
    starts = [0, total[0]]
    rows = [r for i in range(2) for r in range(starts[i], starts[i] + lens[i])]
    out, state = gf.decay_attention(q[rows], k[rows], v[rows], ld, _cu(lens), return_state=True)
    R.assert_within(out, val[rows], tol[rows], 'prompt')
    mid = state.clone()
    for t in range(steps):
        at = [starts[i] + lens[i] + t for i in range(2)]
        R.assert_within(gf.decay_attention_step(q[at], k[at], v[at], ld, state), val[at], tol[at], f'step {t}')
    want, bound = R.decay_state(k, v, ld, total)
    R.assert_within(state, want, bound, 'state')
    rest = [r for i in range(2) for r in range(starts[i] + lens[i], starts[i] + total[i])]
    cont, last = gf.decay_attention(q[rest], k[rest], v[rest], ld, _cu([steps, steps]), initial_state=mid, return_state=True)
    R.assert_within(cont, val[rest], tol[rest], 'continued')
    R.assert_within(last, want, bound, 'continued state')


# ------------------------------------------------------------------------------------------------------------------------------------
# streams, graphs, repeatability, refusals, wrong lengths
# ------------------------------------------------------------------------------------------------------------------------------------
def _everything(q, k, v, g, kc, vc, lengths, ld, state, into, cu):
    gf = _gf()
    a = gf.packed_attention(q, k, v, cu)
    ga = torch.autograd.grad(a, (q, k, v), g)
    b = gf.cached_attention_step(q[:2].detach(), kc, vc, lengths, k[:2].detach(), v[:2].detach())
    h = q.shape[1]
    wide = [t.repeat_interleave(h // t.shape[1], 1) for t in (k, v)]
    c, last = gf.decay_attention(q, *wide, ld, cu, return_state=True)
    gc = torch.autograd.grad(c, (q, k, v), g)
    d = gf.decay_attention_step(q[:2].detach(), wide[0][:2].detach(), wide[1][:2].detach(), ld, state, new_state=into)
    return [a, *ga, b, c, last, *gc, d, into.clone()]


def _everything_inputs(rows, nseq, seed=0):
    hq, hkv, d = 4, 2, 64
    q, k, v = _randn(rows, hq, d, seed=seed).requires_grad_(True), _randn(rows, hkv, d, seed=seed + 1).requires_grad_(True), _randn(rows, hkv, d, seed=seed + 2).requires_grad_(True)
    kc, vc = _cache(2, 2000, hkv, d, seed + 3), _cache(2, 2000, hkv, d, seed + 4)
    state = torch.randn(2, hq, d, d, device='cuda')
    return dict(q=q, k=k, v=v, g=_randn(rows, hq, d, seed=seed + 5), kc=kc, vc=vc, lengths=torch.tensor([5, 1500], dtype=torch.int32, device='cuda'), ld=_decays(hq),
                state=state, into=torch.empty_like(state))


def test_results_repeat_to_the_bit_and_on_another_stream():
    x, cu = _everything_inputs(900, 3), _cu([300, 1, 599])
    first = [t.clone() for t in _everything(**x, cu=cu)]
    for a, b in zip(first, _everything(**x, cu=cu)):
        assert torch.equal(a, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = _everything(**x, cu=cu)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for a, b in zip(first, other):
        assert torch.equal(a, b)


def test_graph_replays_with_other_lengths():
    """One capture, forward and backward, replayed with other sequence lengths and cache lengths in the same buffers; eager work between the replays."""
    x = _everything_inputs(900, 3, seed=200)
    cu = _cu([300, 1, 599])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _everything(**x, cu=cu)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = _everything(**x, cu=cu)
    for lens, lengths in (([300, 1, 599], [5, 1500]), ([0, 0, 900], [0, 1999]), ([10, 20, 30], [700, 1]), ([450, 450, 0], [5, 1500])):
        cu.copy_(_cu(lens))
        x['lengths'].copy_(torch.tensor(lengths, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        kept = [t.clone() for t in got]
        for a, b in zip(kept, _everything(**x, cu=cu)):
            assert torch.equal(a, b)


def test_wrong_sequence_bounds_stay_inside_the_tensors():
    """cu_seqlens that descends, is negative or passes the rows: the entries are clamped -- wrong results, but the call returns and what follows is untouched."""
    gf = _gf()
    x = _everything_inputs(300, 3, seed=300)
    for bad in ([0, 5000, 100, 2 ** 30], [0, -7, 300, 12], [9, 300, 0, 300], [0, 2 ** 31 - 1, -2 ** 31, 300]):
        _everything(**x, cu=torch.tensor(bad, dtype=torch.int64, device='cuda').to(torch.int32))
    torch.cuda.synchronize()
    q = x['q'].detach()
    R.assert_within(gf.packed_attention(q, q, q, _cu([300])), *(t['out'] for t in R.packed_reference(q, q, q, [300], 0.125)), 'after')


def test_refusals():
    gf, d = _gf(), 64
    q, k = _randn(10, 4, d, seed=1), _randn(10, 2, d, seed=2)
    cu = _cu([10])
    for bad, msg in (((q, _randn(10, 3, d, seed=1), _randn(10, 3, d, seed=1), cu), 'no multiple'), ((q, k, k[:9], cu), 'differ'), ((q, k[:9], k[:9], cu), 'rows'),
                     ((q[..., :60].contiguous(), k[..., :60].contiguous(), k[..., :60].contiguous(), cu), 'multiple of 8'),
                     ((q, k, k, cu[None]), '1 axes'), ((q, k, k, cu[:0]), 'leading 0'), ((q, k[..., :32], k[..., :32], cu), 'head widths')):
        with pytest.raises(ValueError, match=msg):
            gf.packed_attention(*bad)
    with pytest.raises(TypeError, match='int32'):
        gf.packed_attention(q, k, k, cu.long())
    with pytest.raises(TypeError, match='bfloat16'):
        gf.packed_attention(q, k.half(), k.half(), cu)
    for s in (0.0, -1.0, math.inf, math.nan):
        with pytest.raises(ValueError, match='scale'):
            gf.packed_attention(q, k, k, cu, scale=s)
    with pytest.raises(ValueError, match='numbers of sequences'):
        gf.packed_attention(q, k, k, cu, cu_seqlens_k=_cu([5, 5]))
    kc, lengths = _cache(10, 20, 2, d, 3), torch.zeros(10, dtype=torch.int32, device='cuda')
    vc = kc.clone()
    with pytest.raises(ValueError, match='come together'):
        gf.cached_attention_step(q, kc, vc, lengths, k)
    with pytest.raises(ValueError, match='same memory'):
        gf.cached_attention_step(q, kc, kc, lengths, k, k)
    with pytest.raises(ValueError, match='expanded'):
        gf.cached_attention_step(q, kc[:1].expand(10, 20, 2, d), vc, lengths, k, k)
    with pytest.raises(ValueError, match='updated in place'):
        gf.cached_attention_step(q, torch.zeros(10, 20, 2, 2 * d, dtype=torch.bfloat16, device='cuda')[..., ::2], vc, lengths, k, k)
    with pytest.raises(RuntimeError, match='no backward'):
        gf.cached_attention_step(q.clone().requires_grad_(), kc, vc, lengths, k, k)
    ld = _decays(4)
    x = _randn(10, 4, d, seed=5)
    with pytest.raises(ValueError, match='each of the 4 heads'):
        gf.decay_attention(x, x, x, ld[:3], cu)
    with pytest.raises(RuntimeError, match='constants'):
        gf.decay_attention(x, x, x, ld.clone().requires_grad_(), cu)
    with pytest.raises(ValueError, match='initial_state must be'):
        gf.decay_attention(x, x, x, ld, cu, initial_state=torch.zeros(2, 4, d, d, device='cuda'))
    s = torch.zeros(10 * 4 * d * d + 64, device='cuda')
    a, b = s[:-64].view(10, 4, d, d), s[64:].view(10, 4, d, d)
    with pytest.raises(ValueError, match='overlaps'):
        gf.decay_attention_step(x, x, x, ld, a, new_state=b)
    with pytest.raises(ValueError, match='contiguous'):
        gf.decay_attention_step(x, x, x, ld, a.transpose(2, 3))
    with pytest.raises(RuntimeError, match='no backward'):
        gf.decay_attention_step(x.clone().requires_grad_(), x, x, ld, a)


def test_offsets_past_32_bits_in_a_long_cache():
    """A cache of over 2^32 bytes and 2^31 elements: the last sequence's last tokens, and the rows of a packed buffer whose strides make it as long."""
    gf, d, hkv, cap = _gf(), 128, 8, 1 << 19
    big = torch.empty((5, cap, hkv, d), dtype=torch.bfloat16, device='cuda')      # 2.7e9 elements, 5.4 GB
    big[4, :100].normal_()
    big[4, cap - 100:].normal_()
    lengths = torch.tensor([-1, -1, -1, -1, cap], dtype=torch.int32, device='cuda')
    view = big[:, cap - 100:]                                                     # the same memory as a cache of 100 tokens
    q = _randn(5, 8, d, seed=1)
    short = lengths.clamp(max=100)
    a = gf.cached_attention_step(q, view, view, short)
    val, tol = R.step_reference(q[4:], big[4:, cap - 100:], big[4:, cap - 100:], [100], d ** -0.5)
    R.assert_within(a[4:], val, tol, 'cache')
    # a packed buffer whose consecutive rows lie 2^20 elements apart
    rows = 2500
    wide = big.view(-1)[:rows << 20].view(rows, 1 << 20)[:, :hkv * d].unflatten(1, (hkv, d))
    wide.copy_(_randn(rows, hkv, d, seed=2))
    dense = wide.contiguous()
    assert torch.equal(gf.packed_attention(wide, wide, wide, _cu([rows])), gf.packed_attention(dense, dense, dense, _cu([rows])))
    ld = _decays(hkv)
    assert torch.equal(gf.decay_attention(wide, wide, wide, ld, _cu([rows])), gf.decay_attention(dense, dense, dense, ld, _cu([rows])))


@pytest.mark.parametrize('lens, spare', [([2, 2, 3], 0), ([1, 0, 31], 5), ([70, 130, 56], 0), ([256], 0)], ids=str)
@pytest.mark.parametrize('d', [32, 64, 80, 128])
def test_few_rows_round_nothing_but_their_results(lens, spare, d):
    """Up to 256 rows the weights go into the products with their rounding's remainder (U^2 of them is left), in the cached form always."""
    gf, w = _gf(), R.U ** 2
    q, k, v, g = _packed_inputs(lens, spare, 4, 2, d, 700)
    cu, rows, tiny = _cu(lens), sum(lens), 2.0 ** -100
    val, tol = R.packed_reference(q, k, v, lens, d ** -0.5, g, w=w)
    for t in (q, k, v):
        t.requires_grad_(True)
    out = gf.packed_attention(q, k, v, cu)
    grads = torch.autograd.grad(out, (q, k, v), g)
    for name, t in zip(('out', 'dq', 'dk', 'dv'), (out, *grads)):
        R.assert_within(t, val[name], tol[name] + tiny, name)
    decay = -torch.linspace(0.01, 0.5, 2, device='cuda')
    a, b, c = (x.detach()[:, :2].clone().requires_grad_(True) for x in (q, k, v))
    out = gf.decay_attention(a, b, c, decay, cu)
    da, db, dc = torch.autograd.grad(out, (a, b, c), g[:, :2])
    z, (a, b, c) = g[:, :2], (x.detach() for x in (a, b, c))       # (no sequence passes 256 tokens: no rounded state in front of a segment)
    for name, got, (ref, tol) in (('decay out', out, R.decay_form(a, b, c, decay, lens, d ** -0.5, w=w)),
                                  ('decay dq', da, R.decay_form(z, c, b, decay, lens, d ** -0.5, w=w)),
                                  ('decay dk', db, R.decay_form(c, z, a, decay, lens, d ** -0.5, reverse=True, w=w)),
                                  ('decay dv', dc, R.decay_form(b, a, z, decay, lens, d ** -0.5, reverse=True, w=w))):
        R.assert_within(got[:rows], ref[:rows], tol[:rows] + tiny, name)
    cache = [_randn(2, 600, 2, d, seed=710 + i) for i in range(2)]
    n = torch.tensor([600, 3], dtype=torch.int32, device='cuda')
    val, tol = R.step_reference(g[:2], cache[0], cache[1], [600, 3], d ** -0.5, w=w)
    R.assert_within(gf.cached_attention_step(g[:2].contiguous(), cache[0], cache[1], n), val, tol + tiny, 'step')


def test_gradients_of_gradients_are_refused():
    """A recorded backward pass gives the same gradients, and says so when they are differentiated in their turn."""
    gf = _gf()
    q, k, v, g = (_randn(40, 2, 32, seed=800 + i).requires_grad_(i < 3) for i in range(4))
    decay = torch.full((2,), -0.1, device='cuda')
    for call in (lambda: gf.packed_attention(q, k, v, _cu([30, 10])), lambda: gf.decay_attention(q, k, v, decay, _cu([30, 10]))):
        plain = torch.autograd.grad(call(), (q, k, v), g)
        recorded = torch.autograd.grad(call(), (q, k, v), g, create_graph=True)
        assert all(torch.equal(a, b) for a, b in zip(plain, recorded))
        with pytest.raises(RuntimeError):
            torch.autograd.grad(recorded[0].float().sum(), q)


@pytest.mark.parametrize('rows', [200, 900])
def test_two_captured_graphs_at_once(rows):
    """Two captures of the same calls replayed at the same time on two streams: nothing is shared between them."""
    cu = _cu([rows // 3, 1, rows - rows // 3 - 1])
    inputs = [_everything_inputs(rows, 3, seed=900 + 10 * i) for i in range(2)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _everything(**inputs[0], cu=cu)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs, got = [], []
    for x in inputs:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            got.append(_everything(**x, cu=cu))
    streams = [torch.cuda.Stream() for _ in inputs]
    for _ in range(3):
        for t in (t for each in got for t in each):
            t.fill_(7.0)
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        kept = [[t.clone() for t in each] for each in got]
        for each, x in zip(kept, inputs):
            for a, b in zip(each, _everything(**x, cu=cu)):
                assert torch.equal(a, b)


def test_calls_from_two_threads():
    """Two host threads, each on its own stream, through the same operators."""
    import threading
    cu = _cu([300, 1, 599])
    inputs = [_everything_inputs(900, 3, seed=950 + 10 * i) for i in range(2)]
    want = [[t.clone() for t in _everything(**x, cu=cu)] for x in inputs]
    torch.cuda.synchronize()
    same = [False, False]

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            runs = [_everything(**inputs[i], cu=cu) for _ in range(5)]
            torch.cuda.current_stream().synchronize()
            same[i] = all(torch.equal(a, b) for r in runs for a, b in zip(r, want[i]))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert same == [True, True]


@pytest.mark.parametrize('lens', [[2200, 2100], [2048, 2048]], ids=str)
@pytest.mark.parametrize('d', [32, 64, 128])
def test_packed_attention_many_blocks(lens, d):
    """Enough blocks that the kernels take their forms for a full chip: tall blocks, whole row tiles per wave."""
    _check_packed(lens, 3, 16, 4, d, 960)


@pytest.mark.parametrize('d', [32, 64, 96, 128])
def test_cached_step_many_short_caches(d):
    """Enough sequences that neither wide blocks nor splits are taken."""
    b, cap, hkv = 300, 100, 2
    q, kc, vc = _randn(b, 4, d, seed=970), _cache(b, cap, hkv, d, 971), _cache(b, cap, hkv, d, 972)
    lengths = [(i * 37) % (cap + 1) for i in range(b)]
    val, tol = R.step_reference(q, kc, vc, lengths, d ** -0.5)
    out = _gf().cached_attention_step(q, kc, vc, torch.tensor(lengths, dtype=torch.int32, device='cuda'))
    R.assert_within(out, val, tol, 'out')


def test_calls_that_look_the_same_but_for_their_addresses():
    """Same types, shapes and strides as an earlier call, other addresses: rows off 16 bytes are copied, a cache or state off 16 bytes or twice the same is refused."""
    gf, d = _gf(), 64

    def odd(t):
        return torch.empty(t.numel() + 3, dtype=t.dtype, device='cuda')[3:].view(t.shape).copy_(t)

    cu, ld = _cu([3, 5]), _decays(2)
    q, k, v = (_randn(8, 2, d, seed=980 + i) for i in range(3))
    kc, vc = _cache(8, 20, 2, d, 984), _cache(8, 20, 2, d, 985)
    n, s = torch.arange(8, dtype=torch.int32, device='cuda'), torch.randn(8, 2, d, d, device='cuda')
    new = torch.empty_like(s)
    calls = (lambda q, k, v: gf.packed_attention(q, k, v, cu), lambda q, k, v: gf.decay_attention(q, k, v, ld, cu), lambda q, k, v: gf.cached_attention_step(q, kc, vc, n, k, v),
             lambda q, k, v: gf.decay_attention_step(q, k, v, ld, s, new_state=new))
    for call in calls:
        want = call(q, k, v)
        for moved in ((odd(q), k, v), (q, odd(k), v), (q, k, odd(v))):
            assert torch.equal(call(*moved), want)
        assert torch.equal(call(q.clone(), k, v), want)
        assert not torch.equal(call(k, q, v), want)
    with pytest.raises(ValueError, match='updated in place'):
        gf.cached_attention_step(q, odd(kc), vc, n, k, v)
    with pytest.raises(ValueError, match='updated in place'):
        gf.cached_attention_step(q, kc, odd(vc), n, k, v)
    with pytest.raises(ValueError, match='same memory'):
        gf.cached_attention_step(q, kc, kc, n, k, v)
    with pytest.raises(ValueError, match='aligned'):
        gf.decay_attention_step(q, k, v, ld, odd(s), new_state=new)
    with pytest.raises(ValueError, match='aligned'):
        gf.decay_attention_step(q, k, v, ld, s, new_state=odd(new))
    with pytest.raises(RuntimeError, match='no backward'):
        gf.decay_attention_step(q.clone().requires_grad_(), k, v, ld, s, new_state=new)
    with pytest.raises(RuntimeError, match='constants'):
        gf.decay_attention(q, k, v, ld.clone().requires_grad_(), cu)
    with torch.no_grad():
        a = gf.decay_attention(q, k, v, ld.clone().requires_grad_(), cu)
    assert torch.equal(a, gf.decay_attention(q, k, v, ld, cu))
    assert not torch.equal(gf.packed_attention(q, k, v, cu, scale=0.5), gf.packed_attention(q, k, v, cu, scale=torch.tensor(0.25)))
