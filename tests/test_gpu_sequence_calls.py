"""The sequence operators (genie/sequence.py) in the surroundings a training or serving program puts them into, on the GPU: hooks on saved tensors, empty batches, the C entries'
own workspaces, versions of tensors that are updated in place, values that are not finite.  Numerics: tests/test_gpu_sequence.py."""
import pytest
import torch

import sequence_ref as R
import util  # noqa: F401  (paths)

pytestmark = pytest.mark.gpu


def _gf():
    from genie import functional
    return functional


def _randn(*shape, seed, scale=1.0):
    return (torch.randn(shape, generator=torch.Generator(device='cuda').manual_seed(seed), device='cuda') * scale).to(torch.bfloat16)


def _cu(lens):
    return torch.tensor([0] + list(lens), dtype=torch.int32, device='cuda').cumsum(0).to(torch.int32)


def _apart(t):
    """The same values, nothing of them contiguous."""
    wide = torch.empty((*t.shape, 2), dtype=t.dtype, device=t.device)
    wide[..., 0] = t
    return wide[..., 0]


def _shifted(t):
    """The same values at an address off 16 bytes."""
    flat = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)[1:].view(t.shape)
    return flat.copy_(t)


@pytest.mark.parametrize('hook', ['on the host', 'apart', 'shifted'])
@pytest.mark.parametrize('lens', [[20, 1, 50], [400, 300]], ids=str)
def test_gradients_after_a_round_trip_of_the_saved_tensors(lens, hook):
    """Slices of a fused projection come back dense, in a layout of their own or off 16 bytes: the gradients are those of the plain call, to the bit."""
    gf, rows, h, d = _gf(), sum(lens), 4, 64
    fused = _randn(rows, 3 * h, d, seed=1).requires_grad_(True)
    g, ld, cu = _randn(rows, h, d, seed=2), -torch.linspace(0.01, 0.5, h, device='cuda'), _cu(lens)
    s0 = torch.randn((len(lens), h, d, d), generator=torch.Generator(device='cuda').manual_seed(3), device='cuda')

    def context():
        if hook == 'on the host':
            return torch.autograd.graph.save_on_cpu()
        return torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach(), _apart if hook == 'apart' else _shifted)

    for call in (lambda q, k, v: gf.packed_attention(q, k[:, :2], v[:, :2], cu), lambda q, k, v: gf.decay_attention(q, k, v, ld, cu),
                 lambda q, k, v: gf.decay_attention(q, k, v, ld, cu, initial_state=s0)):
        want = torch.autograd.grad(call(*fused.split(h, 1)), fused, g)[0]
        with context():
            out = call(*fused.split(h, 1))
        assert torch.equal(torch.autograd.grad(out, fused, g)[0], want)


@pytest.mark.parametrize('rows_q, rows_k', [(5, 0), (0, 16), (0, 5000), (5000, 0)])
@pytest.mark.parametrize('hq, hkv, d', [(16, 1, 64), (8, 8, 128)])
def test_packed_backward_entry_without_rows_on_one_side_stays_in_its_workspace(rows_q, rows_k, hq, hkv, d):
    """The C entry with exactly the workspace it asks for: gradients are zero and nothing behind the workspace changes."""
    from genie import _hip
    lib, st, sk = _hip.load_library(), _hip.i64((hq * d, d)), _hip.i64((hkv * d, d))
    q, k = _randn(rows_q + 1, hq, d, seed=1), _randn(rows_k + 1, hkv, d, seed=2)
    dq, dk, dv = (torch.full_like(t, 3.0) for t in (q, k, k))
    lse = torch.full((hq, rows_q + 1), float('-inf'), device='cuda')
    need, spare = lib.genie_packed_attention_bwd_ws_floats(1, rows_q, rows_k, hq, hkv, d), 1 << 22
    ws = torch.full((need + spare,), 7.0, device='cuda')
    cu_q, cu_k = _cu([rows_q]), _cu([rows_k])
    rc = lib.genie_packed_attention_bwd(*(t.data_ptr() for t in (q, k, k, q, q, q, lse, ws)), need, *(t.data_ptr() for t in (dq, dk, dv, cu_q, cu_k)), 1, rows_q, rows_k, hq, hkv, d,
                                        st, sk, sk, st, 0.125, torch.cuda.current_stream().cuda_stream)
    assert rc == 0, lib.genie_last_error()
    torch.cuda.synchronize()
    assert (ws[need:] == 7.0).all()
    for t, rows in ((dq, rows_q), (dk, rows_k), (dv, rows_k)):
        assert (t[:rows] == 0).all() and (t[rows:] == 3.0).all()


def test_training_calls_without_rows_or_keys():
    gf = _gf()
    ld, s0 = torch.full((4,), -0.1, device='cuda'), torch.randn(1, 4, 64, 64, device='cuda')
    for call in (lambda x: gf.packed_attention(x, x, x, _cu([0])), lambda x: gf.decay_attention(x, x, x, ld, _cu([0])),
                 lambda x: gf.decay_attention(x, x, x, ld, _cu([0]), initial_state=s0)):
        x = torch.zeros(0, 4, 64, dtype=torch.bfloat16, device='cuda', requires_grad=True)
        call(x).sum().backward()
        assert x.grad.shape == x.shape
    q, k = _randn(5, 4, 64, seed=1).requires_grad_(True), torch.zeros(0, 4, 64, dtype=torch.bfloat16, device='cuda', requires_grad=True)
    gf.packed_attention(q, k, k, _cu([5]), cu_seqlens_k=_cu([0])).sum().backward()
    assert torch.equal(q.grad, torch.zeros_like(q)) and k.grad.shape == k.shape


@pytest.mark.parametrize('lens, spare', [([1], 0), ([2, 0, 3], 5), ([70, 130, 56], 0), ([256], 0)], ids=str)
@pytest.mark.parametrize('dk, dv', [(32, 32), (64, 64), (96, 64), (24, 128), (128, 128)])
def test_few_rows_carry_their_state_without_rounding_it(lens, spare, dk, dv):
    """Up to 256 rows a state in front of a sequence enters outputs and dq with its rounding's remainder: U^2 of it is left, as of the weights."""
    gf, rows, h, w = _gf(), sum(lens) + spare, 3, R.U ** 2
    q, k, v, g = (_randn(rows, h, d, seed=20 + i) for i, d in enumerate((dk, dk, dv, dv)))
    for t in (q, k, v, g):
        t[rows - spare:] = float('nan')
    ld = torch.tensor([-0.01, 0.0, -0.7], device='cuda')
    s0 = torch.randn((len(lens), h, dk, dv), generator=torch.Generator(device='cuda').manual_seed(24), device='cuda') * 8
    for t in (q, k, v):
        t.requires_grad_(True)
    out, last = gf.decay_attention(q, k, v, ld, _cu(lens), initial_state=s0, return_state=True)
    dq = torch.autograd.grad(out, q, g)[0]
    used, tiny = sum(lens), 2.0 ** -100
    for name, got, (val, tol) in (('out', out, R.decay_form(q.detach(), k.detach(), v.detach(), ld, lens, dk ** -0.5, state=s0, w=w)),
                                  ('dq', dq, R.decay_form(g, v.detach(), k.detach(), ld, lens, dk ** -0.5, state=s0.transpose(2, 3), w=w))):
        R.assert_within(got[:used], val[:used], tol[:used] + tiny, name)
        assert (got[used:] == 0).all()
    R.assert_within(last, *R.decay_state(k.detach(), v.detach(), ld, lens, s0), 'state')


@pytest.mark.parametrize('lens', [[40, 3], [300, 170]], ids=str)
@pytest.mark.parametrize('d', [64, 128])
@pytest.mark.parametrize('scale', [1e-44, 1e-39, 1e-37, 1e-20, 1e-3, 1.0, 3.0])
def test_packed_gradients_at_any_scale(lens, d, scale, monkeypatch):
    """From scales whose inverse is no fp32 number (all keys weigh the same) to ones that leave a few keys."""
    gf, rows, hq, hkv = _gf(), sum(lens), 4, 2
    q, k, v, g = (_randn(rows, h, d, seed=30 + i) for i, h in enumerate((hq, hkv, hkv, hq)))
    # a score is a sum of d fp32 products: off by d 2^-24 of its magnitudes at worst, in the weight's exponent and in the log-sum-exp's
    most = scale * torch.einsum('ihd,jhd->hij', q.float().abs(), k.float().abs().repeat_interleave(2, 1)).max().item()
    monkeypatch.setattr(R, 'SLACK', R.SLACK + 2 * d * 2.0 ** -24 * most)
    val, tol = R.packed_reference(q, k, v, lens, scale, g)
    for t in (q, k, v):
        t.requires_grad_(True)
    out = gf.packed_attention(q, k, v, _cu(lens), scale=scale)
    for name, t in zip(('out', 'dq', 'dk', 'dv'), (out, *torch.autograd.grad(out, (q, k, v), g))):
        # (results under the smallest normal number may be rounded to their multiples of 2^-133, or to zero)
        R.assert_within(t, torch.where(val[name].abs() < 2.0 ** -126, t.double(), val[name]), tol[name] + 2.0 ** -126, name)
        assert name in ('dq', 'dk') or (t != 0).any()


# ------------------------------------------------------------------------------------------------------------------------------------
# forms and bounds that tests/test_gpu_sequence.py does not reach
# ------------------------------------------------------------------------------------------------------------------------------------
def _state_bound(log_decay, lens, mag):
    """Final states: the decayed operand l^e c is a sum of three bf16 values (U^3 = 2^-24 of it is left) and one fp32 product; its power carries the roundings of log2 l and of
    their product with e (together 2^-23 of the exponent, log2 l e < |log_decay| 1.5 len) and the hardware's 2^-23; the sum over a sequence adds three products a
    token, 2^-24 each.  A state in front of the sequence goes through one such power and one sum."""
    lens = torch.tensor(lens, dtype=torch.float64, device=mag.device)[:, None]
    span = (log_decay.double().clamp(min=-60).abs()[None, :] * 1.5 * lens).clamp(max=90)      # (past 2^-90 the term itself is gone)
    return mag * (2.0 ** -24 * (3 * lens + 8 + 2 * span))[:, :, None, None]


@pytest.mark.parametrize('lens', [[2], [3, 1, 2], [2, 5, 0, 3], [3] * 100, [1 + i % 7 for i in range(90)]], ids=lambda x: f'{len(x)}x{x[0]}')
@pytest.mark.parametrize('dk, dv', [(64, 64), (128, 128), (32, 96), (104, 40), (8, 128)])
@pytest.mark.parametrize('state', [False, True])
def test_final_states_of_short_sequences_are_fp32(lens, dk, dv, state):
    """Both forms (up to 256 rows in one launch, more in three), square and not: the states hold what fp32 holds, not what two bf16 values do."""
    gf, h, n = _gf(), 3, sum(lens)
    q, k, v = (_randn(n, h, d, seed=50 + i) for i, d in enumerate((dk, dk, dv)))
    ld = torch.tensor([-0.3, -1.7, -0.01], device='cuda')
    s0 = torch.randn((len(lens), h, dk, dv), generator=torch.Generator(device='cuda').manual_seed(54), device='cuda') if state else None
    out, last = gf.decay_attention(q, k, v, ld, _cu(lens), initial_state=s0, return_state=True)
    val, bound = R.decay_state(k, v, ld, lens, s0)
    mag = bound / (R.U * R.U + 2.0 ** -18)
    R.assert_within(last, val, _state_bound(ld, lens, mag), 'state')
    R.assert_within(out, *R.decay_form(q, k, v, ld, lens, dk ** -0.5, state=s0), 'out')


@pytest.mark.parametrize('heads', [(20, 1), (40, 2), (4, 4)], ids=str)
@pytest.mark.parametrize('d', [8, 24, 40, 80, 96, 120])
def test_cached_step_split_at_every_width(heads, d):
    """Caches split over blocks, with and without a token to append: joins whose threads do not divide evenly, more query heads to a key head than a product has columns."""
    gf, (hq, hkv), cap = _gf(), heads, 2600
    lengths = [2599, 1300, 0, -1, 33]
    b = len(lengths)
    q, kn, vn = _randn(b, hq, d, seed=60), _randn(b, hkv, d, seed=61), _randn(b, hkv, d, seed=62)
    kc, vc = _randn(b, cap, hkv, d, seed=63), _randn(b, cap, hkv, d, seed=64)
    n = torch.tensor(lengths, dtype=torch.int32, device='cuda')
    val, tol = R.step_reference(q, kc, vc, lengths, d ** -0.5)
    R.assert_within(gf.cached_attention_step(q, kc, vc, n), val, tol, 'without a token')
    out = gf.cached_attention_step(q, kc, vc, n, kn, vn)
    for i, m in enumerate(lengths):
        if m >= 0:
            assert torch.equal(kc[i, m], kn[i]) and torch.equal(vc[i, m], vn[i])
    val, tol = R.step_reference(q, kc, vc, [m + 1 for m in lengths], d ** -0.5)
    R.assert_within(out, val, tol, 'with a token')


@pytest.mark.parametrize('b, cap', [(3, 60), (3, 3000), (300, 90)])
@pytest.mark.parametrize('d', [64, 128])
def test_cached_step_with_values_that_are_not_finite(b, cap, d):
    """One wide block, several parts, four waves: NaN stays in its sequence, key head and (in a value) column; a score of minus infinity is a key that is not there."""
    gf, hq, hkv = _gf(), 4, 2
    q, kc, vc = _randn(b, hq, d, seed=70), _randn(b, cap, hkv, d, seed=71), _randn(b, cap, hkv, d, seed=72)
    full = torch.full((b,), cap, dtype=torch.int32, device='cuda')
    want = gf.cached_attention_step(q, kc, vc, full)
    rest = torch.ones_like(want, dtype=torch.bool)
    rest[1] = False

    def call(q=q, kc=kc, vc=vc, n=full):
        return gf.cached_attention_step(q, kc, vc, n)

    for at in (0, cap // 2, cap - 1):
        bad = kc.clone()
        bad[1, at, 0, 3] = float('nan')
        out = call(kc=bad)
        assert torch.isnan(out[1, :2]).all() and torch.equal(out[1, 2:], want[1, 2:]) and torch.equal(out[rest], want[rest])
        bad = vc.clone()
        bad[1, at, 1, 5] = float('nan')
        out = call(vc=bad)
        assert torch.isnan(out[1, 2:, 5]).all() and torch.equal(out[rest], want[rest]) and torch.equal(out[1, :2], want[1, :2])
        cols = [c for c in range(d) if c != 5]
        assert torch.equal(out[1, 2:][:, cols], want[1, 2:][:, cols])
        bad, sign = kc.clone(), q.clone()
        bad[1, at, 0] = 0
        bad[1, at, 0, 0] = float('inf')
        sign[1, 0, 0], sign[1, 1, 0] = -2.0, 2.0                                  # query head 0: a score of -inf; head 1: +inf, whose softmax is NaN
        out = call(q=sign, kc=bad)
        assert torch.isnan(out[1, 1]).all()
        keep = [j for j in range(cap) if j != at]
        val, tol = R.step_reference(sign[1:2, :1], kc[1:2, keep, :1], vc[1:2, keep, :1], [cap - 1], d ** -0.5)
        R.assert_within(out[1:2, :1], val, tol, 'without the key')
    bad = kc.clone()
    bad[1] = float('nan')                                                         # nothing but NaN, in every wave and part; and as the only key
    out = call(kc=bad)
    assert torch.isnan(out[1]).all() and torch.equal(out[rest], want[rest])
    one = full.clone()
    one[1] = 1
    assert torch.isnan(call(kc=bad, n=one)[1]).all()
    bad = q.clone()
    bad[1, 2] = float('nan')
    out = call(q=bad)
    assert torch.isnan(out[1, 2]).all() and torch.equal(out[rest], want[rest]) and torch.equal(out[1, [0, 1, 3]], want[1, [0, 1, 3]])


@pytest.mark.parametrize('state', [False, True])
@pytest.mark.parametrize('d', [32, 128])
def test_more_sequences_than_one_search_level_in_few_rows(d, state):
    """200 sequences of 0, 1 and 2 tokens in 199 rows: forward, final states and gradients of both operators."""
    gf, h, lens = _gf(), 2, [i % 3 for i in range(200)]
    n, w, tiny = sum(lens), R.U ** 2, 2.0 ** -100
    q, k, v, g = (_randn(n, h, d, seed=90 + i).requires_grad_(i < 3) for i in range(4))
    ld = torch.tensor([-0.2, -1.0], device='cuda')
    s0 = torch.randn((200, h, d, d), generator=torch.Generator(device='cuda').manual_seed(94), device='cuda') if state else None
    out, last = gf.decay_attention(q, k, v, ld, _cu(lens), initial_state=s0, return_state=True)
    grads = torch.autograd.grad(out, (q, k, v), g)
    a, b, c = (t.detach() for t in (q, k, v))
    st = None if s0 is None else s0.transpose(2, 3)
    R.assert_within(last, *R.decay_state(b, c, ld, lens, s0), 'state')
    for name, got, (val, tol) in (('out', out, R.decay_form(a, b, c, ld, lens, d ** -0.5, state=s0, w=w)), ('dq', grads[0], R.decay_form(g, c, b, ld, lens, d ** -0.5, state=st, w=w)),
                                  ('dk', grads[1], R.decay_form(c, g, a, ld, lens, d ** -0.5, reverse=True, w=w)),
                                  ('dv', grads[2], R.decay_form(b, a, g, ld, lens, d ** -0.5, reverse=True, w=w))):
        R.assert_within(got, val, tol + tiny, name)
    out = gf.packed_attention(q, k, v, _cu(lens))
    val, tol = R.packed_reference(a, b, c, lens, d ** -0.5, g, w=w)
    for name, got in zip(('out', 'dq', 'dk', 'dv'), (out, *torch.autograd.grad(out, (q, k, v), g))):
        R.assert_within(got, val[name], tol[name] + tiny, name)


@pytest.mark.parametrize('rows', [150, 3000])
def test_wide_heads_in_a_captured_graph(rows):
    """Heads of 128 (blocks with more than 64 KB of LDS), a state in front, forward and backward captured and replayed with other lengths; eager work between the replays."""
    gf, d = _gf(), 128
    q, k, v, g = (_randn(rows, h, d, seed=100 + i).requires_grad_(i < 3) for i, h in enumerate((4, 2, 2, 4)))
    s0 = torch.randn((3, 2, d, d), generator=torch.Generator(device='cuda').manual_seed(104), device='cuda')
    ld, cu = torch.tensor([-0.02, -0.4], device='cuda'), _cu([rows - 40, 0, 40])
    kc, vc = _randn(3, 500, 2, d, seed=105), _randn(3, 500, 2, d, seed=106)
    n = torch.tensor([3, 499, 70], dtype=torch.int32, device='cuda')

    def everything():
        a = gf.packed_attention(q, k, v, cu)
        b, last = gf.decay_attention(q[:, :2], k, v, ld, cu, initial_state=s0, return_state=True)
        with torch.no_grad():
            step = gf.cached_attention_step(q[:3], kc, vc, n, k[:3], v[:3])
        return [a, *torch.autograd.grad(a, (q, k, v), g), b, last, *torch.autograd.grad(b, (q, k, v), g[:, :2]), step]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        everything()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = everything()
    for lens in ([rows - 40, 0, 40], [0, rows, 0], [5, 6, 7]):
        cu.copy_(_cu(lens))
        graph.replay()
        torch.cuda.synchronize()
        kept = [t.clone() for t in got]
        for a, b in zip(kept, everything()):
            assert torch.equal(a, b)


def test_checkpointed_calls():
    """Activation checkpointing replaces the saved tensors by recomputed ones."""
    from torch.utils.checkpoint import checkpoint
    gf, rows, h, d = _gf(), 300, 2, 64
    fused, g, cu = _randn(rows, 3 * h, d, seed=110).requires_grad_(True), _randn(rows, h, d, seed=111), _cu([170, 130])
    ld = torch.tensor([-0.02, -0.4], device='cuda')

    def block(x):
        q, k, v = (x * 0.5).split(h, 1)
        return gf.packed_attention(q, k, v, cu) + gf.decay_attention(q, k, v, ld, cu)

    want = torch.autograd.grad(block(fused), fused, g)[0]
    assert torch.equal(torch.autograd.grad(checkpoint(block, fused, use_reentrant=False), fused, g)[0], want)
