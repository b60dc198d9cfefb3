"""The host side of the sequence operators (genie/sequence.py) without a GPU: their checks, layouts, saved tensors and autograd nodes run as they do there, the kernels'
launches are written down instead of made."""
import pytest
import torch

import util  # noqa: F401  (paths)


@pytest.fixture
def launches(monkeypatch):
    """CPU tensors pass the operators' device check; [(entry point, arguments)] of the launches they would make."""
    from genie import _hip, sequence
    made = []
    monkeypatch.setattr(_hip, 'require_gpu', lambda *_: None)
    monkeypatch.setattr(sequence, '_PLANS', {})
    monkeypatch.setattr(sequence, '_launch', lambda name, device, *args: made.append((name, args)))
    return made


def _randn(*shape, seed=0):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16)


def _cu(*lens):
    return torch.tensor([0, *lens], dtype=torch.int32).cumsum(0).to(torch.int32)


def _fused(rows, heads, d, seed):
    """q, k and v as slices of one projection."""
    x = _randn(rows, sum(heads), d, seed=seed).requires_grad_(True)
    return x.split(heads, 1)


class _Hooks:
    """Hooks on saved tensors that bring every tensor back at another address, through `back`."""

    def __init__(self, back):
        self.back, self.returned = back, []

    def unpack(self, t):
        self.returned.append(self.back(t))
        return self.returned[-1]

    def __enter__(self):
        self.context = torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach(), self.unpack)
        self.context.__enter__()
        return self

    def __exit__(self, *what):
        self.context.__exit__(*what)

    def covers(self, pointer, strides, shape):
        """Whether a (rows, heads, width) tensor of these strides at this address lies inside what was brought back."""
        last = pointer + 2 * sum((n - 1) * st for n, st in zip(shape, (*strides, 1)))
        for t in self.returned:
            if t.dtype == torch.bfloat16 and pointer == t.data_ptr() and tuple(t.shape) == tuple(shape):
                return tuple(t.stride()) == (*strides, 1) and last < t.data_ptr() + 2 * t.untyped_storage().nbytes()
        return False


def _dense(t):
    return t.clone(memory_format=torch.contiguous_format)


def test_packed_backward_takes_the_layout_its_saved_tensors_come_back_with(launches):
    from genie import functional as GF
    q, k, v = _fused(20, (4, 2, 2), 64, 1)
    assert q.stride() == (512, 64, 1)
    with _Hooks(_dense) as hooks:
        out = GF.packed_attention(q, k, v, _cu(13, 7))
        out.backward(_randn(20, 4, 64, seed=2))
    name, args = launches[-1]
    assert name == 'genie_packed_attention_bwd'
    for at, strides, shape in ((0, 20, (20, 4, 64)), (1, 21, (20, 2, 64)), (2, 22, (20, 2, 64))):
        assert hooks.covers(args[at], list(args[strides]), shape), (at, list(args[strides]))


def test_decay_backward_takes_the_layout_its_saved_tensors_come_back_with(launches):
    from genie import functional as GF
    q, k, v = _fused(20, (2, 2, 2), 64, 1)
    with _Hooks(_dense) as hooks:
        out = GF.decay_attention(q, k, v, torch.full((2,), -0.1), _cu(13, 7))
        out.backward(_randn(20, 2, 64, seed=2))
    name, args = launches[-1]
    assert name == 'genie_decay_attention_bwd'
    for at, strides in ((0, 19), (1, 20), (2, 21)):
        assert hooks.covers(args[at], list(args[strides]), (20, 2, 64)), (at, list(args[strides]))


def _apart(t):
    """The same values, nothing of them contiguous."""
    wide = torch.empty((*t.shape, 2), dtype=t.dtype, device=t.device)
    wide[..., 0] = t
    return wide[..., 0]


def _shifted(t):
    """The same values at an address off 16 bytes."""
    flat = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)[1:].view(t.shape)
    return flat.copy_(t)


@pytest.mark.parametrize('back', [_dense, _apart, _shifted], ids=lambda f: f.__name__)
def test_saved_tensors_that_come_back_in_any_layout_are_laid_out_for_the_kernels(launches, back):
    """Every pointer of the backward launch that the kernels read as 16-byte pieces is aligned, every matrix has the strides given or is dense."""
    from genie import functional as GF
    rows = 300
    q, k, v = _fused(rows, (2, 2, 2), 64, 1)
    for call, bwd, aligned in ((lambda: GF.packed_attention(q, k, v, _cu(250, 50)), 'genie_packed_attention_bwd', (0, 1, 2, 3, 4, 5)),
                               (lambda: GF.decay_attention(q, k, v, torch.full((2,), -0.1), _cu(250, 50)), 'genie_decay_attention_bwd', (0, 1, 2, 3, 7))):
        with _Hooks(back):
            call().backward(_randn(rows, 2, 64, seed=2))
        name, args = launches[-1]
        assert name == bwd and all(args[i] % 16 == 0 for i in aligned), args
        strides = [tuple(a) for a in args if hasattr(a, '_length_')]
        assert len(strides) == 4 and all(st == (128, 64) for st in strides), strides


def test_saved_tensors_that_come_back_as_something_else_are_refused(launches):
    from genie import functional as GF
    q, k, v = _fused(20, (2, 2, 2), 64, 1)
    for call in (lambda: GF.packed_attention(q, k, v, _cu(13, 7)), lambda: GF.decay_attention(q, k, v, torch.full((2,), -0.1), _cu(13, 7))):
        for back in (lambda t: t.double(), lambda t: t[:-1]):
            with _Hooks(back):
                out = call()
            before = len(launches)
            with pytest.raises(RuntimeError, match='came back'):
                out.backward(_randn(20, 2, 64, seed=2))
            assert len(launches) == before


@pytest.mark.parametrize('rows_q, rows_k', [(5, 0), (0, 16), (0, 0), (0, 5000), (5000, 0), (1, 1)])
@pytest.mark.parametrize('hq, hkv, dim', [(16, 1, 64), (8, 8, 128)])
def test_packed_backward_workspace_covers_calls_without_rows_on_one_side(rows_q, rows_k, hq, hkv, dim):
    """delta is written for every query row, keys or not; and one float less than the query asks for is refused."""
    from genie import _hip
    lib, strides = _hip.load_library(), _hip.i64((hq * dim, dim))
    need = lib.genie_packed_attention_bwd_ws_floats(1, rows_q, rows_k, hq, hkv, dim)
    assert need >= hq * rows_q and need > 0
    rc = lib.genie_packed_attention_bwd(*([16] * 8), need - 1, *([16] * 5), 1, rows_q, rows_k, hq, hkv, dim, strides, strides, strides, strides, 1.0, None)
    assert rc == -1 and b'workspace' in lib.genie_last_error()


def _empty(heads, d, kind):
    """(0, heads, d) with the strides that an expanded gradient, a slice of a wider tensor or a row stride without 8 elements would have."""
    if kind == 'expanded':
        return torch.zeros((), dtype=torch.bfloat16).expand(0, heads, d)
    if kind == 'sliced':
        return torch.zeros(0, heads, 2 * d, dtype=torch.bfloat16)[..., ::2]
    return torch.zeros(0, heads, d, dtype=torch.bfloat16).as_strided((0, heads, d), (3, 5, 1))


@pytest.mark.parametrize('kind', ['expanded', 'sliced', 'odd'])
def test_training_calls_without_rows(launches, kind):
    """A batch without tokens: results and gradients are empty, whatever strides the empty tensors have, and nothing is launched."""
    from genie import functional as GF
    ld, s0 = torch.full((4,), -0.1), torch.randn(1, 4, 64, 64)
    for call in (lambda x: GF.packed_attention(x, x, x, _cu(0)), lambda x: GF.decay_attention(x, x, x, ld, _cu(0)), lambda x: GF.decay_attention(x, x, x, ld, _cu(0), initial_state=s0)):
        x = _empty(4, 64, kind).requires_grad_(True)
        out = call(x)
        assert out.shape == (0, 4, 64)
        out.sum().backward()
        assert x.grad.shape == x.shape
        assert call(x.detach()).shape == x.shape
    assert not launches


@pytest.mark.parametrize('kind', ['expanded', 'sliced', 'odd'])
def test_training_calls_without_keys(launches, kind):
    from genie import functional as GF
    q, k = _randn(5, 4, 64, seed=1).requires_grad_(True), _empty(4, 64, kind).requires_grad_(True)
    out = GF.packed_attention(q, k, k, _cu(5), cu_seqlens_k=_cu(0))
    assert torch.equal(out, torch.zeros_like(out))
    out.sum().backward()
    assert torch.equal(q.grad, torch.zeros_like(q)) and k.grad.shape == k.shape
    out = GF.packed_attention(k, q, q, _cu(0), cu_seqlens_k=_cu(5))                 # keys, but no queries
    q.grad = None
    out.sum().backward()
    assert torch.equal(q.grad, torch.zeros_like(q)) and not launches


def test_steps_without_sequences(launches):
    from genie import functional as GF
    for kind in ('expanded', 'sliced', 'odd'):
        x = _empty(4, 64, kind)
        assert GF.cached_attention_step(x, torch.zeros(0, 8, 4, 64, dtype=torch.bfloat16), torch.zeros(0, 8, 4, 64, dtype=torch.bfloat16),
                                        torch.zeros(0, dtype=torch.int32), x, x).shape == (0, 4, 64)
        assert GF.decay_attention_step(x, x, x, torch.zeros(4), torch.zeros(0, 4, 64, 64)).shape == (0, 4, 64)
    assert not launches


def test_dual_tensors_are_refused(launches):
    """Forward-mode differentiation: a result without its tangent would be a silent derivative of zero."""
    from genie import functional as GF
    import torch.autograd.forward_ad as fwad
    x, s, ld = _randn(6, 2, 64, seed=1), torch.randn(6, 2, 64, 64), torch.full((2,), -0.1)
    cache, n = [_randn(6, 10, 2, 64, seed=i) for i in (2, 3)], torch.zeros(6, dtype=torch.int32)
    cu = _cu(6)

    def dual(t):
        return fwad.make_dual(t, torch.ones_like(t))

    calls = [(GF.packed_attention, [x, x, x], lambda a: (*a, cu)), (GF.cached_attention_step, [x, *cache, x, x], lambda a: (*a[:3], n, *a[3:])),
             (GF.decay_attention, [x, x, x, ld, torch.randn(1, 2, 64, 64)], lambda a: (*a[:4], cu, a[4])), (GF.decay_attention_step, [x, x, x, ld, s], lambda a: a)]
    for call, given, order in calls:
        for at in range(len(given)):
            for grad in (False, True):
                with fwad.dual_level(), torch.set_grad_enabled(grad):
                    made = len(launches)
                    with pytest.raises(NotImplementedError, match='forward-mode'):
                        call(*order([dual(t) if i == at else t for i, t in enumerate(given)]))
                    assert len(launches) == made
        with fwad.dual_level():
            call(*order(given))                                                   # (no dual among the arguments)
    leaf = x.clone().requires_grad_(True)                                         # the same where a gradient is recorded as well
    with fwad.dual_level(), pytest.raises(NotImplementedError, match='forward-mode'):
        GF.packed_attention(dual(leaf), x, x, cu)


def test_tensors_updated_in_place_say_so(launches):
    """Caches and states are written by the kernels: autograd sees a new version, and a graph that kept the old values refuses instead of using the new ones."""
    from genie import functional as GF
    x, n = _randn(6, 2, 64, seed=1), torch.zeros(6, dtype=torch.int32)
    kc, vc, ld = _randn(6, 10, 2, 64, seed=2), _randn(6, 10, 2, 64, seed=3), torch.full((2,), -0.1)
    state, into = torch.randn(6, 2, 64, 64), torch.zeros(6, 2, 64, 64)

    def versions():
        return [t._version for t in (x, n, kc, vc, ld, state, into)]

    at = versions()
    GF.cached_attention_step(x, kc, vc, n)                                        # nothing is written
    assert versions() == at
    GF.cached_attention_step(x, kc, vc, n, x, x)
    assert [b - a for a, b in zip(at, versions())] == [0, 0, 1, 1, 0, 0, 0]
    GF.decay_attention_step(x, x, x, ld, state)
    assert [b - a for a, b in zip(at, versions())] == [0, 0, 1, 1, 0, 1, 0]
    GF.decay_attention_step(x, x, x, ld, state, new_state=into)
    assert [b - a for a, b in zip(at, versions())] == [0, 0, 1, 1, 0, 1, 1]
    w = torch.randn(6, 2, 64, 64, requires_grad=True)
    loss = (w * state).sum()
    with torch.no_grad():
        GF.decay_attention_step(x, x, x, ld, state)
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        loss.backward()
    with torch.inference_mode():
        GF.decay_attention_step(x, x, x, ld, torch.zeros(6, 2, 64, 64))             # (tensors without versions)


def _ballot_search(cu, rows, tile, first, slot):
    """The 64 lanes of the longest-first search, level by level as a wave walks them -> (sequence, tile); the sequence behind the last holds the spare rows."""
    lane, nseq = torch.arange(64), len(cu) - 1
    clamped = [0] + [min(max(c, 0), rows) for c in cu[1:]]
    start, after = [clamped[min(i, nseq)] for i in range(64)], [clamped[min(i + 1, nseq)] for i in range(64)]
    n = torch.tensor([(max(0, b - a) + tile - 1) // tile for a, b in zip(start, after)])
    lo, width, above = 0, rows // tile + 2, 0
    while True:
        step = (width + 62) // 63
        c = (n[:nseq, None] - (lo + lane * step)[None, :]).clamp(min=0).sum(0)
        if lo == 0 and slot >= int(c[0]):
            return nseq, slot - int(c[0])
        hits = max(1, int((c > slot).sum()))
        assert hits == 1 or bool((c[:hits] > slot).all())                         # the ballot is a prefix
        lo, above, width = lo + (hits - 1) * step, int(c[min(hits, 63)]), step
        if width <= 1:
            break
    who = [i for i in range(64) if int(n[i]) > lo][slot - above:]
    length = after[who[0]] - start[who[0]]
    return who[0], (length + tile - 1) // tile - 1 - lo if first else lo


@pytest.mark.parametrize('seed', range(12))
@pytest.mark.parametrize('first', [False, True])
def test_longest_first_search_covers_every_tile_once_in_order(seed, first):
    import random
    rng = random.Random(seed)
    tile = rng.choice([64, 128, 256])
    lens = [rng.choice([0, 1, tile - 1, tile, tile + 1, rng.randint(0, 40 * tile)]) for _ in range(rng.choice([1, 2, 7, 62, 63]))]
    if seed == 0:
        lens = [70 * tile + 3, 5, 64 * tile]                                      # more tiles than one level of the search tells apart
    cu, spare = [0], rng.choice([0, 1, 3 * tile + 5])
    for x in lens:
        cu.append(cu[-1] + x)
    rows = cu[-1] + spare
    found = [_ballot_search(cu, rows, tile, first, slot) for slot in range(rows // tile + len(lens) + 1)]
    real = [(s, t) for s, t in found if s < len(lens)]
    assert sorted(real) == [(s, t) for s, n in enumerate(lens) for t in range((n + tile - 1) // tile)]
    work = [((lens[s] + tile - 1) // tile - 1 - t) if first else t for s, t in real]
    assert work == sorted(work, reverse=True)
    behind = [t for s, t in found if s == len(lens)]
    assert behind == list(range(len(behind))) and len(behind) * tile >= spare
