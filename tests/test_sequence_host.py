"""Sequence operators without a GPU: the references' gradients against differences, refusals that come before any device work."""
import ctypes

import pytest
import torch

import util  # noqa: F401  (paths)
import sequence_ref as R


def _rand(*shape, seed=0):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed), dtype=torch.float64)


@pytest.mark.parametrize('lens_k', [None, [6, 1, 3]])
def test_packed_reference_gradients_match_differences(lens_k):
    lens, hq, hkv, d = [4, 0, 5], 4, 2, 3
    q, k, v, g = _rand(9, hq, d, seed=1), _rand(sum(lens_k or lens), hkv, d, seed=2), _rand(sum(lens_k or lens), hkv, d, seed=3), _rand(9, hq, d, seed=4)
    f = lambda *x: float((R.packed_reference(*x, lens, 0.7, None, lens_k)[0]['out'] * g).sum())  # noqa: E731
    grads = R.packed_reference(q, k, v, lens, 0.7, g, lens_k)[0]
    for i, name in enumerate(('dq', 'dk', 'dv')):
        x = [q, k, v]
        flat = grads[name].flatten()
        for at in range(0, flat.numel(), 3):
            e = torch.zeros_like(x[i]).flatten()
            e[at] = 1e-5
            e = e.reshape(x[i].shape)
            up, down = [t + e if j == i else t for j, t in enumerate(x)], [t - e if j == i else t for j, t in enumerate(x)]
            # central difference: truncation ~ 1e-10, rounding ~ 1e-16 / 1e-5
            assert abs((f(*up) - f(*down)) / 2e-5 - flat[at].item()) < 1e-7


def test_decay_reference_gradients_match_differences():
    lens, h, dk, dv = [4, 0, 5], 2, 3, 2
    q, k, v, g = _rand(9, h, dk, seed=1), _rand(9, h, dk, seed=2), _rand(9, h, dv, seed=3), _rand(9, h, dv, seed=4)
    ld, s0 = torch.tensor([-0.1, -1.5]), _rand(3, h, dk, dv, seed=5)
    f = lambda *x: float((R.decay_form(*x, ld, lens, 0.7, state=s0)[0] * g).sum())  # noqa: E731
    grads = [R.decay_form(g, v, k, ld, lens, 0.7, state=s0.transpose(2, 3))[0], R.decay_form(v, g, q, ld, lens, 0.7, reverse=True)[0],
             R.decay_form(k, q, g, ld, lens, 0.7, reverse=True)[0]]
    for i in range(3):
        x = [q, k, v]
        flat = grads[i].flatten()
        for at in range(flat.numel()):
            e = torch.zeros_like(x[i]).flatten()
            e[at] = 1e-5
            e = e.reshape(x[i].shape)
            up, down = [t + e if j == i else t for j, t in enumerate(x)], [t - e if j == i else t for j, t in enumerate(x)]
            assert abs((f(*up) - f(*down)) / 2e-5 - flat[at].item()) < 1e-7


def test_decay_reference_is_the_recurrence():
    lens, h = [5, 0, 3], 2
    q, k, v, s0 = _rand(8, h, 4, seed=1), _rand(8, h, 4, seed=2), _rand(8, h, 3, seed=3), _rand(3, h, 4, 3, seed=4)
    ld = torch.tensor([-0.25, float('-inf')])
    y, last = R.decay_form(q, k, v, ld, lens, 0.5, state=s0)[0], R.decay_state(k, v, ld, lens, s0)[0]
    for i, (a, b) in enumerate(R.bounds(lens)):
        for j in range(h):
            s = s0[i, j].clone()
            for t in range(a, b):
                s = s * torch.exp(ld[j].double()) + k[t, j][:, None] * v[t, j][None, :]
                assert torch.allclose(0.5 * q[t, j] @ s, y[t, j], rtol=1e-12, atol=1e-12)
            assert torch.allclose(s, last[i, j], rtol=1e-12, atol=1e-12)


def test_operators_refuse_cpu_tensors_and_wrong_types():
    from genie import functional as GF
    x = torch.zeros(4, 2, 64, dtype=torch.bfloat16)
    cu = torch.tensor([0, 4], dtype=torch.int32)
    with pytest.raises(RuntimeError, match='MI355X only'):
        GF.packed_attention(x, x, x, cu)
    with pytest.raises(RuntimeError, match='MI355X only'):
        GF.decay_attention(x, x, x, torch.zeros(2), cu)
    with pytest.raises(TypeError, match='bfloat16'):
        GF.packed_attention(x.float(), x, x, cu)
    with pytest.raises(ValueError, match='3 axes'):
        GF.packed_attention(x[0], x, x, cu)
    with pytest.raises(RuntimeError, match='MI355X only'):
        GF.cached_attention_step(x, x[:, None], x[:, None], torch.zeros(4, dtype=torch.int32))
    with pytest.raises(RuntimeError, match='MI355X only'):
        GF.decay_attention_step(x, x, x, torch.zeros(2), torch.zeros(4, 2, 64, 64))


def test_c_entries_refuse_before_any_device_work():
    from genie import _hip
    lib = _hip.load_library()
    two = _hip.i64((512, 64))

    def packed(hq=8, hkv=2, dim=64, strides=two, q=16, scale=1.0):
        rc = lib.genie_packed_attention_fwd(q, 16, 16, 16, None, None, 16, 16, 1, 4, 4, hq, hkv, dim, strides, two, two, scale, None)
        return rc, lib.genie_last_error()

    assert packed(hkv=3)[0] == -1 and b'no multiple' in packed(hkv=3)[1]
    assert packed(dim=60)[0] == -1 and b'head width 60' in packed(dim=60)[1]
    assert packed(dim=136)[0] == -1
    assert packed(strides=_hip.i64((516, 64)))[0] == -1 and b'multiples of 8' in packed(strides=_hip.i64((516, 64)))[1]
    assert packed(strides=_hip.i64((1 << 21, 64)))[0] == -1 and b'row stride' in packed(strides=_hip.i64((1 << 21, 64)))[1]
    assert packed(q=None)[0] == -1 and b'null pointer' in packed(q=None)[1]
    assert packed(scale=0.0)[0] == -1 and packed(scale=float('nan'))[0] == -1
    rc = lib.genie_packed_attention_bwd(*([16] * 8), 1 << 20, *([16] * 4), None, 1, 4, 4, 8, 2, 64, two, two, two, two, 1.0, None)
    assert rc == -1 and b'null pointer' in lib.genie_last_error()
    need = lib.genie_packed_attention_bwd_ws_floats(1, 4096, 4096, 8, 2, 64)
    assert need > 8 * 4096
    rc = lib.genie_packed_attention_bwd(*([16] * 8), need - 1, *([16] * 5), 1, 4096, 4096, 8, 2, 64, two, two, two, two, 1.0, None)
    assert rc == -1 and b'workspace' in lib.genie_last_error()
    three = _hip.i64((8192, 512, 64))
    assert lib.genie_cached_attention_step(16, 16, None, 16, 16, 16, 16, None, 0, 1, 8, 2, 64, 16, two, two, two, three, three, 1.0, None) == -1
    assert b'needs a new value' in lib.genie_last_error()
    need = lib.genie_cached_attention_ws_floats(1, 8, 2, 64, 4096)
    assert need > 0
    assert lib.genie_cached_attention_step(16, None, None, 16, 16, 16, 16, 16, need - 1, 1, 8, 2, 64, 4096, two, None, None, three, three, 1.0, None) == -1
    assert b'workspace' in lib.genie_last_error()
    need = lib.genie_decay_attention_state_elems(1, 4096, 8, 64, 64, 0)
    assert need > 0
    assert lib.genie_decay_attention_fwd(16, 16, 16, 16, 16, None, 16, None, 16, 16, need - 1, 1, 4096, 8, 64, 64, two, two, two, 1.0, None) == -1
    assert b'workspace' in lib.genie_last_error()
    assert lib.genie_decay_attention_step(16, 16, 16, 16, 16, 16, 16, 0, 8, 64, 64, two, two, two, 1.0, None) == -1
    assert isinstance(ctypes.c_int64(need).value, int)


def slots(cu, tile):
    """The kernels' slot -> (sequence, tile) map, sequentially."""
    n, rows = len(cu) - 1, cu[-1]
    starts = [cu[s] // tile + s for s in range(n + 1)]
    for slot in range(rows // tile + n + 1):
        s = max(i for i in range(n + 1) if starts[i] <= slot)
        yield s, slot - starts[s]


@pytest.mark.parametrize('seed', range(20))
def test_slot_map_covers_every_tile_once(seed):
    """f(s) = cu[s] // tile + s gives every sequence at least ceil(len / tile) slots, each tile exactly one."""
    import random
    rng = random.Random(seed)
    tile, lens = rng.choice([64, 128]), [rng.choice([0, 1, 63, 64, 65, 128, rng.randint(0, 700)]) for _ in range(rng.randint(1, 90))]
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    seen = [(s, t) for s, t in slots(cu, tile) if s < len(lens) and t * tile < lens[s]]
    assert sorted(seen) == [(s, t) for s, n in enumerate(lens) for t in range((n + tile - 1) // tile)]
