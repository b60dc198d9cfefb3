"""Plain 64-bit references of the sequence operators (genie/sequence.py), one sequence and head at a time, with the error bounds their tests use.

U = 2^-8 is the most a rounding to bf16 can move a value (half a step).  Every bound below is the sum, over the roundings to bf16 that the operator makes,
of U times the magnitude that is rounded, carried through to the result, plus SLACK times the sum of magnitudes for the fp32 arithmetic in between: at most a
few hundred operations of 2^-24 each and one hardware exp2 of a score below 2^6 in size, whose fp32 error of 2^-18 passes into the weight -- 2^-14 in all."""
import torch

U = 2.0 ** -8
SLACK = 2.0 ** -14


def bounds(lens):
    out, at = [], 0
    for n in lens:
        out.append((at, at + n))
        at += n
    return out


def packed_reference(q, k, v, lens, scale, dout=None, lens_k=None, w=U):
    """out, dq, dk, dv and the largest error each may have (dicts by name).  w: what the roundings of the weights (P, dS) and of the output in delta move them by:
    U, or U^2 where the kernels carry a second bf16 value for what the first left over."""
    q, k, v = q.double(), k.double(), v.double()
    g = None if dout is None else dout.double()
    hq, hkv = q.shape[1], k.shape[1]
    names = ['out'] + ([] if g is None else ['dq', 'dk', 'dv'])
    val = {n: torch.zeros_like(t) for n, t in zip(names, (q, q, k, v))}
    tol = {n: torch.zeros_like(t) for n, t in zip(names, (q, q, k, v))}
    for (a, b), (ka, kb) in zip(bounds(lens), bounds(lens if lens_k is None else lens_k)):
        n, m = b - a, kb - ka
        if n == 0 or m == 0:
            continue
        sees = torch.arange(m, device=q.device)[None, :] <= torch.arange(n, device=q.device)[:, None] + (m - n)
        for h in range(hq):
            j = h // (hq // hkv)
            Q, K, V = q[a:b, h], k[ka:kb, j], v[ka:kb, j]
            s = (scale * (Q @ K.T)).masked_fill(~sees, -torch.inf)
            p = torch.exp(s - s.amax(1, keepdim=True).clamp(min=-1e300))
            p = torch.where(sees, p, torch.zeros_like(p))
            p = p / p.sum(1, keepdim=True).clamp(min=1e-300)
            o = p @ V
            val['out'][a:b, h] = o
            t_o = U * o.abs() + (w + SLACK) * (p @ V.abs())                      # own rounding; weights' rounding
            tol['out'][a:b, h] = t_o
            if g is None:
                continue
            G = g[a:b, h]
            dp, delta = G @ V.T, (G * o).sum(1, keepdim=True)
            ds = p * (dp - delta)
            val['dq'][a:b, h] = scale * (ds @ K)
            val['dk'][ka:kb, j] += scale * (ds.T @ Q)
            val['dv'][ka:kb, j] += p.T @ G
            # dS is rounded; delta comes from the rounded output; SLACK of the magnitudes that dP and delta are sums of
            e_ds = w * ds.abs() + p * (G.abs() * (t_o - (U - w) * o.abs())).sum(1, keepdim=True) + SLACK * p * (G.abs() @ V.abs().T + (G * o).abs().sum(1, keepdim=True))
            tol['dq'][a:b, h] = scale * (e_ds @ K.abs())
            tol['dk'][ka:kb, j] += scale * (e_ds.T @ Q.abs())
            tol['dv'][ka:kb, j] += (w + SLACK) * (p.T @ G.abs())
    for n in names[1:]:
        tol[n] += U * val[n].abs()
    return val, tol


def step_reference(q, k_cache, v_cache, lengths, scale, w=U):
    """One query per sequence against the first lengths[b] places of its cache."""
    val, tol = torch.zeros_like(q, dtype=torch.float64), torch.zeros_like(q, dtype=torch.float64)
    for b, n in enumerate(lengths):
        for h in range(q.shape[1]):
            if n > 0:
                j = h // (q.shape[1] // k_cache.shape[2])
                p = torch.softmax(scale * (k_cache[b, :n, j].double() @ q[b, h].double()), 0)
                V = v_cache[b, :n, j].double()
                val[b, h] = p @ V
                tol[b, h] = U * val[b, h].abs() + (w + SLACK) * (p @ V.abs())
    return val, tol


def decay_form(a, b, c, log_decay, lens, scale, reverse=False, state=None, w=U):
    """y_t = scale sum_{s <= t} l^(t-s) (a_t . b_s) c_s + scale l^(t+1) a_t S, and its bound: the scores (or the state they are summed into) are rounded to
    bf16 as operands (w: by how much), the result is rounded once."""
    a, b, c = a.double(), b.double(), c.double()
    val = torch.zeros(a.shape[:2] + c.shape[2:], dtype=torch.float64, device=a.device)
    tol = torch.zeros_like(val)
    for i, (lo, hi) in enumerate(bounds(lens)):
        t = torch.arange(hi - lo, device=a.device, dtype=torch.float64)
        far = (t[None, :] - t[:, None]) if reverse else (t[:, None] - t[None, :])
        for h in range(a.shape[1]):
            l = float(log_decay[h])
            fade = torch.where(far == 0, torch.ones_like(far), torch.where(far > 0, torch.exp(l * far.clamp(min=1)), torch.zeros_like(far)))
            A, B, C = a[lo:hi, h], b[lo:hi, h], c[lo:hi, h]
            y = ((A @ B.T) * fade) @ C
            mag = ((A.abs() @ B.abs().T) * fade) @ C.abs()
            if state is not None:
                lead = torch.exp(l * (t + 1))[:, None]
                y = y + lead * (A @ state[i, h].double())
                mag = mag + lead * (A.abs() @ state[i, h].double().abs())
            val[lo:hi, h] = scale * y
            tol[lo:hi, h] = scale * (U * y.abs() + (w + SLACK) * mag)
    return val, tol


def decay_state(k, v, log_decay, lens, state=None):
    """State behind each sequence; its fp32 bound: the decayed operand is a sum of two bf16 values (U^2 left), the rest is fp32."""
    n, h = len(lens), k.shape[1]
    val = torch.zeros((n, h, k.shape[2], v.shape[2]), dtype=torch.float64, device=k.device)
    mag = torch.zeros_like(val)
    for i, (lo, hi) in enumerate(bounds(lens)):
        for j in range(h):
            l, L = float(log_decay[j]), hi - lo
            e = torch.arange(L - 1, -1, -1, device=k.device, dtype=torch.float64)
            w = torch.where(e == 0, torch.ones_like(e), torch.exp(l * e.clamp(min=1)))[:, None]
            K, V = k[lo:hi, j].double(), v[lo:hi, j].double()
            val[i, j], mag[i, j] = (K * w).T @ V, (K * w).abs().T @ V.abs()
            if state is not None:
                f = 1.0 if L == 0 else float(torch.exp(torch.tensor(l * L, dtype=torch.float64)))
                val[i, j] += f * state[i, j].double()
                mag[i, j] += f * state[i, j].double().abs()
    return val, mag * (U * U + 2.0 ** -18)


def assert_within(got, want, tol, what):
    got = got.double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert torch.isfinite(got).all(), f'{what}: not finite'
    bad = (got - want).abs() > tol + 1e-30
    if bad.any():
        i = int(((got - want).abs() / (tol + 1e-30)).argmax())
        raise AssertionError(f'{what}: {int(bad.sum())} of {bad.numel()} values outside; worst {got.flatten()[i].item()} for {want.flatten()[i].item()}, allowed '
                             f'{tol.flatten()[i].item()} (index {i})')
    # as a whole: the final rounding is at most U of the norm, the operands' roundings are independent of each other and together at most U of it
    norm = want.norm()
    if norm > 0 and got.dtype.is_floating_point and want.numel() >= 4096 and tol.sum() > 0:
        rel = ((got - want).norm() / norm).item()
        assert rel <= 2 * U, f'{what}: relative error {rel}'
