"""Sequence operators: causal softmax attention and linear attention with a decay per head, over packed sequences and one token at a time.

The attention blocks of ``genie.module.attention`` work on clips of one length with equally many query, key and value heads.  The operators here take
token streams of DIFFERENT lengths packed one behind the other (clips cut at different places, sessions at different points of their context), query heads
that share key / value heads, and have forms for single tokens: against a key / value cache, or through a state of constant size.

=============================  =======================================================================================================
``packed_attention``           softmax attention over packed sequences, differentiable
``cached_attention_step``      one new token per sequence against its cache, the token appended in the same call
``decay_attention``            ``S_t = exp(log_decay) S_{t-1} + k_t v_t^T``, ``o_t = scale q_t S_t`` over packed sequences, differentiable
``decay_attention_step``       the same recurrence for one token per sequence
=============================  =======================================================================================================

Common conventions
  * activations are bf16; scores, softmax statistics, sums and recurrent states are fp32.
  * ``cu_seqlens``: int32 device tensor ``[0, n_0, n_0 + n_1, ...]``; sequence ``s`` owns rows ``cu[s] .. cu[s + 1]``.  It is read on the device only: no call
    synchronises, and a captured graph may be replayed with other lengths in the same buffer.  Its contents are therefore not checked; the kernels clamp
    every entry to the rows that exist, so a wrong one costs wrong results and no access out of bounds.  Rows behind ``cu[-1]`` are padding: never read
    (they may hold anything, NaN included), zero in every result and gradient.
  * a tensor whose rows are not 16-byte aligned, or whose last axis is not contiguous, is copied first; slices of a fused projection are taken as they are.
  * the kernels run on the current stream of the tensors' device; scratch memory is allocated per call (a captured graph owns its own).
  * bitwise reproducible: no atomics, every sum has a fixed order.
  * a non-finite value in a token is not masked out: it may reach any row of its own sequence.
"""
from __future__ import annotations

import contextlib
from typing import Optional, Tuple, Union

import torch
from torch import Tensor
from torch.autograd.function import once_differentiable

from . import _hip

MAX_HEAD_DIM = 128
_MAX_ROWS = 1 << 30
_MAX_STRIDE = 1 << 21


def _need(cond: bool, msg: str, kind=ValueError) -> None:
    if not cond:
        raise kind(msg)


def _check(what: str, t: Tensor, name: str, dim: int, dtype: torch.dtype, device: Optional[torch.device] = None) -> None:
    _need(isinstance(t, Tensor), f'{what}: {name} must be a tensor', TypeError)
    _need(t.dim() == dim, f'{what}: {name} must have {dim} axes, got shape {tuple(t.shape)}')
    _need(t.dtype == dtype, f'{what}: {name} must be {dtype}, got {t.dtype}', TypeError)
    _hip.require_gpu(t, f'{what}: {name}')
    _need(device is None or t.device == device, f'{what}: {name} is on {t.device}, q on {device}')


def _check_width(what: str, d: int, name: str) -> None:
    _need(0 < d <= MAX_HEAD_DIM and d % 8 == 0, f'{what}: the width of {name} must be a multiple of 8 up to {MAX_HEAD_DIM}, got {d}')


def _scale(what: str, scale: Optional[float], d: int) -> float:
    s = d ** -0.5 if scale is None else float(scale)
    _need(0.0 < s < 1e30, f'{what}: scale must be positive and finite, got {scale}')
    return s


def _check_cu(what: str, cu: Tensor, name: str, device: torch.device) -> None:
    _check(what, cu, name, 1, torch.int32, device)
    _need(cu.numel() >= 1, f'{what}: {name} must hold at least the leading 0')
    _need(cu.is_contiguous(), f'{what}: {name} must be contiguous')


def _strides(t: Tensor) -> Optional[Tuple[int, ...]]:
    """Element strides of all axes but the last as the kernels take them, or None where the layout has to be copied."""
    if t.stride(-1) != 1 or t.data_ptr() % 16:
        return None
    dense, out = t.shape[-1], []
    for size, st in zip(reversed(t.shape[:-1]), reversed(t.stride()[:-1])):
        st = dense if size == 1 else st
        if st % 8:
            return None
        out.append(st)
        dense *= size
    return tuple(reversed(out))


def _rows(t: Tensor) -> Tuple[Tensor, Tuple[int, ...]]:
    """(rows, heads, d) or (batch, heads, d) ready for the kernels: the tensor itself where its layout allows, else a contiguous copy."""
    st = _strides(t)
    if st is None or st[0] < t.shape[-1] or st[0] >= _MAX_STRIDE:
        # (a row stride under the head width -- rows that overlap or repeat -- would let a tile's last rows be read past its sequence)
        t = t.contiguous()
        st = _strides(t)
        if st is None:                                            # contiguous, but its storage offset is not 16-byte aligned
            t = t.clone(memory_format=torch.contiguous_format)
            st = _strides(t)
        _need(st[0] < _MAX_STRIDE, f'rows of {st[0]} elements are too long (limit {_MAX_STRIDE})')
    return t, st


def _on(device: torch.device):
    """The tensors' device as the current one (kernels launch there), without the cost of a switch where it already is."""
    return contextlib.nullcontext() if device.index == torch.cuda.current_device() else torch.cuda.device(device)


def _stream(device: torch.device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


def _no_grad_wanted(what: str, *tensors: Optional[Tensor]) -> None:
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError(f'{what} has no backward pass: call it under torch.no_grad(), or on tensors that do not require gradients')


# ------------------------------------------------------------------------------------------------------------------------------------
# causal attention over packed sequences
# ------------------------------------------------------------------------------------------------------------------------------------
class _PackedAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q: Tensor, k: Tensor, v: Tensor, cu_q: Tensor, cu_k: Tensor, scale: float):
        rows, hq, d = q.shape
        rows_k, hkv, _ = k.shape
        (q, sq), (k, sk), (v, sv) = _rows(q), _rows(k), _rows(v)
        keep = any(ctx.needs_input_grad[:3])
        out = torch.empty((rows, hq, d), dtype=torch.bfloat16, device=q.device)
        lse = torch.empty((hq, rows), dtype=torch.float32, device=q.device) if keep else None
        if rows and rows_k:
            P = _hip.ptr
            with _on(q.device):
                _hip.check(_hip.load_library().genie_packed_attention_fwd(P(q), P(k), P(v), P(out), P(lse), P(cu_q), P(cu_k), cu_q.numel() - 1, rows, rows_k, hq, hkv,
                                                                          d, _hip.i64(sq), _hip.i64(sk), _hip.i64(sv), scale, _stream(q.device)),
                           'genie_packed_attention_fwd')
        else:
            out.zero_()
        if keep:
            ctx.save_for_backward(q, k, v, out, lse, cu_q, cu_k)
            ctx.cfg = (sq, sk, sv, scale)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout: Tensor):
        q, k, v, out, lse, cu_q, cu_k = ctx.saved_tensors
        sq, sk, sv, scale = ctx.cfg
        rows, hq, d = q.shape
        rows_k, hkv, _ = k.shape
        dout, sg = _rows(dout)
        dq = torch.empty((rows, hq, d), dtype=torch.bfloat16, device=q.device)
        dk = torch.empty((rows_k, hkv, d), dtype=torch.bfloat16, device=q.device)
        dv = torch.empty_like(dk)
        if rows and rows_k:
            delta = torch.empty((hq, rows), dtype=torch.float32, device=q.device)
            P = _hip.ptr
            with _on(q.device):
                _hip.check(_hip.load_library().genie_packed_attention_bwd(P(q), P(k), P(v), P(out), P(dout), P(lse), P(delta), P(dq), P(dk), P(dv), P(cu_q), P(cu_k),
                                                                          cu_q.numel() - 1, rows, rows_k, hq, hkv, d, _hip.i64(sq), _hip.i64(sk), _hip.i64(sv),
                                                                          _hip.i64(sg), scale, _stream(q.device)), 'genie_packed_attention_bwd')
        else:
            for t in (dq, dk, dv):
                t.zero_()
        need = ctx.needs_input_grad
        return dq if need[0] else None, dk if need[1] else None, dv if need[2] else None, None, None, None


def packed_attention(q: Tensor, k: Tensor, v: Tensor, cu_seqlens: Tensor, scale: Optional[float] = None, cu_seqlens_k: Optional[Tensor] = None) -> Tensor:
    """Causal softmax attention inside each packed sequence.

    ``q`` (rows, Hq, d), ``k`` / ``v`` (rows_k, Hkv, d) bf16 with ``Hq`` a multiple of ``Hkv`` (query head h reads key head ``h // (Hq // Hkv)``), d a multiple of 8 up
    to 128; ``scale`` defaults to ``d ** -0.5``.  Returns (rows, Hq, d) bf16; differentiable in q, k and v.

    ``cu_seqlens_k``: the keys' own packing, where a sequence has other keys than queries -- a prompt that continues a context.  The last query then sees the
    last key: query i of n sees keys ``0 .. i + n_k - n``.  A query that sees no key (``n_k < n``) returns zeros and has zero gradients."""
    what = 'packed_attention'
    _check(what, q, 'q', 3, torch.bfloat16)
    _check(what, k, 'k', 3, torch.bfloat16, q.device)
    _check(what, v, 'v', 3, torch.bfloat16, q.device)
    _need(k.shape == v.shape, f'{what}: k {tuple(k.shape)} and v {tuple(v.shape)} differ')
    _check_width(what, q.shape[2], 'a head')
    _need(k.shape[2] == q.shape[2], f'{what}: q and k have head widths {q.shape[2]} and {k.shape[2]}')
    _need(k.shape[1] > 0 and q.shape[1] > 0 and q.shape[1] % k.shape[1] == 0, f'{what}: {q.shape[1]} query heads are no multiple of {k.shape[1]} key heads')
    _need(q.shape[0] <= _MAX_ROWS and k.shape[0] <= _MAX_ROWS, f'{what}: at most {_MAX_ROWS} rows')
    _check_cu(what, cu_seqlens, 'cu_seqlens', q.device)
    if cu_seqlens_k is None:
        _need(q.shape[0] == k.shape[0], f'{what}: q and k have {q.shape[0]} and {k.shape[0]} rows (pass cu_seqlens_k for keys packed differently)')
        cu_seqlens_k = cu_seqlens
    else:
        _check_cu(what, cu_seqlens_k, 'cu_seqlens_k', q.device)
        _need(cu_seqlens_k.numel() == cu_seqlens.numel(), f'{what}: cu_seqlens and cu_seqlens_k describe different numbers of sequences')
    return _PackedAttention.apply(q, k, v, cu_seqlens, cu_seqlens_k, _scale(what, scale, q.shape[2]))


def cached_attention_step(q: Tensor, k_cache: Tensor, v_cache: Tensor, lengths: Tensor, k_new: Optional[Tensor] = None, v_new: Optional[Tensor] = None,
                          scale: Optional[float] = None) -> Tensor:
    """Softmax attention of one new token per sequence against its cache.

    ``q`` (B, Hq, d); ``k_cache`` / ``v_cache`` (B, capacity, Hkv, d) bf16, any strides with a contiguous last axis; ``lengths`` (B,) int32: tokens already in each cache.
    With ``k_new`` / ``v_new`` (B, Hkv, d) the token is written to place ``lengths[b]`` of the caches and attended to as well -- ``lengths`` itself is left alone (the
    caller advances it once for all layers).  Rows of the caches from the length on are not read.  Returns (B, Hq, d) bf16; no backward pass.

    An unused row of the batch has a negative length (without a new token: or zero): it returns zeros and its caches stay as they are.  A length that leaves no room
    in the cache returns NaN and writes nothing -- the lengths live on the device, so a full cache cannot raise here."""
    what = 'cached_attention_step'
    _check(what, q, 'q', 3, torch.bfloat16)
    b, hq, d = q.shape
    dev = q.device
    for t, name in ((k_cache, 'k_cache'), (v_cache, 'v_cache')):
        _check(what, t, name, 4, torch.bfloat16, dev)
    _need(k_cache.shape == v_cache.shape, f'{what}: k_cache {tuple(k_cache.shape)} and v_cache {tuple(v_cache.shape)} differ')
    _, cap, hkv, dk = k_cache.shape
    _check_width(what, d, 'a head')
    _need(k_cache.shape[0] == b and dk == d, f'{what}: q {tuple(q.shape)} does not fit caches of shape {tuple(k_cache.shape)}')
    _need(hkv > 0 and hq > 0 and hq % hkv == 0, f'{what}: {hq} query heads are no multiple of {hkv} key heads')
    _need(0 < cap <= _MAX_ROWS, f'{what}: capacity {cap}')
    _check(what, lengths, 'lengths', 1, torch.int32, dev)
    _need(lengths.shape[0] == b and lengths.is_contiguous(), f'{what}: lengths must be a contiguous tensor of {b} entries')
    _need((k_new is None) == (v_new is None), f'{what}: k_new and v_new come together')
    _no_grad_wanted(what, q, k_cache, v_cache, k_new, v_new)
    scale = _scale(what, scale, d)
    cst = []
    for t, name in ((k_cache, 'k_cache'), (v_cache, 'v_cache')):
        st = _strides(t)
        _need(st is not None, f'{what}: {name} must have a contiguous last axis and 16-byte aligned rows (it is updated in place and cannot be copied)')
        _need(d <= st[1] < _MAX_STRIDE, f'{what}: consecutive tokens of {name} are {st[1]} elements apart (from the head width up to {_MAX_STRIDE} is supported)')
        cst.append(st)
    skn = svn = None
    if k_new is not None:
        for t, name in ((k_new, 'k_new'), (v_new, 'v_new')):
            _check(what, t, name, 3, torch.bfloat16, dev)
            _need(t.shape == (b, hkv, d), f'{what}: {name} must be {(b, hkv, d)}, got {tuple(t.shape)}')
        for t, name in ((k_cache, 'k_cache'), (v_cache, 'v_cache')):
            _need(all(s != 0 or n == 1 for s, n in zip(t.stride(), t.shape)), f'{what}: {name} is an expanded view; a token cannot be appended to it')
        _need(k_cache.data_ptr() != v_cache.data_ptr(), f'{what}: k_cache and v_cache are the same memory')
        (k_new, skn), (v_new, svn) = _rows(k_new.detach()), _rows(v_new.detach())
    q, sq = _rows(q.detach())
    out = torch.empty((b, hq, d), dtype=torch.bfloat16, device=dev)
    if b == 0:
        return out
    lib = _hip.load_library()
    nws = lib.genie_cached_attention_ws_floats(b, hq, hkv, d, cap)
    ws = torch.empty(nws, dtype=torch.float32, device=dev) if nws else None
    P = _hip.ptr
    with _on(dev):
        _hip.check(lib.genie_cached_attention_step(P(q), P(k_new), P(v_new), P(k_cache), P(v_cache), P(lengths), P(out), P(ws), nws, b, hq, hkv, d, cap, _hip.i64(sq),
                                                   None if skn is None else _hip.i64(skn), None if svn is None else _hip.i64(svn), _hip.i64(cst[0]), _hip.i64(cst[1]),
                                                   scale, _stream(dev)), 'genie_cached_attention_step')
    return out


# ------------------------------------------------------------------------------------------------------------------------------------
# linear attention with a decay per head
# ------------------------------------------------------------------------------------------------------------------------------------
class _DecayAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q: Tensor, k: Tensor, v: Tensor, log_decay: Tensor, cu: Tensor, initial_state: Optional[Tensor], scale: float, return_state: bool):
        rows, h, dk = q.shape
        dv, nseq, dev = v.shape[2], cu.numel() - 1, q.device
        (q, sq), (k, sk), (v, sv) = _rows(q), _rows(k), _rows(v)
        out = torch.empty((rows, h, dv), dtype=torch.bfloat16, device=dev)
        final = torch.empty((nseq, h, dk, dv), dtype=torch.float32, device=dev) if return_state else None
        seg, nws = None, 0
        if rows:
            lib, P = _hip.load_library(), _hip.ptr
            nws = lib.genie_decay_attention_ws_floats(nseq, rows, h, dk, dv)
            seg = torch.empty(nws, dtype=torch.float32, device=dev) if nws else None
            with _on(dev):
                _hip.check(lib.genie_decay_attention_fwd(P(q), P(k), P(v), P(log_decay), P(cu), P(initial_state), P(out), P(final), P(seg), nws, nseq, rows, h, dk, dv,
                                                         _hip.i64(sq), _hip.i64(sk), _hip.i64(sv), scale, _stream(dev)), 'genie_decay_attention_fwd')
        elif return_state:
            final.zero_() if initial_state is None else final.copy_(initial_state)
        if any(ctx.needs_input_grad[:3]):
            ctx.save_for_backward(q, k, v, log_decay, cu, initial_state, seg)
            ctx.cfg = (sq, sk, sv, scale, nws)
        if return_state:
            ctx.mark_non_differentiable(final)
            return out, final
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout: Tensor, *_):
        q, k, v, log_decay, cu, initial_state, seg = ctx.saved_tensors
        sq, sk, sv, scale, nws = ctx.cfg
        rows, h, dk = q.shape
        dv, nseq, dev = v.shape[2], cu.numel() - 1, q.device
        dout, sg = _rows(dout)
        gq, gk = (torch.empty((rows, h, dk), dtype=torch.bfloat16, device=dev) for _ in range(2))
        gv = torch.empty((rows, h, dv), dtype=torch.bfloat16, device=dev)
        if rows:
            rev = torch.empty(nws, dtype=torch.float32, device=dev) if nws else None
            P = _hip.ptr
            with _on(dev):
                _hip.check(_hip.load_library().genie_decay_attention_bwd(P(q), P(k), P(v), P(dout), P(log_decay), P(cu), P(initial_state), P(seg), P(rev), nws, P(gq),
                                                                         P(gk), P(gv), nseq, rows, h, dk, dv, _hip.i64(sq), _hip.i64(sk), _hip.i64(sv), _hip.i64(sg),
                                                                         scale, _stream(dev)), 'genie_decay_attention_bwd')
        need = ctx.needs_input_grad
        return gq if need[0] else None, gk if need[1] else None, gv if need[2] else None, None, None, None, None, None


def _check_decay(what: str, log_decay: Tensor, heads: int, device: torch.device) -> Tensor:
    _check(what, log_decay, 'log_decay', 1, torch.float32, device)
    _need(log_decay.shape[0] == heads, f'{what}: log_decay must hold one value for each of the {heads} heads, got {tuple(log_decay.shape)}')
    _need(not (log_decay.requires_grad and torch.is_grad_enabled()), f'{what}: the decays are constants (no gradient): pass log_decay.detach()', RuntimeError)
    return log_decay.detach().contiguous()


def decay_attention(q: Tensor, k: Tensor, v: Tensor, log_decay: Tensor, cu_seqlens: Tensor, initial_state: Optional[Tensor] = None, scale: Optional[float] = None,
                    return_state: bool = False) -> Union[Tensor, Tuple[Tensor, Tensor]]:
    """Linear attention with a decay for each head over packed sequences: ``S_t = exp(log_decay[h]) S_{t-1} + k_t v_t^T``, ``o_t = scale q_t S_t``.

    ``q`` / ``k`` (rows, H, dk), ``v`` (rows, H, dv) bf16, widths multiples of 8 up to 128; ``log_decay`` (H,) fp32, <= 0 (``-inf``: no memory, 0: none is lost);
    ``scale`` defaults to ``dk ** -0.5``.  Returns (rows, H, dv) bf16, differentiable in q, k and v.

    ``initial_state`` (sequences, H, dk, dv) fp32: the state in front of each sequence's first token.  ``return_state``: also return the state behind each sequence's
    last token, which ``decay_attention_step`` and a later call continue from.  States carry no gradient (truncated backpropagation)."""
    what = 'decay_attention'
    _check(what, q, 'q', 3, torch.bfloat16)
    _check(what, k, 'k', 3, torch.bfloat16, q.device)
    _check(what, v, 'v', 3, torch.bfloat16, q.device)
    rows, h, dk = q.shape
    _need(k.shape == q.shape, f'{what}: q {tuple(q.shape)} and k {tuple(k.shape)} differ')
    _need(v.shape[:2] == q.shape[:2], f'{what}: v {tuple(v.shape)} does not fit q {tuple(q.shape)}')
    _need(h > 0, f'{what}: no heads')
    _need(rows <= _MAX_ROWS, f'{what}: at most {_MAX_ROWS} rows')
    _check_width(what, dk, 'q and k')
    _check_width(what, v.shape[2], 'v')
    log_decay = _check_decay(what, log_decay, h, q.device)
    _check_cu(what, cu_seqlens, 'cu_seqlens', q.device)
    if initial_state is not None:
        _check(what, initial_state, 'initial_state', 4, torch.float32, q.device)
        want = (cu_seqlens.numel() - 1, h, dk, v.shape[2])
        _need(tuple(initial_state.shape) == want, f'{what}: initial_state must be {want}, got {tuple(initial_state.shape)}')
        _need(not (initial_state.requires_grad and torch.is_grad_enabled()), f'{what}: no gradient flows into a state: pass initial_state.detach()', RuntimeError)
        initial_state = initial_state.detach().contiguous()
    return _DecayAttention.apply(q, k, v, log_decay, cu_seqlens, initial_state, _scale(what, scale, dk), bool(return_state))


def decay_attention_step(q: Tensor, k: Tensor, v: Tensor, log_decay: Tensor, state: Tensor, scale: Optional[float] = None, new_state: Optional[Tensor] = None) -> Tensor:
    """``decay_attention`` for one token per sequence: ``q`` / ``k`` (B, H, dk), ``v`` (B, H, dv) bf16, ``state`` (B, H, dk, dv) fp32, contiguous.  The state is advanced in
    place, or into ``new_state`` (the old one then stays).  Returns (B, H, dv) bf16; no backward pass."""
    what = 'decay_attention_step'
    _check(what, q, 'q', 3, torch.bfloat16)
    _check(what, k, 'k', 3, torch.bfloat16, q.device)
    _check(what, v, 'v', 3, torch.bfloat16, q.device)
    b, h, dk = q.shape
    dv = v.shape[2]
    _need(k.shape == q.shape, f'{what}: q {tuple(q.shape)} and k {tuple(k.shape)} differ')
    _need(v.shape[:2] == q.shape[:2], f'{what}: v {tuple(v.shape)} does not fit q {tuple(q.shape)}')
    _need(h > 0, f'{what}: no heads')
    _check_width(what, dk, 'q and k')
    _check_width(what, dv, 'v')
    log_decay = _check_decay(what, log_decay, h, q.device)
    _no_grad_wanted(what, q, k, v, state, new_state)
    new_state = state if new_state is None else new_state
    for t, name in ((state, 'state'), (new_state, 'new_state')):
        _check(what, t, name, 4, torch.float32, q.device)
        _need(tuple(t.shape) == (b, h, dk, dv), f'{what}: {name} must be {(b, h, dk, dv)}, got {tuple(t.shape)}')
        _need(t.is_contiguous() and t.data_ptr() % 16 == 0, f'{what}: {name} must be contiguous and 16-byte aligned')
    lo, hi = sorted((state.data_ptr(), new_state.data_ptr()))
    _need(lo == hi or hi - lo >= state.numel() * 4, f'{what}: new_state overlaps state without being it')
    scale = _scale(what, scale, dk)
    (q, sq), (k, sk), (v, sv) = _rows(q.detach()), _rows(k.detach()), _rows(v.detach())
    out = torch.empty((b, h, dv), dtype=torch.bfloat16, device=q.device)
    if b == 0:
        return out
    P = _hip.ptr
    with _on(q.device):
        _hip.check(_hip.load_library().genie_decay_attention_step(P(q), P(k), P(v), P(log_decay), P(state), P(new_state), P(out), b, h, dk, dv, _hip.i64(sq), _hip.i64(sk),
                                                                  _hip.i64(sv), scale, _stream(q.device)), 'genie_decay_attention_step')
    return out
