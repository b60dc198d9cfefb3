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
    Tensors saved for a backward pass are looked at again as they come back from hooks on saved tensors (``torch.autograd.graph.save_on_cpu`` and its like).
  * the kernels run on the current stream of the tensors' device; scratch memory is allocated per call (a captured graph owns its own).
  * bitwise reproducible: no atomics, every sum has a fixed order.
  * capture of a backward pass into a graph: with no eager autograd graph of the same leaves alive (torch ends the process where it meets a leaf's node of another
    stream inside a capture; this holds for every differentiable operator).
  * gradients of gradients and forward-mode differentiation (dual tensors) are refused.
  * weights (P, dS, decayed scores) and the state in front of a segment are bf16 operands; in calls of up to 256 rows (of the buffers: those behind the last sequence
    count), and in the cached form always, a second bf16 value carries what that left over.  In longer calls a carried state enters outputs and dq as one bf16 value.
  * a non-finite value in a token is not masked out: it may reach any row of its own sequence, and an infinity may arrive as NaN.  Tokens behind a cache's length are not read.
  * softmax exponents are fp32: a weight is off by some 2^-23 of the largest score (scale q.k) in size, and scores from 2^30 on are out of range.
"""
from __future__ import annotations

import functools
from typing import Optional, Tuple, Union

import torch
from torch import Tensor
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _hip

MAX_HEAD_DIM = 128
_MAX_ROWS = 1 << 30
_MAX_STRIDE = 1 << 21


def _check(what: str, t: Tensor, name: str, dim: int, dtype: torch.dtype, device: Optional[torch.device] = None) -> None:
    if not isinstance(t, Tensor):
        raise TypeError(f'{what}: {name} must be a tensor')
    if t.dim() != dim:
        raise ValueError(f'{what}: {name} must have {dim} axes, got shape {tuple(t.shape)}')
    if t.dtype != dtype:
        raise TypeError(f'{what}: {name} must be {dtype}, got {t.dtype}')
    if not t.is_cuda:
        _hip.require_gpu(t, f'{what}: {name}')
    if device is not None and t.device != device:
        raise ValueError(f'{what}: {name} is on {t.device}, q on {device}')


def _check_width(what: str, d: int, name: str) -> None:
    if d % 8 or not 0 < d <= MAX_HEAD_DIM:
        raise ValueError(f'{what}: the width of {name} must be a multiple of 8 up to {MAX_HEAD_DIM}, got {d}')


def _scale(what: str, scale: Optional[float], d: int) -> float:
    s = d ** -0.5 if scale is None else float(scale)
    if not 0.0 < s < 1e30:
        raise ValueError(f'{what}: scale must be positive and finite, got {scale}')
    return s


def _check_cu(what: str, cu: Tensor, name: str, device: torch.device) -> None:
    _check(what, cu, name, 1, torch.int32, device)
    if cu.shape[0] < 1:
        raise ValueError(f'{what}: {name} must hold at least the leading 0')
    if not cu.is_contiguous():
        raise ValueError(f'{what}: {name} must be contiguous')


def _strides(t: Tensor) -> Optional[Tuple[int, ...]]:
    """Element strides of all axes but the last as the kernels take them, or None where the layout (alignment of the first element aside) has to be copied.  An axis
    of one entry takes the stride it would have in a dense tensor."""
    *lead, last = t.stride()
    if last != 1:
        return None
    shape = t.shape
    if 1 in shape:
        dense = shape[-1]
        for i in range(len(lead) - 1, -1, -1):
            if shape[i] == 1:
                lead[i] = dense
            dense *= shape[i]
    for st in lead:
        if st % 8:
            return None
    return tuple(lead)


def _direct(t: Tensor) -> Optional[Tuple[int, ...]]:
    """Strides of (rows, heads, d) or (batch, heads, d) if the kernels can take it as it is, its alignment aside."""
    st = _strides(t)
    # (a row stride under the head width -- rows that overlap or repeat -- would let a tile's last rows be read past its sequence)
    return st if st is not None and t.shape[2] <= st[0] < _MAX_STRIDE else None


def _rows(t: Tensor) -> Tuple[Tensor, Tuple[int, ...]]:
    """(rows, heads, d) or (batch, heads, d) ready for the kernels: the tensor itself where its layout allows, else a contiguous copy."""
    if t.numel() == 0:                                            # (torch calls an empty tensor contiguous whatever its strides are)
        return t, (t.shape[1] * t.shape[2], t.shape[2])
    st = _direct(t)
    if st is None or t.data_ptr() % 16:
        t = t.contiguous() if st is None else t.clone(memory_format=torch.contiguous_format)
        if t.data_ptr() % 16:                                     # contiguous all along, but its storage offset is not 16-byte aligned
            t = t.clone()
        st = _strides(t)
        if st[0] >= _MAX_STRIDE:
            raise ValueError(f'rows of {st[0]} elements are too long (limit {_MAX_STRIDE})')
    return t, st


@functools.lru_cache(maxsize=1024)
def _i64(strides: Tuple[int, ...]):
    return _hip.i64(strides)


def _launch(name: str, device: torch.device, *args) -> None:
    """One C-ABI call on the current stream of the tensors' device, that device being the current one."""
    fn, index = getattr(_hip.load_library(), name), device.index
    if torch._C._cuda_getDevice() == index:
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    if rc:
        _hip.check(rc, name)


def _sig(t: Optional[Tensor]):
    return None if t is None else (t.dtype, t.get_device(), t.shape, t.stride())


_PLANS: dict = {}


def _planned(make, tensors, *rest):
    """``make(*tensors, *rest)``: all checks of a call that its types, devices, shapes and strides decide, and what follows from them for the launch.  Kept for the calls
    that look the same (a token's call: 18 us with the checks, 11 without; a layout's first call
    takes 3 us more than the checks alone; the backward pass of a training call 4 us of 115); nothing in it depends on a tensor's address or contents."""
    try:
        key = (make, *map(_sig, tensors), *rest)
    except AttributeError:                                        # not a tensor: the checks say so
        return make(*tensors, *rest)
    plan = _PLANS.get(key)
    if plan is None:
        plan = make(*tensors, *rest)
        if len(_PLANS) >= 4096:
            _PLANS.clear()
        _PLANS[key] = plan
    return plan


def _came_back(what: str, t: Optional[Tensor], name: str, dtype: torch.dtype, shape: Tuple[int, ...], device: torch.device) -> None:
    """A tensor that the forward pass saved: hooks on saved tensors (``torch.autograd.graph.save_on_cpu`` and its like) may bring it back with other strides, at
    another address, or as something else altogether."""
    if not isinstance(t, Tensor) or t.dtype != dtype or t.shape != shape or t.device != device:
        got = f'{t.dtype} {tuple(t.shape)} on {t.device}' if isinstance(t, Tensor) else repr(t)
        raise RuntimeError(f'{what}: {name} was saved for the backward pass as {dtype} {tuple(shape)} on {device} and came back as {got}')


def _dense(t: Optional[Tensor]) -> Optional[Tensor]:
    """The tensor itself if it is contiguous and 16-byte aligned, else a copy that is."""
    if t is None:
        return None
    t = t.contiguous()
    return t.clone() if t.data_ptr() % 16 else t


def _no_grad_wanted(what: str, *tensors: Optional[Tensor]) -> None:
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError(f'{what} has no backward pass: call it under torch.no_grad(), or on tensors that do not require gradients')


def _no_tangents(what: str, *tensors: Optional[Tensor]) -> None:
    """Forward-mode differentiation has no formula here; a result without its tangent would be a wrong derivative of zero."""
    if forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError(f'{what} has no forward-mode derivative (an argument is a dual tensor)')


def _first_order(backward):
    """``once_differentiable``, whose bookkeeping (3 us of a small training call's 120) only runs where a graph of the backward pass is asked for."""
    recorded = once_differentiable(backward)

    @functools.wraps(backward)
    def run(ctx, *grads):
        return recorded(ctx, *grads) if torch.is_grad_enabled() else backward(ctx, *grads)
    return run


# ------------------------------------------------------------------------------------------------------------------------------------
# causal attention over packed sequences
# ------------------------------------------------------------------------------------------------------------------------------------
def _packed_forward(q: Tensor, k: Tensor, v: Tensor, cu_q: Tensor, cu_k: Tensor, scale: float, sizes, strides, keep: bool):
    """(out, tensors that the backward pass keeps); strides: those of q, k and v where no tensor needs a copy, their alignment aside"""
    _, rows, rows_k, hq, _, d = sizes
    if strides is None or (q.data_ptr() | k.data_ptr() | v.data_ptr()) % 16:
        (q, sq), (k, sk), (v, sv) = _rows(q), _rows(k), _rows(v)
        strides = _i64(sq), _i64(sk), _i64(sv)
    out = q.new_empty((rows, hq, d))
    # for the backward pass, in one buffer: what out's rounding left over (bf16, rows x hq x d), then the log-sum-exps (fp32, hq x rows)
    rest, lo, lse = None, None, None
    if keep:
        rest = torch.empty(rows * hq * (d // 2 + 1), dtype=torch.float32, device=q.device)
        lo = rest.data_ptr()
        lse = lo + rows * hq * d * 2
    if rows and rows_k:
        _launch('genie_packed_attention_fwd', q.device, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lo, lse, cu_q.data_ptr(), cu_k.data_ptr(), *sizes, *strides, scale)
    else:
        out.zero_()
    return out, (q, k, v, out, rest, cu_q, None if cu_k is cu_q else cu_k)


def _packed_bwd_plan(q, k, v, out, rest, cu_q, cu_k, dout, sizes):
    """(None or the strides of q, k, v and dout where no tensor needs a copy, floats of workspace), from the tensors as they came back"""
    what, dev = 'packed_attention', dout.device
    nseq, rows, rows_k, hq, hkv, d = sizes
    for t, name, dtype, shape in ((q, 'q', torch.bfloat16, (rows, hq, d)), (k, 'k', torch.bfloat16, (rows_k, hkv, d)), (v, 'v', torch.bfloat16, (rows_k, hkv, d)),
                                  (out, 'the output', torch.bfloat16, (rows, hq, d)), (rest, 'its remainder', torch.float32, (rows * hq * (d // 2 + 1),)),
                                  (cu_q, 'cu_seqlens', torch.int32, (nseq + 1,)), (cu_q if cu_k is None else cu_k, 'cu_seqlens_k', torch.int32, (nseq + 1,))):
        _came_back(what, t, name, dtype, shape, dev)
    strides = [_direct(t) for t in (q, k, v, dout)]
    direct = None not in strides and all(t is None or t.is_contiguous() for t in (out, rest, cu_q, cu_k))
    return tuple(map(_i64, strides)) if direct else None, _hip.load_library().genie_packed_attention_bwd_ws_floats(*sizes)


class _PackedAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q: Tensor, k: Tensor, v: Tensor, cu_q: Tensor, cu_k: Tensor, scale: float, sizes, strides):
        out, saved = _packed_forward(q, k, v, cu_q, cu_k, scale, sizes, strides, True)
        ctx.sizes, ctx.scale = sizes, scale
        ctx.save_for_backward(*saved)
        return out

    @staticmethod
    @_first_order
    def backward(ctx, dout: Tensor):
        # nothing about the saved tensors' layout is taken over from the forward pass: they are looked at as they came back
        q, k, v, out, rest, cu_q, cu_k = ctx.saved_tensors
        _, rows, rows_k, hq, hkv, d = sizes = ctx.sizes
        strides, nws = _planned(_packed_bwd_plan, (q, k, v, out, rest, cu_q, cu_k, dout), sizes)
        dq, dk, dv = q.new_empty((rows, hq, d)), q.new_empty((rows_k, hkv, d)), q.new_empty((rows_k, hkv, d))
        if rows and rows_k:
            if strides is None or (q.data_ptr() | k.data_ptr() | v.data_ptr() | dout.data_ptr() | out.data_ptr() | rest.data_ptr()) % 16:
                (q, sq), (k, sk), (v, sv), (dout, sg) = _rows(q), _rows(k), _rows(v), _rows(dout)
                strides = _i64(sq), _i64(sk), _i64(sv), _i64(sg)
                out, rest, cu_q, cu_k = _dense(out), _dense(rest), _dense(cu_q), _dense(cu_k)
            cu_k = cu_q if cu_k is None else cu_k
            lo = rest.data_ptr()
            ws = torch.empty(nws, dtype=torch.float32, device=q.device)
            _launch('genie_packed_attention_bwd', q.device, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lo, dout.data_ptr(), lo + rows * hq * d * 2, ws.data_ptr(), nws,
                    dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), cu_q.data_ptr(), cu_k.data_ptr(), *sizes, *strides, ctx.scale)
        else:
            for t in (dq, dk, dv):
                t.zero_()
        need = ctx.needs_input_grad
        return dq if need[0] else None, dk if need[1] else None, dv if need[2] else None, None, None, None, None, None


def _packed_plan(q, k, v, cu_seqlens, cu_seqlens_k, scale):
    """(scale, sizes, None or the strides of q, k and v where they need no copy)"""
    what = 'packed_attention'
    _check(what, q, 'q', 3, torch.bfloat16)
    _check(what, k, 'k', 3, torch.bfloat16, q.device)
    _check(what, v, 'v', 3, torch.bfloat16, q.device)
    if k.shape != v.shape:
        raise ValueError(f'{what}: k {tuple(k.shape)} and v {tuple(v.shape)} differ')
    rows, hq, d = q.shape
    rows_k, hkv, _ = k.shape
    _check_width(what, d, 'a head')
    if k.shape[2] != d:
        raise ValueError(f'{what}: q and k have head widths {q.shape[2]} and {k.shape[2]}')
    if hkv == 0 or hq == 0 or hq % hkv:
        raise ValueError(f'{what}: {q.shape[1]} query heads are no multiple of {k.shape[1]} key heads')
    if rows > _MAX_ROWS or rows_k > _MAX_ROWS:
        raise ValueError(f'{what}: at most {_MAX_ROWS} rows')
    _check_cu(what, cu_seqlens, 'cu_seqlens', q.device)
    if cu_seqlens_k is None:
        if rows != rows_k:
            raise ValueError(f'{what}: q and k have {q.shape[0]} and {k.shape[0]} rows (pass cu_seqlens_k for keys packed differently)')
    else:
        _check_cu(what, cu_seqlens_k, 'cu_seqlens_k', q.device)
        if cu_seqlens_k.shape != cu_seqlens.shape:
            raise ValueError(f'{what}: cu_seqlens and cu_seqlens_k describe different numbers of sequences')
    scale = _scale(what, scale, d)
    strides = [_direct(t) for t in (q, k, v)]
    return scale, (cu_seqlens.shape[0] - 1, rows, rows_k, hq, hkv, d), None if None in strides else tuple(map(_i64, strides))


def packed_attention(q: Tensor, k: Tensor, v: Tensor, cu_seqlens: Tensor, scale: Optional[float] = None, cu_seqlens_k: Optional[Tensor] = None) -> Tensor:
    """Causal softmax attention inside each packed sequence.

    ``q`` (rows, Hq, d), ``k`` / ``v`` (rows_k, Hkv, d) bf16 with ``Hq`` a multiple of ``Hkv`` (query head h reads key head ``h // (Hq // Hkv)``), d a multiple of 8 up
    to 128; ``scale`` defaults to ``d ** -0.5``.  Returns (rows, Hq, d) bf16; differentiable in q, k and v.

    ``cu_seqlens_k``: the keys' own packing, where a sequence has other keys than queries -- a prompt that continues a context.  The last query then sees the
    last key: query i of n sees keys ``0 .. i + n_k - n``.  A query that sees no key (``n_k < n``) returns zeros and has zero gradients."""
    scale, sizes, strides = _planned(_packed_plan, (q, k, v, cu_seqlens, cu_seqlens_k), None if scale is None else float(scale))
    _no_tangents('packed_attention', q, k, v)
    if cu_seqlens_k is None:
        cu_seqlens_k = cu_seqlens
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        return _PackedAttention.apply(q, k, v, cu_seqlens, cu_seqlens_k, scale, sizes, strides)
    return _packed_forward(q, k, v, cu_seqlens, cu_seqlens_k, scale, sizes, strides, False)[0]


def _cached_plan(q, k_cache, v_cache, lengths, k_new, v_new, scale):
    """(device, the output's shape, floats of workspace, None or the strides of tensors that need no copy, (sizes, caches' strides, scale))"""
    what = 'cached_attention_step'
    _check(what, q, 'q', 3, torch.bfloat16)
    b, hq, d = q.shape
    dev = q.device
    for t, name in ((k_cache, 'k_cache'), (v_cache, 'v_cache')):
        _check(what, t, name, 4, torch.bfloat16, dev)
    if k_cache.shape != v_cache.shape:
        raise ValueError(f'{what}: k_cache {tuple(k_cache.shape)} and v_cache {tuple(v_cache.shape)} differ')
    _, cap, hkv, dk = k_cache.shape
    _check_width(what, d, 'a head')
    if k_cache.shape[0] != b or dk != d:
        raise ValueError(f'{what}: q {tuple(q.shape)} does not fit caches of shape {tuple(k_cache.shape)}')
    if hkv == 0 or hq == 0 or hq % hkv:
        raise ValueError(f'{what}: {hq} query heads are no multiple of {hkv} key heads')
    if not 0 < cap <= _MAX_ROWS:
        raise ValueError(f'{what}: capacity {cap}')
    _check(what, lengths, 'lengths', 1, torch.int32, dev)
    if lengths.shape[0] != b or not lengths.is_contiguous():
        raise ValueError(f'{what}: lengths must be a contiguous tensor of {b} entries')
    if (k_new is None) != (v_new is None):
        raise ValueError(f'{what}: k_new and v_new come together')
    scale = _scale(what, scale, d)
    cst = []
    for t, name in ((k_cache, 'k_cache'), (v_cache, 'v_cache')):
        st = _strides(t)
        if st is None:
            raise ValueError(f'{what}: {name} must have a contiguous last axis and 16-byte aligned rows (it is updated in place and cannot be copied)')
        if not d <= st[1] < _MAX_STRIDE:
            raise ValueError(f'{what}: consecutive tokens of {name} are {st[1]} elements apart (from the head width up to {_MAX_STRIDE} is supported)')
        cst.append(st)
    rows = [q]
    if k_new is not None:
        for t, name in ((k_new, 'k_new'), (v_new, 'v_new')):
            _check(what, t, name, 3, torch.bfloat16, dev)
            if t.shape != (b, hkv, d):
                raise ValueError(f'{what}: {name} must be {(b, hkv, d)}, got {tuple(t.shape)}')
        for st, t, name in ((cst[0], k_cache, 'k_cache'), (cst[1], v_cache, 'v_cache')):
            if any(s == 0 and n > 1 for s, n in zip(st, t.shape)):
                raise ValueError(f'{what}: {name} is an expanded view; a token cannot be appended to it')
        rows += [k_new, v_new]
    direct = [_direct(t) for t in rows]
    direct = None if None in direct else (*map(_i64, direct), None, None)[:3]
    nws = _hip.load_library().genie_cached_attention_ws_floats(b, hq, hkv, d, cap)
    return dev, (b, hq, d), nws, direct, ((b, hq, hkv, d, cap), (_i64(cst[0]), _i64(cst[1])), scale)


def cached_attention_step(q: Tensor, k_cache: Tensor, v_cache: Tensor, lengths: Tensor, k_new: Optional[Tensor] = None, v_new: Optional[Tensor] = None,
                          scale: Optional[float] = None) -> Tensor:
    """Softmax attention of one new token per sequence against its cache.

    ``q`` (B, Hq, d); ``k_cache`` / ``v_cache`` (B, capacity, Hkv, d) bf16, any strides with a contiguous last axis; ``lengths`` (B,) int32: tokens already in each cache.
    With ``k_new`` / ``v_new`` (B, Hkv, d) the token is written to place ``lengths[b]`` of the caches and attended to as well -- ``lengths`` itself is left alone (the
    caller advances it once for all layers).  Rows of the caches from the length on are not read.  Returns (B, Hq, d) bf16; no backward pass.

    An unused row of the batch has a negative length (without a new token: or zero): it returns zeros and its caches stay as they are.  A length that leaves no room
    in the cache returns NaN and writes nothing -- the lengths live on the device, so a full cache cannot raise here."""
    what = 'cached_attention_step'
    new = k_new is not None
    device, shape, nws, direct, tail = _planned(_cached_plan, (q, k_cache, v_cache, lengths, k_new, v_new), None if scale is None else float(scale))
    _no_grad_wanted(what, q, k_cache, v_cache, k_new, v_new)
    _no_tangents(what, q, k_cache, v_cache, k_new, v_new)
    if shape[0] == 0:
        return q.new_empty(shape)
    kc, vc = k_cache.data_ptr(), v_cache.data_ptr()
    if (kc | vc) % 16:
        raise ValueError(f'{what}: {"k_cache" if kc % 16 else "v_cache"} must have a contiguous last axis and 16-byte aligned rows (it is updated in place and cannot be copied)')
    if new and kc == vc:
        raise ValueError(f'{what}: k_cache and v_cache are the same memory')
    out = q.new_empty(shape)
    ws = torch.empty(nws, dtype=torch.float32, device=device) if nws else None
    P = _hip.ptr
    sizes, cst, scale = tail
    if direct is None or (q.data_ptr() | (k_new.data_ptr() | v_new.data_ptr() if new else 0)) % 16:
        q, sq = _rows(q)
        direct = _i64(sq), None, None
        if new:
            (k_new, skn), (v_new, svn) = _rows(k_new), _rows(v_new)
            direct = _i64(sq), _i64(skn), _i64(svn)
    _launch('genie_cached_attention_step', device, P(q), P(k_new), P(v_new), kc, vc, P(lengths), P(out), P(ws), nws, *sizes, *direct, *cst, scale)
    if new:
        torch._C._increment_version((k_cache, v_cache))           # (written behind autograd's back: a graph that kept the old values must not use these)
    return out


# ------------------------------------------------------------------------------------------------------------------------------------
# linear attention with a decay per head
# ------------------------------------------------------------------------------------------------------------------------------------
def _decay_forward(q: Tensor, k: Tensor, v: Tensor, log_decay: Tensor, cu: Tensor, initial_state: Optional[Tensor], scale: float, return_state: bool,
                   direct):
    """(out, final states or None, what the backward pass keeps); direct: strides of q, k and v if only their alignment is open"""
    rows, h, dk = q.shape
    dv, nseq, dev = v.shape[2], cu.shape[0] - 1, q.device
    if direct is not None and not (q.data_ptr() | k.data_ptr() | v.data_ptr()) % 16:
        sq, sk, sv = direct
    else:
        (q, sq), (k, sk), (v, sv) = _rows(q), _rows(k), _rows(v)
    out = q.new_empty((rows, h, dv))
    final = torch.empty((nseq, h, dk, dv), dtype=torch.float32, device=dev) if return_state else None
    states = ws = None
    if rows:
        P = _hip.ptr
        n = _hip.load_library().genie_decay_attention_state_elems(nseq, rows, h, dk, dv, initial_state is not None)
        if n:
            states, ws = torch.empty(n, dtype=torch.bfloat16, device=dev), torch.empty(n, dtype=torch.float32, device=dev)
        _launch('genie_decay_attention_fwd', dev, P(q), P(k), P(v), P(log_decay), P(cu), P(initial_state), P(out), P(final), P(states), P(ws), n, nseq, rows, h, dk, dv,
                _i64(sq), _i64(sk), _i64(sv), scale)
    elif return_state:
        final.zero_() if initial_state is None else final.copy_(initial_state)
    return out, final, (q, k, v, log_decay, cu, states)


def _decay_bwd_plan(q, k, v, log_decay, cu, states, dout, sizes, has_initial):
    """(None or the strides of q, k, v and dout where no tensor needs a copy, elements of states and workspace), from the tensors as they came back"""
    what, dev = 'decay_attention', dout.device
    nseq, rows, h, dk, dv = sizes
    elems = _hip.load_library().genie_decay_attention_state_elems
    kept = elems(*sizes, has_initial) if rows else 0
    for t, name, dtype, shape in ((q, 'q', torch.bfloat16, (rows, h, dk)), (k, 'k', torch.bfloat16, (rows, h, dk)), (v, 'v', torch.bfloat16, (rows, h, dv)),
                                  (log_decay, 'log_decay', torch.float32, (h,)), (cu, 'cu_seqlens', torch.int32, (nseq + 1,)),
                                  *(((states, 'the states', torch.bfloat16, (kept,)),) if kept else ())):
        _came_back(what, t, name, dtype, shape, dev)
    strides = [_direct(t) for t in (q, k, v, dout)]
    direct = None not in strides and all(t is None or t.is_contiguous() for t in (log_decay, cu, states))
    return tuple(map(_i64, strides)) if direct else None, elems(*sizes, 0) if rows else 0


class _DecayAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q: Tensor, k: Tensor, v: Tensor, log_decay: Tensor, cu: Tensor, initial_state: Optional[Tensor], scale: float, return_state: bool, direct):
        out, final, saved = _decay_forward(q, k, v, log_decay, cu, initial_state, scale, return_state, direct)
        ctx.sizes, ctx.scale, ctx.has_initial = (cu.shape[0] - 1, *q.shape, v.shape[2]), scale, int(initial_state is not None)
        ctx.save_for_backward(*saved)
        if return_state:
            ctx.mark_non_differentiable(final)
            return out, final
        return out

    @staticmethod
    @_first_order
    def backward(ctx, dout: Tensor, *_):
        q, k, v, log_decay, cu, states = ctx.saved_tensors
        _, rows, h, dk, dv = sizes = ctx.sizes
        strides, n = _planned(_decay_bwd_plan, (q, k, v, log_decay, cu, states, dout), sizes, ctx.has_initial)
        gq, gk, gv = q.new_empty((rows, h, dk)), q.new_empty((rows, h, dk)), q.new_empty((rows, h, dv))
        if rows:
            rev, ws, P, dev = None, None, _hip.ptr, q.device
            if strides is None or (q.data_ptr() | k.data_ptr() | v.data_ptr() | dout.data_ptr() | (P(states) or 0)) % 16:
                (q, sq), (k, sk), (v, sv), (dout, sg) = _rows(q), _rows(k), _rows(v), _rows(dout)
                strides = _i64(sq), _i64(sk), _i64(sv), _i64(sg)
                log_decay, cu, states = _dense(log_decay), _dense(cu), _dense(states)
            if n:
                rev, ws = torch.empty(n, dtype=torch.bfloat16, device=dev), torch.empty(n, dtype=torch.float32, device=dev)
            _launch('genie_decay_attention_bwd', dev, P(q), P(k), P(v), P(dout), P(log_decay), P(cu), ctx.has_initial, P(states), P(rev), P(ws), n, P(gq), P(gk), P(gv),
                    *sizes, *strides, ctx.scale)
        need = ctx.needs_input_grad
        return gq if need[0] else None, gk if need[1] else None, gv if need[2] else None, None, None, None, None, None, None


def _check_decay(what: str, log_decay: Tensor, heads: int, device: torch.device) -> None:
    _check(what, log_decay, 'log_decay', 1, torch.float32, device)
    if log_decay.shape[0] != heads:
        raise ValueError(f'{what}: log_decay must hold one value for each of the {heads} heads, got {tuple(log_decay.shape)}')


def _constant(what: str, why: str, t: Tensor) -> Tensor:
    if t.requires_grad:
        if torch.is_grad_enabled():
            raise RuntimeError(f'{what}: {why}')
        t = t.detach()
    return t if t.is_contiguous() else t.contiguous()


def _decay_plan(q, k, v, log_decay, cu_seqlens, initial_state, scale):
    """(scale, None or the strides of q, k and v where they need no copy)"""
    what = 'decay_attention'
    _check(what, q, 'q', 3, torch.bfloat16)
    _check(what, k, 'k', 3, torch.bfloat16, q.device)
    _check(what, v, 'v', 3, torch.bfloat16, q.device)
    rows, h, dk = q.shape
    if k.shape != q.shape:
        raise ValueError(f'{what}: q {tuple(q.shape)} and k {tuple(k.shape)} differ')
    if v.shape[:2] != q.shape[:2]:
        raise ValueError(f'{what}: v {tuple(v.shape)} does not fit q {tuple(q.shape)}')
    if h == 0:
        raise ValueError(f'{what}: no heads')
    if rows > _MAX_ROWS:
        raise ValueError(f'{what}: at most {_MAX_ROWS} rows')
    _check_width(what, dk, 'q and k')
    _check_width(what, v.shape[2], 'v')
    _check_decay(what, log_decay, h, q.device)
    _check_cu(what, cu_seqlens, 'cu_seqlens', q.device)
    if initial_state is not None:
        _check(what, initial_state, 'initial_state', 4, torch.float32, q.device)
        want = (cu_seqlens.shape[0] - 1, h, dk, v.shape[2])
        if initial_state.shape != want:
            raise ValueError(f'{what}: initial_state must be {want}, got {tuple(initial_state.shape)}')
    strides = tuple(_direct(t) for t in (q, k, v))
    return _scale(what, scale, dk), None if None in strides else strides


def decay_attention(q: Tensor, k: Tensor, v: Tensor, log_decay: Tensor, cu_seqlens: Tensor, initial_state: Optional[Tensor] = None, scale: Optional[float] = None,
                    return_state: bool = False) -> Union[Tensor, Tuple[Tensor, Tensor]]:
    """Linear attention with a decay for each head over packed sequences: ``S_t = exp(log_decay[h]) S_{t-1} + k_t v_t^T``, ``o_t = scale q_t S_t``.

    ``q`` / ``k`` (rows, H, dk), ``v`` (rows, H, dv) bf16, widths multiples of 8 up to 128; ``log_decay`` (H,) fp32, <= 0 (``-inf``: no memory, 0: none is lost);
    ``scale`` defaults to ``dk ** -0.5``.  Returns (rows, H, dv) bf16, differentiable in q, k and v.

    ``initial_state`` (sequences, H, dk, dv) fp32: the state in front of each sequence's first token.  ``return_state``: also return the state behind each sequence's
    last token, which ``decay_attention_step`` and a later call continue from.  States carry no gradient (truncated backpropagation)."""
    what = 'decay_attention'
    scale, direct = _planned(_decay_plan, (q, k, v, log_decay, cu_seqlens, initial_state), None if scale is None else float(scale))
    _no_tangents(what, q, k, v, log_decay, initial_state)
    log_decay = _constant(what, 'the decays are constants (no gradient): pass log_decay.detach()', log_decay)
    if initial_state is not None:
        initial_state = _constant(what, 'no gradient flows into a state: pass initial_state.detach()', initial_state)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        return _DecayAttention.apply(q, k, v, log_decay, cu_seqlens, initial_state, scale, bool(return_state), direct)
    out, final, _ = _decay_forward(q, k, v, log_decay, cu_seqlens, initial_state, scale, return_state, direct)
    return (out, final) if return_state else out


def _decay_step_plan(q, k, v, log_decay, state, new_state, scale):
    """(device, the output's shape, None or the strides of tensors that need no copy, sizes, scale)"""
    what = 'decay_attention_step'
    _check(what, q, 'q', 3, torch.bfloat16)
    _check(what, k, 'k', 3, torch.bfloat16, q.device)
    _check(what, v, 'v', 3, torch.bfloat16, q.device)
    b, h, dk = q.shape
    dv = v.shape[2]
    if k.shape != q.shape:
        raise ValueError(f'{what}: q {tuple(q.shape)} and k {tuple(k.shape)} differ')
    if v.shape[:2] != q.shape[:2]:
        raise ValueError(f'{what}: v {tuple(v.shape)} does not fit q {tuple(q.shape)}')
    if h == 0:
        raise ValueError(f'{what}: no heads')
    _check_width(what, dk, 'q and k')
    _check_width(what, dv, 'v')
    _check_decay(what, log_decay, h, q.device)
    for t, name in ((state, 'state'), (new_state, 'new_state')):
        if t is None and name == 'new_state':
            continue
        _check(what, t, name, 4, torch.float32, q.device)
        if t.shape != (b, h, dk, dv):
            raise ValueError(f'{what}: {name} must be {(b, h, dk, dv)}, got {tuple(t.shape)}')
        if not t.is_contiguous():
            raise ValueError(f'{what}: {name} must be contiguous and 16-byte aligned')
    direct = [_direct(t) for t in (q, k, v)]
    return q.device, (b, h, dv), None if None in direct else tuple(map(_i64, direct)), (b, h, dk, dv), _scale(what, scale, dk)


def decay_attention_step(q: Tensor, k: Tensor, v: Tensor, log_decay: Tensor, state: Tensor, scale: Optional[float] = None, new_state: Optional[Tensor] = None) -> Tensor:
    """``decay_attention`` for one token per sequence: ``q`` / ``k`` (B, H, dk), ``v`` (B, H, dv) bf16, ``state`` (B, H, dk, dv) fp32, contiguous.  The state is advanced in
    place, or into ``new_state`` (the old one then stays).  Returns (B, H, dv) bf16; no backward pass."""
    what = 'decay_attention_step'
    device, shape, direct, sizes, scale = _planned(_decay_step_plan, (q, k, v, log_decay, state, new_state), None if scale is None else float(scale))
    _no_tangents(what, q, k, v, log_decay, state, new_state)
    log_decay = _constant(what, 'the decays are constants (no gradient): pass log_decay.detach()', log_decay)
    _no_grad_wanted(what, q, k, v, state, new_state)
    old = state.data_ptr()
    new = old if new_state is None else new_state.data_ptr()
    if (old | new) % 16:
        raise ValueError(f'{what}: {"state" if old % 16 else "new_state"} must be contiguous and 16-byte aligned')
    if old != new and abs(old - new) < state.numel() * 4:
        raise ValueError(f'{what}: new_state overlaps state without being it')
    out = q.new_empty(shape)
    if shape[0] == 0:
        return out
    if direct is None or (q.data_ptr() | k.data_ptr() | v.data_ptr()) % 16:
        (q, sq), (k, sk), (v, sv) = _rows(q), _rows(k), _rows(v)
        direct = _i64(sq), _i64(sk), _i64(sv)
    _launch('genie_decay_attention_step', device, q.data_ptr(), k.data_ptr(), v.data_ptr(), log_decay.data_ptr(), old, new, out.data_ptr(), *sizes, *direct, scale)
    torch._C._increment_version((state if new_state is None else new_state,))
    return out
