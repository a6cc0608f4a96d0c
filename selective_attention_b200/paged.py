"""Served selective attention: a paged 8-bit key/value cache for many requests, and attention
over packed prompts (C-ABI ``sattn_paged_*`` and ``sattn_prefill_packed``).

The reference serves a batch from a dense full-precision cache with one write index
(``inference/selective_attn_cache.py:10-42``) and pads its prompts. Here requests of any lengths
share one pool of pages: :func:`sattn_paged_plan` gives new tokens their slots,
:func:`sattn_paged_append` writes their keys, values and log-gates as 8-bit codes,
:func:`sattn_paged_decode` attends to them with one query token for each request,
:func:`sattn_paged_read` reads them back, and :func:`sattn_prefill_packed` attends within whole
prompts. Query heads may share key heads. :class:`PagedSelectiveCache` keeps the pool of one
layer stack and makes these calls in order.

Every launch goes on the current torch stream of the inputs' device; nothing synchronizes.
"""
from __future__ import annotations

from ctypes import byref, c_void_p
from typing import Optional

import torch

from . import _lib
from .kernels import _aligned16, _stream
from .utils import check_cuda, check_ndim, check_shape, to_contiguous

PAGE_SIZES = (16, 32, 64, 128)
CACHE_HEAD_DIMS = (32, 64, 128, 256)


def _int32(t: torch.Tensor, name: str, shape=None) -> None:
    if t.dtype != torch.int32 or not t.is_contiguous():
        raise ValueError(f"[{name}] expected a contiguous int32 tensor")
    if shape is not None:
        check_shape(t, shape, name)


def sattn_paged_plan(lengths, new_lengths, block_table, free_pages, free_state, num_tokens: int, page_size: int):
    """Slots for the next call's tokens, from request lengths alone (C-ABI ``sattn_paged_plan``).

    Request ``r`` holds ``lengths[r]`` tokens in the pages ``block_table[r]`` and is to take
    ``new_lengths[r]`` more; pages come from the ring ``free_pages``, of which those counted
    ``free_state[0]`` to ``free_state[1]`` (int64; handed out, returned) are free. ``lengths``,
    ``new_lengths`` ``(R,)``, ``block_table`` ``(R, W)`` and ``free_pages`` ``(F,)`` are int32;
    ``num_tokens`` is the number of rows to plan (the new tokens, or more: padding). New entries of
    ``block_table`` are written in place; nothing else of the inputs changes.

    Returns ``(lengths_out, cu_new, slots, positions, free_state_out)``: ``(R,)`` int32 lengths
    with the new tokens, ``(R + 1,)`` int32 offsets of each request's tokens, ``(num_tokens,)`` int64
    slots (page * page_size + place) and int32 positions, and the ring's new state. A request whose
    pages are not to be had keeps its length and gets slots of -1.
    """
    check_ndim(lengths, 1, "lengths")
    check_ndim(block_table, 2, "block_table")
    check_ndim(free_pages, 1, "free_pages")
    R, W = block_table.shape
    dev = check_cuda([lengths, new_lengths, block_table, free_pages, free_state],
                     ["lengths", "new_lengths", "block_table", "free_pages", "free_state"])
    _int32(lengths, "lengths", (R,))
    _int32(new_lengths, "new_lengths", (R,))
    _int32(block_table, "block_table")
    _int32(free_pages, "free_pages")
    if free_state.dtype != torch.int64 or not free_state.is_contiguous():
        raise ValueError("[free_state] expected a contiguous int64 tensor")
    check_shape(free_state, (2,), "free_state")
    if page_size not in PAGE_SIZES:
        raise ValueError(f"[page_size] {page_size} is not one of {PAGE_SIZES}")
    if num_tokens < 0:
        raise ValueError(f"[num_tokens] {num_tokens} is negative")
    # the int32 outputs are parts of one allocation, as are the int64 ones
    small = torch.empty(2 * R + 1 + num_tokens, device=dev, dtype=torch.int32)
    large = torch.empty(num_tokens + 2, device=dev, dtype=torch.int64)
    lengths_out, cu_new, positions = small[:R], small[R:2 * R + 1], small[2 * R + 1:]
    slots, state_out = large[:num_tokens], large[num_tokens:]
    with torch.cuda.device(dev):
        st = _lib.lib().sattn_paged_plan(
            _lib.ptr(lengths), _lib.ptr(new_lengths), _lib.ptr(block_table), _lib.ptr(free_pages),
            _lib.ptr(free_state), _lib.ptr(lengths_out), _lib.ptr(cu_new), _lib.ptr(slots), _lib.ptr(positions),
            _lib.ptr(state_out), R, W, free_pages.numel(), num_tokens, page_size, _stream(dev))
    _lib.check(st, "sattn_paged_plan")
    return lengths_out, cu_new, slots, positions, state_out


def _cache(k_cache, v_cache, k_scale, v_scale, log_gate_cache) -> _lib.SattnCache:
    """Checks a cache's tensors and describes them."""
    check_ndim(k_cache, 4, "k_cache")
    P, H, page, D = k_cache.shape
    if k_cache.dtype not in _lib.CACHE_CODES:
        raise ValueError(f"[k_cache] unsupported dtype {k_cache.dtype}; expected int8 or float8_e4m3fn")
    if v_cache.dtype != k_cache.dtype:
        raise ValueError(f"[v_cache] dtype {v_cache.dtype} differs from k_cache's {k_cache.dtype}")
    if page not in PAGE_SIZES or D not in CACHE_HEAD_DIMS:
        raise ValueError(f"[k_cache] expected (pages, heads, page size in {PAGE_SIZES}, head dim in "
                         f"{CACHE_HEAD_DIMS}), got {tuple(k_cache.shape)}")
    check_shape(v_cache, (P, H, page, D), "v_cache")
    check_shape(log_gate_cache, (P, H, page), "log_gate_cache", optional=True)
    for t, n in ((k_scale, "k_scale"), (v_scale, "v_scale")):
        check_shape(t, (P, H), n)
    for t, n in ((k_scale, "k_scale"), (v_scale, "v_scale"), (log_gate_cache, "log_gate_cache")):
        if t is not None and t.dtype != torch.float32:
            raise ValueError(f"[{n}] expected float32, got {t.dtype}")
    for t, n in ((k_cache, "k_cache"), (v_cache, "v_cache"), (k_scale, "k_scale"), (v_scale, "v_scale"),
                 (log_gate_cache, "log_gate_cache")):
        if t is not None and not t.is_contiguous():
            raise ValueError(f"[{n}] must be contiguous (it is used in place)")
    for t, n in ((k_cache, "k_cache"), (v_cache, "v_cache"), (log_gate_cache, "log_gate_cache")):
        if t is not None and t.data_ptr() % 16:
            raise ValueError(f"[{n}] must start on a 16-byte boundary")
    return _lib.SattnCache(num_pages=P, nkv=H, page_size=page, head_dim=D, code=_lib.CACHE_CODES[k_cache.dtype],
                           k_codes=_lib.ptr(k_cache), v_codes=_lib.ptr(v_cache), k_scale=_lib.ptr(k_scale),
                           v_scale=_lib.ptr(v_scale), log_gate=_lib.ptr(log_gate_cache))


_CACHE_NAMES = ["k_cache", "v_cache", "k_scale", "v_scale", "log_gate_cache"]


def _slots(slots) -> torch.Tensor:
    check_ndim(slots, 1, "slots")
    if slots.dtype != torch.int64:
        raise ValueError(f"[slots] expected int64, got {slots.dtype}")
    return to_contiguous(slots)


def _rows(t: torch.Tensor):
    """``(tensor, token stride, head stride)`` of a (tokens, heads, D) tensor whose rows of D lie
    together; strides of dimensions of size one do not count and a broadcast one is written out."""
    if (t.stride(2) != 1 and t.shape[2] > 1) or any(t.stride(i) == 0 and t.shape[i] > 1 for i in (0, 1)):
        t = t.contiguous()
    hs = t.stride(1) if t.shape[1] > 1 else t.shape[2]
    ts = t.stride(0) if t.shape[0] > 1 else t.shape[1] * hs
    return t, ts, hs


def sattn_paged_append(k, v, slots, k_cache, v_cache, k_scale, v_scale, log_gate=None, log_gate_cache=None) -> None:
    """Writes tokens into a paged cache at their slots, in place (C-ABI ``sattn_paged_append``).

    ``k``, ``v`` ``(T, Hkv, D)`` float32, bfloat16 or float16 with any token and head strides;
    ``slots`` ``(T,)`` int64 as :func:`sattn_paged_plan` gives them (-1: not written); ``k_cache``,
    ``v_cache`` ``(pages, Hkv, page_size, D)`` int8 or float8_e4m3fn; ``k_scale``, ``v_scale``
    ``(pages, Hkv)`` float32; ``log_gate`` ``(T, Hkv)`` and ``log_gate_cache`` ``(pages, Hkv, page_size)``
    float32, both or neither. A page's scale is the largest magnitude that it has held (finite ones
    count) times the reciprocal of the largest code, 127 or 448: where new tokens raise it, the page's earlier codes are
    rounded anew.
    """
    dev = check_cuda([k, v, slots, k_cache, v_cache, k_scale, v_scale, log_gate, log_gate_cache],
                     ["k", "v", "slots"] + _CACHE_NAMES[:4] + ["log_gate", "log_gate_cache"])
    c = _cache(k_cache, v_cache, k_scale, v_scale, log_gate_cache)
    check_ndim(k, 3, "k")
    T = k.shape[0]
    check_shape(k, (T, c.nkv, c.head_dim), "k")
    check_shape(v, (T, c.nkv, c.head_dim), "v")
    if v.dtype != k.dtype:
        raise ValueError(f"[v] dtype {v.dtype} differs from k's {k.dtype}")
    code = _lib.dtype_code(k.dtype, "k")
    slots = _slots(slots)
    check_shape(slots, (T,), "slots")
    if (log_gate is None) != (log_gate_cache is None):
        raise ValueError("[log_gate] a cache with log-gates takes them, and one without does not")
    if log_gate is not None:
        check_shape(log_gate, (T, c.nkv), "log_gate")
        log_gate = to_contiguous(log_gate.float())
    k, k_ts, k_hs = _rows(k)
    v, v_ts, v_hs = _rows(v)
    with torch.cuda.device(dev):
        st = _lib.lib().sattn_paged_append(byref(c), _lib.ptr(k), _lib.ptr(v), _lib.ptr(log_gate), _lib.ptr(slots), T,
                                           k_ts, k_hs, v_ts, v_hs, code, _stream(dev))
    _lib.check(st, "sattn_paged_append")


def sattn_paged_read(slots, k_cache, v_cache, k_scale, v_scale, dtype: torch.dtype = torch.float32):
    """Values of slots of a paged cache (C-ABI ``sattn_paged_read``): ``(k, v)``, each
    ``(len(slots), Hkv, D)`` in ``dtype``; zeros where a slot is not the cache's (-1)."""
    dev = check_cuda([slots, k_cache, v_cache, k_scale, v_scale], ["slots"] + _CACHE_NAMES[:4])
    c = _cache(k_cache, v_cache, k_scale, v_scale, None)
    code = _lib.dtype_code(dtype, "dtype")
    slots = _slots(slots)
    k = torch.empty(slots.numel(), c.nkv, c.head_dim, device=dev, dtype=dtype)
    v = torch.empty_like(k)
    with torch.cuda.device(dev):
        st = _lib.lib().sattn_paged_read(byref(c), _lib.ptr(slots), slots.numel(), _lib.ptr(k), _lib.ptr(v), code,
                                         _stream(dev))
    _lib.check(st, "sattn_paged_read")
    return k, v


def sattn_paged_decode(q, k_cache, v_cache, k_scale, v_scale, block_table, lengths, log_gate_cache=None, scale=None,
                       out=None, workspace: Optional[torch.Tensor] = None):
    """One decode step's attention over a paged cache (C-ABI ``sattn_paged_decode``).

    ``q`` ``(R, Hq, D)``, ``Hq`` a multiple of the cache's heads; ``block_table`` ``(R, W)`` and
    ``lengths`` ``(R,)`` int32. Request ``r``'s own token is the last of its ``lengths[r]`` (it was
    appended before): the pos-mode gated softmax of :func:`~.kernels.sattn_decode_step`
    (``modules/selective_attention.py:399-404``), in which every key but the own one adds its log-gate
    and a log-gate of ``-inf`` drops the key. A length of 0 gives zeros. ``scale`` defaults to
    ``D ** -0.5``. Returns ``(R, Hq, D)`` in ``q``'s dtype. ``workspace`` (uint8) is allocated when it
    is ``None`` or too small; calls that overlap on the GPU need one each.
    """
    dev = check_cuda([q, k_cache, v_cache, k_scale, v_scale, block_table, lengths, log_gate_cache],
                     ["q"] + _CACHE_NAMES[:4] + ["block_table", "lengths", "log_gate_cache"])
    c = _cache(k_cache, v_cache, k_scale, v_scale, log_gate_cache)
    check_ndim(q, 3, "q")
    check_ndim(block_table, 2, "block_table")
    R, Hq, D = q.shape
    if D != c.head_dim or Hq == 0 or Hq % c.nkv:
        raise ValueError(f"[q] expected (requests, a multiple of {c.nkv} heads, {c.head_dim}), got {tuple(q.shape)}")
    code = _lib.dtype_code(q.dtype, "q")
    W = block_table.shape[1]
    _int32(block_table, "block_table", (R, W))
    _int32(lengths, "lengths", (R,))
    q = _aligned16(to_contiguous(q))
    if out is None:
        out = torch.empty(R, Hq, D, device=dev, dtype=q.dtype)
    else:
        check_cuda([q, out], ["q", "out"])
        check_shape(out, (R, Hq, D), "out")
        if out.dtype != q.dtype or not out.is_contiguous() or out.data_ptr() % 16:
            raise ValueError("[out] expected a contiguous, 16-byte aligned tensor of q's dtype")
    if R == 0:
        return out
    if W == 0:
        return out.zero_()
    need = int(_lib.lib().sattn_paged_decode_workspace_size(byref(c), R, W, Hq))
    if need and (workspace is None or workspace.numel() * workspace.element_size() < need):
        workspace = torch.empty(need, device=dev, dtype=torch.uint8)
    elif need:
        check_cuda([q, workspace], ["q", "workspace"])
    with torch.cuda.device(dev):
        st = _lib.lib().sattn_paged_decode(byref(c), _lib.ptr(q), _lib.ptr(block_table), _lib.ptr(lengths),
                                           _lib.ptr(out), R, W, Hq, float(D ** -0.5 if scale is None else scale), code,
                                           c_void_p(_lib.ptr(workspace) if need else None), need, _stream(dev))
    _lib.check(st, "sattn_paged_decode")
    return out


def sattn_prefill_packed(q, k, v, cu_seqlens, log_gate=None, scale=None, out=None, impl: str = "auto"):
    """Selective attention over packed prompts, causal (C-ABI ``sattn_prefill_packed``).

    ``q`` ``(T, Hq, D)``, ``k``, ``v`` ``(T, Hkv, D)`` (slices of one projection's output are taken as
    they are); ``cu_seqlens`` ``(R + 1,)`` int32 offsets of the sequences, from 0; ``log_gate``
    ``(T, Hkv)`` or ``None``. Within a sequence it is :func:`~.kernels.sattn_prefill`: every
    earlier key adds its log-gate, the own one does not, ``-inf`` drops a key
    (``modules/selective_attention.py:27-144``, ``:270-280``). Returns ``(T, Hq, D)`` in ``q``'s dtype, zeros
    past the last sequence. ``scale`` defaults to ``D ** -0.5``. ``impl``: ``"auto"`` (tensor cores for
    16-bit types with ``D`` 64 or 128), ``"tc"`` or ``"simt"``.
    """
    check_ndim(q, 3, "q")
    check_ndim(k, 3, "k")
    check_ndim(cu_seqlens, 1, "cu_seqlens")
    T, Hq, D = q.shape
    Hk = k.shape[1]
    dev = check_cuda([q, k, v, cu_seqlens, log_gate, out], ["q", "k", "v", "cu_seqlens", "log_gate", "out"])
    if Hk == 0 or Hq == 0 or Hq % Hk:
        raise ValueError(f"[k] {Hq} query heads are not a multiple of {Hk} key heads")
    for t, n in ((k, "k"), (v, "v")):
        check_shape(t, (T, Hk, D), n)
        if t.dtype != q.dtype:
            raise ValueError(f"[{n}] dtype {t.dtype} differs from q's {q.dtype}")
    check_shape(log_gate, (T, Hk), "log_gate", optional=True)
    if cu_seqlens.numel() == 0:
        raise ValueError("[cu_seqlens] expected the offsets of the sequences, from 0")
    _int32(cu_seqlens, "cu_seqlens")
    code = _lib.dtype_code(q.dtype, "q")
    per = 16 // q.element_size()

    def rows(t):
        t, ts, hs = _rows(t)
        if ts % per or hs % per or t.data_ptr() % 16:
            t, ts, hs = _rows(t.contiguous() if not t.is_contiguous() else t.clone())
        return t, ts, hs

    (q, q_ts, q_hs), (k, k_ts, k_hs), (v, v_ts, v_hs) = rows(q), rows(k), rows(v)
    log_gate = None if log_gate is None else to_contiguous(log_gate.float())
    if out is None:
        out = torch.empty(T, Hq, D, device=dev, dtype=q.dtype)
    else:
        check_shape(out, (T, Hq, D), "out")
        if out.dtype != q.dtype or not out.is_contiguous() or out.data_ptr() % 16:
            raise ValueError("[out] expected a contiguous, 16-byte aligned tensor of q's dtype")
    p = _lib.SattnPackedParams(
        num_tokens=T, num_seqs=cu_seqlens.numel() - 1, nheads=Hq, nkv=Hk, head_dim=D, q_token_stride=q_ts,
        q_head_stride=q_hs, k_token_stride=k_ts, k_head_stride=k_hs, v_token_stride=v_ts, v_head_stride=v_hs,
        dtype=code, impl=_lib.IMPLS[impl], scale=float(D ** -0.5 if scale is None else scale), q=_lib.ptr(q),
        k=_lib.ptr(k), v=_lib.ptr(v), log_gate=_lib.ptr(log_gate), cu_seqlens=_lib.ptr(cu_seqlens),
        out=_lib.ptr(out))
    with torch.cuda.device(dev):
        st = _lib.lib().sattn_prefill_packed(byref(p), _stream(dev))
    _lib.check(st, "sattn_prefill_packed")
    return out
