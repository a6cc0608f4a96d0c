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

import functools
import struct
from typing import Optional

import torch

from . import _lib
from .kernels import _aligned16
from .utils import check_cuda, check_ndim, check_shape, to_contiguous

PAGE_SIZES = (16, 32, 64, 128)
CACHE_HEAD_DIMS = (32, 64, 128, 256)
_I32, _I64, _F32 = torch.int32, torch.int64, torch.float32
_FUNCTIONS = {}  # the C entries by name
_current_device, _current_stream = torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream


# Each call looks its arguments over in one expression, and where that fails goes through them one by
# one for the message: on small inputs the checks would otherwise take longer than the kernel.

# The C structs as bytes: building them field by field through ctypes takes longer than these calls'
# kernels do on such inputs. (A test holds them against the ctypes mirrors.)
_CACHE = struct.Struct("@qqqqi4xPPPPP")
_PACKED = struct.Struct("@qqqqqqqqqqqiif4xPPPPPP")


def _int32(t: torch.Tensor, name: str, shape=None) -> None:
    if t.dtype != torch.int32 or not t.is_contiguous():
        raise ValueError(f"[{name}] expected a contiguous int32 tensor")
    if shape is not None:
        check_shape(t, shape, name)


def _call(name: str, d: int, *args) -> None:
    """One C entry with the tensors' device as the current one (it mostly is), on its current stream."""
    fn = _FUNCTIONS.get(name)
    if fn is None:
        fn = _FUNCTIONS[name] = getattr(_lib.lib(), name)
    if _current_device() == d:
        status = fn(*args, _current_stream(d))
    else:
        with torch.cuda.device(d):
            status = fn(*args, _current_stream(d))
    if status:
        _lib.check(status, name)


def _plan_faults(lengths, new_lengths, block_table, free_pages, free_state, num_tokens, page_size) -> None:
    check_ndim(lengths, 1, "lengths")
    check_ndim(block_table, 2, "block_table")
    check_ndim(free_pages, 1, "free_pages")
    check_cuda((lengths, new_lengths, block_table, free_pages, free_state),
               ("lengths", "new_lengths", "block_table", "free_pages", "free_state"))
    R = block_table.shape[0]
    _int32(lengths, "lengths", (R,))
    _int32(new_lengths, "new_lengths", (R,))
    _int32(block_table, "block_table")
    _int32(free_pages, "free_pages")
    if free_state.dtype != _I64 or not free_state.is_contiguous():
        raise ValueError("[free_state] expected a contiguous int64 tensor")
    check_shape(free_state, (2,), "free_state")
    if page_size not in PAGE_SIZES:
        raise ValueError(f"[page_size] {page_size} is not one of {PAGE_SIZES}")
    raise ValueError(f"[num_tokens] {num_tokens} is negative")


def sattn_paged_plan(lengths, new_lengths, block_table, free_pages, free_state, num_tokens: int, page_size: int):
    """Slots for the next call's tokens, from request lengths alone (C-ABI ``sattn_paged_plan``).

    Request ``r`` holds ``lengths[r]`` tokens in the pages ``block_table[r]`` and is to take
    ``new_lengths[r]`` more; pages come from the ring ``free_pages``, of which those counted
    ``free_state[0]`` to ``free_state[1]`` (int64; handed out, returned) are free. ``lengths``,
    ``new_lengths`` ``(R,)``, ``block_table`` ``(R, W)`` and ``free_pages`` ``(F,)`` are int32;
    ``num_tokens`` is the number of rows to plan: the new tokens, or more (padding). New entries of
    ``block_table`` are written in place; nothing else of the inputs changes.

    Returns ``(lengths_out, cu_new, slots, positions, free_state_out)``: ``(R,)`` int32 lengths
    with the new tokens, ``(R + 1,)`` int32 offsets of each request's tokens, ``(num_tokens,)`` int64
    slots (page * page_size + place) and int32 positions, and the ring's new state. A request whose
    pages are not to be had, or whose tokens do not all lie within ``num_tokens``, keeps its length and gets
    slots of -1.
    """
    d = lengths.get_device()
    shape = block_table.shape
    if not (d >= 0 and len(shape) == 2 and lengths.shape == new_lengths.shape == shape[:1]
            and lengths.dtype == new_lengths.dtype == block_table.dtype == free_pages.dtype == _I32
            and free_state.dtype == _I64 and free_state.shape == (2,) and len(free_pages.shape) == 1
            and new_lengths.get_device() == block_table.get_device() == free_pages.get_device()
            == free_state.get_device() == d and lengths.is_contiguous() and new_lengths.is_contiguous()
            and block_table.is_contiguous() and free_pages.is_contiguous() and free_state.is_contiguous()
            and page_size in PAGE_SIZES and num_tokens >= 0):
        _plan_faults(lengths, new_lengths, block_table, free_pages, free_state, num_tokens, page_size)
    R, W = shape
    dev = lengths.device
    # the int32 outputs are parts of one allocation, as are the int64 ones
    small = torch.empty(2 * R + 1 + num_tokens, device=dev, dtype=_I32)
    wide = torch.empty(num_tokens + 2, device=dev, dtype=_I64)
    lengths_out, cu_new, positions = small.split_with_sizes((R, R + 1, num_tokens))
    slots, state_out = wide.split_with_sizes((num_tokens, 2))
    at, large = small.data_ptr(), wide.data_ptr()
    _call("sattn_paged_plan", d, lengths.data_ptr(), new_lengths.data_ptr(), block_table.data_ptr(),
          free_pages.data_ptr(), free_state.data_ptr(), at, at + 4 * R, large, at + 8 * R + 4, large + 8 * num_tokens, R,
          W, free_pages.shape[0], num_tokens, page_size)
    return lengths_out, cu_new, slots, positions, state_out


def _cache_faults(k_cache, v_cache, k_scale, v_scale, log_gate_cache) -> None:
    """Says what is wrong with a cache's tensors."""
    check_cuda((k_cache, v_cache, k_scale, v_scale, log_gate_cache), _CACHE_NAMES + ("log_gate_cache",))
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


def _cache(k_cache, v_cache, k_scale, v_scale, log_gate_cache):
    """``(sattn_cache as bytes, heads, page size, head dim, device index)`` of checked tensors."""
    shape, kind, dev = k_cache.shape, k_cache.dtype, k_cache.get_device()
    kp, vp = k_cache.data_ptr(), v_cache.data_ptr()
    gp = 0 if log_gate_cache is None else log_gate_cache.data_ptr()
    good = (dev >= 0 and v_cache.get_device() == k_scale.get_device() == v_scale.get_device() == dev
            and len(shape) == 4 and shape[2] in PAGE_SIZES and shape[3] in CACHE_HEAD_DIMS and v_cache.shape == shape
            and kind in _lib.CACHE_CODES and v_cache.dtype == kind and k_scale.shape == shape[:2]
            and v_scale.shape == shape[:2] and k_scale.dtype == _F32 and v_scale.dtype == _F32
            and k_cache.is_contiguous() and v_cache.is_contiguous() and k_scale.is_contiguous()
            and v_scale.is_contiguous() and not (kp | vp | gp) & 15)
    if good and log_gate_cache is not None:
        good = (log_gate_cache.shape == shape[:3] and log_gate_cache.dtype == _F32
                and log_gate_cache.is_contiguous() and log_gate_cache.get_device() == dev)
    if not good:
        _cache_faults(k_cache, v_cache, k_scale, v_scale, log_gate_cache)
    P, H, page, D = shape
    return _CACHE.pack(P, H, page, D, _lib.CACHE_CODES[kind], kp, vp, k_scale.data_ptr(), v_scale.data_ptr(), gp), \
        H, page, D, dev


_CACHE_NAMES = ("k_cache", "v_cache", "k_scale", "v_scale")


def _rows(t: torch.Tensor):
    """``(tensor, token stride, head stride)`` of a (tokens, heads, D) tensor whose rows of D lie
    together; strides of dimensions of size one do not count and a broadcast one is written out."""
    (n, h, d), (ts, hs, ds) = t.shape, t.stride()
    if (ds != 1 and d > 1) or (ts == 0 and n > 1) or (hs == 0 and h > 1):
        t = t.contiguous()
        ts, hs, _ = t.stride()
    if h == 1:
        hs = d
    if n == 1:
        ts = h * hs
    return t, ts, hs


def _append_faults(k, v, slots, k_cache, log_gate, log_gate_cache, H, D) -> None:
    check_cuda((k_cache, k, v, slots, log_gate), ("k_cache", "k", "v", "slots", "log_gate"))
    check_ndim(k, 3, "k")
    T = k.shape[0]
    check_shape(k, (T, H, D), "k")
    check_shape(v, (T, H, D), "v")
    if v.dtype != k.dtype:
        raise ValueError(f"[v] dtype {v.dtype} differs from k's {k.dtype}")
    _lib.dtype_code(k.dtype, "k")
    if slots.dtype != _I64:
        raise ValueError(f"[slots] expected int64, got {slots.dtype}")
    check_shape(slots, (T,), "slots")
    if (log_gate is None) != (log_gate_cache is None):
        raise ValueError("[log_gate] a cache with log-gates takes them, and one without does not")
    check_shape(log_gate, (T, H), "log_gate")


def sattn_paged_append(k, v, slots, k_cache, v_cache, k_scale, v_scale, log_gate=None, log_gate_cache=None) -> None:
    """Writes tokens into a paged cache at their slots, in place (C-ABI ``sattn_paged_append``).

    ``k``, ``v`` ``(T, Hkv, D)`` float32, bfloat16 or float16 with any token and head strides;
    ``slots`` ``(T,)`` int64 as :func:`sattn_paged_plan` gives them (-1: not written); ``k_cache``,
    ``v_cache`` ``(pages, Hkv, page_size, D)`` int8 or float8_e4m3fn; ``k_scale``, ``v_scale``
    ``(pages, Hkv)`` float32; ``log_gate`` ``(T, Hkv)`` and ``log_gate_cache`` ``(pages, Hkv, page_size)``
    float32, both or neither. A page's scale is the largest magnitude that it has held (finite ones
    count) times the reciprocal of the largest code, 127 or 448: where new tokens raise it, the page's
    earlier codes are rounded anew.
    """
    c, H, _, D, d = _cache(k_cache, v_cache, k_scale, v_scale, log_gate_cache)
    shape = k.shape
    T = shape[0] if len(shape) == 3 else -1
    if not (shape == v.shape == (T, H, D) and k.dtype == v.dtype and k.dtype in _lib.DTYPE_CODES
            and slots.dtype == _I64 and slots.shape == (T,)
            and k.get_device() == v.get_device() == slots.get_device() == d
            and (log_gate is None) == (log_gate_cache is None)
            and (log_gate is None or (log_gate.shape == (T, H) and log_gate.get_device() == d))):
        _append_faults(k, v, slots, k_cache, log_gate, log_gate_cache, H, D)
    code = _lib.DTYPE_CODES[k.dtype]
    slots = to_contiguous(slots)
    if log_gate is not None:
        log_gate = to_contiguous(log_gate.float())
    k, k_ts, k_hs = _rows(k)
    v, v_ts, v_hs = _rows(v)
    _call("sattn_paged_append", d, c, k.data_ptr(), v.data_ptr(), None if log_gate is None else log_gate.data_ptr(),
          slots.data_ptr(), T, k_ts, k_hs, v_ts, v_hs, code)


def sattn_paged_read(slots, k_cache, v_cache, k_scale, v_scale, dtype: torch.dtype = torch.float32):
    """Values of slots of a paged cache (C-ABI ``sattn_paged_read``): ``(k, v)``, each
    ``(len(slots), Hkv, D)`` in ``dtype``; zeros where a slot is not the cache's (-1)."""
    c, H, _, D, d = _cache(k_cache, v_cache, k_scale, v_scale, None)
    code = _lib.dtype_code(dtype, "dtype")
    if not (slots.dtype == _I64 and len(slots.shape) == 1 and slots.get_device() == d):
        check_cuda((k_cache, slots), ("k_cache", "slots"))
        check_ndim(slots, 1, "slots")
        raise ValueError(f"[slots] expected int64, got {slots.dtype}")
    slots = to_contiguous(slots)
    dev = slots.device
    n = slots.shape[0]
    k = torch.empty((n, H, D), device=dev, dtype=dtype)
    v = torch.empty((n, H, D), device=dev, dtype=dtype)
    _call("sattn_paged_read", d, c, slots.data_ptr(), n, k.data_ptr(), v.data_ptr(), code)
    return k, v


@functools.lru_cache(maxsize=None)
def _decode_workspace(heads: int, page: int, head_dim: int, nheads: int) -> int:
    """Bytes of workspace of a decode step; they go by the head geometry alone."""
    c = _CACHE.pack(1, heads, page, head_dim, 0, 16, 16, 16, 16, 0)
    return int(_lib.lib().sattn_paged_decode_workspace_size(c, 1, 1, nheads))


def _decode_faults(q, k_cache, block_table, lengths, H, D) -> None:
    check_cuda((k_cache, q, block_table, lengths), ("k_cache", "q", "block_table", "lengths"))
    check_ndim(q, 3, "q")
    check_ndim(block_table, 2, "block_table")
    R, Hq, d = q.shape
    if d != D or Hq == 0 or Hq % H:
        raise ValueError(f"[q] expected (requests, a multiple of {H} heads, {D}), got {tuple(q.shape)}")
    _lib.dtype_code(q.dtype, "q")
    _int32(block_table, "block_table", (R, block_table.shape[1]))
    _int32(lengths, "lengths", (R,))


def sattn_paged_decode(q, k_cache, v_cache, k_scale, v_scale, block_table, lengths, log_gate_cache=None, scale=None,
                       out=None, workspace: Optional[torch.Tensor] = None):
    """One decode step's attention over a paged cache (C-ABI ``sattn_paged_decode``).

    ``q`` ``(R, Hq, D)``, ``Hq`` a multiple of the cache's heads; ``block_table`` ``(R, W)`` and
    ``lengths`` ``(R,)`` int32. Request ``r``'s own token is the last of its ``lengths[r]`` (it was
    appended before): the pos-mode gated softmax of :func:`~.kernels.sattn_decode_step`
    (``modules/selective_attention.py:399-404``), in which every key but the own one adds its log-gate
    and a log-gate of ``-inf`` drops the key. A length of 0 gives zeros. At most 65535
    requests. ``scale`` defaults to ``D ** -0.5``. Returns ``(R, Hq, D)`` in ``q``'s dtype. ``workspace`` (contiguous uint8) is
    allocated when it is ``None`` or does not do; calls that overlap on the GPU need one each.
    """
    c, H, page, D, d = _cache(k_cache, v_cache, k_scale, v_scale, log_gate_cache)
    shape, table = q.shape, block_table.shape
    R, Hq = shape[:2] if len(shape) == 3 else (-1, 0)
    W = table[1] if len(table) == 2 else -1
    if not (Hq and shape[2] == D and Hq % H == 0 and q.dtype in _lib.DTYPE_CODES
            and table == (R, W) and lengths.shape == (R,) and block_table.dtype == lengths.dtype == _I32
            and block_table.is_contiguous() and lengths.is_contiguous()
            and q.get_device() == block_table.get_device() == lengths.get_device() == d):
        _decode_faults(q, k_cache, block_table, lengths, H, D)
    if out is not None or workspace is not None:
        check_cuda((q, out, workspace), ("q", "out", "workspace"))
    code = _lib.DTYPE_CODES[q.dtype]
    dev = q.device
    q = _aligned16(to_contiguous(q))
    if out is None:
        out = torch.empty_like(q)
    else:
        check_shape(out, (R, Hq, D), "out")
        if out.dtype != q.dtype or not out.is_contiguous() or out.data_ptr() % 16:
            raise ValueError("[out] expected a contiguous, 16-byte aligned tensor of q's dtype")
    if R == 0:
        return out
    if W == 0:
        return out.zero_()
    need = _decode_workspace(H, page, D, Hq)
    if (workspace is None or workspace.numel() * workspace.element_size() < need or workspace.data_ptr() % 16
            or not workspace.is_contiguous()):
        workspace = torch.empty(need, device=dev, dtype=torch.uint8)
    _call("sattn_paged_decode", d, c, q.data_ptr(), block_table.data_ptr(), lengths.data_ptr(), out.data_ptr(), R, W, Hq,
          D ** -0.5 if scale is None else float(scale), code, workspace.data_ptr(), need)
    return out


def _packed_faults(q, k, v, cu_seqlens, log_gate) -> None:
    check_ndim(q, 3, "q")
    check_ndim(k, 3, "k")
    check_ndim(cu_seqlens, 1, "cu_seqlens")
    check_cuda((q, k, v, cu_seqlens, log_gate), ("q", "k", "v", "cu_seqlens", "log_gate"))
    T, Hq, D = q.shape
    Hk = k.shape[1]
    if Hk == 0 or Hq == 0 or Hq % Hk:
        raise ValueError(f"[k] {Hq} query heads are not a multiple of {Hk} key heads")
    for t, n in ((k, "k"), (v, "v")):
        check_shape(t, (T, Hk, D), n)
        if t.dtype != q.dtype:
            raise ValueError(f"[{n}] dtype {t.dtype} differs from q's {q.dtype}")
    check_shape(log_gate, (T, Hk), "log_gate", optional=True)
    if cu_seqlens.shape[0] == 0:
        raise ValueError("[cu_seqlens] expected the offsets of the sequences, from 0")
    _int32(cu_seqlens, "cu_seqlens")
    _lib.dtype_code(q.dtype, "q")


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
    d = q.get_device()
    shape = q.shape
    if not (d >= 0 and len(shape) == 3 and len(k.shape) == 3 and k.shape == v.shape and k.shape[0] == shape[0]
            and k.shape[2] == shape[2] and k.shape[1] and shape[1] and shape[1] % k.shape[1] == 0
            and q.dtype == k.dtype == v.dtype and q.dtype in _lib.DTYPE_CODES and cu_seqlens.dtype == _I32
            and len(cu_seqlens.shape) == 1 and cu_seqlens.shape[0] and cu_seqlens.is_contiguous()
            and k.get_device() == v.get_device() == cu_seqlens.get_device() == d
            and (log_gate is None or (log_gate.shape == k.shape[:2] and log_gate.get_device() == d))):
        _packed_faults(q, k, v, cu_seqlens, log_gate)
    if out is not None:
        check_cuda((q, out), ("q", "out"))
    T, Hq, D = shape
    Hk = k.shape[1]
    dev = q.device
    code = _lib.DTYPE_CODES[q.dtype]
    per = 16 // q.element_size()

    def rows(t):
        t, ts, hs = _rows(t)
        if ts % per or hs % per or t.data_ptr() % 16:
            t, ts, hs = _rows(t.contiguous() if not t.is_contiguous() else t.clone())
        return t, ts, hs

    (q, q_ts, q_hs), (k, k_ts, k_hs), (v, v_ts, v_hs) = rows(q), rows(k), rows(v)
    log_gate = None if log_gate is None else to_contiguous(log_gate.float())
    if out is None:
        out = torch.empty((T, Hq, D), device=dev, dtype=q.dtype)
    else:
        check_shape(out, (T, Hq, D), "out")
        if out.dtype != q.dtype or not out.is_contiguous() or out.data_ptr() % 16:
            raise ValueError("[out] expected a contiguous, 16-byte aligned tensor of q's dtype")
    p = _PACKED.pack(T, cu_seqlens.shape[0] - 1, Hq, Hk, D, q_ts, q_hs, k_ts, k_hs, v_ts, v_hs, code, _lib.IMPLS[impl],
                     D ** -0.5 if scale is None else float(scale), q.data_ptr(), k.data_ptr(), v.data_ptr(),
                     0 if log_gate is None else log_gate.data_ptr(), cu_seqlens.data_ptr(), out.data_ptr())
    _call("sattn_prefill_packed", d, p)
    return out


class PagedSelectiveCache:
    """The paged caches of a stack of selective-attention layers and the requests that they hold.

    ``requests`` rows, each up to ``max_tokens`` tokens, share ``num_pages`` pages of ``page_size``
    tokens in every layer (a page has the same number in all of them). A step is: :meth:`plan` for the
    numbers of new tokens, then for each layer :meth:`append` of their keys, values and log-gates and
    either :func:`sattn_prefill_packed` (whole prompts, packed by the plan's ``cu_seqlens``) or
    :meth:`decode` (one token for each request); :meth:`release` gives a finished request's pages
    back. Nothing synchronizes: which requests a plan served is read from its ``lengths`` when the
    host wants to know. :meth:`plan` and :meth:`release` put new tensors in the place of ``lengths`` and
    ``free_state``: what is captured in a graph once and replayed is a step's appends and its attention, not these.
    """

    def __init__(self, layers: int, requests: int, max_tokens: int, num_pages: int, heads: int, head_dim: int,
                 page_size: int = 16, dtype: torch.dtype = torch.int8, gated: bool = True, device="cuda"):
        if page_size not in PAGE_SIZES or head_dim not in CACHE_HEAD_DIMS or dtype not in _lib.CACHE_CODES:
            raise ValueError(f"expected a page size in {PAGE_SIZES}, a head dim in {CACHE_HEAD_DIMS} and a dtype in "
                             f"{tuple(_lib.CACHE_CODES)}, got {page_size}, {head_dim}, {dtype}")
        shape = (layers, num_pages, heads, page_size, head_dim)
        self.page_size = page_size
        self.k_cache = torch.zeros(shape, dtype=dtype, device=device)
        self.v_cache = torch.zeros(shape, dtype=dtype, device=device)
        self.k_scale = torch.zeros(shape[:3], device=device)
        self.v_scale = torch.zeros(shape[:3], device=device)
        self.log_gate_cache = torch.zeros(shape[:4], device=device) if gated else None
        self.block_table = torch.full((requests, -(-max_tokens // page_size)), -1, dtype=_I32, device=device)
        self.lengths = torch.zeros(requests, dtype=_I32, device=device)
        # the ring of free pages, and a place past it for what release() does not return
        self._ring = torch.arange(num_pages + 1, dtype=_I32, device=device)
        self.free_state = torch.tensor([0, num_pages], dtype=_I64, device=device)

    @property
    def free_pages(self) -> torch.Tensor:
        return self._ring[:-1]

    def layer(self, i: int) -> dict:
        """Layer ``i``'s cache, as the functions of this module take it."""
        return dict(k_cache=self.k_cache[i], v_cache=self.v_cache[i], k_scale=self.k_scale[i],
                    v_scale=self.v_scale[i],
                    log_gate_cache=None if self.log_gate_cache is None else self.log_gate_cache[i])

    def plan(self, new_lengths: torch.Tensor, num_tokens: int):
        """Pages for ``new_lengths`` ``(requests,)`` int32 more tokens (0: the request takes no part);
        ``num_tokens`` is their sum, or more (requests past it are not served). Returns ``(cu_seqlens, slots, positions)``."""
        self.lengths, cu, slots, positions, self.free_state = sattn_paged_plan(
            self.lengths, new_lengths, self.block_table, self.free_pages, self.free_state, num_tokens, self.page_size)
        return cu, slots, positions

    def append(self, layer: int, k, v, slots, log_gate=None) -> None:
        sattn_paged_append(k, v, slots, log_gate=log_gate, **self.layer(layer))

    def decode(self, layer: int, q, scale=None, out=None, workspace=None):
        """Attention of one token for each request (``q`` ``(requests, Hq, D)``) over all that it holds."""
        return sattn_paged_decode(q, block_table=self.block_table, lengths=self.lengths, scale=scale, out=out,
                                  workspace=workspace, **self.layer(layer))

    def release(self, rows: torch.Tensor) -> None:
        """Gives back the pages of the requests ``rows`` (int64 indices, each once)."""
        held = (self.lengths[rows].long() + self.page_size - 1) // self.page_size
        at = torch.arange(self.block_table.shape[1], device=rows.device)
        there = at[None, :] < held[:, None]
        place = (self.free_state[1] + (held.cumsum(0) - held)[:, None] + at) % (self._ring.shape[0] - 1)
        place = torch.where(there, place, self._ring.shape[0] - 1)
        self._ring[place] = self.block_table[rows]
        self.free_state = self.free_state + torch.stack([torch.zeros_like(held[:1]).sum(), held.sum()])
        self.block_table[rows] = -1
        self.lengths = self.lengths.index_fill(0, rows, 0)
