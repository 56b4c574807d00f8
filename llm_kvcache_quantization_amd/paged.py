"""A cache in pages, bounded by a sliding window or a budget: its operators.

* :func:`append_paged` -- new K / V rows of a ragged batch into their pages, as they are (fp16, bf16)
  or in INT8 with an fp16 scale per (token, group);
* :func:`decode_attn_paged` -- attention of one new token a sequence over its pages, split over the
  length and joined, whole or through a sliding window with a few first tokens that stay visible
  (sinks), and optionally adding the softmax to accumulated weights;
* :func:`prefill_attn_window` -- attention of a prompt, or of a chunk of one, through the same window;
* :func:`evict_paged` -- cuts the cache down to a budget of tokens per KV head by accumulated weight.

:class:`PagedKVCache` (:mod:`paged_cache`) is the cache engine over them.

Layout.  A layer's cache is ``k_pages`` and ``v_pages`` [num_pages, Hkv, page_size, 128] (any strides
with contiguous, 16-byte aligned rows), with ``k_scale`` / ``v_scale`` fp16 [num_pages, Hkv, page_size, G]
beside INT8 pages (G = 128 / group_size, group_size 32, 64 or 128).  ``block_table`` int32 [B, max_pages] names
the pages of each sequence: token t lies in page ``block_table[b, t // page_size]``.  page_size is 16, 32,
64, 128 or 256.

Lengths, positions and page numbers stay on the GPU: nothing here waits for it.  Lengths are clamped to
what the table can hold.  A page number outside [0, num_pages) stands for a page that is not there: its
tokens are left out of the attention, nothing is written to it, and a sequence that has one among its
tokens is not evicted.

Everything is enqueued on the current stream of the tensors' device.  Scratch memory comes from torch's
allocator, call by call, so that calls on several streams and captured graphs share none.  There is no
backward pass: the operators serve inference, as the rest of this package does, and refuse tensors that
require a gradient while gradients are recorded, and tensors with a tangent of forward differentiation.

The reference has no counterpart: its caches are dense and unbounded (src/cache/int8_cache.py,
src/cache/fp16_cache.py).
"""
from __future__ import annotations

import ctypes
import functools
import math
import struct
from typing import Optional, Tuple

import torch
from torch import Tensor
from torch.autograd import forward_ad

from . import _capi as C

HEAD_DIM = 128
PAGE_SIZES = (16, 32, 64, 128, 256)
_INTEGERS = (torch.int8, torch.uint8, torch.int16, torch.uint16, torch.int32, torch.uint32, torch.int64)
_TYPES = {torch.float16: C.KVQ_PAGED_F16, torch.bfloat16: C.KVQ_PAGED_BF16}


def _leaves(cls):
    for _, t in cls._fields_:
        if issubclass(t, ctypes.Structure):
            yield from _leaves(t)
        else:
            yield {C.c_vp: "P", C.c_i64: "q", C.c_i32: "i", C.c_f32: "f"}[t]


def _packer(cls) -> struct.Struct:
    """The parameter block's fields in order, in C's alignment: one pack() fills a block."""
    return struct.Struct("@" + "".join(_leaves(cls)))


_SM = 1.0 / math.sqrt(HEAD_DIM)
_APPEND, _DECODE, _PREFILL, _EVICT = (_packer(c) for c in (
    C.PagedAppendParams, C.PagedDecodeParams, C.PrefillParams, C.PagedEvictParams))


def _no_grad(*tensors: Optional[Tensor]) -> None:
    """Refuses tensors of a recorded graph, and those with a tangent: either derivative would be lost in silence."""
    grad, dual = torch.is_grad_enabled(), forward_ad._current_level >= 0
    if grad or dual:
        for t in tensors:
            if t is None:
                continue
            if grad and t.requires_grad:
                raise NotImplementedError("the paged operators have no backward pass: call them under torch.no_grad()")
            if dual and forward_ad.unpack_dual(t).tangent is not None:
                raise NotImplementedError("the paged operators have no forward derivative: they take no tensor with a tangent")


_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


def _call(fn, block: bytes, device: torch.device) -> None:
    if device.index != _current_device():
        with torch.cuda.device(device):
            C.check(fn(block, C.stream_handle(device)))
    else:
        C.check(fn(block, C.stream_handle(device)))


def _i32(t: Tensor, name: str, batch: int, device: torch.device) -> Tensor:
    """A [B] tensor of lengths or positions as contiguous int32 on the device."""
    if t.ndim != 1 or t.shape[0] != batch:
        raise ValueError(f"{name} must be [B] = [{batch}], got {tuple(t.shape)}")
    if t.dtype != torch.int32 or t.device != device:
        if t.dtype not in _INTEGERS:
            raise ValueError(f"{name} must be integers of at most 64 bits with a sign, got {t.dtype}")
        if t.dtype in (torch.int64, torch.uint32):  # to int32's ends, which lie behind every table
            t = t.to(torch.int64).clamp(-1 << 31, (1 << 31) - 1)
        t = t.to(device=device, dtype=torch.int32)
    return t.contiguous()


def _cache_fields(k_pages: Tensor, v_pages: Tensor, k_scale: Optional[Tensor], v_scale: Optional[Tensor],
                  table: Tensor, batch: Optional[int] = None) -> tuple:
    """The checked fields of kvq_paged_cache."""
    shape = k_pages.shape
    if len(shape) != 4 or shape[3] != HEAD_DIM:
        raise ValueError(f"pages must be [num_pages, Hkv, page_size, {HEAD_DIM}], got {tuple(shape)}")
    if v_pages.shape != shape:
        raise ValueError(f"k/v pages differ in shape: {tuple(shape)} vs {tuple(v_pages.shape)}")
    pages, heads, size, _ = shape
    dtype, index = k_pages.dtype, k_pages.get_device()
    if not k_pages.is_cuda:
        raise ValueError("the paged operators need GPU (ROCm) tensors")
    if v_pages.dtype != dtype or v_pages.get_device() != index:
        raise ValueError(f"k/v pages differ: {dtype} on {k_pages.device} vs {v_pages.dtype} on {v_pages.device}")
    if size not in PAGE_SIZES:
        raise ValueError(f"page_size must be one of {PAGE_SIZES}, got {size}")
    if heads == 0:
        raise ValueError("pages must have a KV head")
    if dtype == torch.int8:
        fmt, item = C.KVQ_PAGED_INT8, 1
        if k_scale is None or v_scale is None:
            raise ValueError("INT8 pages need k_scale and v_scale")
        groups = k_scale.shape[-1]
        for name, s in (("k_scale", k_scale), ("v_scale", v_scale)):
            if s.dtype != torch.float16 or s.get_device() != index or s.shape != (pages, heads, size, groups) or \
                    groups not in (1, 2, 4):
                raise ValueError(f"{name} must be fp16 [{pages}, {heads}, {size}, G] with G 1, 2 or 4 on {k_pages.device}, got "
                                 f"{s.dtype} {tuple(s.shape)} on {s.device}")
        ks, vs = k_scale.stride(), v_scale.stride()
        if pages and (ks[2] != groups or vs[2] != groups or groups > 1 and (ks[3] != 1 or vs[3] != 1)):
            raise ValueError(f"a page's scales must be dense, got strides {ks} and {vs}")
        group = HEAD_DIM // groups
        scales = (k_scale.data_ptr(), v_scale.data_ptr(), 2 * ks[0], 2 * ks[1], 2 * vs[0], 2 * vs[1])
    else:
        fmt, item, group = _TYPES.get(dtype), 2, 0
        if fmt is None:
            raise ValueError(f"pages must be float16, bfloat16 or int8, got {dtype}")
        if k_scale is not None or v_scale is not None:
            raise ValueError(f"{dtype} pages take no scales")
        scales = (0, 0, 0, 0, 0, 0)
    k, v = k_pages.stride(), v_pages.stride()
    if k[3] != 1 or v[3] != 1:
        raise ValueError("page rows must be contiguous")
    if table.ndim != 2 or table.dtype != torch.int32 or table.get_device() != index:
        raise ValueError(f"block_table must be int32 [B, max_pages] on {k_pages.device}, got {table.dtype} "
                         f"{tuple(table.shape)} on {table.device}")
    rows, cols = table.shape
    step, inner = table.stride()
    if cols > 1 and inner != 1:
        raise ValueError("block_table rows must be contiguous")
    if batch is not None and rows != batch:
        raise ValueError(f"block_table has {rows} rows for a batch of {batch}")
    return (k_pages.data_ptr(), v_pages.data_ptr(), item * k[0], item * k[1], item * k[2], item * v[0], item * v[1],
            item * v[2], *scales, table.data_ptr(), step, pages, cols, size, fmt, group, rows, heads, 0)


def _rows16(x: Tensor) -> Tensor:
    """x itself if its rows of 128 are contiguous and 16-byte aligned, else a copy."""
    *outer, inner = x.stride()
    if inner != 1 or x.data_ptr() & 15 or any([v & 7 for v in outer]):
        return x.clone(memory_format=torch.contiguous_format)
    return x


def _tau(inv_tau: Tensor, heads: int, device: torch.device) -> Tensor:
    if inv_tau.shape != (heads,):
        raise ValueError(f"inv_tau must be [{heads}] (one per query head), got {tuple(inv_tau.shape)}")
    return inv_tau.to(device=device, dtype=torch.float32).contiguous()


def _window(window: Optional[int], sinks: int) -> Tuple[int, int]:
    if window is None:
        window = 0
    elif window < 1:
        raise ValueError(f"window must be at least 1 (or None), got {window}")
    if sinks < 0:
        raise ValueError(f"sinks must be >= 0, got {sinks}")
    return min(int(window), 1 << 30), min(int(sinks), 1 << 30)


@functools.lru_cache(maxsize=256)
def _decode_scratch(pages: int, cols: int, size: int, rows: int, heads: int, q_heads: int, window: int, sinks: int,
                    weights: bool) -> int:
    """Bytes of scratch of a decode call: a matter of its sizes alone."""
    p = C.PagedDecodeParams()
    c = p.cache
    c.k_stride_t = c.v_stride_t = 2 * HEAD_DIM
    c.num_pages, c.max_pages, c.page_size, c.batch, c.kv_heads = pages, cols, size, rows, heads
    c.k = c.v = c.table = p.weights = 16  # not read
    if not weights:
        p.weights = None
    p.window, p.sinks, p.q_heads = window, sinks, q_heads
    return C.lib().kvq_paged_decode_workspace_bytes(ctypes.byref(p))


@functools.lru_cache(maxsize=256)
def _prefill_scratch(batch: int, q_heads: int, heads: int, seq: int, total: int, window: int, sinks: int) -> int:
    p = C.PrefillParams()
    p.batch, p.q_heads, p.kv_heads, p.seq_q, p.seq_kv, p.window, p.sinks = batch, q_heads, heads, seq, total, window, sinks
    return C.lib().kvq_prefill_workspace_bytes(ctypes.byref(p))


def append_paged(k: Tensor, v: Tensor, k_pages: Tensor, v_pages: Tensor, block_table: Tensor, write_pos: Tensor,
                 new_lens: Optional[Tensor] = None, *, k_scale: Optional[Tensor] = None,
                 v_scale: Optional[Tensor] = None) -> None:
    """Appends k, v [B, Hkv, S, 128] (fp16 or bf16) into the pages: token i of sequence b goes to slot
    ``write_pos[b] + i`` for i < ``new_lens[b]`` (default: all S; a padded batch passes its lengths).

    fp16 / bf16 pages take the rows as they are and must have their type.  INT8 pages take codes and fp16
    scales per (token, group), bit for bit those of :class:`INT8KVCache` with ``clip_percentile=100``: scale =
    fp16(max(absmax, 1e-5) / 127), code = round(fp16(x / scale)) clamped to +-127.  A group with a NaN or an
    Inf gets the scale NaN (whoever attends to the token gets NaN, as from fp16 pages).  Group maxima from
    65,500 up read back as infinite.

    Slots past the table's end, and pages that are not there, are not written.  Pages that two sequences
    share, or one has twice, may be read but not appended to.
    """
    if k.ndim != 4 or k.shape[3] != HEAD_DIM or k.shape != v.shape:
        raise ValueError(f"k and v must be [B, Hkv, S, {HEAD_DIM}] alike, got {tuple(k.shape)} / {tuple(v.shape)}")
    batch, heads, seq, _ = k.shape
    cache = _cache_fields(k_pages, v_pages, k_scale, v_scale, block_table, batch)
    device = k_pages.device
    if k.dtype not in _TYPES or v.dtype != k.dtype or (k_pages.dtype != torch.int8 and k.dtype != k_pages.dtype):
        raise ValueError(f"k/v must be fp16 or bf16 and of the pages' type: got {k.dtype} / {v.dtype} for {k_pages.dtype} pages")
    if k.device != device or v.device != device:
        raise ValueError(f"k/v must lie on {device}, got {k.device} / {v.device}")
    if heads != k_pages.shape[1]:
        raise ValueError(f"k/v have {heads} heads, the pages {k_pages.shape[1]}")
    _no_grad(k, v, k_pages, v_pages, k_scale, v_scale)
    pos = _i32(write_pos, "write_pos", batch, device)
    lens = None if new_lens is None else _i32(new_lens, "new_lens", batch, device)
    k, v = _rows16(k), _rows16(v)
    _call(C.lib().kvq_paged_append, _APPEND.pack(
        *cache, k.data_ptr(), v.data_ptr(), *k.stride()[:3], *v.stride()[:3], pos.data_ptr(),
        0 if lens is None else lens.data_ptr(), seq, _TYPES[k.dtype]), device)


def decode_attn_paged(q: Tensor, k_pages: Tensor, v_pages: Tensor, block_table: Tensor, context_lens: Tensor,
                      sm_scale: Optional[float] = None, *, k_scale: Optional[Tensor] = None,
                      v_scale: Optional[Tensor] = None, inv_tau: Optional[Tensor] = None,
                      window: Optional[int] = None, sinks: int = 0, weights: Optional[Tensor] = None) -> Tensor:
    """Attention of one query token a sequence, q [B, Hq, 128] (fp16 or bf16), over its pages; returns [B, Hq,
    128] in q's type.

    With n = ``context_lens[b]`` (the new token included) token t is seen where t < n and, with a window, t >= n -
    window or t < sinks:  out = softmax_t(sm_scale * inv_tau[h] * q . k_t) @ v_t, statistics and sums in fp32.
    Sequences that see nothing are zero.  fp16 / bf16 pages must have q's type; INT8 pages serve both (V's values
    code * scale are used in fp16).  Hq / Hkv is at most 16, B at most 4096.

    ``weights`` (fp32 [B, Hkv, >= max_pages * page_size], tokens contiguous) accumulates in place what each token
    was given: weights[b, g, t] += the softmax summed over the query heads of KV head g.
    """
    if q.ndim != 3 or q.shape[2] != HEAD_DIM:
        raise ValueError(f"q must be [B, Hq, {HEAD_DIM}], got {tuple(q.shape)}")
    batch, q_heads, _ = q.shape
    cache = _cache_fields(k_pages, v_pages, k_scale, v_scale, block_table, batch)
    device, heads = k_pages.device, k_pages.shape[1]
    if q.dtype not in _TYPES or (k_pages.dtype != torch.int8 and q.dtype != k_pages.dtype):
        raise ValueError(f"q must be fp16 or bf16 and of the pages' type: got {q.dtype} for {k_pages.dtype} pages")
    if q.device != device:
        raise ValueError(f"q must lie on {device}, got {q.device}")
    if q_heads == 0 or q_heads % heads:
        raise ValueError(f"q_heads={q_heads} must be a multiple of kv_heads={heads}")
    _no_grad(q, k_pages, v_pages, k_scale, v_scale, inv_tau, weights)
    lens = _i32(context_lens, "context_lens", batch, device)
    window, sinks = _window(window, sinks)
    w = (0, 0, 0)
    if weights is not None:
        if weights.ndim != 3 or weights.shape[:2] != (batch, heads) or weights.dtype != torch.float32 or \
                weights.device != device or weights.shape[2] < block_table.shape[1] * k_pages.shape[2]:
            raise ValueError(f"weights must be fp32 [{batch}, {heads}, >= {block_table.shape[1] * k_pages.shape[2]}] on "
                             f"{device}, got {weights.dtype} {tuple(weights.shape)} on {weights.device}")
        if weights.shape[2] > 1 and weights.stride(2) != 1:
            raise ValueError("weights must be contiguous over the tokens")
        ws = weights.stride()
        if batch > 1 and ws[0] == 0 or heads > 1 and ws[1] == 0:
            raise ValueError("weights must have memory of their own for every sequence and head")
        w = (weights.data_ptr(), ws[0], ws[1])
    tau = None if inv_tau is None else _tau(inv_tau, q_heads, device)
    q = _rows16(q)
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    if batch == 0:
        return out
    # (the sizes' limits are checked in the library, by both calls)
    nbytes = _decode_scratch(k_pages.shape[0], block_table.shape[1], k_pages.shape[2], batch, heads, q_heads, window, sinks, weights is not None)
    scratch = q.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
    _call(C.lib().kvq_paged_decode, _DECODE.pack(
        *cache, q.data_ptr(), *q.stride()[:2], out.data_ptr(), lens.data_ptr(), 0 if tau is None else tau.data_ptr(), *w,
        0 if scratch is None else scratch.data_ptr(), nbytes, _SM if sm_scale is None else sm_scale, window, sinks, q_heads,
        _TYPES[q.dtype], 0), device)
    return out


def prefill_attn_window(q: Tensor, k: Tensor, v: Tensor, sm_scale: Optional[float] = None, *,
                        window: Optional[int] = None, sinks: int = 0, q_lens: Optional[Tensor] = None,
                        kv_lens: Optional[Tensor] = None, inv_tau: Optional[Tensor] = None) -> Tensor:
    """Causal attention of a prompt, or of a chunk of one: q [B, Hq, S, 128] over k, v [B, Hkv, T, 128] (all fp16 or
    all bf16, any strides); returns [B, Hq, S, 128].

    Query i of sequence b, i < ``q_lens[b]`` (default S), stands at position p = ``kv_lens[b]`` - ``q_lens[b]`` + i
    (``kv_lens`` default T) and sees key j where j <= p and, with a window, j > p - window or j < sinks.  Padded
    queries, and those that see nothing, are zero; keys at or past ``kv_lens[b]`` may hold anything.  Softmax
    statistics and sums in fp32, the probabilities enter the product with V in the inputs' type.
    """
    if q.ndim != 4 or q.shape[3] != HEAD_DIM:
        raise ValueError(f"q must be [B, Hq, S, {HEAD_DIM}], got {tuple(q.shape)}")
    batch, q_heads, seq, _ = q.shape
    if k.ndim != 4 or k.shape[0] != batch or k.shape[3] != HEAD_DIM or v.shape != k.shape:
        raise ValueError(f"k and v must be [{batch}, Hkv, T, {HEAD_DIM}] alike, got {tuple(k.shape)} / {tuple(v.shape)}")
    heads, total = k.shape[1], k.shape[2]
    device = q.device
    if not q.is_cuda or k.device != device or v.device != device:
        raise ValueError(f"q, k and v must lie on one GPU, got {q.device} / {k.device} / {v.device}")
    if q.dtype not in _TYPES or k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError(f"q, k and v must be all fp16 or all bf16, got {q.dtype} / {k.dtype} / {v.dtype}")
    if q_heads == 0 or heads == 0 or q_heads % heads:
        raise ValueError(f"q_heads={q_heads} must be a multiple of kv_heads={heads}")
    _no_grad(q, k, v, inv_tau)
    ql = None if q_lens is None else _i32(q_lens, "q_lens", batch, device)
    kl = None if kv_lens is None else _i32(kv_lens, "kv_lens", batch, device)
    window, sinks = _window(window, sinks)
    tau = None if inv_tau is None else _tau(inv_tau, q_heads, device)
    q, k, v = _rows16(q), _rows16(k), _rows16(v)
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    if batch == 0 or seq == 0:
        return out
    nbytes = _prefill_scratch(batch, q_heads, heads, seq, total, window, sinks)
    scratch = q.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
    _call(C.lib().kvq_prefill_attn, _PREFILL.pack(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), *q.stride()[:3], *k.stride()[:3], *v.stride()[:3], out.data_ptr(),
        *out.stride()[:3], 0 if ql is None else ql.data_ptr(), 0 if kl is None else kl.data_ptr(),
        0 if tau is None else tau.data_ptr(), 0 if scratch is None else scratch.data_ptr(), nbytes,
        _SM if sm_scale is None else sm_scale, batch, q_heads, heads, seq, total, window, sinks, _TYPES[q.dtype], 0), device)
    return out


def evict_paged(k_pages: Tensor, v_pages: Tensor, block_table: Tensor, context_lens: Tensor, weights: Tensor,
                budget: int, *, sinks: int = 0, recent: int = 0, k_scale: Optional[Tensor] = None,
                v_scale: Optional[Tensor] = None) -> Tuple[Tensor, Tensor, Tensor]:
    """Cuts every sequence of more than ``budget`` tokens down to ``budget`` per KV head: its first ``sinks``, its last
    ``recent`` and, of the others, those of the largest weight (equal weights go to the earlier token, NaN is lower
    than all).  Kept tokens move, in order, to slots 0 .. budget - 1 of the sequence's pages, in place; what lies behind
    is left as it was.

    ``weights``: fp32 [B, Hkv, >= max_pages * page_size], as :func:`decode_attn_paged` accumulates them; not changed.
    Returns (new_lens int32 [B], kept int32 [B, Hkv, budget], new_weights fp32 like weights): the sequences' new
    lengths, the old token of every slot (-1 behind the last), and the kept tokens' weights (0 behind the last).

    Sequences of at most ``budget`` tokens stay as they are.  So do sequences with a page that is not there
    (``kept`` is -1 for them).  No page may serve two sequences, or two places of one.
    """
    cache = _cache_fields(k_pages, v_pages, k_scale, v_scale, block_table)
    device, heads, batch = k_pages.device, k_pages.shape[1], block_table.shape[0]
    lens = _i32(context_lens, "context_lens", batch, device)
    if weights.ndim != 3 or weights.shape[:2] != (batch, heads) or weights.dtype != torch.float32 or \
            weights.device != device or weights.shape[2] < block_table.shape[1] * k_pages.shape[2]:
        raise ValueError(f"weights must be fp32 [{batch}, {heads}, >= {block_table.shape[1] * k_pages.shape[2]}] on {device}, "
                         f"got {weights.dtype} {tuple(weights.shape)} on {weights.device}")
    if weights.shape[2] > 1 and weights.stride(2) != 1:
        raise ValueError("weights must be contiguous over the tokens")
    _no_grad(k_pages, v_pages, k_scale, v_scale, weights)
    if budget < 1 or sinks < 0 or recent < 0 or sinks + recent > budget:
        raise ValueError(f"budget must be positive and hold sinks + recent, got {budget}, {sinks} + {recent}")
    if budget > 1 << 30 or weights.shape[2] > 1 << 30:  # before an output of that size is made
        raise ValueError(f"budget and weights may have at most 2^30 tokens, got {budget} and {weights.shape[2]}")
    new_lens = torch.empty_like(lens)
    kept = lens.new_empty((batch, heads, budget))
    new_weights = torch.empty_like(weights, memory_format=torch.contiguous_format)
    if weights.shape[2] == 0:  # no slots: no tokens
        return new_lens.zero_(), kept.fill_(-1), new_weights
    if batch:
        _call(C.lib().kvq_paged_evict, _EVICT.pack(
            *cache, lens.data_ptr(), weights.data_ptr(), *weights.stride()[:2], new_lens.data_ptr(), kept.data_ptr(),
            new_weights.data_ptr(), weights.shape[2], budget, sinks, recent), device)
    return new_lens, kept, new_weights
