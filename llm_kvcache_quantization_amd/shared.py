"""Several answers from one prompt on a paged cache: copied pages, and attention over a shared prefix.

* :func:`copy_paged` -- pages onto others, in the pools of all layers at once: the page that a forked sequence
  goes on writing, or all that is held into another pool;
* :func:`decode_attn_shared` -- attention of one new token a sequence, where the sequences of a group continue one
  prompt whose pages they share: K and V of the prompt are read once for all of them.

:class:`PagePools` and :class:`SharedPrefix` are what a program keeps for them from call to call: the pools' layout,
and how the sequences share their first tokens.  Layouts, devices, streams and what a page number outside the pool
means are as in :mod:`paged`; there is no backward pass.  :meth:`PagedKVCache.fork` is what puts the two to use.

The reference has no counterpart: each of its caches holds one dense row a sequence (src/cache/int8_cache.py:29).
"""
from __future__ import annotations

import ctypes
import functools
from bisect import bisect_left
from typing import Dict, List, Optional, Sequence, Tuple, Union

import torch
from torch import Tensor
from torch.autograd import forward_ad

from . import _capi as C
from .paged import _SM, _TYPES, HEAD_DIM, PAGE_SIZES, _cache_fields, _call, _i32, _no_grad, _packer, _rows16, _tau

MAX_ROWS = 4096  # of a call of decode_attn_shared

_COPY, _SHARED = _packer(C.CopyPagesParams), _packer(C.SharedDecodeParams)


class PagePools:
    """Tensors of pages that are copied together: [num_pages, heads, page_size, X] alike but for X and type, such as
    K, V and their scales of every layer.  Rows (X elements, 2 to 1024 bytes, a power of two) are contiguous, and one behind
    the other where they have less than 16 bytes; pages and heads begin at multiples of 16 bytes.  Holds the tensors; layout, and whether they require a
    gradient, are looked at here, once."""

    def __init__(self, tensors: Sequence[Tensor]):
        self.tensors = tuple(tensors)
        if not self.tensors:
            raise ValueError("pools must be at least one tensor of pages")
        first = self.tensors[0]
        if first.ndim != 4 or not first.is_cuda:
            raise ValueError(f"pools must be [num_pages, heads, page_size, X] on a GPU, got {tuple(first.shape)} on {first.device}")
        self.device, (self.num_pages, self.heads, self.page_size) = first.device, first.shape[:3]
        if self.page_size not in PAGE_SIZES or self.heads == 0:
            raise ValueError(f"page_size must be one of {PAGE_SIZES} and heads positive, got {self.page_size} and {self.heads}")
        rows = []
        self.written = True  # whether every page and head has memory of its own
        for t in self.tensors:
            if t.ndim != 4 or t.device != self.device or t.shape[:3] != first.shape[:3]:
                raise ValueError(f"pools must be alike in device and their first three sizes: {tuple(first.shape)} on {first.device} "
                                 f"and {tuple(t.shape)} on {t.device}")
            item, (sp, sh, st, sx) = t.element_size(), t.stride()
            row = item * t.shape[3]
            if not 2 <= row <= 1024 or row & (row - 1):
                raise ValueError(f"a row must have 2 to 1024 bytes, a power of two, got {row}")
            if t.shape[3] > 1 and sx != 1:
                raise ValueError("page rows must be contiguous")
            if row < 16 and st * item != row:
                raise ValueError("rows of less than 16 bytes must lie one behind the other within a page")
            if t.data_ptr() % 16 or self.num_pages > 1 and sp * item % 16 or self.heads > 1 and sh * item % 16 or st * item % min(row, 16):
                raise ValueError("pages, heads and rows must begin at multiples of 16 bytes")
            self.written &= (self.num_pages < 2 or sp > 0) and (self.heads < 2 or sh > 0) and st > 0
            # the stride of a dimension of one is not used, whatever it is
            rows.append((t.data_ptr(), sp * item if self.num_pages > 1 else 0, sh * item if self.heads > 1 else 0, st * item, row, 0))
        self._grad = any(t.requires_grad for t in self.tensors)
        self.layout = tuple((t.shape[3], t.dtype) for t in self.tensors)
        self._blocks = (C.PagePool * len(rows))(*rows)
        self._at = ctypes.addressof(self._blocks)

    @functools.cached_property
    def _grids(self) -> Tuple[Dict[Tuple[int, int], List[int]], List[int]]:
        """Where the tensors' pages begin, to find those that two tensors have in common: of each (page stride, address of a page
        modulo it) the tensors' first pages as multiples of the stride, rising; and the addresses of those that repeat one page."""
        grids: Dict[Tuple[int, int], List[int]] = {}
        fixed = []
        for t in self.tensors:
            at, step = t.data_ptr(), t.stride(0) * t.element_size()
            if step:
                grids.setdefault((step, at % step), []).append(at // step)
            else:
                fixed.append(at)
        for firsts in grids.values():
            firsts.sort()
        return grids, fixed


@functools.lru_cache(maxsize=256)
def _scratch(info: Tuple[int, ...], cols: int, size: int, rows: int, heads: int, q_heads: int) -> int:
    """Bytes of scratch of a call: a matter of its sizes alone."""
    p = C.SharedDecodeParams()
    c = p.cache
    c.k_stride_t = c.v_stride_t = 2 * HEAD_DIM
    c.max_pages, c.page_size, c.batch, c.kv_heads = cols, size, rows, heads
    c.k = c.v = c.table = 16  # not read
    p.plan, p.q_heads = C.SharedPlanInfo(*info), q_heads
    return C.lib().kvq_shared_decode_workspace_bytes(ctypes.byref(p))


Pages = Union[Tensor, Sequence[int]]


def _apart(pools: PagePools, src: Optional[List[int]], to: PagePools, dst: List[int]) -> None:
    """Refuses pages that are written twice, or written and read (`src` None: not known here)."""
    written = set(dst)
    if len(written) < len(dst):
        raise ValueError("no page may be written twice")
    if not written:
        return
    low, high = min(written), max(written)
    (reads, fixed), (writes, _) = pools._grids, to._grids
    for grid, firsts in writes.items():
        for i, a in enumerate(firsts):  # page d of a tensor is page d - k of one that begins k pages behind it
            for b in firsts[i + 1 :]:
                if b - a > high - low:
                    break
                # (a tensor that the pools name twice is written twice, with the same)
                if (b > a or to is not pools) and any(d + b - a in written for d in dst):
                    raise ValueError("no page may be written twice: tensors that are written share their memory")
        if not src:
            continue
        least, most = low - max(src), high - min(src)
        for r in reads.get(grid, ()):  # page s of a tensor is page s + r - w of one that begins at w
            for w in firsts[bisect_left(firsts, r - most) :]:
                if r - w < least:
                    break
                if any(s + r - w in written for s in src):
                    raise ValueError("no page may be written by one pair and read by another")
        for at in fixed:
            if at % grid[0] == grid[1] and any(at // grid[0] - w in written for w in firsts):
                raise ValueError("no page may be written by one pair and read by another")


def _page_numbers(x: Union[Tensor, List[int]], name: str, pages: int, device: torch.device) -> Tensor:
    if isinstance(x, Tensor):
        if x.ndim != 1:
            raise ValueError(f"{name} must be [n], got {tuple(x.shape)}")
        return _i32(x, name, x.shape[0], device)
    if any(not 0 <= v < pages for v in x):
        raise ValueError(f"{name} must be pages of the pool, 0 to {pages - 1}")
    return torch.tensor(x, dtype=torch.int32, device=device)


def copy_paged(pools: Union[PagePools, Sequence[Tensor]], src: Pages, dst: Pages, lens: Optional[Tensor] = None, *,
               into: Union[PagePools, Sequence[Tensor], None] = None) -> None:
    """Copies page ``src[i]`` of every tensor of ``pools`` onto page ``dst[i]`` of the same tensor, or of its counterpart
    in ``into``: the first ``lens[i]`` slots of it (default: all); what lies behind is left as it was.

    ``src`` and ``dst`` [n] are integer tensors, or whole numbers from the host, which are checked; of tensors, pairs with a
    page that is not there are left out.  No page may be written by two pairs, or written by one and read by another.
    (Of numbers from the host that is refused too, where pages are the same because the pools' tensors and those of
    ``into`` are the same or slices of one another's pages; memory that is cut into pages in two ways is not looked for.)
    ``into`` has the pools' heads, page size, row sizes and types; its number of pages may differ.
    """
    pools = pools if isinstance(pools, PagePools) else PagePools(pools)
    to = pools if into is None else into if isinstance(into, PagePools) else PagePools(into)
    if to is not pools:
        if to.device != pools.device or to.heads != pools.heads or to.page_size != pools.page_size or to.layout != pools.layout:
            raise ValueError("into must have the pools' device, heads, page size, row sizes and types")
    if not to.written:
        raise ValueError("pages that are written must have memory of their own, got a stride of 0")
    if pools._grad or to._grad or forward_ad._current_level >= 0:
        _no_grad(*pools.tensors, *to.tensors)
    device = pools.device
    if not isinstance(src, Tensor):
        src = [int(v) for v in src]
    if not isinstance(dst, Tensor):
        dst = [int(v) for v in dst]
        _apart(pools, None if isinstance(src, Tensor) else src, to, dst)
    src, dst = _page_numbers(src, "src", pools.num_pages, device), _page_numbers(dst, "dst", to.num_pages, device)
    n = src.shape[0]
    if dst.shape[0] != n:
        raise ValueError(f"src and dst must be of one length, got {n} and {dst.shape[0]}")
    if lens is not None:
        lens = _i32(lens, "lens", n, device)
    if n:
        _call(C.lib().kvq_copy_pages, _COPY.pack(
            pools._at, to._at, src.data_ptr(), dst.data_ptr(), 0 if lens is None else lens.data_ptr(), len(pools.tensors), n,
            pools.page_size, pools.heads, pools.num_pages, to.num_pages), device)


class SharedPrefix:
    """How the sequences of a batch share their first tokens: group g is the next ``sizes[g]`` sequences, and the first
    ``lens[g]`` tokens of each of them are those of the group's first one (0: none shared).  Made for a model's head
    counts; holds for any pages and contexts, so that a program makes it once for as long as the groups last."""

    def __init__(self, sizes: Sequence[int], lens: Sequence[int], q_heads: int, kv_heads: int,
                 device: Union[str, torch.device] = "cuda"):
        self.sizes, self.lens = tuple(int(s) for s in sizes), tuple(int(n) for n in lens)
        if len(self.sizes) != len(self.lens):
            raise ValueError(f"sizes and lens must be of one length, got {len(self.sizes)} and {len(self.lens)}")
        if any(not -(1 << 31) <= v < 1 << 31 for v in self.sizes + self.lens):
            raise ValueError("sizes and lens must fit 32 bits")
        self.q_heads, self.kv_heads = int(q_heads), int(kv_heads)
        n, info = len(self.sizes), C.SharedPlanInfo()
        sizes_c, lens_c = (C.c_i32 * n)(*self.sizes), (C.c_i32 * n)(*self.lens)
        plan = C.lib().kvq_shared_plan
        C.check(plan(sizes_c, lens_c, n, self.q_heads, self.kv_heads, ctypes.byref(info), None, 0))
        words = torch.empty(info.words, dtype=torch.int32)
        C.check(plan(sizes_c, lens_c, n, self.q_heads, self.kv_heads, ctypes.byref(info), words.data_ptr(), info.words))
        self._info = (info.rows, info.units, info.slots, info.words)
        device = torch.device(device)
        if device.type == "cuda" and device.index is None:
            device = torch.device("cuda", torch.cuda.current_device())
        self.device = device
        self._words = words.to(device)
        self._stream = C.stream_handle(device) if device.type == "cuda" else None

    @property
    def rows(self) -> int:
        return self._info[0]

    def __repr__(self) -> str:
        return f"SharedPrefix(sizes={list(self.sizes)}, lens={list(self.lens)}, heads={self.q_heads}/{self.kv_heads})"


def decode_attn_shared(q: Tensor, k_pages: Tensor, v_pages: Tensor, block_table: Tensor, context_lens: Tensor,
                       prefix: SharedPrefix, sm_scale: Optional[float] = None, *, k_scale: Optional[Tensor] = None,
                       v_scale: Optional[Tensor] = None, inv_tau: Optional[Tensor] = None) -> Tensor:
    """Attention of one query token a sequence, q [B, Hq, 128] (fp16 or bf16), over its pages; returns [B, Hq, 128] in q's
    type.  What :func:`decode_attn_paged` computes without a window, with K and V of a group's prefix read once for all
    its sequences:

    with n = ``context_lens[b]`` (the new token included), out = softmax_t(sm_scale * inv_tau[h] * q . k_t) @ v_t over t < n,
    statistics and sums in fp32; token t < ``prefix.lens[g]`` lies in the pages of the group's first sequence, whatever
    b's own table says there.  Sequences that see nothing are zero.  fp16 / bf16 pages must have q's type; INT8 pages
    serve both (V's values code * scale are used in fp16).  Hq / Hkv is at most 128, B at most 4096, and a page stride below 2^32 bytes.
    """
    if q.ndim != 3 or q.shape[2] != HEAD_DIM:
        raise ValueError(f"q must be [B, Hq, {HEAD_DIM}], got {tuple(q.shape)}")
    batch, q_heads, _ = q.shape
    cache = _cache_fields(k_pages, v_pages, k_scale, v_scale, block_table, batch)
    device, heads = k_pages.device, k_pages.shape[1]
    if q.dtype not in _TYPES or (k_pages.dtype != torch.int8 and q.dtype != k_pages.dtype):
        raise ValueError(f"q must be fp16 or bf16 and of the pages' type: got {q.dtype} for {k_pages.dtype} pages")
    if q.device != device or prefix.device != device:
        raise ValueError(f"q and prefix must lie on {device}, got {q.device} and {prefix.device}")
    if prefix.rows != batch or prefix.q_heads != q_heads or prefix.kv_heads != heads:
        raise ValueError(f"prefix is made for {prefix.rows} sequences and {prefix.q_heads} / {prefix.kv_heads} heads, got {batch} "
                         f"and {q_heads} / {heads}")
    _no_grad(q, k_pages, v_pages, k_scale, v_scale, inv_tau)
    lens = _i32(context_lens, "context_lens", batch, device)
    tau = None if inv_tau is None else _tau(inv_tau, q_heads, device)
    q = _rows16(q)
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    if batch == 0:
        return out
    if prefix._stream != C.stream_handle(device):  # not given back while this stream still reads it
        prefix._words.record_stream(torch.cuda.current_stream(device))
    nbytes = _scratch(prefix._info, block_table.shape[1], k_pages.shape[2], batch, heads, q_heads)
    scratch = q.new_empty(nbytes, dtype=torch.uint8)
    _call(C.lib().kvq_shared_decode, _SHARED.pack(
        *cache, q.data_ptr(), *q.stride()[:2], out.data_ptr(), lens.data_ptr(), 0 if tau is None else tau.data_ptr(),
        prefix._words.data_ptr(), scratch.data_ptr(), nbytes, *prefix._info, _SM if sm_scale is None else sm_scale, q_heads,
        _TYPES[q.dtype], 0), device)
    return out
