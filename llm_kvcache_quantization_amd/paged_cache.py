"""The paged KV-cache engine over the operators of :mod:`paged`.

:class:`PagedKVCache` keeps the method names of the dense engines (``append``, ``append_decode_attn``,
``get_kv``, ``get_seq_len``, ``clear``, ``release``, ``get_memory_mb``, the decode statistics), so that the
attention hook drives it through :class:`INT8CacheWrapperContainer` like any of them, and adds

* pages: sequences of different lengths share one pool per layer, and memory follows what is held;
* ``prefill_attn``: a prompt, or the next chunk of one, is appended and attended in one call;
* a bound: ``window`` (sliding window, with ``sinks`` first tokens that stay visible; pages that
  nothing can see any more go back to the pool) or ``budget`` (eviction by accumulated attention
  weight, keeping ``sinks`` first and ``recent`` last tokens, once a sequence is ``slack`` tokens over).

The reference has no counterpart: its caches are dense and unbounded (src/cache/int8_cache.py:29,
src/cache/fp16_cache.py).
"""
from __future__ import annotations

import math
from typing import List, Optional, Sequence, Tuple

import torch
from torch import Tensor

from .cache import _EngineBase
from .paged import HEAD_DIM, PAGE_SIZES, append_paged, decode_attn_paged, evict_paged, prefill_attn_window


class PagedKVCache(_EngineBase):
    """A paged cache of fp16, bf16 or INT8 pages (``dtype``; INT8 with fp16 scales per (token, ``group_size``)).

    ``num_pages`` fixes the pool (``RuntimeError`` when it is used up); without it the pool grows by doubling.
    ``max_seq_len`` bounds the tokens that a sequence holds (those of pages given back no longer count).  Layers share the
    block table: call them in the same order with the same token counts, as a model's forward does (those in use: a
    layer that never appends needs no pages, and one that begins late takes pages of its own for what the others
    gave back).  K and V are fp16 or bf16; float pages have their
    type, INT8 pages take either.  What the engine keeps (pools, table, lengths) belongs to the stream it was made on:
    use it on one stream, or make the other wait before and after.
    """

    def __init__(self, num_layers: int, device: str = "cuda", dtype: torch.dtype = torch.float16, page_size: int = 64,
                 num_pages: Optional[int] = None, group_size: int = 32, max_seq_len: Optional[int] = None,
                 window: Optional[int] = None, sinks: int = 0, budget: Optional[int] = None, recent: Optional[int] = None,
                 slack: Optional[int] = None, inv_tau: Optional[Tensor] = None, use_attn_temperature: bool = True,
                 decode_attn_impl: str = "hip_fused"):
        self._init_common(num_layers, device, max_seq_len, decode_attn_impl, False)
        if dtype not in (torch.float16, torch.bfloat16, torch.int8):
            raise ValueError(f"dtype must be float16, bfloat16 or int8, got {dtype}")
        if page_size not in PAGE_SIZES:
            raise ValueError(f"page_size must be one of {PAGE_SIZES}, got {page_size}")
        if group_size not in (32, 64, 128):
            raise ValueError(f"group_size must be 32, 64 or 128, got {group_size}")
        if num_pages is not None and num_pages < 1:
            raise ValueError(f"num_pages must be positive, got {num_pages}")
        if window is not None and window < 1:
            raise ValueError(f"window must be at least 1, got {window}")
        if sinks < 0:
            raise ValueError(f"sinks must be >= 0, got {sinks}")
        if decode_attn_impl not in ("hip_fused", "triton_fused"):
            raise ValueError(f"decode_attn_impl={decode_attn_impl!r}: a paged cache decodes with its HIP kernels "
                             "('hip_fused', or the reference's name 'triton_fused')")
        if budget is None:
            if recent is not None or slack is not None:
                raise ValueError("recent and slack belong to a budget")
        else:
            if window is not None:
                raise ValueError("window and budget bound the cache in two ways: give one of them")
            recent = budget // 4 if recent is None else recent
            slack = page_size if slack is None else slack
            if budget < 1 or recent < 0 or sinks + recent > budget or slack < 0:
                raise ValueError(f"budget must be positive and hold sinks + recent, slack >= 0: got budget {budget}, sinks "
                                 f"{sinks}, recent {recent}, slack {slack}")
        self.dtype, self.page_size, self.num_pages, self.group_size = dtype, page_size, num_pages, group_size
        self.window, self.sinks, self.budget, self.recent, self.slack = window, sinks, budget, recent, slack
        self.inv_tau, self.use_attn_temperature = inv_tau, use_attn_temperature
        self._drop()

    def _drop(self) -> None:
        n = self.num_layers
        self._pools: List[Optional[tuple]] = [None] * n       # (k, v, k_scale, v_scale) of each layer
        self._weights: List[Optional[Tensor]] = [None] * n
        self._batch = self._heads = 0
        self._total = 0                                        # pages of a pool
        self._forget()

    def _forget(self) -> None:
        n = self.num_layers
        self._held: List[List[int]] = [[] for _ in range(n)]   # tokens held of each sequence, per layer
        self._seen: List[List[int]] = [[] for _ in range(n)]   # tokens appended to each sequence, per layer
        self._rows: List[List[int]] = [[] for _ in range(self._batch)]  # pages of each sequence, -1: given back
        self._gone: dict = {}                                  # sequence: its pages before this, but the sinks', are given back,
        self._holes: dict = {}                                 # and some before this
        self._lost: List[dict] = [{} for _ in range(n)]        # the same of a layer's tokens, whoever has taken pages there since
        self._lead: Optional[int] = None                       # the layer that a step begins with
        self._free: List[int] = list(range(self._total - 1, -1, -1))
        self._table: Optional[Tensor] = None
        self._lens: dict = {}                                  # device copies of token counts, by value
        self._layer_seq_lens = [0] * n
        self._seq_len = 0

    # ---------------------------------------------------------------- bookkeeping (host)

    def _check(self, layer_id: int, k: Tensor, v: Tensor) -> None:
        if not 0 <= layer_id < self.num_layers:
            raise ValueError(f"layer_id {layer_id} out of range")
        if k.ndim != 4 or k.shape[3] != HEAD_DIM or k.shape != v.shape:
            raise ValueError(f"k and v must be [B, Hkv, S, {HEAD_DIM}] alike, got {tuple(k.shape)} / {tuple(v.shape)}")
        if not k.is_cuda:
            raise ValueError("the paged engine needs GPU (ROCm) tensors")
        if k.dtype != v.dtype or k.dtype not in (torch.float16, torch.bfloat16) or self.dtype not in (torch.int8, k.dtype):
            raise ValueError(f"K and V must be fp16 or bf16 and of the pages' type {self.dtype}, got {k.dtype} / {v.dtype}")
        if self._batch and (k.shape[0] != self._batch or k.shape[1] != self._heads):
            raise ValueError(f"the cache holds {self._batch} sequences of {self._heads} heads, got {k.shape[0]} of {k.shape[1]}")

    def _counts(self, counts: Optional[Sequence[int]], batch: int, seq: int) -> List[int]:
        if counts is None:
            return [seq] * batch
        counts = [int(c) for c in counts]
        if len(counts) != batch or any(c < 0 or c > seq for c in counts):
            raise ValueError(f"lens must give {batch} token counts in [0, {seq}], got {counts}")
        return counts

    def _device_ints(self, values: List[int], device) -> Tensor:
        """int32 [B] on the device; layers ask for the same values, so the last few are kept."""
        key = tuple(values)
        t = self._lens.get(key)
        if t is None:
            if len(self._lens) >= 8:
                self._lens.pop(next(iter(self._lens)))
            t = self._lens[key] = torch.tensor(values, dtype=torch.int32, device=device)
        return t

    def _give_back(self, counts: Optional[List[int]] = None) -> None:
        """Returns pages that no layer in use needs: behind the longest held length, or out of the window's sight, that of
        the next token where a sequence takes one (`counts`; None: all do), else of its last.  (A layer that begins later
        takes pages of its own.)"""
        begun = [h for h in self._held if h]
        if not begun:
            return
        least = most = begun[0]
        if any(h != least for h in begun):
            least, most = [min(x) for x in zip(*begun)], [max(x) for x in zip(*begun)]
        ps, changed = self.page_size, False
        for row, hi in zip(self._rows, most):
            while len(row) > -(-hi // ps):
                page = row.pop()
                changed = True
                if page >= 0:
                    self._free.append(page)
        if self.window is not None:
            keep = -(-self.sinks // ps)
            for b, (row, lo) in enumerate(zip(self._rows, least)):
                # the next token's query stands at lo or later and sees no token before lo + 1 - window but the sinks
                end = max(lo + (1 if counts is None or counts[b] else 0) - self.window, 0) // ps
                for i in range(max(self._gone.get(b, 0), keep), end):
                    if row[i] >= 0:
                        self._free.append(row[i])
                        row[i] = -1
                        changed = True
                if end > max(self._gone.get(b, 0), keep):
                    self._gone[b] = end
                    self._holes[b] = max(self._holes.get(b, 0), end)
                    for held, lost in zip(self._held, self._lost):
                        if held:
                            lost[b] = max(lost.get(b, 0), end)
        if changed:
            self._table = None

    def _needs(self, held: List[int], target: List[int]) -> List[Tuple[int, int]]:
        """(sequence, place) of the pages that tokens held .. target - 1 lack: at the end of a row, and where a layer begins
        in pages that were given back."""
        ps, out = self.page_size, []
        for b, (row, h, t) in enumerate(zip(self._rows, held, target)):
            if h // ps < self._holes.get(b, 0):
                out += [(b, i) for i in range(h // ps, min(len(row), -(-t // ps))) if row[i] < 0]
            out += [(b, i) for i in range(len(row), -(-t // ps))]
        return out

    def _reserve(self, layer_id: int, counts: List[int], device) -> None:
        """Pages for `counts` more tokens of each sequence."""
        held = self._held[layer_id] or [0] * self._batch
        target = [h + c for h, c in zip(held, counts)]
        if self.max_seq_len is not None:
            keep, lost = -(-self.sinks // self.page_size), self._lost[layer_id]
            most = max((t - max(lost.get(b, 0) - keep, 0) * self.page_size for b, t in enumerate(target)), default=0)
            if most > self.max_seq_len:
                raise ValueError(f"target_len {most} exceeds max_seq_len {self.max_seq_len} for layer {layer_id}")
        need = self._needs(held, target)
        if len(need) > len(self._free):
            self._give_back(counts)  # short of pages: all that the new tokens do not see
            need = self._needs(held, target)
        short = len(need) - len(self._free)
        if short > 0:
            if self.num_pages is not None:
                raise RuntimeError(f"out of pages: {len(need)} needed, {len(self._free)} of {self.num_pages} free")
            self._grow(self._total + max(short, self._total))
        for b, i in need:
            row = self._rows[b]
            if i == len(row):
                row.append(self._free.pop())
            else:
                row[i] = self._free.pop()
                self._gone[b] = min(self._gone.get(b, 0), i)
        if need:
            self._table = None

    def _grow(self, total: int) -> None:
        for i, pool in enumerate(self._pools):
            if pool is not None:
                self._pools[i] = tuple(None if x is None else torch.cat([x, x.new_empty((total - self._total, *x.shape[1:]))])
                                       for x in pool)
        self._free = list(range(total - 1, self._total - 1, -1)) + self._free
        self._total = total

    def _pool(self, layer_id: int, device) -> tuple:
        pool = self._pools[layer_id]
        if pool is None:
            shape = (self._total, self._heads, self.page_size)
            rows = [torch.empty((*shape, HEAD_DIM), dtype=self.dtype, device=device) for _ in range(2)]
            scales = [torch.empty((*shape, HEAD_DIM // self.group_size), dtype=torch.float16, device=device)
                      if self.dtype == torch.int8 else None for _ in range(2)]
            pool = self._pools[layer_id] = (*rows, *scales)
        return pool

    def _block_table(self, device) -> Tensor:
        if self._table is None:
            cols = max([len(r) for r in self._rows] + [1])
            self._table = torch.tensor([r + [-1] * (cols - len(r)) for r in self._rows], dtype=torch.int32, device=device)
        return self._table

    def _layer_weights(self, layer_id: int, device) -> Optional[Tensor]:
        if self.budget is None:
            return None
        cap = self._block_table(device).shape[1] * self.page_size
        w = self._weights[layer_id]
        if w is None or w.shape[0] != self._batch or w.shape[2] < cap:
            grown = torch.zeros((self._batch, self._heads, max(cap, 2 * (0 if w is None else w.shape[2]))), device=device)
            if w is not None and w.shape[0] == self._batch:
                grown[:, :, : w.shape[2]] = w
            w = self._weights[layer_id] = grown
        return w

    # A call that is refused leaves the cache as it was: what an append changed is put back (slots behind the tokens
    # held may hold anything, and a first call that did not come about fixes no batch).

    def _state(self, layer_id: int) -> tuple:
        return self._held[layer_id], self._seen[layer_id], self._batch

    def _put_back(self, layer_id: int, state: tuple) -> None:
        self._held[layer_id], self._seen[layer_id], batch = state
        if not batch:
            self._drop()
            return
        self._layer_seq_lens[layer_id] = max(self._seen[layer_id], default=0)
        self._seq_len = max(self._layer_seq_lens)

    # ---------------------------------------------------------------- the cache

    def append(self, layer_id: int, k: Tensor, v: Tensor, lens: Optional[Sequence[int]] = None) -> None:
        """Appends k, v [B, Hkv, S, 128]; ``lens``: the real tokens of each sequence of a padded batch."""
        self._check(layer_id, k, v)
        batch, heads, seq, _ = k.shape
        counts = self._counts(lens, batch, seq)
        if not batch:
            return
        before = self._state(layer_id)
        try:
            self._append(layer_id, k, v, counts, lens is not None)
        except BaseException:
            self._put_back(layer_id, before)
            raise

    def _append(self, layer_id: int, k: Tensor, v: Tensor, counts: List[int], ragged: bool) -> None:
        batch, heads = k.shape[:2]
        if not self._batch:
            self._batch, self._heads = batch, heads
            self._rows = [[] for _ in range(batch)]
            if self.num_pages is not None:
                self._total = self.num_pages
                self._free = list(range(self._total - 1, -1, -1))
        if layer_id == self._lead and (self.window is not None or self.budget is not None):
            self._give_back([0] * batch)  # the call may yet be refused: what the last token sees stays
        self._reserve(layer_id, counts, k.device)
        held = self._held[layer_id] or [0] * batch
        kp, vp, ks, vs = self._pool(layer_id, k.device)
        table = self._block_table(k.device)
        append_paged(k, v, kp, vp, table, self._device_ints(held, k.device),
                     self._device_ints(counts, k.device) if ragged else None, k_scale=ks, v_scale=vs)
        if self._lead is None:
            self._lead = layer_id
        self._held[layer_id] = [h + c for h, c in zip(held, counts)]
        self._seen[layer_id] = [s + c for s, c in zip(self._seen[layer_id] or [0] * batch, counts)]
        self._layer_seq_lens[layer_id] = max(self._seen[layer_id], default=0)
        self._seq_len = max(self._layer_seq_lens)

    def get_seq_lens(self, layer_id: int = 0) -> List[int]:
        """Token slots of each sequence, those of pages given back among them (``get_seq_len`` counts all that the
        longest was given, the position of its next token)."""
        return list(self._held[layer_id])

    def get_paged_tensors(self, layer_id: int):
        """(k_pages, v_pages, k_scale, v_scale, block_table, lens) as the operators take them: the pools themselves, the
        table and the lengths as copies of the caller's own."""
        *pool, table, lens = self._tensors(layer_id)
        return (*pool, table.clone(), lens.clone())

    def _tensors(self, layer_id: int) -> tuple:
        """get_paged_tensors with the engine's own table and lengths, which other layers and calls share."""
        if not 0 <= layer_id < self.num_layers or not self._held[layer_id]:
            raise ValueError(f"Layer {layer_id} cache is empty")
        pool = self._pools[layer_id]
        device = pool[0].device
        return (*pool, self._block_table(device), self._device_ints(self._held[layer_id], device))

    def get_kv(self, layer_id: int) -> Tuple[Tensor, Tensor]:
        """Dense K, V [B, Hkv, n, 128] of what is held (INT8: fp16 values), n the longest sequence's tokens; slots
        past a shorter sequence's end, and those of pages given back to the pool, are zero."""
        *_, table, _ = self._tensors(layer_id)
        held = self._held[layer_id]
        table = table[:, : -(-max(held, default=0) // self.page_size)]
        if self._lost[layer_id]:  # a layer that began later may have pages where this one gave its own back
            place = torch.arange(table.shape[1], device=table.device)
            lost = self._device_ints([self._lost[layer_id].get(b, 0) for b in range(self._batch)], table.device)
            table = table.masked_fill((place < lost.unsqueeze(1)) & (place >= -(-self.sinks // self.page_size)), -1)
        return self._dense(layer_id, table, held)

    def _dense(self, layer_id: int, table: Tensor, lens: List[int]) -> Tuple[Tensor, Tensor]:
        """Dense K, V [B, Hkv, max(lens), 128] of the pages that a table [B, cols] names, sequence b's first lens[b] slots; the
        others, and pages that are not there, are zero."""
        t = table.long()
        slot = torch.arange(t.shape[1] * self.page_size, device=t.device)
        there = (t >= 0).repeat_interleave(self.page_size, dim=1) & (slot < self._device_ints(lens, t.device).unsqueeze(1))

        def dense(pages, scale):
            x = pages[t.clamp(min=0)]
            if scale is not None:
                g = scale[t.clamp(min=0)].float().unsqueeze(-1)
                x = (x.float().unflatten(-1, (-1, self.group_size)) * g).flatten(-2).half()
            x = x.permute(0, 2, 1, 3, 4).flatten(2, 3)
            return x.masked_fill(~there[:, None, :, None], 0.0)[:, :, : max(lens, default=0)]

        kp, vp, ks, vs = self._pools[layer_id]
        return dense(kp, ks), dense(vp, vs)

    # ---------------------------------------------------------------- attention

    def _attend_one(self, layer_id: int, q: Tensor, sm_scale: Optional[float], tau: Optional[Tensor],
                    weights: Optional[Tensor], held: Optional[List[int]] = None) -> Tensor:
        kp, vp, ks, vs, table, lens = self._tensors(layer_id)
        if held is not None:
            lens = self._device_ints(held, q.device)
        return decode_attn_paged(q, kp, vp, table, lens, sm_scale, k_scale=ks, v_scale=vs, inv_tau=tau, window=self.window,
                                 sinks=self.sinks, weights=weights)

    def decode_attn(self, layer_id: int, q: Tensor, sm_scale: Optional[float] = None) -> Tensor:
        """Attention of q [B, Hq, 128] over the layer's cache as it is, with the engine's ``inv_tau``."""
        if self.window is not None and 0 <= layer_id < self.num_layers:
            for b, end in self._lost[layer_id].items():  # another layer's next token may have come already
                if end * self.page_size > max(self._held[layer_id][b] - self.window, 0):
                    raise RuntimeError(f"sequence {b} sees tokens whose pages were given back for its next one: append that first")
        tau = self.inv_tau[layer_id] if self.use_attn_temperature and self.inv_tau is not None else None
        return self._attend_one(layer_id, q, sm_scale, tau, None)

    def append_decode_attn(self, layer_id: int, q: Tensor, k: Tensor, v: Tensor, sm_scale: Optional[float] = None,
                           inv_tau: Optional[Tensor] = None) -> Tensor:
        """The decode step: appends one token a sequence, attends, and with a budget accumulates the weights and
        evicts where a sequence has grown ``slack`` over it.  q [B, Hq, 128], fp16 or bf16 whatever the pages (float pages
        attend, and return, in their own type); k, v [B, Hkv, 1, 128] as ``append`` takes them; ``inv_tau`` as given
        (the hook passes the engine's)."""
        if k.ndim != 4 or k.shape[2] != 1:
            raise ValueError(f"a decode step appends one token, got k {tuple(k.shape)}")
        if q.ndim != 3 or q.shape[0] != k.shape[0] or q.shape[1] % max(k.shape[1], 1):
            raise ValueError(f"q must be [B, Hq, {HEAD_DIM}] for k {tuple(k.shape)}, got {tuple(q.shape)}")
        # refused before anything is appended
        if q.shape[1] > 16 * k.shape[1]:
            raise NotImplementedError(f"more than 16 query heads a KV head: {q.shape[1]} / {k.shape[1]}")
        if q.shape[2] != HEAD_DIM or q.shape[1] == 0 or q.device != k.device or \
                q.dtype not in (torch.float16, torch.bfloat16):
            raise ValueError(f"q must be fp16 or bf16 [B, Hq, {HEAD_DIM}] on {k.device}, got {q.dtype} {tuple(q.shape)} on {q.device}")
        if self.dtype != torch.int8:  # q alone: what is stored has the pages' type already, or append refuses it
            q = q.to(self.dtype)
        before = self._state(layer_id)
        self.append(layer_id, k, v)
        try:
            out = self._attend_one(layer_id, q, sm_scale, inv_tau, self._layer_weights(layer_id, k.device))
        except BaseException:
            self._put_back(layer_id, before)
            raise
        self._evict(layer_id, self.slack)
        return out

    def prefill_attn(self, layer_id: int, q: Tensor, k: Tensor, v: Tensor, sm_scale: Optional[float] = None,
                     inv_tau: Optional[Tensor] = None, lens: Optional[Sequence[int]] = None) -> Tensor:
        """A prompt, or the next chunk of one: appends k, v [B, Hkv, S, 128] and returns the causal attention of q [B,
        Hq, S, 128] over what was held and the new tokens (``lens``: the real ones of each sequence of a padded
        batch).  The new tokens are attended as given, those of earlier calls as the cache holds them.  With a
        budget each sequence's last query begins the accumulated weights, and longer ones are cut down at once."""
        if q.ndim != 4 or k.ndim != 4 or q.shape[0] != k.shape[0] or q.shape[2] != k.shape[2]:
            raise ValueError(f"q must be [B, Hq, S, {HEAD_DIM}] for k {tuple(k.shape)}, got {tuple(q.shape)}")
        self._check(layer_id, k, v)
        batch, _, seq, _ = k.shape
        counts = self._counts(lens, batch, seq)
        held = list(self._held[layer_id]) or [0] * batch
        kk, vv = k, v
        if any(held):
            kk, vv, held = self._with_past(layer_id, k, v, held, counts)
        ragged = lens is not None or len(set(held)) > 1
        out = prefill_attn_window(
            q, kk, vv, sm_scale, window=self.window, sinks=self.sinks, inv_tau=inv_tau,
            q_lens=self._device_ints(counts, k.device) if ragged else None,
            kv_lens=self._device_ints([h + c for h, c in zip(held, counts)], k.device) if ragged else None)
        before = self._state(layer_id)
        self.append(layer_id, k, v, lens)
        if self.budget is not None and batch and seq:
            try:
                last = self._device_ints([max(c - 1, 0) for c in counts], k.device).long()
                ql = q.gather(2, last.view(-1, 1, 1, 1).expand(-1, q.shape[1], 1, HEAD_DIM)).squeeze(2)
                self._attend_one(layer_id, ql, sm_scale, inv_tau, self._layer_weights(layer_id, k.device),
                                 [h if c else 0 for h, c in zip(self._held[layer_id], counts)])
            except BaseException:
                self._put_back(layer_id, before)
                raise
            self._evict(layer_id, 0)
        return out

    def _with_past(self, layer_id: int, k: Tensor, v: Tensor, held: List[int],
                   counts: List[int]) -> Tuple[Tensor, Tensor, List[int]]:
        """What each sequence holds, then its new tokens, dense [B, Hkv, max, 128], and how many of the first there are.

        Through a window that is the sinks' pages and those that the first new token sees: tokens between them are seen
        by none of the queries, and those behind them lie as far from the queries as they did, so that the same window
        and sinks hold."""
        table, ps = self._block_table(k.device), self.page_size
        if self.window is not None:
            keep = -(-self.sinks // ps)
            left_out = [max(max(h + 1 - self.window, 0) // ps - keep, 0) for h in held]
            held = [h - n * ps for h, n in zip(held, left_out)]
            place = torch.arange(-(-max(held) // ps), device=k.device)
            place = place + (place >= keep) * self._device_ints(left_out, k.device).unsqueeze(1)
            table = table.gather(1, place.clamp(max=table.shape[1] - 1))
        total = max(h + c for h, c in zip(held, counts))
        out = []
        for past, new in zip(self._dense(layer_id, table[:, : -(-max(held) // ps)], held), (k, v)):
            x = new.new_zeros((new.shape[0], new.shape[1], total, HEAD_DIM))
            if len(set(held)) == 1 and len(set(counts)) == 1:
                x[:, :, : held[0]] = past.to(new.dtype)
                x[:, :, held[0] :] = new[:, :, : counts[0]]
            else:
                for b, (h, c) in enumerate(zip(held, counts)):
                    x[b, :, :h] = past[b, :, :h].to(new.dtype)
                    x[b, :, h : h + c] = new[b, :, :c]
            out.append(x)
        return out[0], out[1], held

    def _evict(self, layer_id: int, slack: int) -> None:
        if self.budget is None:
            return
        held = self._held[layer_id]
        if max(held, default=0) <= self.budget + slack:
            return
        kp, vp, ks, vs, table, lens = self._tensors(layer_id)
        w = self._layer_weights(layer_id, kp.device)
        _, _, self._weights[layer_id] = evict_paged(kp, vp, table, lens, w, self.budget, sinks=self.sinks, recent=self.recent,
                                                    k_scale=ks, v_scale=vs)
        self._held[layer_id] = [min(h, self.budget) for h in held]

    # ---------------------------------------------------------------- the rest of an engine

    def clear(self) -> None:
        """Forgets every sequence; the pools stay, for a batch of the same size."""
        self._forget()
        for w in self._weights:
            if w is not None:
                w.zero_()

    def release(self) -> None:
        """Frees the pools; the next append may bring another batch size."""
        self._drop()

    def get_memory_mb(self) -> float:
        tensors = [x for pool in self._pools if pool is not None for x in pool if x is not None]
        tensors += [w for w in self._weights if w is not None]
        return sum(x.numel() * x.element_size() for x in tensors) / 2 ** 20

    def to_tuple(self) -> Tuple[Tuple[Tensor, Tensor], ...]:
        return tuple(self.get_kv(i) for i in range(self.num_layers))

    def __repr__(self) -> str:
        kind = {torch.float16: "fp16", torch.bfloat16: "bf16", torch.int8: "int8"}[self.dtype]
        return (f"PagedKVCache(num_layers={self.num_layers}, {kind}, page_size={self.page_size}, seq_len={self._seq_len}, "
                f"memory={self.get_memory_mb():.2f}MB)")
