"""PagedKVCache.fork and compact on the CPU, the operators stood in for by torch: what every sequence holds after any run of
appends, forks, decode steps and compactions, that no page is written that another sequence sees, and that no page is lost."""
import random

import pytest
import torch

import llm_kvcache_quantization_amd.paged_cache as M
from test_paged_engine_cpu import tensor


class Handle:
    def __init__(self, tensors):
        self.tensors = list(tensors)


def append_paged(k, v, kp, vp, table, pos, lens=None, k_scale=None, v_scale=None):
    ps = kp.shape[2]
    for b in range(k.shape[0]):
        for i in range(k.shape[2] if lens is None else int(lens[b])):
            t = int(pos[b]) + i
            kp[int(table[b, t // ps]), :, t % ps] = torch.Tensor(k[b, :, i].float()).to(kp.dtype)
            vp[int(table[b, t // ps]), :, t % ps] = torch.Tensor(v[b, :, i].float()).to(vp.dtype)


def copy_paged(pools, src, dst, lens=None, into=None):
    pools = pools.tensors if isinstance(pools, Handle) else list(pools)
    to = pools if into is None else into.tensors
    src, dst = [int(x) for x in src], [int(x) for x in dst]
    assert len(set(dst)) == len(dst) and (into is not None or not set(dst) & set(src))
    for x, y in zip(pools, to):
        for i, (s, d) in enumerate(zip(src, dst)):
            n = x.shape[2] if lens is None else int(lens[i])
            y[d, :, :n] = x[s, :, :n]


class Prefix:
    def __init__(self, sizes, lens, q_heads, heads, device):
        self.sizes, self.lens = list(sizes), list(lens)


@pytest.fixture
def calls(monkeypatch):
    log = []

    def note(name, fn):
        def run(*args, **kw):
            log.append((name, args, kw))
            return fn(*args, **kw)
        monkeypatch.setattr(M, name, run)

    note("append_paged", append_paged)
    note("copy_paged", copy_paged)
    note("decode_attn_paged", lambda q, *a, **kw: q.clone())
    note("decode_attn_shared", lambda q, *a, **kw: q.clone())
    note("prefill_attn_window", lambda q, *a, **kw: q.clone())
    monkeypatch.setattr(M, "PagePools", Handle)
    monkeypatch.setattr(M, "SharedPrefix", Prefix)
    return log


def make(layers=2, **kw):
    return M.PagedKVCache(layers, device="cpu", **dict(dict(page_size=16), **kw))


class Model:
    """What each sequence holds: a list of tokens' values per layer."""

    def __init__(self, cache, layers=2, heads=1):
        self.c, self.layers, self.heads, self.rows, self.next = cache, layers, heads, None, 0

    def append(self, counts, decode=False):
        seq = max(counts)
        batch = len(counts)
        if self.rows is None:
            self.rows = [[[] for _ in range(self.layers)] for _ in range(batch)]
        for layer in range(self.layers):
            x = torch.zeros(batch, self.heads, seq, 128)
            for b, n in enumerate(counts):
                for i in range(n):
                    self.next += 1
                    x[b, :, i] = self.next % 2039  # whole numbers that fp16 holds
                    self.rows[b][layer].append(self.next % 2039)
            from test_paged_engine_cpu import OnGpu
            k = x.half().as_subclass(OnGpu)
            if decode:
                self.c.append_decode_attn(layer, tensor(batch, 2 * self.heads, 128), k, k)
            else:
                self.c.append(layer, k, k, counts)

    def fork(self, parents):
        self.rows = [[list(t) for t in self.rows[p]] for p in parents]
        self.c.fork(parents)

    def check(self):
        c = self.c
        for layer in range(self.layers):
            pool, table = c._pools[layer][0], c._block_table("cpu")
            assert c.get_seq_lens(layer) == [len(r[layer]) for r in self.rows]
            for b, row in enumerate(self.rows):
                got = [float(pool[int(table[b, t // 16]), 0, t % 16, 5]) for t in range(len(row[layer]))]
                assert got == [float(x) for x in row[layer]], (layer, b)
        pages = [p for r in c._rows for p in r if p >= 0]
        count = {p: pages.count(p) for p in pages}
        assert {p: n for p, n in count.items() if n > 1} == c._refs
        assert sorted(c._free + list(count)) == list(range(c._total))


def test_fork_shares_pages_and_copies_the_last_when_it_is_written(calls):
    c = make()
    m = Model(c)
    m.append([40])
    m.fork([0, 0, 0])
    m.check()
    assert len(set(map(tuple, c._rows))) == 1 and c.get_seq_len() == 40 and not [x for x in calls if x[0] == "copy_paged"]
    m.append([1, 1, 1], decode=True)
    m.check()
    copies = [x for x in calls if x[0] == "copy_paged"]
    assert len(copies) == 1 and len(copies[0][1][1]) == 2 and copies[0][1][3].tolist() == [8, 8]  # all layers, once
    assert [r[:2] for r in c._rows] == [c._rows[0][:2]] * 3 and len({r[2] for r in c._rows}) == 3
    m.append([1, 1, 1], decode=True)
    assert len([x for x in calls if x[0] == "copy_paged"]) == 1
    m.check()


def test_full_pages_need_no_copy(calls):
    c = make()
    m = Model(c)
    m.append([32])
    m.fork([0, 0])
    m.append([1, 1])
    m.check()
    assert not [x for x in calls if x[0] == "copy_paged"]


def test_ending_and_reordering(calls):
    c = make()
    m = Model(c)
    m.append([20, 5, 33])
    used = c._total - len(c._free)
    m.fork([2, 0])
    m.check()
    assert c._total - len(c._free) == used - 1 and c.get_seq_lens() == [33, 20] and c.get_seq_len() == 33
    m.fork([1, 0])
    m.append([3, 1])
    m.check()
    m.fork([0])
    assert c.get_seq_len() == 23
    m.check()


@pytest.mark.parametrize("seed", range(24))
def test_any_run_of_calls(calls, monkeypatch, seed):
    """Random appends, steps, forks (beams: some twice, some ended) and compactions; tables laid out or changed."""
    monkeypatch.setattr(M, "_PATCHED", 1 if seed % 2 else 1 << 30)
    rng = random.Random(seed)
    c = make()
    m = Model(c)
    m.append([rng.randint(1, 50) for _ in range(rng.randint(1, 3))])
    m.check()
    for _ in range(25):
        n = len(m.rows)
        what = rng.choice(("append", "step", "step", "fork", "fork", "compact"))
        if what == "append":
            m.append([rng.randint(0, 20) for _ in range(n - 1)] + [rng.randint(1, 20)])
        elif what == "step":
            m.append([1] * n, decode=True)
        elif what == "fork":
            m.fork([rng.randrange(n) for _ in range(rng.randint(1, 5))])
        else:
            c.compact()
            assert c._total == len({p for r in c._rows for p in r})
        m.check()


def test_fixed_pools_refuse_and_stay(calls):
    c = make(num_pages=4)
    m = Model(c)
    m.append([40])
    m.fork([0, 0, 0])
    rows, free = [list(r) for r in c._rows], list(c._free)
    from test_paged_engine_cpu import OnGpu
    k = torch.zeros(3, 1, 1, 128).half().as_subclass(OnGpu)
    with pytest.raises(RuntimeError, match="out of pages: 2 needed, 1"):
        c.append(0, k, k)
    assert c._rows == rows and c._free == free
    m.check()
    m.fork([0, 1])
    m.append([1, 1])
    m.check()
    c.compact()  # keeps a fixed pool
    assert c._total == 4


def test_budget_copies_all_pages(calls, monkeypatch):
    monkeypatch.setattr(M, "evict_paged", lambda k, v, table, lens, w, budget, **kw: (lens, None, w))
    c = make(budget=100)
    m = Model(c)
    m.append([40])
    for layer in range(2):
        c._layer_weights(layer, "cpu").copy_(torch.arange(48.0))
    m.fork([0, 0])
    m.append([1, 1], decode=True)
    m.check()
    assert not c._refs and len({p for r in c._rows for p in r}) == 6
    assert all(w.shape[0] == 2 and torch.equal(w[0], w[1]) and float(w[0, 0, 7]) == 7 for w in c._weights)
    assert not [x for x in calls if x[0] == "decode_attn_shared"]


def test_window_gives_back_each_sequences_pages(calls):
    c = make(window=20)
    m = Model(c)
    m.append([64])
    m.fork([0, 0])
    for _ in range(20):
        m.append([1, 1], decode=True)
    for row in c._rows:
        assert row[:2] == [-1, -1]
    pages = [p for r in c._rows for p in r if p >= 0]
    assert sorted(c._free + sorted(set(pages))) == list(range(c._total))
    assert {p: pages.count(p) for p in pages if pages.count(p) > 1} == c._refs
    assert not [x for x in calls if x[0] == "decode_attn_shared"]


def test_a_layer_that_begins_after_a_fork_writes_to_pages_of_its_own(calls):
    c = make()
    m = Model(c, layers=1)
    m.append([40])
    m.fork([0, 0])
    from test_paged_engine_cpu import OnGpu
    k = torch.arange(2.0).view(2, 1, 1, 1).expand(2, 1, 20, 128).half().as_subclass(OnGpu)
    c.append(1, k, k)
    m.check()
    table = c._block_table("cpu")
    assert [float(c._pools[1][0][int(table[b, 1]), 0, 2, 0]) for b in range(2)] == [0.0, 1.0]


def test_attention_reads_a_shared_prefix_once(calls, monkeypatch):
    monkeypatch.setattr(M, "_MIN_SAVED", 32)
    c = make()
    m = Model(c)
    m.append([70, 20])
    m.fork([0, 0, 0, 1, 1])
    del calls[:]
    m.append([1] * 5, decode=True)
    shared = [x for x in calls if x[0] == "decode_attn_shared"]
    assert len(shared) == 2 and shared[0][1][5] is shared[1][1][5]
    assert shared[0][1][5].sizes == [3, 2] and shared[0][1][5].lens == [64, 16]
    m.append([1] * 5, decode=True)
    assert [x for x in calls if x[0] == "decode_attn_shared"][-1][1][5] is shared[0][1][5]  # kept while the groups last
    m.fork([0, 3, 1])
    m.append([1] * 3, decode=True)
    assert calls[-1][0] == "decode_attn_paged"  # no neighbours share any more
    m.fork([0, 2, 1])
    m.append([1] * 3, decode=True)
    assert calls[-1][0] == "decode_attn_shared" and calls[-1][1][5].sizes == [2, 1]
    monkeypatch.setattr(M, "_MIN_SAVED", 65)
    m.append([1] * 3, decode=True)
    assert calls[-1][0] == "decode_attn_paged"  # 64 tokens of one head are too few


@pytest.mark.parametrize("dtype,last", [(torch.float16, 104), (torch.bfloat16, 104), (torch.int8, 14)])
def test_long_tails_are_read_by_themselves(calls, monkeypatch, dtype, last):
    """Four sequences share 64 tokens: each by itself reads 4 (64 + n), the shared attention 64 + 4 n; `last` is the greatest n
    at which the former is 1.4 times as much, or 2.6 times for INT8 pages."""
    monkeypatch.setattr(M, "_MIN_SAVED", 1)
    times = {torch.int8: 2.6}.get(dtype, 1.4)
    assert 4 * (64 + last) >= times * (64 + 4 * last) and 4 * (65 + last) < times * (68 + 4 * last)
    c = make(layers=1, dtype=dtype)
    kv = torch.bfloat16 if dtype == torch.bfloat16 else torch.float16
    k = tensor(1, 1, 64, 128).to(kv)
    c.append(0, k, k)
    c.fork([0] * 4)
    k = tensor(4, 1, last - 1, 128).to(kv)
    c.append(0, k, k)
    k = tensor(4, 1, 1, 128).to(kv)
    for name in ("decode_attn_shared", "decode_attn_paged"):
        c.append_decode_attn(0, k[:, :, 0], k, k)
        assert calls[-1][0] == name


@pytest.mark.parametrize("rows,name", [(4096, "decode_attn_shared"), (4097, "decode_attn_paged")])
def test_more_rows_than_the_shared_attention_takes(calls, rows, name):
    c = make(layers=1)
    k = tensor(1, 1, 32, 128)
    c.append(0, k, k)
    c.fork([0] * rows)
    k = tensor(rows, 1, 1, 128)
    c.append_decode_attn(0, k[:, :, 0], k, k)
    assert calls[-1][0] == name and c.get_seq_lens(0) == [33] * rows


def test_refusals(calls):
    c = make()
    with pytest.raises(ValueError):
        c.fork([0])
    m = Model(c)
    m.append([5, 5])
    for bad in ([], [2], [-1], [0, 5]):
        with pytest.raises(ValueError):
            c.fork(bad)
    m.check()
    with pytest.raises(ValueError):  # the batch is another now
        m.c.fork([0])
        k = tensor(2, 1, 1, 128)
        c.append(0, k, k)


def test_clear_and_release_after_a_fork(calls):
    c = make()
    m = Model(c)
    m.append([40])
    m.fork([0, 0, 0])
    c.clear()
    assert not c._refs and sorted(c._free) == list(range(c._total))
    m = Model(c)
    m.append([5, 6, 7])
    m.check()
    c.clear()
    c.compact()
    assert c.get_memory_mb() == 0
    m = Model(c)
    m.append([5, 6, 7])
    m.check()
    c.release()
    m = Model(c)
    m.append([9])
    m.check()


def test_groups_that_save_most():
    a, b = list(range(10)), list(range(5)) + [20, 21, 22]
    assert M.shared_groups([a, a, b, b]) == ([2, 2], [10, 8])
    assert M.shared_groups([a, b, [0, 1, 2, 3, 4, 9], [50]]) == ([3, 1], [5, 0])
    assert M.shared_groups([a, a[:3]]) == ([2], [3])
    assert M.shared_groups([a, [9], a]) == ([1, 1, 1], [0, 0, 0])
    assert M.shared_groups([a]) == ([1], [0])
    assert M.shared_groups([[], []]) == ([1, 1], [0, 0])
    assert M.shared_groups([a[:1] + [7]] * 2 + [a] * 3) == ([2, 3], [2, 10])
