"""PagedKVCache on the CPU with its operators stood in for: what it counts, refuses and hands over."""
import pytest
import torch

import llm_kvcache_quantization_amd.paged_cache as M


class OnGpu(torch.Tensor):
    """A CPU tensor that passes for one of a GPU."""

    is_cuda = True


def tensor(*shape, dtype=torch.float16):
    return torch.randn(shape).to(dtype).as_subclass(OnGpu)


class Calls(list):
    """The operators' calls in order, as (name, args, kwargs)."""

    def named(self, name):
        return [c for c in self if c[0] == name]


@pytest.fixture
def calls(monkeypatch):
    """The operators do nothing but record; attention returns its queries, eviction its weights."""
    log = Calls()

    def stand_in(name, result):
        def fn(*args, **kw):
            log.append((name, args, kw))
            return result(*args)

        monkeypatch.setattr(M, name, fn)

    stand_in("append_paged", lambda *a: None)
    stand_in("decode_attn_paged", lambda q, *a: q.clone())
    stand_in("prefill_attn_window", lambda q, *a: q.clone())
    stand_in("evict_paged", lambda k, v, table, lens, w, budget: (lens, None, w))
    return log


def make(layers=1, **kw):
    return M.PagedKVCache(layers, device="cpu", **dict(dict(page_size=16), **kw))


def append(c, lens, layer=0, heads=2, seq=None):
    x = tensor(len(lens), heads, seq or max(lens), 128)
    c.append(layer, x, x, lens)


def test_seq_len_is_the_longest_sequences(calls):
    """Chunks in which another sequence is the longest: the next position follows the tokens a sequence was given, not
    the chunks' longest."""
    c = make(2)
    for layer in (0, 1):
        append(c, [3, 5], layer)
        assert c.get_seq_len() == 5
    append(c, [5, 3])
    assert c.get_seq_lens() == [8, 8] and c.get_seq_len() == 8
    append(c, [0, 1])
    assert c.get_seq_lens() == [8, 9] and c.get_seq_len() == 9
    assert c._layer_seq_lens == [9, 5]
    c.clear()
    assert c.get_seq_len() == 0
    append(c, [2, 1])
    assert c.get_seq_len() == 2


def test_evicted_tokens_count_as_positions(calls):
    c = make(budget=8, recent=2, slack=0)
    append(c, [20, 3])
    c._evict(0, 0)
    assert c.get_seq_lens() == [8, 3] and c.get_seq_len() == 20
    append(c, [1, 1])
    assert c.get_seq_len() == 21


def snapshot(c):
    return [list(h) for h in c._held], c.get_seq_len(), list(c._layer_seq_lens), c._batch


def refuse(monkeypatch, name, after=0):
    """From now on the operator refuses its calls, after so many that it takes."""
    taken, left = getattr(M, name), [after]

    def fn(*args, **kw):
        if left[0] == 0:
            raise ValueError("refused here")
        left[0] -= 1
        return taken(*args, **kw)

    monkeypatch.setattr(M, name, fn)


@pytest.mark.parametrize("budget", [None, 40])
@pytest.mark.parametrize("held", [0, 13])
@pytest.mark.parametrize("name", ["append_paged", "decode_attn_paged", "prefill_attn_window"])
def test_a_refused_call_changes_nothing(calls, monkeypatch, budget, held, name):
    """Whichever operator refuses a prompt, a chunk or a step, the cache is as it was, and one that has not begun takes
    another batch."""
    c = make(2, budget=budget)
    if held:
        append(c, [held, held])
        append(c, [held, held], 1)
    was = snapshot(c)
    refuse(monkeypatch, name)
    q, k = tensor(2, 4, 5, 128), tensor(2, 2, 5, 128)
    tries = {"append_paged": ("append", "prompt", "step"), "decode_attn_paged": ("step",) + (("prompt",) if budget else ()),
             "prefill_attn_window": ("prompt",)}[name]
    for t in tries:
        with pytest.raises(ValueError, match="refused here"):
            if t == "append":
                c.append(1, k, k)
            elif t == "prompt":
                c.prefill_attn(1, q, k, k, lens=[5, 2])
            else:
                c.append_decode_attn(1, q[:, :, 0], k[:, :, :1], k[:, :, :1])
        assert snapshot(c) == was, t
    monkeypatch.undo()
    monkeypatch.setattr(M, "append_paged", lambda *a, **kw: None)
    if held:
        append(c, [1, 2], 1)
        assert c.get_seq_lens(1) == [held + 1, held + 2]
    else:
        append(c, [4, 1, 7], heads=3)
        assert c.get_seq_lens() == [4, 1, 7] and c._pools[0][0].shape[1] == 3


def test_a_refused_first_call_fixes_no_batch(calls):
    """Out of pages, or of max_seq_len, or with wrong lengths: the next call may bring another batch."""
    for kw in (dict(num_pages=3), dict(max_seq_len=40)):
        c = make(**kw)
        with pytest.raises((RuntimeError, ValueError)):
            append(c, [50, 50])
        with pytest.raises(ValueError, match="token counts"):
            append(c, [50, 50], seq=3)
        assert snapshot(c) == ([[]], 0, [0], 0)
        append(c, [30], heads=4)
        assert c.get_seq_lens() == [30] and len(c._rows[0]) == 2
    c = make(num_pages=3)
    append(c, [], seq=5)  # no sequences: nothing to do, and nothing fixed
    append(c, [48])
    assert c._pools[0][0].shape[0] == 3


def test_prompts_attend_before_they_append(calls):
    c = make()
    q, k = tensor(2, 4, 5, 128), tensor(2, 2, 5, 128)
    c.prefill_attn(0, q, k, k)
    assert [x[0] for x in calls] == ["prefill_attn_window", "append_paged"]
    assert c.get_seq_lens() == [5, 5]


@pytest.mark.parametrize("pages", [torch.float16, torch.bfloat16, torch.int8])
def test_a_step_takes_the_keys_that_append_takes(calls, pages):
    """K and V of another type than the pages' are refused by a step as by an append; q is brought to float pages' type."""
    for kt in (torch.float16, torch.bfloat16, torch.float32, torch.int32):
        for qt in (torch.float16, torch.bfloat16):
            c = make(dtype=pages)
            q, k = tensor(2, 4, 128, dtype=qt), tensor(2, 2, 1, 128, dtype=kt)
            if kt == pages or pages == torch.int8 and kt in (torch.float16, torch.bfloat16):
                out = c.append_decode_attn(0, q, k, k)
                assert out.dtype == (qt if pages == torch.int8 else pages)
                stored = calls.named("append_paged")[-1][1]
                assert stored[0].dtype == stored[1].dtype == kt
            else:
                for call in (lambda: c.append_decode_attn(0, q, k, k), lambda: c.append(0, k, k),
                             lambda: c.append_decode_attn(0, q, tensor(2, 2, 1, 128, dtype=pages if pages != torch.int8 else torch.half), k)):
                    with pytest.raises(ValueError, match="pages' type"):
                        call()
                    assert snapshot(c) == ([[]], 0, [0], 0)


def test_tensors_handed_out_are_the_callers(calls):
    """Whoever counts on in the lengths, or edits the table, does not reach other layers' calls."""
    c = make(2)
    for layer in (0, 1):
        append(c, [20, 7], layer)
    *_, table, lens = c.get_paged_tensors(0)
    want = table.clone()
    lens += 1
    table.fill_(-1)
    for layer in (0, 1):
        *_, t, n = c.get_paged_tensors(layer)
        assert n.tolist() == [20, 7] and torch.equal(t, want)
    c.decode_attn(1, tensor(2, 4, 128))
    _, (_, _, _, t, n, _), _ = calls[-1]
    assert n.tolist() == [20, 7] and torch.equal(t, want)


# ---------------------------------------------------------------- pages given back


def write(k, v, kp, vp, table, pos, lens=None, **kw):
    """append_paged, token by token."""
    for b in range(k.shape[0]):
        for i in range(k.shape[2] if lens is None else int(lens[b])):
            t = int(pos[b]) + i
            page = int(table[b, t // kp.shape[2]])
            assert page >= 0, "a token is written to a page that is not there"
            kp[page, :, t % kp.shape[2]], vp[page, :, t % kp.shape[2]] = k[b, :, i], v[b, :, i]


class Filled:
    """A cache of layers whose token t of sequence b is (layer, b, t), and what each should still hold of them."""

    def __init__(self, monkeypatch, layers, **kw):
        monkeypatch.setattr(M, "append_paged", write)
        self.c = make(layers, **kw)
        self.n = [[0, 0, 0] for _ in range(layers)]

    def append(self, layer, counts):
        k = torch.zeros(3, 1, max(counts), 128)
        for b, m in enumerate(counts):
            k[b, 0, :m, 0], k[b, 0, :m, 1] = layer, b
            k[b, 0, :m, 2] = torch.arange(self.n[layer][b], self.n[layer][b] + m)
            self.n[layer][b] += m
        k = k.half().as_subclass(OnGpu)
        self.c.append(layer, k, -k, counts)
        self.check()

    def check(self):
        c = self.c
        owned = [p for r in c._rows for p in r if p >= 0]
        assert len(owned) == len(set(owned)) and sorted(owned + c._free) == list(range(c._total))
        for layer, lens in enumerate(self.n):
            if not any(lens):
                continue
            assert c.get_seq_lens(layer) == lens
            k, v = c.get_kv(layer)
            assert torch.equal(k, -v)
            for b, n in enumerate(lens):
                t = torch.arange(k.shape[2])
                there = k[b, 0, :, 0] + k[b, 0, :, 1] + k[b, 0, :, 2] != 0
                right = (t < n) & (k[b, 0, :, 0] == layer) & (k[b, 0, :, 1] == b) & (k[b, 0, :, 2] == t)
                # nothing but the tokens themselves, or zeros where pages were given back; what the next query sees is all there
                assert (right | ~there).all(), (layer, b)
                seen = (t < n) & ((t >= n + 1 - c.window) | (t < c.sinks)) if c.window else t < n
                assert right[seen].all(), (layer, b)

    def pages(self):
        return [sum(p >= 0 for p in r) for r in self.c._rows]


def test_layers_that_are_not_used_hold_no_pages_back(calls, monkeypatch):
    """Only layers 1 and 3 of 4 append: the window gives pages back all the same, and a budget's eviction does."""
    f = Filled(monkeypatch, 4, window=20, sinks=4)
    for n in ([30, 5, 40], [30, 30, 0], [1, 1, 1], [100, 1, 60], [1, 1, 1]):
        for layer in (1, 3):
            f.append(layer, n)
    # the next query sees the sinks' page and 20 tokens that end inside a page: 4 pages at most, and the last append's
    assert max(f.pages()) <= 1 + 2 + 8 and f.pages()[1] <= 5
    f.append(1, [1, 1, 1])
    f.append(3, [1, 1, 1])
    assert max(f.pages()) <= 4
    c = make(4, budget=16, recent=4, slack=0)
    for _ in range(3):
        append(c, [60, 8], 2)
        c._evict(2, 0)
    append(c, [1, 1], 2)
    assert [len(r) for r in c._rows] == [2, 2]


def test_layers_one_after_the_other(calls, monkeypatch):
    """Every chunk of a layer before the next layer's first: later layers take pages of their own where the first gave
    back, in a fixed pool too."""
    f = Filled(monkeypatch, 3, window=24, sinks=20, num_pages=40)
    chunks = ([20, 50, 3], [40, 7, 0], [33, 33, 33], [1, 0, 1], [60, 2, 64], [1, 1, 1])
    for layer in range(3):
        for n in chunks:
            f.append(layer, n)
    for _ in range(40):
        for layer in range(3):
            f.append(layer, [1, 1, 1])
    assert max(f.pages()) <= 2 + 3


@pytest.mark.parametrize("seed", range(6))
def test_pages_whatever_the_order(calls, monkeypatch, seed):
    """Chunks and steps of three layers in orders of all kinds, layers that begin late among them."""
    g = torch.Generator().manual_seed(seed)
    pick = lambda n: int(torch.randint(0, n, (1,), generator=g))  # noqa: E731
    f = Filled(monkeypatch, 3, window=(1, 5, 16, 33, 40, 7)[seed], sinks=(0, 3, 16, 17, 1, 40)[seed])
    plan = [[pick(40), pick(40), pick(40)] if pick(2) else [1, 1, 1] for _ in range(25)]
    plan = [n if max(n) else [1, 0, 0] for n in plan]
    at = [0, 0, 0]
    while min(at) < len(plan):
        layer = pick(3) if seed % 2 else min(range(3), key=lambda x: (at[x] + (5 * x if at[x] == 0 and at[0] < 8 * x else 0), x))
        if at[layer] < len(plan):
            f.append(layer, plan[at[layer]])
            at[layer] += 1


def test_a_sequence_that_takes_nothing_keeps_what_it_sees(calls, monkeypatch):
    """A row of a padded batch with no new token still sees `window` tokens: they stay, and one whose next token another
    layer has taken already, for want of pages, is refused."""
    f = Filled(monkeypatch, 2, window=16, num_pages=9)
    for layer in (0, 1):
        f.append(layer, [47, 47, 47])
    assert not f.c._free
    f.append(0, [0, 50, 1])
    # row 0 sees token 31, the last of page 1; the others' next query saw token 32 first
    assert f.c._rows[0][0] < 0 <= f.c._rows[0][1] and f.c._rows[1][1] < 0
    with pytest.raises(RuntimeError, match="sequence 1 "):
        f.c.decode_attn(1, tensor(3, 2, 128))
    f.c.decode_attn(0, tensor(3, 2, 128))
    f.append(1, [0, 50, 1])
    for layer in (0, 1):
        f.c.decode_attn(layer, tensor(3, 2, 128))


@pytest.mark.parametrize("held", range(40, 60))
def test_a_refused_step_keeps_what_the_last_token_sees(calls, monkeypatch, held):
    f = Filled(monkeypatch, 1, window=16)
    f.append(0, [held, 20, 1])
    refuse(monkeypatch, "decode_attn_paged")
    x = torch.zeros(3, 1, 1, 128).half().as_subclass(OnGpu)
    with pytest.raises(ValueError, match="refused here"):
        f.c.append_decode_attn(0, tensor(3, 2, 128), x, x)
    k, _ = f.c.get_kv(0)
    for b, n in enumerate(f.n[0]):
        t = torch.arange(max(n - 16, 0), n)
        assert torch.equal(k[b, 0, t, 2].float(), t.float()) and (k[b, 0, t, 1] == b).all()
    monkeypatch.setattr(M, "decode_attn_paged", lambda q, *a, **kw: q)
    f.c.decode_attn(0, tensor(3, 2, 128))


def test_max_seq_len_counts_what_is_held(calls, monkeypatch):
    """A stream through a window goes on past max_seq_len; a chunk that would have more than it in pages is refused."""
    f = Filled(monkeypatch, 2, window=20, sinks=4, max_seq_len=96)
    for _ in range(8):
        for layer in (0, 1):
            f.append(layer, [40, 1, 0])
    assert f.c.get_seq_lens() == [320, 8, 0]
    with pytest.raises(ValueError, match="max_seq_len"):
        append(f.c, [90, 1, 1], heads=1)
    with pytest.raises(ValueError, match="max_seq_len"):
        append(f.c, [1, 95, 1], heads=1)
    c = make(max_seq_len=96)
    append(c, [96])
    with pytest.raises(ValueError, match="max_seq_len"):
        append(c, [1])


def test_giving_back_looks_at_new_pages_only(calls):
    """A step's bookkeeping does not grow with the tokens that a window has left behind."""
    c = make(window=20)
    append(c, [2000, 1, 1])
    append(c, [1, 1, 1])
    looked = []

    class Row(list):
        def __getitem__(self, i):
            looked.append(i)
            return list.__getitem__(self, i)

    c._rows = [Row(r) for r in c._rows]
    for _ in range(64):
        append(c, [1, 1, 1])
    assert 0 < len(looked) <= 2 * 3 * (64 // 16 + 1), looked  # whether a page is there, and which


# ---------------------------------------------------------------- chunks


def attend(q, k, v, sm=None, window=None, sinks=0, q_lens=None, kv_lens=None, inv_tau=None):
    """prefill_attn_window in float64 (heads alike)."""
    out = torch.zeros(q.shape, dtype=torch.float64)
    for b in range(q.shape[0]):
        m = q.shape[2] if q_lens is None else int(q_lens[b])
        n = k.shape[2] if kv_lens is None else int(kv_lens[b])
        if not m:
            continue
        pos, key = torch.arange(n - m, n)[:, None], torch.arange(n)[None]
        vis = key <= pos
        if window:
            vis &= (key > pos - window) | (key < sinks)
        s = (q[b, :, :m].double() @ k[b, :, :n].double().transpose(1, 2)).masked_fill(~vis, -float("inf"))
        out[b, :, :m] = torch.softmax(s, -1) @ v[b, :, :n].double()
    return out.as_subclass(torch.Tensor)


@pytest.mark.parametrize("window,sinks", [(None, 0), (1, 0), (1, 3), (16, 0), (17, 16), (40, 5), (33, 40), (500, 4)])
@pytest.mark.parametrize("late", [False, True])
def test_chunks_through_a_window_touch_the_window(calls, monkeypatch, window, sinks, late):
    """What a chunk attends over is the sinks' pages, the window's and its own tokens, however much was held, and what comes
    out is the attention over all tokens."""
    monkeypatch.setattr(M, "append_paged", write)
    seen = []

    def stand_in(q, k, v, *args, **kw):
        seen.append(k.shape[2])
        return attend(q, k, v, *args, **kw)

    monkeypatch.setattr(M, "prefill_attn_window", stand_in)
    g = torch.Generator().manual_seed(1)
    c = make(2, window=window, sinks=sinks)
    plans = ([200, 200, 200], [1, 1, 1], [30, 30, 30], [33, 7, 50], [20, 0, 300], [15, 15, 15]), ([64, 64, 64], [16, 16, 16], [8, 8, 8])
    for plan in plans:
        lens = [[0, 0, 0], [0, 0, 0]]
        kept = [[[torch.zeros(1, 0, 128).half() for _ in range(2)] for _ in range(3)] for _ in range(2)]
        order = [(n, layer) for layer in (0, 1) for n in plan] if late else [(n, layer) for n in plan for layer in (0, 1)]
        for counts, layer in order:
            S = max(counts)
            q, k, v = (torch.randn(3, 1, S, 128, generator=g).mul(0.3).half().as_subclass(OnGpu) for _ in range(3))
            out = c.prefill_attn(layer, q, k, v, lens=None if len(set(counts)) == 1 else counts)
            bound = S + (max(lens[layer]) if window is None else -(-sinks // 16) * 16 + window + 15)
            assert seen[-1] <= max(bound, S), (counts, layer)
            for b, n in enumerate(counts):
                both = [torch.cat([kept[layer][b][i], torch.Tensor(x[b, :, :n]).half()], 1) for i, x in enumerate((k, v))]
                kept[layer][b] = both
                lens[layer][b] += n
                if n:
                    want = attend(q[b : b + 1, :, :n], both[0][None], both[1][None], window=window, sinks=sinks)[0]
                    assert torch.allclose(out[b, :, :n], want, rtol=0, atol=1e-12), (counts, layer, b)
        assert c.get_seq_lens(1) == lens[1]
        c.clear()


def test_a_chunk_leaves_the_cache_as_an_append_does(calls, monkeypatch):
    f = Filled(monkeypatch, 1, window=20, sinks=4)
    f.append(0, [50, 3, 0])
    x = torch.zeros(3, 1, 7, 128).half().as_subclass(OnGpu)
    for b in range(3):
        x[b, 0, :, 1], x[b, 0, :, 2] = b, torch.arange(f.n[0][b], f.n[0][b] + 7)
    f.c.prefill_attn(0, x, x, -x, lens=[7, 5, 1])
    f.n[0] = [57, 8, 1]
    f.check()


def test_a_refused_layer_does_not_lead(calls):
    """After clear() another layer than the one that was refused begins the steps: pages still go back."""
    c = make(2, window=20, max_seq_len=200, num_pages=100)  # never short of pages
    append(c, [5])
    c.clear()
    with pytest.raises(ValueError, match="max_seq_len"):
        append(c, [300])
    for _ in range(3):
        append(c, [64], 1)
    assert sum(p >= 0 for p in c._rows[0]) <= 2 + 4
