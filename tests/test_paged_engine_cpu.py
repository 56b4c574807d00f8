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
