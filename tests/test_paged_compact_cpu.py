"""PagedKVCache.compact on the CPU, the operators stood in for as in test_paged_fork_cpu: what a cache does that holds nothing."""
import pytest
import torch

from test_paged_engine_cpu import tensor
from test_paged_fork_cpu import Model, calls, make  # noqa: F401


def ended(c):
    """A cache whose only sequence with tokens has ended."""
    m = Model(c)
    m.append([20, 0])
    m.fork([1])
    return m


def test_a_cache_that_holds_nothing_is_compacted_and_goes_on(calls):  # noqa: F811
    c = make()
    m = ended(c)
    c.compact()
    assert c.get_memory_mb() == 0 and c.get_seq_lens(0) == [0]
    k, v = c.get_kv(0)
    assert k.shape == v.shape == (1, 1, 0, 128)
    assert c.get_paged_tensors(0)[0].shape == (0, 1, 16, 128)
    assert torch.equal(c.decode_attn(0, tensor(1, 2, 128)), calls[-1][1][0])
    assert c.to_tuple()[1][0].shape == (1, 1, 0, 128)
    c.compact()
    m.append([18])
    m.check()
    c.compact()
    m.append([1], decode=True)
    m.check()


@pytest.mark.parametrize("n", [1, 3])
def test_forks_of_nothing(calls, n):  # noqa: F811
    c = make()
    m = ended(c)
    c.compact()
    m.fork([0] * n)
    m.append([17] * n)
    m.check()


def test_a_new_cache_has_nothing_to_compact(calls):  # noqa: F811
    c = make()
    c.compact()
    m = Model(c)
    m.append([5])
    m.check()


def owned(c):
    """Whether every pool's memory is what it holds."""
    return all(x.untyped_storage().nbytes() == x.nbytes for pool in c._pools for x in pool if x is not None)


def test_pools_shrink_one_after_another(calls, monkeypatch):  # noqa: F811
    """Never are two layers' new pools made before the first one's old pool is let go."""
    c = make(layers=3)
    m = Model(c, layers=3)
    m.append([60, 33, 20])
    m.fork([2, 0])
    old = [{x.data_ptr() for x in pool if x is not None} for pool in c._pools]
    alive = []

    def note(fn):
        def run(*args, **kw):
            alive.append(sum(x is not None and x.data_ptr() in ats for pool, ats in zip(c._pools, old) for x in pool))
            return fn(*args, **kw)
        return run

    for name in ("clone", "new_empty"):
        monkeypatch.setattr(torch.Tensor, name, note(getattr(torch.Tensor, name)))
    c.compact()
    m.check()
    assert owned(c) and c._total == 6
    assert alive and all(left <= 6 - i // 2 * 2 for i, left in enumerate(alive)), alive


@pytest.mark.parametrize("at", range(1, 5))
def test_short_of_memory(calls, monkeypatch, at):  # noqa: F811
    """An allocation that fails, whichever: what is held can be read and goes on, and the next call gives the rest back."""
    c = make()
    m = Model(c)
    m.append([60, 33, 20])
    m.fork([2, 0, 0])
    count, real, empty = [0], torch.Tensor.clone, torch.Tensor.new_empty

    def failing(fn):
        def run(*args, **kw):
            count[0] += 1
            if count[0] == at:
                raise torch.OutOfMemoryError("no memory left")
            return fn(*args, **kw)
        return run

    monkeypatch.setattr(torch.Tensor, "clone", failing(real))
    monkeypatch.setattr(torch.Tensor, "new_empty", failing(empty))
    with pytest.raises(torch.OutOfMemoryError):
        c.compact()
    m.check()
    assert c._total == 6 and not owned(c)
    c.compact()
    m.check()
    assert owned(c)
    m.append([1, 1, 1], decode=True)
    m.check()


def test_pages_that_are_low_enough_stay(calls):  # noqa: F811
    c = make()
    m = Model(c)
    m.append([60, 33, 20])
    m.fork([2, 0])
    rows, n = [list(r) for r in c._rows], 6
    c.compact()
    copies = [x for x in calls if x[0] == "copy_paged"]
    assert len(copies) == 1 and all(p >= n for p in copies[0][1][1])
    assert all(b == a or a >= n for r, s in zip(rows, c._rows) for a, b in zip(r, s))
    del calls[:]
    c.compact()
    assert not calls
    m.check()
