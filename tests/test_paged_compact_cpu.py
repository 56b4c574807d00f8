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
