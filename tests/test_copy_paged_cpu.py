"""What copy_paged refuses of page numbers from the host, on the CPU with the kernel stood in for: pages written twice, and
pages written by one pair and read by another, however the same memory is named."""
import pytest
import torch

import llm_kvcache_quantization_amd.shared as S
from llm_kvcache_quantization_amd import PagePools, copy_paged
from test_paged_engine_cpu import tensor


@pytest.fixture
def launched(monkeypatch):
    log = []
    monkeypatch.setattr(S, "_call", lambda fn, block, device: log.append(block))
    return log


def pool(pages=8):
    return tensor(pages, 2, 16, 128)


def refused(launched, *args, **kw):
    with pytest.raises(ValueError, match="written"):
        copy_paged(*args, **kw)
    assert not launched


def test_a_page_is_written_once_whatever_src_is(launched):
    a, src = pool(), torch.tensor([0, 1], dtype=torch.int32)
    refused(launched, [a], src, [2, 2])
    refused(launched, [a], src, [2, 2], into=[pool()])
    refused(launched, [a], [0, 1], [2, 2], into=[pool()])
    copy_paged([a], src, [2, 3])
    copy_paged([a], [0, 0], torch.tensor([2, 3], dtype=torch.int32))
    assert len(launched) == 2


def test_the_same_tensors_as_into_are_the_same_pages(launched):
    a, b = pool(), pool()
    handle = PagePools([a, b])
    for pools in ([a, b], handle):
        for into in ([a, b], PagePools([a, b]), [b, a], [a, pool()], [pool(), a], [a.view(a.shape), pool()]):
            refused(launched, pools, [0, 1], [1, 2], into=into)
            refused(launched, pools, [3], [3], into=into)
    refused(launched, handle, [0, 1], [1, 2], into=handle)
    copy_paged([a, b], [0, 1], [2, 3], into=[a, b])
    copy_paged([a, b], [0, 1], [2, 3], into=[b, a])
    copy_paged([a, b], [0, 1], [1, 2], into=[pool(), pool()])
    assert len(launched) == 3


def test_slices_are_other_numbers_of_the_same_pages(launched):
    a = pool(10)
    refused(launched, [a], [5], [1], into=[a[4:]])  # page 5 of a
    refused(launched, [a[4:]], [1], [5], into=[a])
    refused(launched, [a[:4]], [0, 3], [2, 0], into=[a[3:]])
    refused(launched, [a[4:5]], [0], [4], into=[a])  # one page: a stride that is not used
    refused(launched, [a], [4], [0], into=[a[4:5]])
    refused(launched, [a[:1].expand(8, -1, -1, -1)], [5], [0], into=[a])  # all are page 0
    copy_paged([a], [1], [1], into=[a[4:]])
    copy_paged([a[:5]], [0, 1, 2], [2, 1, 0], into=[a[5:]])
    copy_paged([a[:1].expand(8, -1, -1, -1)], [5], [1], into=[a])
    assert len(launched) == 3


def test_pages_side_by_side_in_one_tensor_are_apart(launched):
    """K and V of a page in one tensor: pages of one between those of the other."""
    kv = tensor(8, 2, 2, 16, 128)
    k, v = kv[:, 0], kv[:, 1]
    copy_paged([k], [0, 1], [1, 2], into=[v])
    copy_paged([k, v], [0, 1], [2, 3])
    assert len(launched) == 2
    refused(launched[:0], [k, v], [0, 1], [1, 2], into=[v, k])


def test_two_tensors_of_into_that_share_pages(launched):
    a, b, c = pool(), pool(), pool(10)
    refused(launched, [a, b], [0], [1], into=[c, c])
    refused(launched, [a, b], [0, 1], [0, 4], into=[c[:6], c[4:]])
    copy_paged([a, b], [0, 1], [0, 1], into=[c[:5], c[5:]])
    copy_paged([a, a], [0], [1])  # the same onto the same
    assert len(launched) == 2


def test_numbers_are_whole_before_they_are_compared(launched):
    a = pool()
    refused(launched, [a], [0, 1], [2, 2.5])
    refused(launched, [a], [0.5, 1], [0, 3])
    copy_paged([a], iter([0, 1]), range(2, 4))
    assert len(launched) == 1
