"""PagedKVCache.compact on a GPU: what is held, and the memory that it takes."""
import pytest
import torch

from test_gpu_paged import BF16, D, DEV, F16, SM

pytestmark = pytest.mark.gpu


def _k():
    import llm_kvcache_quantization_amd as K

    return K


def randn(*shape, dtype, g):
    return torch.randn(shape, generator=g).to(dtype).to(DEV)


@pytest.mark.parametrize("dtype,pages", [(F16, F16), (BF16, BF16), (F16, torch.int8)])
def test_a_cache_that_holds_nothing(dtype, pages):
    """The sequence with tokens ends, the pools shrink to nothing: attention of nothing is zero, and the cache goes on."""
    K = _k()
    g = torch.Generator().manual_seed(1)
    c = K.PagedKVCache(2, device=DEV, dtype=pages, page_size=16)
    for layer in range(2):
        k, v = (randn(2, 2, 40, D, dtype=dtype, g=g) for _ in range(2))
        c.append(layer, k, v, lens=[40, 0])
    c.fork([1])
    c.compact()
    assert c.get_memory_mb() == 0
    for layer in range(2):
        assert c.get_kv(layer)[0].shape == (1, 2, 0, D)
        assert not c.decode_attn(layer, randn(1, 12, D, dtype=dtype, g=g), SM).any()
    c.fork([0, 0])
    for layer in range(2):
        q, k, v = (randn(2, n, 1, D, dtype=dtype, g=g) for n in (12, 2, 2))
        out = c.append_decode_attn(layer, q.squeeze(2), k, v, SM)
        want = c.get_kv(layer)[1].repeat_interleave(6, 1).squeeze(2)  # of one token: its V
        assert torch.equal(out, want.to(dtype))


@pytest.mark.parametrize("pages", [F16, torch.int8])
def test_memory(pages):
    """Most pages are held: the call needs room for one layer's new pool beside the old ones, and gives back the rest; what
    is held is the same, bit for bit."""
    K = _k()
    g = torch.Generator().manual_seed(2)
    layers, page = 6, 64
    c = K.PagedKVCache(layers, device=DEV, dtype=pages, page_size=page)
    for layer in range(layers):
        k, v = (randn(4, 4, 900, D, dtype=F16, g=g) for _ in range(2))
        c.append(layer, k, v, lens=[900, 100, 850, 700])
    c.fork([2, 0, 3, 0])
    before = [c.get_kv(layer) for layer in range(layers)]
    k = v = None
    total = c.get_memory_mb() * 2 ** 20
    used = len({p for row in c._rows for p in row})
    one = total / c._total * used / layers
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    base = torch.cuda.memory_allocated()
    c.compact()
    peak = torch.cuda.max_memory_allocated() - base
    left = torch.cuda.memory_allocated() - base
    assert c.get_memory_mb() * 2 ** 20 == pytest.approx(one * layers)
    assert peak <= one + 2 ** 20 and left <= one * layers - total + 2 ** 20, (peak, left, one)
    for layer in range(layers):
        for a, b in zip(before[layer], c.get_kv(layer)):
            assert torch.equal(a, b)
    out = c.append_decode_attn(0, *(randn(4, n, 1, D, dtype=F16, g=g).squeeze(2) if n == 12 else randn(4, n, 1, D, dtype=F16, g=g)
                                    for n in (12, 4, 4)), SM)
    assert not out.isnan().any()
