"""Copies of pages (copy_paged) against indexed assignment, bit for bit: what is copied, and that nothing else changes."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _k():
    import llm_kvcache_quantization_amd as K

    return K


def bits(shape, dtype, g):
    """Random bit patterns, NaN among them: a copy does not look at values."""
    item = torch.tensor([], dtype=dtype).element_size()
    return torch.randint(-128, 128, (*shape[:-1], shape[-1] * item), dtype=torch.int8, generator=g).view(dtype)


def raw(x):
    return x.contiguous().view(torch.int8)


def want(pools, into, src, dst, lens):
    out = [x.clone() for x in into]
    for x, y in zip(pools, out):
        for i, (s, d) in enumerate(zip(src, dst)):
            n = x.shape[2] if lens is None else min(max(lens[i], 0), x.shape[2])
            if 0 <= s < x.shape[0] and 0 <= d < y.shape[0]:
                y[d, :, :n] = x[s, :, :n]
    return out


def layers(n, pages, heads, page, kind, g, layout="dense"):
    if kind == "int8":
        shapes = [(torch.int8, 128)] * 2 + [(torch.float16, 4)] * 2
    elif kind == "int8_128":
        shapes = [(torch.int8, 128)] * 2 + [(torch.float16, 1)] * 2
    else:
        shapes = [(kind, 128)] * 2
    out = []
    for _ in range(n):
        for dtype, x in shapes:
            if layout == "tokens_first" and x == 128:
                t = bits((pages, page, heads, x), dtype, g).permute(0, 2, 1, 3)
            elif layout == "padded":
                t = bits((pages, heads + 1, page, x), dtype, g)[:, :heads]
            else:
                t = bits((pages, heads, page, x), dtype, g)
            out.append(t)
    return out


def cuda(ts):
    out = []
    for t in ts:
        base = torch.empty_strided(t.size(), t.stride(), dtype=t.dtype, device=DEV)
        out.append(base.copy_(t))
    return out


@pytest.mark.parametrize("kind", [torch.float16, torch.bfloat16, "int8", "int8_128"], ids=str)
@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("part", [False, True])
@pytest.mark.parametrize("other", [False, True])
def test_copies(kind, page, part, other):
    print(f"[copy] {kind} page {page} part {part} other {other}", flush=True)
    g = torch.Generator().manual_seed(page + part)
    pools = layers(3, 21, 3, page, kind, g)
    into = layers(3, 11, 3, page, kind, g) if other else pools
    order = torch.randperm(21, generator=g).tolist()
    src, dst = order[:9], torch.randperm(11, generator=g).tolist()[:9] if other else order[9:18]
    lens = [0, 1, page - 1, page, page + 5, -2, 3, page // 2, 5] if part else None
    src[4], dst[5] = 21, -1  # pages that are not there
    expect = want(pools, into, src, dst, lens)
    a = cuda(pools)
    b = cuda(into) if other else a
    dev = [torch.tensor(x, dtype=torch.int32, device=DEV) for x in (src, dst)]
    _k().copy_paged(a, *dev, None if lens is None else torch.tensor(lens, device=DEV), into=b if other else None)
    for x, y in zip(b, expect):
        assert torch.equal(raw(x.cpu()), raw(y))
    if other:
        for x, y in zip(a, pools):
            assert torch.equal(raw(x.cpu()), raw(y))


@pytest.mark.parametrize("layout", ["tokens_first", "padded"])
@pytest.mark.parametrize("kind", [torch.float16, "int8"], ids=str)
@pytest.mark.parametrize("part", [False, True])
def test_strides(layout, kind, part):
    """Pages with tokens before heads, and pages with room between them, which stays as it was."""
    g = torch.Generator().manual_seed(5)
    pools = layers(2, 9, 5, 32, kind, g, layout)
    src, dst = [0, 3, 8], [1, 2, 7]
    lens = [7, 32, 19] if part else None
    expect = want(pools, pools, src, dst, lens)
    a = cuda(pools)
    whole = [x if layout != "padded" else torch.empty(0) for x in a]
    _k().copy_paged(a, torch.tensor(src, device=DEV), torch.tensor(dst, device=DEV),
                    None if lens is None else torch.tensor(lens, device=DEV))
    for x, y in zip(a, expect):
        assert torch.equal(raw(x.cpu()), raw(y))
    # from one layout into another
    b = cuda(layers(2, 9, 5, 32, kind, g))
    expect = want(pools, [x.cpu() for x in b], src, dst, lens)
    _k().copy_paged(cuda(pools), src, dst, None if lens is None else torch.tensor(lens, device=DEV), into=b)
    for x, y in zip(b, expect):
        assert torch.equal(raw(x.cpu()), raw(y))
    assert len(whole) == len(a)


def test_many_pools_and_pairs():
    """More pools than one launch takes, and more pairs than a grid's second dimension has."""
    g = torch.Generator().manual_seed(7)
    pools = cuda(layers(70, 6, 2, 16, torch.float16, g))
    expect = want([x.cpu() for x in pools], [x.cpu() for x in pools], [0, 1], [4, 5], [9, 16])
    _k().copy_paged(_k().PagePools(pools), [0, 1], [4, 5], torch.tensor([9, 16], device=DEV))
    for x, y in zip(pools, expect):
        assert torch.equal(raw(x.cpu()), raw(y))
    n = 70001
    a = torch.arange(n, dtype=torch.int32, device=DEV).view(n, 1, 1, 1).expand(n, 1, 16, 4).contiguous()
    b = torch.zeros_like(a)
    perm = torch.randperm(n, device=DEV)
    _k().copy_paged([a], torch.arange(n, device=DEV), perm, into=[b])
    assert torch.equal(b[perm], a)


def test_pages_past_32_bits():
    """Pages behind the first 4 GiB of a pool."""
    a = torch.zeros(70000, 4, 64, 128, dtype=torch.float16, device=DEV)  # 64 KiB a page
    a[69999] = torch.randn(4, 64, 128, device=DEV).half()
    _k().copy_paged([a], [69999, 69999], [69998, 3])
    assert torch.equal(a[69998], a[69999]) and torch.equal(a[3], a[69999]) and not a[69997].any() and not a[4].any()


def test_captured_and_on_another_stream():
    K = _k()
    g = torch.Generator().manual_seed(9)
    pools = cuda(layers(4, 12, 2, 16, "int8", g))
    handle = K.PagePools(pools)
    src, dst = torch.tensor([0, 1, 2], dtype=torch.int32, device=DEV), torch.tensor([5, 6, 7], dtype=torch.int32, device=DEV)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        K.copy_paged(handle, src, dst)
    for i in range(4):
        for x in pools:
            x[:3] = (x[:3].float() + 1).to(x.dtype) if x.dtype != torch.int8 else x[:3] + 1
        src.copy_(torch.tensor([[0, 1, 2], [2, 1, 0], [1, 0, 2], [0, 2, 1]][i], dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        for x in pools:
            assert torch.equal(raw(x[5:8]), raw(x[src.long()])), i
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        K.copy_paged(handle, [0, 1], [8, 9])
    side.synchronize()
    for x in pools:
        assert torch.equal(raw(x[8:10]), raw(x[:2]))


def test_refusals():
    K = _k()
    a = torch.zeros(8, 2, 16, 128, dtype=torch.float16, device=DEV)
    copy = K.copy_paged
    copy([a], [], [])
    copy([a], torch.empty(0, dtype=torch.int32, device=DEV), torch.empty(0, dtype=torch.int32, device=DEV))
    for src, dst in (([0], [0, 1]), ([0, 1], [2, 2]), ([0, 1], [1, 2]), ([8], [0]), ([-1], [0]), ([0], [8])):
        with pytest.raises(ValueError):
            copy([a], src, dst)
    copy([a], [0, 1], [1, 2], into=[torch.zeros_like(a)])  # another pool: the same numbers are other pages
    for bad in ([], [a.cpu()], [a[0]], [a[:, :, :8]], [a, a[:4]], [a, a[:, :1]], [a[..., :96]], [a[..., ::2]],
                [torch.zeros(8, 2, 16, 129, dtype=torch.float16, device=DEV)[..., 1:]],
                [torch.zeros(8, 2, 16, 8, dtype=torch.float16, device=DEV)[..., :4]]):
        with pytest.raises(ValueError):
            copy(bad, [0], [1])
    for into in ([a, a], [a.float()], [a[:, :1]], [torch.zeros(8, 2, 32, 128, dtype=torch.float16, device=DEV)],
                 [a[:1].expand(8, -1, -1, -1)], [a[:, :1].expand(-1, 2, -1, -1)]):
        with pytest.raises(ValueError):
            copy([a], [0], [1], into=into)
    copy([a[:1].expand(8, -1, -1, -1)], [5], [1], into=[a])  # read, it may share its memory
    with pytest.raises(ValueError):
        copy([a], [0], [1], torch.tensor([1, 2], device=DEV))
    with pytest.raises(ValueError):
        copy([a], torch.tensor([0.0], device=DEV), torch.tensor([1], device=DEV))
    with pytest.raises(NotImplementedError):
        copy([a.clone().requires_grad_()], [0], [1])
