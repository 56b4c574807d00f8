"""copy_paged leaves what lies between and behind pages as it was: pools that are slices of filled tensors, compared whole, bit
for bit."""
import pytest
import torch

from test_gpu_copy_paged import DEV, _k, bits, raw

pytestmark = pytest.mark.gpu

# a slice [pages, heads, page, X] of a larger tensor, and that tensor's shape
LAYOUTS = {
    "a head more": (lambda p, h, s, x: (p, h + 1, s, x), lambda t: t[:, :-1]),
    "a head before": (lambda p, h, s, x: (p, h + 1, s, x), lambda t: t[:, 1:]),
    "every second page": (lambda p, h, s, x: (2 * p, h, s, x), lambda t: t[1::2]),
    "pages in the middle": (lambda p, h, s, x: (p + 2, h, s, x), lambda t: t[1:-1]),
    "tokens before heads, a head more": (lambda p, h, s, x: (p, s, h + 1, x), lambda t: t[:, :, :-1].permute(0, 2, 1, 3)),
    "rows of twice the length": (lambda p, h, s, x: (p, h, s, 2 * x), lambda t: t[..., : t.shape[3] // 2]),
}
DENSE_TOKENS = ("a head more", "a head before", "every second page", "pages in the middle")  # what rows below 16 bytes need


@pytest.mark.parametrize("layout,dtype,x", [(k, t, x) for t, x in ((torch.float16, 128), (torch.int8, 128), (torch.float16, 4), (torch.float16, 1))
                                            for k in (LAYOUTS if x > 4 else DENSE_TOKENS)])
@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("part", [False, True])
@pytest.mark.parametrize("other", [False, True])
def test_gaps_stay(layout, dtype, x, page, part, other):
    g = torch.Generator().manual_seed(page + x)
    shape, cut = LAYOUTS[layout]
    whole = [bits(shape(9, 3, page, x), dtype, g) for _ in range(4)]
    device = [t.to(DEV) for t in whole]
    src, dst = [0, 3, 8, 5], [1, 2, 7, 4]
    lens = [page // 2 + 1, page, 3, 0] if part else None
    reads, writes = (whole[:2], whole[2:]) if other else (whole, whole)
    for a, b in zip(reads, writes):
        for i, (s, d) in enumerate(zip(src, dst)):
            n = page if lens is None else lens[i]
            cut(b)[d, :, :n] = cut(a)[s, :, :n]
    pools = [cut(t) for t in (device[:2] if other else device)]
    _k().copy_paged(pools, src, dst, None if lens is None else torch.tensor(lens, device=DEV),
                    into=[cut(t) for t in device[2:]] if other else None)
    for got, want in zip(device, whole):
        assert torch.equal(raw(got.cpu()), raw(want))
