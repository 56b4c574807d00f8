"""bf16 queries over INT8 pages, where one large channel meets codes that are zero, so that the scores are what the small
channels say: each attention against float64.

The queries enter the matrix instructions in fp16, scaled so that the largest lies in [2^14, 2^15): bf16 values down to
2^-31 of that power of two are exact (8 bits above fp16's least step, 2^-24), and smaller ones off by at most half a step, 2^-39
of it, which moves a score by at most sm sum |k| 2^-39 Q.  To that comes the tolerance that test_gpu_paged derives, with d the scores'
error."""
import pytest
import torch

from test_gpu_paged import BF16, D, DEV, F16, SM, check, reference

pytestmark = pytest.mark.gpu

LENS, SHARED, PAGE = [256, 300, 333], 256, 64


def cache(group, g, heads=2):
    """Codes with a zero channel 0 and scales about 16; a table whose first SHARED tokens are everybody's."""
    cols = -(-max(LENS) // PAGE)
    table = torch.stack([torch.cat([torch.arange(SHARED // PAGE), 4 + 2 * b + torch.arange(cols - SHARED // PAGE)]) for b in range(3)])
    pages = int(table.max()) + 1
    out = []
    for size in (16.0, 0.01):
        codes = torch.randint(-127, 128, (pages, heads, PAGE, D), generator=g).to(torch.int8)
        out += [codes, ((0.5 + torch.rand(pages, heads, PAGE, D // group, generator=g)) * size).half()]
    ck, sk, cv, sv = out
    ck[..., 0] = 0

    def dense(c, s):
        x = c.double() * s.double().repeat_interleave(group, -1)
        return x[table].permute(0, 2, 1, 3, 4).flatten(2, 3)  # [B, H, T, 128]

    return (ck, cv, sk, sv, table.int()), dense(ck, sk), dense(cv, sv).half().double()


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("ratio", [-3, 0, 12, 17, 20, 26, 30, 33])
@pytest.mark.parametrize("shared", [False, True])
def test_small_channels_beside_a_large_one(shared, ratio, group):
    import llm_kvcache_quantization_amd as K

    g = torch.Generator().manual_seed(group + ratio)
    (ck, cv, sk, sv, table), kd, vd = cache(group, g)
    q = ((1 + torch.rand(3, 12, D, generator=g)) * 2.0 ** -11 * torch.randn(3, 12, D, generator=g).sign()).to(BF16)
    q[..., 0] = 2.0 ** (ratio - 10)
    lens = torch.tensor(LENS, dtype=torch.int32, device=DEV)
    args = [x.to(DEV) for x in (q, ck, cv, table)] + [lens]
    kw = dict(k_scale=sk.to(DEV), v_scale=sv.to(DEV))
    if shared:
        out = K.decode_attn_shared(*args, K.SharedPrefix([3], [SHARED], 12, 2, DEV), SM, **kw)
    else:
        out = K.decode_attn_paged(*args, SM, **kw)
    Q = 2.0 ** max(ratio - 10, -10)  # at or above the power of two at the largest
    for b, n in enumerate(LENS):
        # (over V rounded to fp16 after its scale, as the shared attention takes it; the other's own rounding of V counts
        # with the flag)
        ref, tol, _, _ = reference(q[b], kd[b], vd[b], torch.arange(kd.shape[2]) < n, SM, BF16, F16, 0 if shared else group)
        d = SM * kd[b, :, :n].abs().sum(-1).max() * 2.0 ** -39 * Q if ratio > 30 else 0.0  # small ones are from 2^-(ratio + 1) Q on
        spread = vd[b].abs().amax()
        check(out[b], ref, tol + 2 * d * spread, (shared, ratio, group, b))


@pytest.mark.parametrize("shared", [False, True])
@pytest.mark.parametrize("top", [-133, -127, -126, -125, -113, -112, -60, 0, 60, 100])
def test_queries_of_any_size(shared, top):
    """Queries whose largest is 2^top, from subnormal ones on: no scale passes fp32, and a score's error is that of fp32 sums (of
    subnormal queries the scores are below 2^-100; above 2^7, past fp16's least scales, they meet codes that are zero)."""
    import llm_kvcache_quantization_amd as K

    g = torch.Generator().manual_seed(7)
    (ck, cv, sk, sv, table), _, vd = cache(32, g)
    sk = (torch.ones_like(sk) * 2.0 ** min(-top - 7, 15)).half() if top > -20 else sk
    sk = sk.clamp(min=2.0 ** -14)
    if top > 7:
        ck = torch.zeros_like(ck)
    kd = (ck.double() * sk.double().repeat_interleave(32, -1))[table.long()].permute(0, 2, 1, 3, 4).flatten(2, 3)
    q = torch.randn(3, 12, D, generator=g, dtype=torch.float64).clamp(-1, 1)
    q[..., 5] = 1.0
    q = (q * 2.0 ** top).to(BF16)
    lens = torch.tensor(LENS, dtype=torch.int32, device=DEV)
    args = [x.to(DEV) for x in (q, ck, cv, table)] + [lens]
    kw = dict(k_scale=sk.to(DEV), v_scale=sv.to(DEV))
    out = K.decode_attn_shared(*args, K.SharedPrefix([3], [SHARED], 12, 2, DEV), SM, **kw) if shared else K.decode_attn_paged(*args, SM, **kw)
    for b, n in enumerate(LENS):
        ref, tol, _, _ = reference(q[b], kd[b], vd[b], torch.arange(kd.shape[2]) < n, SM, BF16, F16, 0 if shared else 32)
        check(out[b], ref, tol, (shared, top, b))
