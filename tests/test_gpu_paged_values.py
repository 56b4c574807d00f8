"""The paged operators at values that a softmax has none for, and at those far below its largest, against float64."""
import math

import pytest
import torch

from test_gpu_paged import BF16, F16, SM, Pool, visible

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
D = 128


def _k():
    import llm_kvcache_quantization_amd as K

    return K


@pytest.mark.parametrize("int8", [0, 64])
@pytest.mark.parametrize("slots", [None, 4000])  # one work-group a row, and split
def test_weights_of_tokens_that_are_not_seen(int8, slots):
    """A row whose softmax is none (a NaN, an infinite score) gives NaN weights to the tokens it sees; those outside its window
    and on pages that are not there get nothing, in its tiles too."""
    K = _k()
    print(f"[unseen] {int8} {slots}", flush=True)
    lens, window, sinks = [90, 90, 90, 90], 50, 3
    pool = Pool(lens, 2, 16, F16, int8, seed=3, slots=slots)
    T = pool.cols * 16
    vis = [visible(n, T, window, sinks) for n in lens]
    pool.fill(lambda b: vis[b])
    vis[2][48:64] = False  # its page is gone
    pool.table[2, 3] = -1
    q = torch.randn(4, 6, D, generator=torch.Generator().manual_seed(4)).half()
    q[0, 1, 5] = math.nan   # one head of a row
    q[1] = math.inf
    q[2, :, 7] = -math.inf
    pool.cuda()
    w = torch.rand(4, 2, T + 4, generator=torch.Generator().manual_seed(5)).to(DEV)
    was = w.clone()
    K.decode_attn_paged(q.to(DEV), *pool.args(), torch.tensor(lens, device=DEV), SM, **pool.scales(), window=window, sinks=sinks, weights=w)
    torch.cuda.synchronize()
    for b in range(4):
        seen = torch.nn.functional.pad(vis[b], (0, 4)).to(DEV)
        assert torch.equal(w[b][:, ~seen], was[b][:, ~seen]), b
        nan = torch.isnan(w[b][:, seen])
        if b == 0:  # query heads 0 to 2 are KV head 0's
            assert nan[0].all() and not nan[1].any()
        elif b == 3:
            assert not nan.any() and (w[b][:, seen] > was[b][:, seen]).all()
        else:
            assert nan.all()


def faint(n, bits, seed):
    """K, V [1, n, 128] and q [2, 128] (float64): token 0 scores 0 and has no value, the others score `bits` (log2) below it, give
    or take one, and have values around 1."""
    g = torch.Generator().manual_seed(seed)
    q = torch.ones(2, D, dtype=torch.float64)
    f = math.log(2) / (D * SM)
    k = (-(bits + 2 * torch.rand(n, 1, generator=g, dtype=torch.float64) - 1) * f).expand(n, D).clone()
    v = 1 + 0.5 * torch.randn(n, D, generator=g, dtype=torch.float64)
    k[0] = v[0] = 0
    return q, k[None], v[None]


def exact_and_tolerance(q, k, v, u_out, u_p, u_v, up):
    """float64 attention of q [Hq, 128] over k, v [1, n, 128], and how far off a kernel may be, as derived in test_gpu_paged.py
    but for P: in fp16 its steps below 2^-14 are 2^-24, and a score's P is 2^up times its share of the largest's at least, so
    that it is off by 2^-25-up of it at most.  An fp16 output below 2^-14 has steps of 2^-24 itself, so that rounding it is off by
    up to 2^-25 whatever the kernel does: 2^-20 of a value around 1 lies there (bf16, of fp32's range, has no such end)."""
    s = q @ k[0].t() * SM
    e = torch.exp(s - s.max())
    p = e / e.sum(1, keepdim=True)
    out, A = p @ v[0], p @ v[0].abs()
    d = 130 * 2.0 ** -23 * float((q.abs() @ k[0].abs().t() * SM).max())
    tol = u_out * out.abs() + (u_p + u_v + 2 * d + k.shape[1] * 2.0 ** -23 + 2.0 ** -20) * A
    last = 2.0 ** -25 if u_out == 2.0 ** -11 else 0.0
    return out, tol + 2.0 ** (-25 - up) * v[0].abs().sum(0) / e.sum(1, keepdim=True) + last + 1e-12


@pytest.mark.parametrize("dtype,int8", [(F16, 0), (F16, 32), (BF16, 128), (BF16, 0)])
@pytest.mark.parametrize("n", [600, 65536])  # one work-group a row, and split
@pytest.mark.parametrize("bits", [20, 25, 28])
def test_decode_many_faint_tokens(dtype, int8, n, bits):
    """A first token that takes nearly all the softmax and has no value: the result is what the many others add up to."""
    K = _k()
    print(f"[faint] decode {dtype} {int8} {n} {bits}", flush=True)
    q, k, v = faint(n, bits, 7)
    pool = Pool([n], 1, 64, dtype, int8)
    T = pool.cols * 64
    k, v = (torch.nn.functional.pad(x.to(dtype), (0, 0, 0, T - n)) for x in (k, v))
    pool.dense_k, pool.dense_v = k[None], v[None]
    if int8:
        from test_gpu_paged import quantize

        pool.ck, pool.sk = quantize(pool.dense_k, int8)
        pool.cv, pool.sv = quantize(pool.dense_v, int8)
    pool.fill(lambda b: visible(n, T, None, 0)).cuda()
    w = torch.zeros(1, 1, T, device=DEV)
    out = K.decode_attn_paged(q.to(dtype).to(DEV)[None], *pool.args(), torch.tensor([n], device=DEV), SM, **pool.scales(), weights=w)
    kd, vd = (x[0, :, :n] for x in pool.values())
    ref, tol = exact_and_tolerance(q, kd, vd, 2.0 ** -11 if dtype == F16 else 2.0 ** -8, 2.0 ** -8 if dtype == BF16 and not int8 else 2.0 ** -11,
                                   2.0 ** -11 if int8 else 0, 100 if dtype == BF16 and not int8 else 9)
    err = (out[0].double().cpu() - ref).abs()
    assert (err <= tol).all(), (float((err / ref.abs()).max()), float((tol / ref.abs()).max()))
    # the softmax itself is fp32 throughout
    p = torch.softmax(q @ kd[0].t() * SM, 1).sum(0)
    d = 130 * 2.0 ** -23 * float((q.abs() @ kd[0].abs().t() * SM).max())
    assert ((w[0, 0, :n].double().cpu() - p).abs() <= p * (2 * d + n * 2.0 ** -23 + 2.0 ** -20)).all()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("S,T", [(500, 500), (40, 700), (3, 40000)])  # whole, and split over the keys
@pytest.mark.parametrize("bits", [20, 25, 28])
def test_prompt_many_faint_tokens(dtype, S, T, bits):
    K = _k()
    print(f"[faint] prompt {dtype} {S} {T} {bits}", flush=True)
    q, k, v = faint(T, bits, 8)
    q, k, v = (x.to(dtype) for x in (q[:, None].expand(-1, S, -1), k, v))
    out = K.prefill_attn_window(q[None].to(DEV), k[None].to(DEV), v[None].to(DEV), SM)[0].double().cpu()
    for i in {0, 1, S // 2, S - 1}:
        n = T - S + i + 1
        ref, tol = exact_and_tolerance(q[:, i].double(), k[:, :n].double(), v[:, :n].double(), *[2.0 ** -11 if dtype == F16 else 2.0 ** -8] * 2,
                                       0, 9 if dtype == F16 else 100)
        err = (out[:, i] - ref).abs()
        assert (err <= tol).all(), (i, float((err / ref.abs()).max()), float((tol / ref.abs()).max()))


@pytest.mark.parametrize("slots", [2048, 2064, 16384, 16400, 32768, 32784])
def test_evict_at_the_variants_ends(slots):
    """Tables on either side of where the selection changes, full and nearly empty rows in each."""
    from test_gpu_paged import run_evict

    run_evict([slots, 700, slots - 1], 1, 16, F16, 0, 600, 4, 100, slots=slots)
    zeros = lambda w, g: torch.where(torch.rand(w.shape, generator=g) < 0.9, 0.0, w)  # noqa: E731
    run_evict([slots - 5, 601], 2, 16, F16, 64, 600, 0, 7, slots=slots, w=zeros)
