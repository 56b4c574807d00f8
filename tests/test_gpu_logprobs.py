"""Log probabilities, entropy and the likeliest tokens (token_logprobs) against float64, the tokens whole number for whole
number (ties to the lower one).

Tolerances, in nats: with e = 2^-23 (fp32) and t = (x - max) / T of at most about 200 where its exponential is no 0, an
exponential is off by 2^-22 + 2 |t| e of itself (its argument is rounded as a difference and as a product); n of them are added in
chains of at most n / 256 + 10 with e each.  So l is off by r = 2^-22 + A e + (n / 256 + 12) e of itself, A = sum p |t| (weighted), log l by r and an
fp32 rounding, log p_t by that and 2 |t| e; the entropy log l - sum p t by r, its own sum's r (A + 1) and the roundings."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
E = 2.0 ** -23
TYPES = [torch.float16, torch.bfloat16, torch.float32]


def _k():
    import llm_kvcache_quantization_amd as K

    return K


def best_of(x, k):
    """Indices of the k largest of each row, the lower first among equal ones, NaN least (x on the CPU)."""
    x = x.float()
    key = torch.where(torch.isnan(x), torch.tensor(-math.inf), x)
    nan = torch.isnan(x)
    out = []
    for row, bad in zip(key, nan):
        order = sorted(range(len(row)), key=lambda i: (bool(bad[i]), -float(row[i]), i)) if len(row) <= 3000 else None
        if order is None:
            s = torch.sort(row, descending=True, stable=True).indices
            order = torch.cat([s[~bad[s]], s[bad[s]]]).tolist()
        out.append(order[:k])
    return torch.tensor(out, dtype=torch.int64).view(len(out), k)


def check(x, tokens, top, temperature=1.0, out=None):
    K = _k()
    print(f"[logprobs] {tuple(x.shape)} {x.dtype} top {top} T {temperature}", flush=True)
    got = out or K.token_logprobs(x.to(DEV), None if tokens is None else tokens.to(DEV), top, temperature=temperature)
    torch.cuda.synchronize()
    rows, v = x.reshape(-1, x.shape[-1]), x.shape[-1]
    y = rows.double() / temperature
    none = torch.isnan(y).any(1) | (y == math.inf).any(1) | (y == -math.inf).all(1)
    t = y - y.amax(1, keepdim=True)
    p = t.exp()
    l = p.sum(1)
    log_l = l.log()
    tz = torch.where(p > 0, t, torch.zeros(()).double())
    A = (p * tz.abs()).sum(1) / l
    H = log_l + A
    r = 2.0 ** -22 + A * 2 * E + (v / 256 + 12) * E
    tol_l = r + E * log_l.abs() + E
    ent = got.entropy.cpu().double().reshape(-1)
    assert torch.isnan(ent[none]).all()
    assert ((ent - H).abs()[~none] <= (tol_l + r * (A + 1) + E * (H + 1))[~none]).all(), (ent - H).abs()[~none].max()

    def close(lp, at, rows_t):
        want = rows_t - log_l.view(-1, *([1] * (rows_t.ndim - 1)))
        tol = tol_l.view(-1, *([1] * (rows_t.ndim - 1))) + 3 * E * rows_t.abs() + E * want.abs()
        lp = lp.cpu().double().reshape(want.shape)
        keep = ~none
        assert torch.isnan(lp[none]).all(), at
        same = (lp == want) | ((lp - want).abs() <= tol)
        assert same[keep].all(), (at, (lp - want)[keep].abs().max())

    if tokens is None:
        assert got.logprobs is None
    else:
        tk = tokens.cpu().reshape(-1).long()
        inside = (tk >= 0) & (tk < v)
        lp = got.logprobs.cpu().reshape(-1)
        assert torch.isnan(lp[~inside]).all()
        some = t.gather(1, tk.clamp(0, v - 1).unsqueeze(1)).squeeze(1)
        lp = torch.where(inside, lp, (some - log_l).float())
        close(lp, "token", some)
    if not top:
        assert got.top_tokens is None and got.top_logprobs is None
    else:
        want = best_of(rows.cpu(), top)
        ids = got.top_tokens.cpu().reshape(-1, top)
        assert ids.dtype == torch.int64 and torch.equal(ids, want), (ids - want).nonzero()[:5]
        close(got.top_logprobs, "top", t.gather(1, want))
    return got


def draw(rows, v, dtype, seed=0, spread=2.5):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, v, generator=g) * spread
    for i in range(rows):
        x[i, torch.randint(v, (min(9, v),), generator=g)] += 9 * torch.rand(min(9, v), generator=g)
    return x.to(dtype), torch.randint(v, (rows,), generator=g)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("v", [1, 2, 7, 8, 15, 16, 17, 31, 33, 63, 64, 65, 127, 255, 1000, 2047, 2048, 2049, 8191, 8192, 8193, 16390])
def test_vocabularies(dtype, v):
    x, t = draw(3, v, dtype, v)
    for top in {0, 1, min(5, v), min(32, v)}:
        check(x, t, top)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,v", [(1, 151936), (2, 152064), (33, 50257), (2100, 1000), (2047, 515), (1, 400001)])
def test_rows(dtype, rows, v):
    x, t = draw(rows, v, dtype, rows)
    check(x, t, 20)
    check(x, None, 0)


@pytest.mark.parametrize("dtype", TYPES)
def test_ties(dtype):
    """Equal logits go to the lower token: constant rows, rows of few values, zeros of both signs; sorted rows of either way
    fill the lists again and again."""
    v = 9001
    flat = torch.full((1, v), 1.5)
    steps = (torch.arange(v) % 7).float().view(1, v)
    zeros = torch.where(torch.arange(v) % 2 == 0, 0.0, -0.0).view(1, v)
    up = torch.arange(v).float().view(1, v) / 64
    late = torch.zeros(1, v)
    late[0, -40:] = 3
    early = torch.zeros(1, v)
    early[0, :40] = 3
    x = torch.cat([flat, steps, zeros, up, up.flip(1), late, early]).to(dtype)
    for top in (1, 2, 31, 32):
        check(x, torch.tensor([0, 6, 1, v - 1, 0, v - 1, 0]), top)
    long = (torch.arange(200000).float() / 1000).view(1, -1).to(dtype)
    check(long, torch.tensor([199999]), 32)
    check(long.flip(1).contiguous(), torch.tensor([199999]), 32)
    check(torch.zeros(2, 150001, dtype=dtype), torch.tensor([5, 150000]), 32)


@pytest.mark.parametrize("dtype", TYPES)
def test_masks(dtype):
    """-Inf and the type's lowest value as masks, nearly all and all of a row; NaN and +Inf; top beyond what is left."""
    v = 5003
    x, t = draw(10, v, dtype, 3)
    low = torch.finfo(dtype).min
    x[0, :] = -math.inf
    x[1, :] = low
    x[2, :] = -math.inf
    x[2, [17, 4000]] = torch.tensor([1.0, 2.0], dtype=dtype)
    x[3, 1:] = -math.inf
    x[4, :] = low
    x[4, 77] = 3.0
    x[5, 100] = math.nan
    x[6, 4999] = math.inf
    x[7, :] = math.nan
    x[8, ::2] = low
    x[8, 1::2] = -math.inf
    t[:5] = torch.tensor([5, 6, 17, 0, 77])
    t[8] = 3
    for top in (0, 1, 3, 20):
        check(x, t, top)
    got = _k().token_logprobs(x.to(DEV), t.to(DEV), 3)
    assert math.isclose(float(got.entropy[1]), math.log(v), rel_tol=1e-6) and float(got.logprobs[8]) == -math.inf
    wide = x.new_full((3, 160001), -math.inf)
    wide[0, 12345], wide[1, :], wide[2, 159999:] = 1.0, low, low
    check(wide, torch.tensor([12345, 8, 160000]), 5)


@pytest.mark.parametrize("dtype", TYPES)
def test_masks_begin_and_end_anywhere(dtype):
    """Long rows, several steps a thread and several work-groups a row, whose masked runs lie anywhere."""
    v = 70001
    x, t = draw(8, v, dtype, 5)
    runs = [(0, 1), (v - 1, v), (0, 20000), (20000, 45000), (45000, v), (1, v), (33333, 33334), (8, v - 8)]
    for row, (a, b) in enumerate(runs):
        x[row, a:b] = -math.inf
    t[:] = torch.tensor([0, 0, 30000, 30000, 0, 0, 33333, 3])
    check(x, t, 9)
    check(x.repeat(60, 1)[:, :9001].contiguous(), t.repeat(60).clamp(max=9000), 2)  # a work-group a row


@pytest.mark.parametrize("rows", [383, 384])
def test_rows_of_one_and_several_work_groups(rows):
    x, t = draw(rows, 20011, torch.bfloat16, rows)
    check(x, t, 3)


def test_rows_past_32_bits():
    """Rows whose begins lie more than 2^32 bytes apart."""
    v, step = 5003, (1 << 31) + 8
    x, t = draw(3, v, torch.bfloat16, 6)
    room = torch.empty(2 * step + v, dtype=torch.bfloat16, device=DEV)
    rows = room.as_strided((3, v), (step, 1))
    rows.copy_(x)
    check(x, t, 4, out=_k().token_logprobs(rows, t.to(DEV), 4))


def test_confident_rows_keep_their_small_logarithms():
    """log p of a token that has nearly all of the probability is the others' sum, not a difference of large numbers."""
    x = torch.full((2, 40000), -10.0)
    x[0, 39999] = 20.0
    x[1, 3] = 1000.0
    got = _k().token_logprobs(x.to(DEV), torch.tensor([39999, 3], device=DEV), 1)
    rest = 39999 * math.exp(-30)
    # l = 1 + rest in fp32: off by at most 2^-24, of which rest is the small part
    assert abs(float(got.logprobs[0]) + math.log1p(rest)) <= 2.0 ** -23
    assert float(got.logprobs[1]) == 0.0 and float(got.entropy[1]) == 0.0


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("temperature", [0.05, 0.7, 1.0, 3.0, 100.0])
def test_temperatures(dtype, temperature):
    x, t = draw(5, 3001, dtype, 8)
    check(x, t, 7, temperature)


@pytest.mark.parametrize("dtype", TYPES)
def test_layouts(dtype):
    """Rows that begin anywhere, the last position of a [B, S, V] batch, transposed rows, more dimensions, token types."""
    x, t = draw(6, 1021, dtype, 9)
    big = torch.zeros(6, 1100, dtype=dtype, device=DEV)
    for off in (0, 1, 3, 7):
        view = big[:, off : off + 1021]
        view.copy_(x)
        check(x, t, 4, out=_k().token_logprobs(view, t.to(DEV), 4))
    seq = torch.randn(6, 3, 1021, device=DEV).to(dtype)
    seq[:, -1] = x.to(DEV)
    check(x, t, 4, out=_k().token_logprobs(seq[:, -1], t.to(DEV), 4))
    check(x, t, 4, out=_k().token_logprobs(x.to(DEV).t().contiguous().t(), t.to(DEV), 4))
    check(x.view(2, 3, 1021), t.view(2, 3), 4)
    check(x[0], t[0], 4)
    for kind in (torch.int32, torch.int16, torch.uint8):
        tk = t.clamp(max=200).to(kind)
        check(x, tk, 0)
    check(x, torch.tensor([-1, 1021, -100, 2 ** 40, 0, 1020]), 2)
    check(x[:1].expand(4, -1), t[:4], 3)


def test_empty_and_other_streams_and_graphs():
    K = _k()
    none = K.token_logprobs(torch.empty(0, 100, device=DEV), torch.empty(0, dtype=torch.int64, device=DEV), 3)
    assert none.logprobs.shape == none.entropy.shape == (0,) and none.top_tokens.shape == (0, 3)
    x = torch.randn(4, 60000, device=DEV)
    t = torch.arange(4, device=DEV)
    K.token_logprobs(x, t, 5)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got = K.token_logprobs(x, t, 5)
        graphs.append((g, got))
    for i in range(6):
        x.copy_(torch.randn(4, 60000, device=DEV))
        want = K.token_logprobs(x, t, 5)
        g, got = graphs[i % 2]
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), i
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = K.token_logprobs(x, t, 5)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_refusals():
    K = _k()
    x = torch.randn(3, 50, device=DEV)
    t = torch.zeros(3, dtype=torch.int64, device=DEV)
    for args in ((x.cpu(),), (x.double(),), (x.int(),), (x[:, :0],), (x, t[:2]), (x, t.float()), (x, t.view(3, 1)), (x, t, 33),
                 (x, t, -1), (x[:, :4].contiguous(), t, 5)):
        with pytest.raises(ValueError):
            K.token_logprobs(*args)
    for temperature in (0.0, -1.0, math.inf, math.nan, 1e-31):
        with pytest.raises(ValueError):
            K.token_logprobs(x, t, temperature=temperature)
    with pytest.raises(NotImplementedError):
        K.token_logprobs(x.clone().requires_grad_(), t)
