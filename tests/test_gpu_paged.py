"""The paged cache's operators (append_paged, decode_attn_paged, evict_paged) against plain
implementations: attention in float64 over the visible tokens, codes and moved rows bit for bit.

Everything a call must not look at is poisoned: slots at or past a sequence's length, tokens
outside its window, pages of nobody hold NaN (INT8: NaN scales).

Tolerance of an attention output, u being half a step of a type (fp16 2^-11, bf16 2^-8):
``u_out |out|`` for the output's own rounding; ``u_p A`` with A = sum p |v| for the probabilities' in the
product (fp16 over INT8 pages), plus ``2^-25 sum |v| / L`` for those below fp16's normal range (L = sum exp(s -
max) >= 1 scales them); ``2^-11 A`` for INT8 values code * scale in fp16; scores of 128 fp32 products are off by
at most d = 130 * 2^-23 sm sum |q k|, which moves p by a factor exp(+-2 d): ``2 d A``; n fp32 additions:
``n 2^-23 A``."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
D = 128
SM = 1 / math.sqrt(D)
U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
F16, BF16 = torch.float16, torch.bfloat16


def _k():
    import llm_kvcache_quantization_amd as K

    return K


def quantize(x, group):
    """INT8 codes and scales of rows [..., 128]: the formula of append_paged, in torch on the CPU."""
    x = x.float().cpu().unflatten(-1, (D // group, group))
    odd = ~torch.isfinite(x).all(-1)
    top = x.abs().amax(-1).clamp(min=1e-5)
    s = (top / torch.full_like(top, 127.0)).clamp(max=65504.0).half()
    c = (x / s.float().unsqueeze(-1)).half().float().round().clamp(-127, 127)
    c[odd] = 0
    s[odd] = math.nan
    return c.flatten(-2).to(torch.int8), s


class Pool:
    """Pages of B sequences with `caps` token slots each in random order, values drawn, the rest NaN."""

    def __init__(self, lens, heads, page, dtype, int8=0, seed=0, slots=None, tokens_first=False, spare=2):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.heads, self.page, self.dtype, self.int8 = lens, heads, page, dtype, int8
        cols = max(1, -(-max(max(lens), slots or 1) // page))
        self.cols = cols
        B = len(lens)
        n = B * cols + spare
        self.table = torch.randperm(n, generator=g)[: B * cols].view(B, cols).int()
        shape = (n, page, heads, D) if tokens_first else (n, heads, page, D)

        def pages():
            x = torch.full(shape, math.nan, dtype=dtype)
            return x.permute(0, 2, 1, 3) if tokens_first else x

        self.k, self.v = pages(), pages()
        T = cols * page
        kd = torch.randn(B, heads, T, D, generator=g)
        kd[..., torch.randperm(D, generator=g)[:4]] *= 8
        vd = torch.randn(B, heads, T, D, generator=g)
        self.dense_k, self.dense_v = kd.to(dtype), vd.to(dtype)
        self.ks = self.vs = None
        if int8:
            self.ck, self.sk = quantize(self.dense_k, int8)
            self.cv, self.sv = quantize(self.dense_v, int8)
            self.k = torch.randint(-128, 128, self.k.shape, dtype=torch.int8, generator=g)
            self.v = torch.randint(-128, 128, self.k.shape, dtype=torch.int8, generator=g)
            self.ks = torch.full((n, heads, page, D // int8), math.nan, dtype=F16)
            self.vs = self.ks.clone()

    def fill(self, visible):
        """Writes the tokens of sequence b where visible(b) says so."""
        for b in range(len(self.lens)):
            t = torch.nonzero(visible(b)).flatten()
            p, s = self.table[b, t // self.page].long(), t % self.page
            if self.int8:
                self.k[p, :, s], self.v[p, :, s] = self.ck[b, :, t].transpose(0, 1), self.cv[b, :, t].transpose(0, 1)
                self.ks[p, :, s], self.vs[p, :, s] = self.sk[b, :, t].transpose(0, 1), self.sv[b, :, t].transpose(0, 1)
            else:
                self.k[p, :, s], self.v[p, :, s] = self.dense_k[b, :, t].transpose(0, 1), self.dense_v[b, :, t].transpose(0, 1)
        return self

    def cuda(self):
        for n in ("k", "v", "ks", "vs", "table"):
            x = getattr(self, n)
            if x is not None:
                setattr(self, n, x.to(DEV))
        return self

    def values(self):
        """float64 K, V [B, H, T, 128] as the pages hold them."""
        if not self.int8:
            return self.dense_k.double(), self.dense_v.double()

        def deq(c, s):
            return (c.double().unflatten(-1, (-1, self.int8)) * s.double().unsqueeze(-1)).flatten(-2)

        return deq(self.ck, self.sk), deq(self.cv, self.sv)

    def args(self):
        return self.k, self.v, self.table

    def scales(self):
        return dict(k_scale=self.ks, v_scale=self.vs)


def visible(n, T, window, sinks):
    t = torch.arange(T)
    seen = t < n
    return seen & ((t >= n - window) | (t < sinks)) if window else seen


def reference(q, k, v, vis, sm, out_type, p_type, int8, tau=None):
    """float64 attention of q [Hq, 128] over one sequence's K, V [H, T, 128]: (out, tolerance, p)."""
    hq, h = q.shape[0], k.shape[0]
    idx = torch.nonzero(vis).flatten()
    out, tol = torch.zeros(hq, D, dtype=torch.float64), torch.zeros(hq, D, dtype=torch.float64)
    probs = torch.zeros(h, k.shape[1], dtype=torch.float64)
    ptol = torch.zeros_like(probs)
    if not len(idx):
        return out, tol, probs, ptol
    for x in range(hq):
        f = sm * (1.0 if tau is None else float(tau[x]))
        kk, vv = k[x * h // hq, idx], v[x * h // hq, idx]
        s = kk @ q[x].double() * f
        e = torch.exp(s - s.max())
        p = e / e.sum()
        out[x] = p @ vv
        d = 130 * 2.0 ** -23 * (kk.abs() @ q[x].double().abs() * abs(f)).max()
        A = p @ vv.abs()
        rel = U[p_type] + (2.0 ** -11 if int8 else 0) + 2 * d + len(idx) * 2.0 ** -23 + 2.0 ** -20
        tol[x] = U[out_type] * out[x].abs() + rel * A + 2.0 ** -25 * vv.abs().sum(0) / e.sum() + 1e-7
        probs[x * h // hq, idx] += p
        ptol[x * h // hq, idx] += p * (2 * d + len(idx) * 2.0 ** -23 + 2.0 ** -20)
    return out, tol, probs, ptol


def check(out, ref, tol, what):
    bad = (out.double().cpu() - ref).abs() - tol
    assert not torch.isnan(out).any(), what
    assert bad.max() <= 0, (what, float(bad.max()), float((out.double().cpu() - ref).abs().max()), float(tol.max()))


def run_decode(lens, hq, hkv, page, dtype, int8=0, window=None, sinks=0, seed=1, tau=False, weights=False, slots=None,
               tokens_first=False, q_pad=0):
    K = _k()
    print(f"[decode] lens {lens} heads {hq}/{hkv} page {page} {dtype} int8 {int8} window {window} sinks {sinks}", flush=True)
    pool = Pool(lens, hkv, page, dtype, int8, seed, slots=slots, tokens_first=tokens_first)
    T = pool.cols * page
    vis = [visible(n, T, window, sinks) for n in lens]
    pool.fill(lambda b: vis[b]).cuda()
    g = torch.Generator().manual_seed(seed + 1)
    q = torch.randn(len(lens), hq, D, generator=g).to(dtype)
    t = (0.5 + torch.rand(hq, generator=g)) if tau else None
    w0 = torch.rand(len(lens), hkv, T + 5, generator=g) if weights else None
    w = w0.to(DEV) if weights else None
    out = K.decode_attn_paged(torch.nn.functional.pad(q.to(DEV), (0, q_pad))[..., :D],
                              *pool.args(), torch.tensor(lens, dtype=torch.int32, device=DEV), SM, **pool.scales(),
                              inv_tau=None if t is None else t.to(DEV), window=window, sinks=sinks, weights=w)
    torch.cuda.synchronize()
    assert out.dtype == dtype and out.shape == (len(lens), hq, D)
    kd, vd = pool.values()
    for b in range(len(lens)):
        ref, tol, p, ptol = reference(q[b], kd[b], vd[b], vis[b], SM, dtype, F16 if int8 else dtype, int8, t)
        check(out[b], ref, tol, ("row", b))
        if weights:
            add = torch.zeros_like(w0[b]).double()
            pad = torch.zeros_like(add)
            add[:, :T], pad[:, :T] = p, ptol
            want = w0[b].double() + add
            err = (w[b].double().cpu() - want).abs() - (pad + 2.0 ** -23 * want)
            assert err.max() <= 0, ("weights", b, float(err.max()))
    return pool, q, out


TYPES = [(F16, 0), (BF16, 0), (F16, 32), (BF16, 32), (F16, 64), (BF16, 128), (F16, 128), (BF16, 64)]


@pytest.mark.parametrize("dtype,int8", TYPES)
@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
def test_decode_short_rows(dtype, int8, page):
    run_decode([0, 1, 15, 16, 17, 31, 32, 33, 63, 200], 12, 2, page, dtype, int8)


@pytest.mark.parametrize("dtype,int8", TYPES)
@pytest.mark.parametrize("page", [16, 64])
def test_decode_split_rows(dtype, int8, page):
    run_decode([2500, 0, 1, 4097, 33, 1300], 28, 4, page, dtype, int8)


@pytest.mark.parametrize("dtype,int8", [(F16, 0), (BF16, 32)])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 4), (33, 40), (100, 0), (700, 4), (5000, 4)])
def test_decode_window(dtype, int8, window, sinks):
    run_decode([0, 1, 16, 17, 48, 101, 1333, 2049], 10, 2, 16, dtype, int8, window=window, sinks=sinks)
    run_decode([1333, 2049], 10, 2, 64, dtype, int8, window=window, sinks=sinks)


@pytest.mark.parametrize("hq,hkv", [(1, 1), (16, 1), (3, 3), (40, 8), (2, 1)])
def test_decode_head_layouts(hq, hkv):
    run_decode([70, 1500], hq, hkv, 32, F16)
    run_decode([70, 1500], hq, hkv, 32, BF16, 32)


@pytest.mark.parametrize("dtype,int8", [(F16, 0), (BF16, 0), (F16, 32), (BF16, 128)])
@pytest.mark.parametrize("window,sinks", [(None, 0), (50, 3)])
def test_decode_weights(dtype, int8, window, sinks):
    run_decode([0, 1, 33, 300], 12, 2, 16, dtype, int8, weights=True, window=window, sinks=sinks)
    run_decode([0, 1999, 33, 3500, 1], 28, 4, 16, dtype, int8, weights=True, window=window, sinks=sinks)


def test_decode_inv_tau_and_strides():
    run_decode([70, 1500], 12, 2, 64, F16, tau=True)
    run_decode([70, 1500], 12, 2, 64, BF16, 32, tau=True)
    run_decode([70, 1500], 12, 2, 64, F16, tokens_first=True, q_pad=4)
    run_decode([70, 1500], 12, 2, 16, BF16, tokens_first=True, q_pad=8)


def test_decode_one_long_row_and_many_rows():
    run_decode([40000], 12, 2, 64, F16)
    run_decode([65536 + 31], 5, 1, 256, F16, 128)
    run_decode([i % 37 for i in range(300)], 2, 1, 16, F16)
    run_decode([(i * 7919) % 1500 for i in range(90)], 2, 1, 16, BF16)


@pytest.mark.parametrize("rows", [63, 64, 65, 127, 4096])
@pytest.mark.parametrize("split", [False, True])
@pytest.mark.parametrize("weights", [False, True])
def test_decode_many_rows(rows, split, weights):
    """Rows at and past a wave's lanes, up to the most of a call; a table of many columns has the rows' tiles shared
    out over work-groups that know nothing of rows."""
    K = _k()
    print(f"[decode] rows {rows} split {split} weights {weights}", flush=True)
    g = torch.Generator().manual_seed(rows)
    lens = torch.randint(0, 49, (rows,), generator=g)
    lens[torch.rand(rows, generator=g) < 0.3] = 0
    lens[0], lens[-1] = 0, 48
    lens = lens.tolist()
    pool = Pool(lens, 1, 16, F16)
    T = pool.cols * 16
    vis = [visible(n, T, None, 0) for n in lens]
    pool.fill(lambda b: vis[b]).cuda()
    q = torch.randn(rows, 2, D, generator=g).to(F16)
    table = torch.cat([pool.table, torch.full((rows, 70), -1, dtype=torch.int32, device=DEV)], 1) if split else pool.table
    w = torch.zeros(rows, 1, table.shape[1] * 16, device=DEV) if weights else None
    out = K.decode_attn_paged(q.to(DEV), pool.k, pool.v, table, torch.tensor(lens, dtype=torch.int32, device=DEV), SM, weights=w)
    torch.cuda.synchronize()
    kd, vd = pool.values()
    for b in range(rows):
        ref, tol, p, ptol = reference(q[b], kd[b], vd[b], vis[b], SM, F16, F16, 0)
        check(out[b], ref, tol, ("row", b))
        if weights:
            got = w[b].double().cpu()
            assert ((got[:, :T] - p).abs() - ptol - 2.0 ** -23 * p).max() <= 0, ("weights", b)
            assert not got[:, T:].any()


@pytest.mark.parametrize("dtype,int8", [(F16, 0), (BF16, 64)])
@pytest.mark.parametrize("lens", [[600] * 13, [530, 0, 0, 1100, 40, 0, 640, 3, 1025, 0], [577] * 40, [0] * 20 + [900, 0, 1] * 12])
def test_decode_shares_of_rows(dtype, int8, lens):
    """Even and uneven rows, fewer and more of them than work-groups a KV head: work-groups of one row, and those
    that end a row and begin another."""
    for hq, hkv in ((5, 5), (16, 16)):
        run_decode(lens, hq, hkv, 32, dtype, int8, weights=int8 == 0)


def test_decode_default_scale_and_long_lens():
    """No sm_scale means 1/sqrt(128); int64 lengths are taken; lengths past the table are clamped to it."""
    K = _k()
    pool, q, out = run_decode([64, 40], 12, 2, 32, F16, slots=64)
    ln = torch.tensor([64, 40], device=DEV)
    a = K.decode_attn_paged(q.to(DEV), *pool.args(), ln)
    assert torch.equal(a, out)
    b = K.decode_attn_paged(q.to(DEV)[:1], pool.k, pool.v, pool.table[:1], torch.tensor([1 << 30], device=DEV), SM)
    assert torch.equal(b, out[:1])
    z = K.decode_attn_paged(q.to(DEV)[:1], pool.k, pool.v, pool.table[:1], torch.tensor([-5], device=DEV), SM)
    assert not z.any()


def test_decode_missing_pages():
    """Pages outside the pool: their tokens are left out, a row of nothing else is zero."""
    K = _k()
    for int8 in (0, 32):
        for lens, page in (([100, 64, 2000], 16), ([100, 64, 2000], 64)):
            pool = Pool(lens, 2, page, F16, int8, seed=5)
            T = pool.cols * page
            gone = {0: [1], 1: list(range(pool.cols)), 2: [0, 3, 1999 // page]}
            vis = [visible(n, T, None, 0) for n in lens]
            for b, cols in gone.items():
                for c in cols:
                    vis[b][c * page : (c + 1) * page] = False
            pool.fill(lambda b: vis[b])
            for b, cols in gone.items():
                for i, c in enumerate(cols):
                    pool.table[b, c] = (-1, pool.k.shape[0], 2 ** 31 - 1)[i % 3]
            pool.cuda()
            q = torch.randn(3, 12, D, generator=torch.Generator().manual_seed(3)).half()
            out = K.decode_attn_paged(q.to(DEV), *pool.args(), torch.tensor(lens, device=DEV), SM, **pool.scales())
            kd, vd = pool.values()
            assert not out[1].any()
            for b in (0, 2):
                ref, tol, _, _ = reference(q[b], kd[b], vd[b], vis[b], SM, F16, F16, int8)
                check(out[b], ref, tol, (int8, page, b))


def test_decode_infinities():
    """Inf and NaN where they are seen reach the row that sees them, and no other."""
    K = _k()
    pool = Pool([40, 40, 40], 1, 32, F16, seed=6)
    pool.fill(lambda b: visible(40, 64, None, 0))
    q = torch.randn(3, 4, D, generator=torch.Generator().manual_seed(3)).half()
    pool.v[pool.table[0, 0].long(), 0, 3, 7] = math.nan
    pool.k[pool.table[2, 0].long(), 0, 3] = 0
    pool.k[pool.table[2, 0].long(), 0, 3, 0] = -math.inf  # score -inf for a positive q, +inf for a negative one
    q[2, :, 0] = torch.tensor([1.0, 2.0, 0.5, 3.0])
    pool.cuda()
    out = K.decode_attn_paged(q.to(DEV), *pool.args(), torch.tensor([40] * 3, device=DEV), SM).cpu()
    assert torch.isnan(out[0, :, 7]).all() and not torch.isnan(out[0, :, 8:]).any()
    assert not torch.isnan(out[1]).any() and not torch.isnan(out[2]).any()
    kd, vd = pool.values()
    vis = visible(40, 64, None, 0)
    vis[3] = False
    ref, tol, _, _ = reference(q[2], kd[2], vd[2], vis, SM, F16, F16, 0)
    check(out[2], ref, tol, "-inf score")
    # a row whose scores are all -inf has no softmax
    k = torch.full_like(pool.k, 0)
    k[..., 0] = -math.inf
    q2 = torch.ones(1, 4, D, dtype=F16, device=DEV)
    out = K.decode_attn_paged(q2, k, torch.ones_like(k), pool.table[:1], torch.tensor([40], device=DEV), SM)
    assert torch.isnan(out).all()


def test_decode_large_scores():
    """Scores that grow along the row by more than fp16's range: the maximum follows."""
    K = _k()
    n = 600
    pool = Pool([n], 1, 64, F16, seed=8)
    ramp = torch.linspace(-60, 60, pool.dense_k.shape[2])
    for sign in (1, -1):
        pool.dense_k[:] = (sign * ramp.view(1, 1, -1, 1) / 8).half()
        p2 = Pool([n], 1, 64, F16, seed=8)
        p2.dense_k = pool.dense_k
        vis = visible(n, p2.cols * 64, None, 0)
        p2.fill(lambda b: vis).cuda()
        q = torch.ones(1, 3, D).half()
        out = K.decode_attn_paged(q.to(DEV), *p2.args(), torch.tensor([n], device=DEV), SM)
        kd, vd = p2.values()
        ref, tol, _, _ = reference(q[0], kd[0], vd[0], vis, SM, F16, F16, 0)
        check(out[0], ref, tol, sign)


def test_decode_small_and_large_queries_over_int8():
    """bf16 queries outside fp16's range over INT8 pages."""
    K = _k()
    for f in (2.0 ** -40, 2.0 ** 30, 1.0):
        pool = Pool([77], 2, 16, BF16, 64, seed=9)
        vis = visible(77, pool.cols * 16, None, 0)
        pool.fill(lambda b: vis).cuda()
        q = (torch.randn(1, 6, D, generator=torch.Generator().manual_seed(1)) * f).to(BF16)
        sm = SM / f
        out = K.decode_attn_paged(q.to(DEV), *pool.args(), torch.tensor([77], device=DEV), sm, **pool.scales())
        kd, vd = pool.values()
        ref, tol, _, _ = reference(q[0], kd[0], vd[0], vis, sm, BF16, F16, 64)
        check(out[0], ref, tol, f)


# ---------------------------------------------------------------- append


def torch_append(pool, k, v, pos, lens):
    """The pages after an append, on the CPU."""
    kp, vp = pool.k.clone(), pool.v.clone()
    ks = None if pool.ks is None else pool.ks.clone()
    vs = None if pool.vs is None else pool.vs.clone()
    if pool.int8:
        (ck, sk), (cv, sv) = quantize(k, pool.int8), quantize(v, pool.int8)
    for b in range(k.shape[0]):
        for i in range(lens[b]):
            t = pos[b] + i
            if t < 0 or t >= pool.cols * pool.page:
                continue
            p, s = int(pool.table[b, t // pool.page]), t % pool.page
            if not 0 <= p < kp.shape[0]:
                continue
            if pool.int8:
                kp[p, :, s], vp[p, :, s], ks[p, :, s], vs[p, :, s] = ck[b, :, i], cv[b, :, i], sk[b, :, i], sv[b, :, i]
            else:
                kp[p, :, s], vp[p, :, s] = k[b, :, i], v[b, :, i]
    return kp, vp, ks, vs


def same_bits(a, b):
    if a is None or b is None:
        return a is b
    w = {1: torch.int8, 2: torch.int16, 4: torch.int32}[a.element_size()]
    a, b = a.cpu(), b.cpu()
    nan = torch.isnan(a) & torch.isnan(b) if a.is_floating_point() else torch.zeros(a.shape, dtype=torch.bool)
    return bool(((a.contiguous().view(w) == b.contiguous().view(w)) | nan).all())


def run_append(B, H, S, page, dtype, int8, pos, lens=None, seed=0, slots=None, layout="bhsd", table=None, edit=None, pages="own"):
    K = _k()
    print(f"[append] {B} {H} {S} page {page} {dtype} int8 {int8} pos {pos} lens {lens}", flush=True)
    pool = Pool([1] * B, H, page, dtype, int8, seed, slots=slots or max(p + S for p in pos), tokens_first=pages == "tokens" and not int8)
    if table is not None:
        table(pool.table)
    g = torch.Generator().manual_seed(seed + 3)
    k, v = (torch.randn(B, H, S, D, generator=g) * 3).to(dtype), torch.randn(B, H, S, D, generator=g).to(dtype)
    k[..., 5] *= 20
    if edit:
        edit(k, v)
    want = torch_append(pool, k, v, pos, lens or [S] * B)
    pool.cuda()
    kd, vd = k.to(DEV), v.to(DEV)
    if layout == "bshd":
        kd, vd = (x.transpose(1, 2).contiguous().transpose(1, 2) for x in (kd, vd))
    if layout == "odd":  # rows that are not 16-byte aligned
        kd, vd = (torch.nn.functional.pad(x, (0, 3))[..., :D] for x in (kd, vd))
    K.append_paged(kd, vd, *pool.args(), torch.tensor(pos, device=DEV),
                   None if lens is None else torch.tensor(lens, dtype=torch.int32, device=DEV), **pool.scales())
    torch.cuda.synchronize()
    for name, a, b in zip(("k", "v", "k_scale", "v_scale"), (pool.k, pool.v, pool.ks, pool.vs), want):
        assert same_bits(a, b), name
    return pool


@pytest.mark.parametrize("dtype,int8", TYPES)
@pytest.mark.parametrize("page", [16, 128])
def test_append(dtype, int8, page):
    run_append(1, 2, 1, page, dtype, int8, [517])
    run_append(3, 4, 1, page, dtype, int8, [0, page - 1, page])
    run_append(3, 4, 37, page, dtype, int8, [0, 9, 200], lens=[37, 0, 20])
    run_append(2, 5, 333, page, dtype, int8, [1, 40])


@pytest.mark.parametrize("layout,pages", [("bshd", "own"), ("odd", "own"), ("bhsd", "tokens")])
def test_append_layouts(layout, pages):
    for dtype, int8 in ((F16, 0), (BF16, 32)):
        run_append(2, 3, 21, 16, dtype, int8, [3, 30], layout=layout, pages=pages)


def test_append_out_of_the_table():
    """Slots past the table, negative positions and pages that are not there are left alone."""
    def table(t):
        t[0, 1] = -1
        t[1, 0] = 10 ** 6

    for int8 in (0, 64):
        run_append(2, 2, 50, 16, F16, int8, [0, 3], slots=40, table=table)
        run_append(2, 2, 5, 16, F16, int8, [-3, 2 ** 31 - 2], slots=40)
        run_append(2, 2, 5, 16, F16, int8, [0, 0], lens=[-1, 100][:1] + [5], slots=40)


def test_append_values():
    """Zeros, subnormals, the largest values, ties and non-finite groups."""
    def edit(k, v):
        k[0, 0, 0] = 0
        k[0, 0, 1] = 6e-8
        k[0, 0, 2, :] = 65000.0
        k[0, 0, 3, 1] = math.nan
        k[0, 0, 4, 40] = math.inf
        k[0, 0, 5, 127] = -math.inf
        v[0, 0, 0] = torch.arange(D) - 63.5
        v[0, 0, 1] = (torch.arange(D) - 64) * 2.0 ** -14

    for dtype in (F16, BF16):
        for int8 in (0, 32, 64, 128):
            run_append(1, 1, 6, 16, dtype, int8, [0], edit=edit)


@pytest.mark.parametrize("dtype,int8", TYPES)
def test_append_long(dtype, int8):
    """Prompts of 64 and more new tokens: about the work-groups' share of them, padded, at the ends of the table."""
    def table(t):
        t[0, 2] = -1
        t[1, 3] = 10 ** 6

    for S in (63, 64, 65, 129):
        run_append(2, 3, S, 16, dtype, int8, [0, 37])
    run_append(4, 3, 150, 32, dtype, int8, [5, 0, 64, 31], lens=[150, 0, 65, 1], layout="bshd", pages="tokens")
    run_append(2, 2, 100, 16, dtype, int8, [0, 3], slots=90, table=table, layout="odd")
    run_append(3, 2, 70, 16, dtype, int8, [-3, -70, 2 ** 31 - 80], slots=80, lens=[70, -5, 1000])


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_append_every_value(dtype, group):
    """Every 16-bit pattern beside a largest value of its group of each magnitude: the codes are those of the IEEE
    quotient."""
    bits = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(dtype)
    g = torch.Generator().manual_seed(group)

    def edit(k, v):
        for x in (k, v):
            rows = bits[torch.randperm(65536, generator=g)].view(4, 2, 64, D)
            x.copy_(rows)
            top = bits[torch.randint(0, 0x7800, (4, 2, 64, D // group), generator=g)]
            keep = x.unflatten(-1, (-1, group)).abs() <= top.abs().unsqueeze(-1)
            x.copy_(torch.where(keep, x.unflatten(-1, (-1, group)), top.unsqueeze(-1)).flatten(-2))

    for seed in range(8):
        run_append(4, 2, 64, 16, dtype, group, [0, 1, 2, 3], seed=seed, edit=edit)


@pytest.mark.parametrize("group", [32, 64, 128])
def test_append_codes_are_the_dense_engines(group):
    K = _k()
    eng = K.INT8KVCache(1, device=DEV, clip_percentile=100.0, group_size=group)
    k = (torch.randn(1, 2, 80, D, generator=torch.Generator().manual_seed(group)) * 2).half().to(DEV)
    v = torch.randn(1, 2, 80, D, generator=torch.Generator().manual_seed(1)).half().to(DEV)
    eng.append(0, k, v)
    kq, vq, ks, vs = eng.get_int8_tensors(0)
    kp = torch.zeros(5, 2, 16, D, dtype=torch.int8, device=DEV)
    vp = torch.zeros_like(kp)
    sk = torch.zeros(5, 2, 16, D // group, dtype=F16, device=DEV)
    sv = torch.zeros_like(sk)
    table = torch.arange(5, dtype=torch.int32, device=DEV).view(1, 5)
    K.append_paged(k, v, kp, vp, table, torch.zeros(1, dtype=torch.int32, device=DEV), k_scale=sk, v_scale=sv)
    for a, b in ((kp, kq), (vp, vq), (sk, ks), (sv, vs)):
        assert torch.equal(a.transpose(0, 1).flatten(1, 2), b[0])


# ---------------------------------------------------------------- eviction


def torch_evict(pool, lens, w, budget, sinks, recent):
    """(pages..., new lens, kept, new weights) on the CPU, token by token."""
    B, H = w.shape[:2]
    pools = [x.clone() for x in (pool.k, pool.v, pool.ks, pool.vs) if x is not None]
    was = [x.clone() for x in pools]
    kept = torch.full((B, H, budget), -1, dtype=torch.int32)
    nw = torch.zeros_like(w)
    new = []
    cap = pool.cols * pool.page
    for b in range(B):
        n = min(max(lens[b], 0), cap)
        pages = pool.table[b, : -(-n // pool.page)]
        gone = n > budget and bool(((pages < 0) | (pages >= pool.k.shape[0])).any())
        new.append(n if gone else min(n, budget))
        for h in range(H):
            if n <= budget or gone:
                nw[b, h, :n] = w[b, h, :n]
                if not gone:
                    kept[b, h, :n] = torch.arange(n)
                continue
            mid = list(range(sinks, n - recent))
            x = w[b, h].tolist()
            order = sorted(mid, key=lambda t: (0, -x[t], t) if x[t] == x[t] else (1, 0.0, t))
            keep = sorted(list(range(sinks)) + order[: budget - sinks - recent] + list(range(n - recent, n)))
            kept[b, h] = torch.tensor(keep)
            for j, t in enumerate(keep):
                nw[b, h, j] = w[b, h, t]
                for dst, src in zip(pools, was):
                    dst[pool.table[b, j // pool.page].long(), h, j % pool.page] = \
                        src[pool.table[b, t // pool.page].long(), h, t % pool.page]
    return pools, torch.tensor(new, dtype=torch.int32), kept, nw


def run_evict(lens, heads, page, dtype, int8, budget, sinks=0, recent=0, seed=0, w=None, table=None, tokens_first=False, slots=None):
    K = _k()
    print(f"[evict] {lens} heads {heads} page {page} {dtype} int8 {int8} budget {budget} {sinks}+{recent}", flush=True)
    pool = Pool(lens, heads, page, dtype, int8, seed, tokens_first=tokens_first and not int8, slots=slots)
    pool.fill(lambda b: visible(lens[b], pool.cols * page, None, 0))
    if table is not None:
        table(pool.table)
    T = pool.cols * page
    g = torch.Generator().manual_seed(seed + 11)
    weights = torch.rand(len(lens), heads, T + 3, generator=g) ** 6
    if w is not None:
        weights = w(weights, g)
    want, new, kept, nw = torch_evict(pool, lens, weights, budget, sinks, recent)
    pool.cuda()
    wd = weights.to(DEV)
    a, b, c = K.evict_paged(*pool.args(), torch.tensor(lens, device=DEV), wd, budget, sinks=sinks, recent=recent, **pool.scales())
    torch.cuda.synchronize()
    assert torch.equal(a.cpu(), new), (a, new)
    assert torch.equal(b.cpu(), kept)
    assert same_bits(c, nw)
    assert same_bits(wd, weights)
    for x, y in zip([t for t in (pool.k, pool.v, pool.ks, pool.vs) if t is not None], want):
        assert same_bits(x, y)


@pytest.mark.parametrize("dtype,int8", TYPES)
@pytest.mark.parametrize("page", [16, 64])
def test_evict(dtype, int8, page):
    run_evict([0, 1, 50, 51, 200, 777], 2, page, dtype, int8, 50, sinks=4, recent=16)


@pytest.mark.parametrize("budget,sinks,recent", [(1, 0, 0), (1, 1, 0), (1, 0, 1), (20, 10, 10), (20, 0, 0), (20, 0, 20), (299, 3, 5), (300, 3, 5)])
def test_evict_protected(budget, sinks, recent):
    run_evict([300, 64], 3, 32, F16, 0, budget, sinks, recent)


def test_evict_long_rows():
    run_evict([5000, 700, 3001], 2, 16, F16, 0, 2100, 4, 100)
    run_evict([9000], 1, 64, BF16, 32, 4000, 0, 0)
    run_evict([32768, 20000], 1, 256, BF16, 128, 3000, 4, 100)
    run_evict([40000, 3001], 1, 256, F16, 128, 5000, 4, 100)  # more weights than a work-group's registers hold


def test_evict_ties_and_special_weights():
    run_evict([500], 2, 16, F16, 0, 100, 2, 8, w=lambda w, g: torch.zeros_like(w))
    run_evict([500], 2, 16, F16, 0, 100, 2, 8, w=lambda w, g: torch.randint(0, 4, w.shape, generator=g).float())
    run_evict([500], 2, 16, F16, 0, 100, 2, 8, w=lambda w, g: torch.where(torch.rand(w.shape, generator=g) < 0.5, -0.0, 0.0))

    def odd(w, g):
        r = torch.rand(w.shape, generator=g)
        w = w - 0.1
        w[r < 0.3] = math.nan
        w[(r > 0.3) & (r < 0.35)] = math.inf
        w[(r > 0.35) & (r < 0.6)] = -math.inf
        w[(r > 0.6) & (r < 0.65)] = 1e-42
        return w

    for budget in (30, 100, 300, 480):
        run_evict([500, 499], 2, 16, F16, 0, budget, 2, 8, w=odd)
    # neighbouring floats: every bit of the key counts
    run_evict([900], 2, 16, F16, 0, 300, 0, 0, w=lambda w, g: (0x3F800000 + torch.randint(0, 700, w.shape, generator=g)).int().view(torch.float32))


def test_evict_missing_pages_and_layout():
    def table(t):
        t[1, 2] = -1
        t[2, t.shape[1] - 1] = 10 ** 8  # behind the row's last token: not looked at

    run_evict([300, 300, 100], 2, 16, F16, 0, 90, 4, 10, table=table)
    run_evict([300, 300, 100], 2, 16, F16, 0, 90, 4, 10, tokens_first=True)
    run_evict([300, 300, 100], 2, 16, F16, 32, 90, 4, 10, table=table)


def test_evict_budget_of_whole_cap():
    run_evict([64, 70], 2, 16, F16, 0, 500)
