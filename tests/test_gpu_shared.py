"""Attention over a shared prefix (decode_attn_shared) against float64 attention of each sequence by itself, and the same
call without sharing (decode_attn_paged).

What a call must not look at is poisoned: a sequence's own slots below its prefix, slots at or past its length and pages
of nobody hold NaN (INT8: NaN scales); table entries of the prefix of all but a group's first sequence name no page.

Tolerances are those derived in test_gpu_paged (output, probabilities, scores, sums), over the values that the call
works with: K's codes x scale, V's code x scale rounded to fp16, so that their rounding adds nothing."""
import math

import pytest
import torch

from test_gpu_paged import BF16, D, DEV, F16, SM, Pool, check, reference, visible

pytestmark = pytest.mark.gpu


def _k():
    import llm_kvcache_quantization_amd as K

    return K


class Groups(Pool):
    """Pages of groups of sequences: sizes, shared tokens of each group, tokens of each sequence."""

    def __init__(self, sizes, shared, lens, heads, page, dtype, int8=0, seed=0, slots=None, tokens_first=False):
        super().__init__(lens, heads, page, dtype, int8, seed, slots=slots or max(max(lens), max(shared, default=1), 1),
                         tokens_first=tokens_first)
        self.sizes, self.shared = sizes, shared
        self.first, self.prefix = [], []
        for n, p in zip(sizes, shared):
            self.first += [len(self.first)] * n
            self.prefix += [p] * n
        T = self.cols * page
        t = torch.arange(T)
        self.fill(lambda b: (t < self.lens[b]) & (t >= self.prefix[b]) if b != self.first[b] else
                  t < max([self.lens[b]] + [min(self.prefix[b], T)]))
        for b, f in enumerate(self.first):
            if b != f:
                for x in ("dense_k", "dense_v") if not int8 else ("ck", "cv", "sk", "sv"):
                    getattr(self, x)[b, :, : self.prefix[b]] = getattr(self, x)[f, :, : self.prefix[b]]
                whole = self.prefix[b] // page if self.lens[b] >= self.prefix[b] else self.cols
                self.table[b, :whole] = torch.tensor([(-1, self.k.shape[0], 2 ** 30)[i % 3] for i in range(whole)], dtype=torch.int32)

    def values(self):
        k, v = super().values()
        return (k, v.half().double()) if self.int8 else (k, v)


def call(pool, q, **kw):
    K = _k()
    prefix = K.SharedPrefix(pool.sizes, pool.shared, q.shape[1], pool.heads, DEV)
    return K.decode_attn_shared(q, *pool.args(), torch.tensor(pool.lens, dtype=torch.int32, device=DEV), prefix, SM,
                                **pool.scales(), **kw)


def run(sizes, shared, lens, hq, hkv, page, dtype, int8=0, seed=1, tau=False, q_pad=0, slots=None, tokens_first=False):
    print(f"[shared] sizes {sizes} shared {shared} lens {lens[:8]} heads {hq}/{hkv} page {page} {dtype} int8 {int8}", flush=True)
    pool = Groups(sizes, shared, lens, hkv, page, dtype, int8, seed, slots, tokens_first).cuda()
    g = torch.Generator().manual_seed(seed + 1)
    q = torch.randn(len(lens), hq, D, generator=g).to(dtype)
    t = (0.5 + torch.rand(hq, generator=g)) if tau else None
    out = call(pool, torch.nn.functional.pad(q.to(DEV), (0, q_pad))[..., :D], inv_tau=None if t is None else t.to(DEV))
    torch.cuda.synchronize()
    assert out.dtype == dtype and out.shape == q.shape
    kd, vd = pool.values()
    for b, n in enumerate(lens):
        ref, tol, _, _ = reference(q[b], kd[b], vd[b], visible(n, kd.shape[2], None, 0), SM, dtype, F16 if int8 else dtype, 0, t)
        check(out[b], ref, tol, ("row", b, n))
    return pool, q.to(DEV), out


TYPES = [(F16, 0), (BF16, 0), (F16, 32), (BF16, 32), (F16, 64), (BF16, 128)]


@pytest.mark.parametrize("dtype,int8", TYPES)
@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
def test_pages_and_types(dtype, int8, page):
    run([3, 2], [300 // page * page, 64 // page * page], [300, 333, 512, 64, 130], 12, 2, page, dtype, int8)


@pytest.mark.parametrize("dtype,int8", [(F16, 0), (BF16, 0), (F16, 32)])
@pytest.mark.parametrize("shared", [0, 1, 15, 16, 17, 31, 63, 64, 65, 127, 129, 200])
def test_prefix_lengths(dtype, int8, shared):
    """A prefix of any number of tokens, none among them; sequences that end with it, one past it, and before it."""
    run([6], [shared], [shared, shared + 1, shared + 63, shared + 70, max(shared - 1, 0), shared // 2], 12, 2, 16, dtype, int8)


@pytest.mark.parametrize("dtype,int8", [(F16, 0), (BF16, 0), (BF16, 64)])
@pytest.mark.parametrize("rows", [1, 2, 3, 5, 6, 10, 11, 16, 22, 33, 64])
def test_columns(dtype, int8, rows):
    """Rows x heads of a KV head from fewer than a wave's 32 columns over the work-group's 128 to several of them."""
    run([rows], [192], [192 + 5 * i % 77 for i in range(rows)], 12, 2, 64, dtype, int8)


@pytest.mark.parametrize("hq,hkv", [(1, 1), (3, 3), (16, 1), (40, 8), (40, 1), (128, 1), (7, 1)])
def test_head_layouts(hq, hkv):
    run([3, 1, 2], [130, 40, 0], [130, 200, 131, 90, 77, 1], hq, hkv, 32, F16)
    run([3, 1, 2], [130, 40, 0], [130, 200, 131, 90, 77, 1], hq, hkv, 32, BF16, 32)


@pytest.mark.parametrize("dtype,int8", TYPES)
def test_long_prefixes(dtype, int8):
    run([4], [4096], [4096, 4600, 5003, 4097], 28, 4, 16, dtype, int8)
    run([2, 3, 1], [2500, 1000, 3001], [2500, 4000, 1000, 0, 3000, 3500], 10, 2, 64, dtype, int8)


def test_many_groups_and_rows():
    run([1] * 40, [i * 13 % 200 for i in range(40)], [(i * 13 % 200) + i for i in range(40)], 2, 1, 16, F16)
    run([7] * 30, [64 + 16 * (i % 3) for i in range(30)], [64 + i % 100 for i in range(210)], 4, 2, 16, BF16)
    run([300], [64], [64 + i % 50 for i in range(300)], 2, 1, 16, F16, 128)


def test_most_rows():
    lens = [48 + i % 40 for i in range(4096)]
    K = _k()
    pool = Groups([4000, 96], [48, 32], lens, 1, 16, F16).cuda()
    q = torch.randn(4096, 2, D, generator=torch.Generator().manual_seed(1)).half()
    out = call(pool, q.to(DEV))
    kd, vd = pool.values()
    for b in list(range(0, 4096, 97)) + [3999, 4000, 4095]:
        ref, tol, _, _ = reference(q[b], kd[b], vd[b], visible(lens[b], kd.shape[2], None, 0), SM, F16, F16, 0)
        check(out[b], ref, tol, ("row", b))


@pytest.mark.parametrize("dtype,int8", [(F16, 0), (BF16, 64)])
def test_ragged_tails_of_many_rows(dtype, int8):
    """More than 64 rows: one of them long, some with nothing of their own, some shorter than their prefix or empty."""
    lens = [64 + 7 * (i % 5) for i in range(90)]
    lens[3], lens[20], lens[21], lens[50], lens[51] = 4000, 0, 13, 64, 1
    run([60, 1, 29], [64, 0, 48], lens, 4, 2, 16, dtype, int8)
    run([257], [128], [128 + (3000 if i in (0, 255, 256) else i % 3) for i in range(257)], 2, 1, 32, dtype, int8)


def test_long_tails():
    run([2, 1], [100, 20], [9000, 100, 5000], 12, 2, 16, F16)
    run([2], [64], [30000, 64], 5, 1, 128, BF16, 32)


@pytest.mark.parametrize("shared", [0, 1 << 29])
def test_longest_rows(shared):
    """2^30 tokens, all in one page: the products of tiles and work-groups pass 32 bits.  Every token of the page stands as
    often, so that the attention is the page's."""
    g = torch.Generator().manual_seed(4)
    k, v = (torch.randn(1, 1, 256, D, generator=g).to(F16) for _ in range(2))
    q = torch.randn(1, 4, D, generator=g).to(F16)
    K = _k()
    table = torch.zeros(1, 1 << 22, dtype=torch.int32, device=DEV)
    out = K.decode_attn_shared(q.to(DEV), k.to(DEV), v.to(DEV), table, torch.tensor([1 << 30], dtype=torch.int32, device=DEV),
                               K.SharedPrefix([1], [shared], 4, 1, DEV), SM)
    torch.cuda.synchronize()
    p = torch.softmax(q[0].double() @ k[0, 0].double().T * SM, -1)
    ref, size = p @ v[0, 0].double(), p @ v[0, 0].double().abs()
    # Sums of up to 2^29 / 256 tokens a work-group in fp32, 16 a step, and of all of them: 2^17 steps and 2^11 parts of 2^-24 each,
    # in numerator and denominator; fp16's P (2^-11), scores (2^-21 of |q| |k| sm, below 2^4) and output (2^-11)
    tol = size * (2 * (2.0 ** 17 + 2.0 ** 11) * 2.0 ** -24 + 2.0 ** -11 + 2 * 2.0 ** -17) + ref.abs() * 2.0 ** -11
    assert ((out[0].cpu().double() - ref).abs() <= tol).all()


def test_strides_and_temperatures():
    run([3], [130], [140, 150, 131], 12, 2, 64, F16, tau=True)
    run([3], [130], [140, 150, 131], 12, 2, 64, BF16, 32, tau=True)
    run([3], [130], [140, 150, 131], 12, 2, 64, F16, tokens_first=True, q_pad=4)
    run([3], [130], [140, 150, 131], 12, 2, 16, BF16, tokens_first=True, q_pad=8)


def test_lengths_past_the_table_and_negative():
    """Lengths are clamped to what the table holds; a prefix longer than the table is seen as far as that."""
    K = _k()
    pool, q, out = run([2], [64], [128, 128], 12, 2, 32, F16, slots=128)
    prefix = K.SharedPrefix([2], [64], 12, 2, DEV)
    args = (q, *pool.args())
    assert torch.equal(K.decode_attn_shared(*args, torch.tensor([1 << 40, 128], device=DEV), prefix, SM), out)
    assert not K.decode_attn_shared(*args, torch.tensor([-3, 0], device=DEV), prefix).any()
    longer = K.SharedPrefix([2], [100000], 12, 2, DEV)
    pool.table[1] = pool.table[0]
    a = K.decode_attn_shared(q, *pool.args(), torch.tensor([128, 1 << 30], device=DEV), longer)
    b = K.decode_attn_paged(q, *pool.args(), torch.tensor([128, 128], device=DEV))
    assert (a.float() - b.float()).abs().max() < 4e-3


def test_missing_pages():
    """Tokens of pages that are not there are left out, of the prefix for the whole group; nothing else is zero."""
    for int8 in (0, 32):
        for page in (16, 64):
            pool = Groups([2, 1], [256, 128], [300, 400, 128], 2, page, F16, int8, seed=5)
            vis = [visible(n, pool.cols * page, None, 0) for n in pool.lens]
            gone = [(0, 1, (0, 1)), (0, 256 // page - 1, (0, 1)), (1, 300 // page, (1,))] + [(2, i, (2,)) for i in range(128 // page)]
            for i, (b, c, rows) in enumerate(gone):
                pool.table[b, c] = (-1, pool.k.shape[0], 2 ** 31 - 1)[i % 3]
                for r in rows:
                    vis[r][c * page : (c + 1) * page] = False
            pool.cuda()
            q = torch.randn(3, 12, D, generator=torch.Generator().manual_seed(3)).half()
            out = call(pool, q.to(DEV))
            kd, vd = pool.values()
            assert not out[2].any()
            for b in (0, 1):
                ref, tol, _, _ = reference(q[b], kd[b], vd[b], vis[b], SM, F16, F16, 0)
                check(out[b], ref, tol, (int8, page, b))


def test_infinities_reach_who_sees_them():
    """A NaN in a prefix reaches its group, one in a sequence's own tokens that sequence alone; all scores -Inf: NaN."""
    pool = Groups([2, 2], [64, 64], [100, 100, 100, 100], 1, 32, F16, seed=6)
    pool.v[pool.table[0, 1].long(), 0, 3, 7] = math.nan       # token 35 of the first prefix
    pool.v[pool.table[3, 2].long(), 0, 30, 9] = math.inf      # token 94 of the last sequence
    pool.cuda()
    q = torch.randn(4, 4, D, generator=torch.Generator().manual_seed(3)).half()
    out = call(pool, q.to(DEV)).cpu()
    assert torch.isnan(out[:2, :, 7]).all() and torch.isfinite(out[:2, :, :7]).all() and torch.isfinite(out[:2, :, 8:]).all()
    assert torch.isfinite(out[2]).all() and (out[3, :, 9] == math.inf).all()
    ones = torch.zeros_like(pool.k)
    ones[..., 0] = -math.inf
    q[:, :, 0] = 1
    assert torch.isnan(_k().decode_attn_shared(q.to(DEV), ones, pool.v.nan_to_num(0, 0, 0), pool.table,
                                               torch.tensor([100] * 4, device=DEV), _k().SharedPrefix([2, 2], [64, 64], 4, 1, DEV))).all()


def test_faint_tokens_count_in_fp16():
    """Many tokens far below a row's largest score, in the prefix and behind it, keep their part of the result."""
    K = _k()
    n, page = 16384, 64
    k = torch.zeros(n // page, 1, page, D, dtype=F16, device=DEV)
    v = torch.ones_like(k)
    k[0, 0, 0, 0] = 1.0
    v[0, 0, 0] = 0.0
    q = torch.zeros(2, 1, D, dtype=F16, device=DEV)
    q[:, 0, 0] = 12.0  # the first token's score is 12 above the others': p = e^-12 each, 16383 of them
    table = torch.arange(n // page, dtype=torch.int32, device=DEV).expand(2, -1).contiguous()
    lens = torch.tensor([n, n], device=DEV)
    want = (n - 1) * math.exp(-12) / (1 + (n - 1) * math.exp(-12))
    for shared in (n, n // 2, 64, 0):
        out = K.decode_attn_shared(q, k, v, table, lens, K.SharedPrefix([2], [shared], 1, 1, DEV), 1.0).double()
        # fp32 sums of 2^14 values, exponentials at 2^-20, the output's half step
        assert (out - want).abs().max() <= want * (2.0 ** -11 + 2.0 ** -9 * 2.0 ** -2 + 2.0 ** -18), (shared, out[0, 0, 0], want)


@pytest.mark.parametrize("dtype,int8", [(F16, 0), (BF16, 32)])
def test_same_bits_again_and_in_a_graph(dtype, int8):
    """Results do not depend on timing; a captured call, replayed with eager work between, gives the eager bits; two graphs
    in turn too."""
    K = _k()
    pool = Groups([5, 4], [1500, 700], [1500 + 40 * i for i in range(5)] + [700 + 90 * i for i in range(4)], 2, 16, dtype, int8).cuda()
    q = torch.randn(9, 12, D, device=DEV).to(dtype)
    lens = torch.tensor(pool.lens, dtype=torch.int32, device=DEV)
    prefix = K.SharedPrefix(pool.sizes, pool.shared, 12, 2, DEV)

    def go():
        return K.decode_attn_shared(q, *pool.args(), lens, prefix, SM, **pool.scales())

    want = go()
    for _ in range(5):
        assert torch.equal(go(), want)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got = go()
        graphs.append((g, got))
    for i in range(6):
        q.copy_(torch.randn(9, 12, D, device=DEV).to(dtype))
        lens.sub_(1)
        want = go()
        g, got = graphs[i % 2]
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want), i


def test_many_rows_in_a_graph():
    """More than 64 rows, whose tails a launch of their own shares out: replays follow the lengths of the moment."""
    K = _k()
    pool = Groups([70], [128], [129 + 11 * i for i in range(70)], 2, 16, F16).cuda()
    q = torch.randn(70, 4, D, device=DEV).half()
    lens = torch.tensor(pool.lens, dtype=torch.int32, device=DEV)
    prefix = K.SharedPrefix(pool.sizes, pool.shared, 4, 2, DEV)
    K.decode_attn_shared(q, *pool.args(), lens, prefix, SM)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = K.decode_attn_shared(q, *pool.args(), lens, prefix, SM)
    for i in range(4):
        lens.copy_((torch.tensor(pool.lens, device=DEV) - 37 * i).clamp(min=128 if i < 3 else 0))
        want = K.decode_attn_shared(q, *pool.args(), lens, prefix, SM)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want), i


def test_another_stream():
    K = _k()
    pool = Groups([3], [640], [700, 640, 900], 2, 16, F16).cuda()
    q = torch.randn(3, 12, D, device=DEV).half()
    want = call(pool, q)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = call(pool, q)
        junk = [torch.full((1 << 16,), -1, dtype=torch.int32, device=DEV) for _ in range(4)]
    prefix = K.SharedPrefix(pool.sizes, pool.shared, 12, 2, DEV)
    with torch.cuda.stream(side):
        again = K.decode_attn_shared(q, *pool.args(), torch.tensor(pool.lens, device=DEV), prefix, SM)
    del prefix
    junk += [torch.full((1 << 10,), -1, dtype=torch.int32, device=DEV) for _ in range(64)]
    side.synchronize()
    assert torch.equal(got, want) and torch.equal(again, want)


def test_refusals():
    K = _k()
    pool = Groups([2], [32], [40, 50], 2, 16, F16).cuda()
    q = torch.randn(2, 12, D, device=DEV).half()
    lens = torch.tensor([40, 50], device=DEV)
    prefix = K.SharedPrefix([2], [32], 12, 2, DEV)
    ok = (q, *pool.args(), lens, prefix)
    K.decode_attn_shared(*ok)
    for i, bad in ((0, q[:1]), (0, q.float()), (0, q.bfloat16()), (0, q[:, :10]), (0, q[..., :64]), (0, q.cpu()), (3, pool.table[:1]),
                   (4, lens[:1]), (4, lens.float()), (5, K.SharedPrefix([2], [32], 12, 2, "cpu")), (5, K.SharedPrefix([1], [32], 12, 2, DEV)),
                   (5, K.SharedPrefix([2], [32], 6, 2, DEV)), (5, K.SharedPrefix([2], [32], 12, 1, DEV))):
        with pytest.raises((ValueError, TypeError)):
            K.decode_attn_shared(*[bad if j == i else x for j, x in enumerate(ok)])
    with pytest.raises(ValueError):
        K.decode_attn_shared(*ok, inv_tau=torch.ones(2, device=DEV))
    with pytest.raises(NotImplementedError):
        K.decode_attn_shared(q.clone().requires_grad_(), *ok[1:])
    empty = K.decode_attn_shared(q[:0], pool.k, pool.v, pool.table[:0], lens[:0], K.SharedPrefix([], [], 12, 2, DEV))
    assert empty.shape == (0, 12, D)
