"""PagedKVCache as it is used: prompts, chunks, decode steps, windows, eviction, the attention hook; and the
paged operators on other streams and in captured graphs.  Attention is compared with float64 over what the
cache should hold, with the tolerances derived in test_gpu_paged.py."""
import math

import pytest
import torch

from test_gpu_paged import BF16, F16, SM, Pool, check, quantize, reference, visible
from test_gpu_prefill_window import reference as prompt_reference

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
D = 128


def _k():
    import llm_kvcache_quantization_amd as K

    return K


def stored(x, int8):
    """float64 values of rows as the cache holds them."""
    if not int8:
        return x.double()
    c, s = quantize(x, int8)
    return (c.double().unflatten(-1, (-1, int8)) * s.double().unsqueeze(-1)).flatten(-2)


class Model:
    """What a cache of one layer should hold: K, V (as stored) and weights of every (sequence, head)."""

    def __init__(self, batch, heads, int8, budget=None, sinks=0, recent=0, slack=0):
        self.k = [[torch.empty(0, D, dtype=torch.float64) for _ in range(heads)] for _ in range(batch)]
        self.v = [[torch.empty(0, D, dtype=torch.float64) for _ in range(heads)] for _ in range(batch)]
        self.w = [[torch.empty(0, dtype=torch.float64) for _ in range(heads)] for _ in range(batch)]
        self.int8, self.budget, self.sinks, self.recent, self.slack = int8, budget, sinks, recent, slack

    def append(self, k, v, counts):
        k, v = stored(k.cpu(), self.int8), stored(v.cpu(), self.int8)
        for b, n in enumerate(counts):
            for h in range(k.shape[1]):
                self.k[b][h] = torch.cat([self.k[b][h], k[b, h, :n]])
                self.v[b][h] = torch.cat([self.v[b][h], v[b, h, :n]])
                self.w[b][h] = torch.cat([self.w[b][h], torch.zeros(n, dtype=torch.float64)])

    def held(self):
        return [len(r[0]) for r in self.k]

    def weigh(self, b, q, sm):
        rep = q.shape[0] // len(self.k[b])
        for h in range(len(self.k[b])):
            p = torch.softmax(q[h * rep : (h + 1) * rep].double() @ self.k[b][h].t() * sm, 1)
            self.w[b][h] += p.sum(0)

    def evict(self, slack):
        if self.budget is None or max(self.held()) <= self.budget + slack:
            return
        for b, n in enumerate(self.held()):
            if n <= self.budget:
                continue
            for h in range(len(self.k[b])):
                mid = torch.arange(self.sinks, n - self.recent)
                best = mid[self.w[b][h][mid].sort(descending=True, stable=True).indices[: self.budget - self.sinks - self.recent]]
                keep = torch.cat([torch.arange(self.sinks), best.sort().values, torch.arange(n - self.recent, n)])
                for x in (self.k, self.v, self.w):
                    x[b][h] = x[b][h][keep]


def same_rows(cache, model, int8):
    k, v = (x.cpu() for x in cache.get_kv(0))
    for b, n in enumerate(model.held()):
        for h in range(k.shape[1]):
            for got, want in ((k[b, h, :n], model.k[b][h]), (v[b, h, :n], model.v[b][h])):
                want = want.half() if int8 else want.to(k.dtype)
                assert torch.equal(got, want), (b, h)
        assert not k[b, :, n:].any() and not v[b, :, n:].any()


def draws(g, B, hq, hkv, S, dtype):
    q = torch.randn(B, hq, S, D, generator=g, device=DEV).to(dtype)
    k = (torch.randn(B, hkv, S, D, generator=g, device=DEV) * 1.5).to(dtype)
    v = torch.randn(B, hkv, S, D, generator=g, device=DEV).to(dtype)
    return q, k, v


@pytest.mark.parametrize("dtype,int8", [(F16, 0), (BF16, 0), (F16, 32), (BF16, 128)])
@pytest.mark.parametrize("window,sinks", [(None, 0), (40, 3)])
def test_prompt_chunk_and_steps(dtype, int8, window, sinks):
    K = _k()
    print(f"[engine] {dtype} {int8} {window}", flush=True)
    B, hq, hkv = 3, 6, 2
    c = K.PagedKVCache(1, device=DEV, dtype=torch.int8 if int8 else dtype, page_size=16, group_size=int8 or 32, window=window, sinks=sinks)
    m = Model(B, hkv, int8)
    g = torch.Generator(device=DEV).manual_seed(4)
    for S, lens in ((100, [100, 7, 55]), (30, [30, 30, 0])):
        q, k, v = draws(g, B, hq, hkv, S, dtype)
        before = m.held()
        out = c.prefill_attn(0, q, k, v, SM, lens=lens)
        for b, n in enumerate(lens):
            # earlier tokens as the cache holds them, the new ones as given
            kk = torch.cat([torch.stack(m.k[b]).to(DEV, torch.float32).half().double() if int8 else torch.stack(m.k[b]).to(DEV),
                            k[b, :, :n].double()], 1)
            vv = torch.cat([torch.stack(m.v[b]).to(DEV, torch.float32).half().double() if int8 else torch.stack(m.v[b]).to(DEV),
                            v[b, :, :n].double()], 1)
            if dtype == BF16 and int8 and before[b]:
                kk, vv = (torch.cat([x[:, : before[b]].to(BF16).double(), x[:, before[b]:]], 1) for x in (kk, vv))
            ref, tol = prompt_reference(q[b], kk.to(torch.float64), vv, n, before[b] + n, window, sinks)
            bad = (out[b].double() - ref).abs() - tol
            assert bad.max() <= 0, (S, b, float(bad.max()))
        m.append(k, v, lens)
        assert c.get_seq_lens() == m.held()
    for step in range(20):
        q, k, v = draws(g, B, hq, hkv, 1, dtype)
        out = c.append_decode_attn(0, q[:, :, 0], k, v, SM)
        m.append(k, v, [1] * B)
        if step % 5 == 4:
            for b, n in enumerate(m.held()):
                ref, tol, _, _ = reference(q[b, :, 0].cpu(), torch.stack(m.k[b]), torch.stack(m.v[b]), visible(n, n, window, sinks), SM, dtype,
                                           F16 if int8 else dtype, int8)
                check(out[b], ref, tol, (step, b))
    if window is None:
        same_rows(c, m, int8)
    else:  # pages out of sight went back to the pool
        assert any(p < 0 for r in c._rows for p in r)
        assert sum(p >= 0 for r in c._rows for p in r) + len(c._free) == c._total
    assert c.get_seq_len() == 150
    c.clear()
    assert c.get_seq_len() == 0 and c.get_memory_mb() > 0
    c.release()
    assert c.get_memory_mb() == 0


@pytest.mark.parametrize("dtype,int8", [(F16, 0), (F16, 64)])
def test_budget(dtype, int8):
    """The cache keeps what a float64 simulation of its weights keeps, step by step."""
    K = _k()
    print(f"[engine] budget {dtype} {int8}", flush=True)
    B, hq, hkv = 2, 4, 2
    kw = dict(budget=48, sinks=4, recent=12, slack=8)
    c = K.PagedKVCache(1, device=DEV, dtype=torch.int8 if int8 else dtype, page_size=16, group_size=int8 or 32, **kw)
    m = Model(B, hkv, int8, **kw)
    g = torch.Generator(device=DEV).manual_seed(5)
    q, k, v = draws(g, B, hq, hkv, 70, dtype)
    lens = [70, 33]
    c.prefill_attn(0, q, k, v, SM, lens=lens)
    m.append(k, v, lens)
    for b, n in enumerate(lens):
        m.weigh(b, q[b, :, n - 1].cpu(), SM)
    m.evict(0)
    assert c.get_seq_lens() == m.held() == [48, 33]
    same_rows(c, m, int8)
    for step in range(60):
        q, k, v = draws(g, B, hq, hkv, 1, dtype)
        out = c.append_decode_attn(0, q[:, :, 0], k, v, SM)
        m.append(k, v, [1] * B)
        for b, n in enumerate(m.held()):
            if step % 7 == 0:
                ref, tol, _, _ = reference(q[b, :, 0].cpu(), torch.stack(m.k[b]), torch.stack(m.v[b]), visible(n, n, None, 0), SM, dtype, F16, int8)
                check(out[b], ref, tol, (step, b))
            m.weigh(b, q[b, :, 0].cpu(), SM)
        m.evict(kw["slack"])
        assert c.get_seq_lens() == m.held(), step
    same_rows(c, m, int8)
    assert c.get_seq_len() == 130 and max(c.get_seq_lens()) <= 56
    assert len(c._rows[0]) <= 5  # pages behind the budget went back


def test_layers_share_the_table_and_the_pool_grows():
    K = _k()
    c = K.PagedKVCache(3, device=DEV, page_size=16)
    g = torch.Generator(device=DEV).manual_seed(6)
    parts = [[] for _ in range(3)]
    for S in (5, 40, 1, 1, 200):
        for layer in range(3):
            _, k, v = draws(g, 2, 2, 2, S, F16)
            c.append(layer, k, v)
            parts[layer].append((k, v))
    for layer in range(3):
        k, v = c.get_kv(layer)
        assert torch.equal(k, torch.cat([p[0] for p in parts[layer]], 2))
        assert torch.equal(v, torch.cat([p[1] for p in parts[layer]], 2))
    assert len(c.to_tuple()) == 3


def test_engine_refusals():
    K = _k()
    c = K.PagedKVCache(1, device=DEV, num_pages=2, page_size=16)
    x = torch.zeros(1, 2, 20, D, device=DEV, dtype=F16)
    c.append(0, x, x)
    with pytest.raises(RuntimeError, match="out of pages"):
        c.append(0, x, x)
    assert c.get_seq_lens() == [20]
    with pytest.raises(ValueError, match="sequences"):
        c.append(0, x.expand(2, -1, -1, -1), x.expand(2, -1, -1, -1))
    with pytest.raises(ValueError, match="pages' type"):
        c.append(0, x.bfloat16(), x.bfloat16())
    with pytest.raises(ValueError, match="one token"):
        c.append_decode_attn(0, x[:, :, 0], x, x)
    with pytest.raises(ValueError, match="q must be"):
        c.prefill_attn(0, x[:, :, :3], x, x)


def test_refused_step_appends_nothing():
    K = _k()
    eng = K.PagedKVCache(1, dtype=torch.int8)
    k = torch.randn(2, 2, 5, 128, device=DEV, dtype=torch.float16)
    eng.append(0, k, k)
    one = k[:, :, :1]
    for q, error in ((k.new_zeros(2, 34, 128), NotImplementedError), (k.new_zeros(2, 4, 64), ValueError),
                     (k.new_zeros(2, 3, 128), ValueError), (torch.zeros(2, 4, 128), ValueError), (k.new_zeros(1, 4, 128), ValueError),
                     (torch.zeros(2, 4, 128, device=DEV), ValueError)):
        with pytest.raises(error):
            eng.append_decode_attn(0, q, one, one)
        assert eng.get_seq_lens(0) == [5, 5] and eng.get_seq_len() == 5
    out = eng.append_decode_attn(0, k.new_zeros(2, 4, 128), one, one)
    torch.cuda.synchronize()
    assert eng.get_seq_lens(0) == [6, 6] and torch.isfinite(out).all()


def test_operator_refusals():
    """What needs GPU tensors to be seen."""
    K = _k()
    k = torch.zeros(4, 2, 16, D, device=DEV, dtype=F16)
    table = torch.zeros(1, 2, device=DEV, dtype=torch.int32)
    lens = torch.ones(1, device=DEV, dtype=torch.int32)
    q = torch.zeros(1, 4, D, device=DEV, dtype=F16)
    x = torch.zeros(1, 2, 3, D, device=DEV, dtype=F16)
    i8 = k.to(torch.int8)
    sc = torch.ones(4, 2, 16, 4, device=DEV, dtype=F16)
    w = torch.zeros(1, 2, 32, device=DEV)
    dec = K.decode_attn_paged
    for bad in (lambda: dec(q.bfloat16(), k, k, table, lens), lambda: dec(q.float(), k, k, table, lens),
                lambda: dec(q[:, :3], k, k, table, lens), lambda: dec(q, k.float(), k.float(), table, lens),
                lambda: dec(q, k[:, :, :12], k[:, :, :12], table, lens), lambda: dec(q, k, k.bfloat16(), table, lens),
                lambda: dec(q, k, k, table.long(), lens), lambda: dec(q, k, k, table.cpu(), lens),
                lambda: dec(q, k, k, table[0], lens), lambda: dec(q, k, k, table.expand(2, -1), lens),
                lambda: dec(q, k, k, table, lens[:0]), lambda: dec(q, k, k, table, lens.float()),
                lambda: dec(q, i8, i8, table, lens), lambda: dec(q, i8, i8, table, lens, k_scale=sc, v_scale=sc.float()),
                lambda: dec(q, i8, i8, table, lens, k_scale=sc[..., :3], v_scale=sc[..., :3]),
                lambda: dec(q, i8, i8, table, lens, k_scale=sc.transpose(0, 1).contiguous().transpose(0, 1)[..., ::2], v_scale=sc),
                lambda: dec(q, k, k, table, lens, k_scale=sc, v_scale=sc), lambda: dec(q, k, k, table, lens, window=0),
                lambda: dec(q, k, k, table, lens, sinks=-1), lambda: dec(q, k, k, table, lens, weights=w[:, :, :31]),
                lambda: dec(q, k, k, table, lens, weights=w.half()), lambda: dec(q, k, k, table, lens, weights=w[:, :1].expand(-1, 2, -1)),
                lambda: dec(q, k, k, table, lens, inv_tau=torch.ones(3, device=DEV)),
                lambda: dec(q, torch.zeros(4, 2, 16, D + 4, device=DEV, dtype=F16)[..., 4:], k, table, lens),
                lambda: dec(q, k.transpose(2, 3).contiguous().transpose(2, 3), k, table, lens),
                lambda: K.append_paged(x.float(), x.float(), k, k.clone(), table, lens),
                lambda: K.append_paged(x.bfloat16(), x.bfloat16(), k, k.clone(), table, lens),
                lambda: K.append_paged(x[:, :1], x[:, :1], k, k.clone(), table, lens),
                lambda: K.append_paged(x, x, k, k.clone(), table, lens, lens[:0]),
                lambda: K.evict_paged(k, k, table, lens, w, 0), lambda: K.evict_paged(k, k, table, lens, w, 4, sinks=3, recent=2),
                lambda: K.evict_paged(k, k, table, lens, w[:, :1], 4),
                lambda: K.prefill_attn_window(x.bfloat16(), x, x), lambda: K.prefill_attn_window(x, x, x, window=0),
                lambda: K.prefill_attn_window(x, x, x, q_lens=lens.expand(2)),
                lambda: K.prefill_attn_window(torch.cat([x, x[:, :1]], 1), x, x)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(NotImplementedError):
        dec(torch.zeros(1, 34, D, device=DEV, dtype=F16), k, k, table, lens)  # 17 query heads a KV head
    with pytest.raises(NotImplementedError, match="backward"):
        dec(q.clone().requires_grad_(), k, k, table, lens)
    with torch.no_grad():
        dec(q.clone().requires_grad_(), k, k, table, lens)
    with pytest.raises(NotImplementedError, match="4096"):
        dec(q.expand(4097, -1, -1), k, k, table.expand(4097, -1).contiguous(), lens.expand(4097).contiguous())


# ---------------------------------------------------------------- streams and graphs


def _operands(seed, weights=True):
    lens = [900, 33, 0, 2100]
    pool = Pool(lens, 2, 16, F16, 0, seed)
    T = pool.cols * 16
    pool.fill(lambda b: visible(lens[b], T, None, 0)).cuda()
    g = torch.Generator().manual_seed(seed)
    q = torch.randn(4, 8, D, generator=g).half().to(DEV)
    w = torch.rand(4, 2, T, generator=g).to(DEV) if weights else None
    new = torch.randn(2, 4, 2, 1, D, generator=g).half().to(DEV)
    return pool, q, torch.tensor(lens, dtype=torch.int32, device=DEV), w, new


def _step(pool, q, lens, w, new, budget=500):
    """One token appended, attended with weights, and the cache cut down: all four outputs."""
    K = _k()
    K.append_paged(new[0], new[1], *pool.args(), lens)
    n = lens + 1
    out = K.decode_attn_paged(q, *pool.args(), n, SM, weights=w)
    return (out, *K.evict_paged(*pool.args(), n, w, budget, sinks=4, recent=50))


def test_no_gradients():
    """Whatever would want a gradient is refused where autograd records, and taken as data where it does not."""
    K = _k()
    q = torch.randn(1, 2, 128, device=DEV, dtype=torch.float16)
    pages = [torch.randn(3, 2, 16, 128, device=DEV, dtype=torch.float16) for _ in range(2)]
    x = torch.randn(1, 2, 4, 128, device=DEV, dtype=torch.float16)
    table, lens = torch.tensor([[2, 0]], dtype=torch.int32, device=DEV), torch.tensor([20], device=DEV)
    w, tau = torch.zeros(1, 2, 32, device=DEV), torch.ones(2, device=DEV)

    def calls(grad):
        def g(name, t):
            return t.clone().requires_grad_(name == grad)

        k, v = g("k_pages", pages[0]), g("v_pages", pages[1])
        return {"append": (lambda: K.append_paged(g("x", x), x, k, v, table, lens), ("x", "k_pages", "v_pages")),
                "decode": (lambda: K.decode_attn_paged(g("q", q), k, v, table, lens, inv_tau=g("tau", tau), weights=g("w", w)),
                           ("q", "k_pages", "v_pages", "tau", "w")),
                "prefill": (lambda: K.prefill_attn_window(g("x", x), x, x, inv_tau=g("tau", tau)), ("x", "tau")),
                "evict": (lambda: K.evict_paged(k, v, table, lens, g("w", w), 8), ("k_pages", "v_pages", "w"))}

    for name in calls(""):
        for grad in calls("")[name][1]:
            with pytest.raises(NotImplementedError):
                calls(grad)[name][0]()
            with torch.no_grad():
                calls(grad)[name][0]()
    torch.cuda.synchronize()


def test_other_streams_and_two_calls_at_once():
    print("[streams]", flush=True)
    want = []
    for seed in (1, 2):
        ops = _operands(seed)
        want.append([x.clone() for x in _step(*ops)] + [ops[0].k.clone(), ops[0].v.clone()])
    torch.cuda.synchronize()
    for _ in range(3):
        got, streams = [], [torch.cuda.Stream(), torch.cuda.Stream()]
        all_ops = [_operands(1), _operands(2)]
        torch.cuda.synchronize()
        for s, ops in zip(streams, all_ops):
            with torch.cuda.stream(s):
                got.append(_step(*ops))
        torch.cuda.synchronize()
        for g, w, ops in zip(got, want, all_ops):
            for a, b in zip((*g, ops[0].k, ops[0].v), w):
                assert torch.equal(torch.nan_to_num(a.float()), torch.nan_to_num(b.float()))


def test_captured_graphs():
    """Two graphs of a step and one of a prompt, replayed in turn between eager calls: every replay gives the
    eager results for the inputs it finds."""
    K = _k()
    print("[graphs]", flush=True)
    a, b = _operands(3), _operands(4)
    q, k, v = draws(torch.Generator(device=DEV).manual_seed(9), 1, 4, 2, 70, F16)
    long_k, long_v = (torch.randn(1, 2, 5000, D, device=DEV).half() for _ in range(2))
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):  # warm-up
        _step(*_operands(5))
        K.prefill_attn_window(q, long_k, long_v, SM)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for ops in (a, b):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(_step(*ops))
        graphs.append(g)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        prompt = K.prefill_attn_window(q, long_k, long_v, SM)
    for rnd in range(4):
        for i, (graph, ops, seed) in enumerate(zip(graphs, (a, b), (3, 4))):
            fresh = _operands(seed + 10 * rnd)
            for dst, src in zip((ops[0].k, ops[0].v, ops[0].table, *ops[1:]), (fresh[0].k, fresh[0].v, fresh[0].table, *fresh[1:])):
                dst.copy_(src)
            want = _step(*fresh)
            graph.replay()
            torch.cuda.synchronize()
            for x, y in zip(outs[i], want):
                assert torch.equal(x, y), (rnd, i)
            assert torch.equal(torch.nan_to_num(ops[0].k), torch.nan_to_num(fresh[0].k))
        q.normal_()
        want = K.prefill_attn_window(q, long_k, long_v, SM)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(prompt, want)


def test_same_inputs_same_bits():
    pool, q, lens, _, _ = _operands(7, weights=False)
    K = _k()
    outs = [K.decode_attn_paged(q, *pool.args(), lens, SM) for _ in range(5)]
    assert all(torch.equal(o, outs[0]) for o in outs)


# ---------------------------------------------------------------- the attention hook


def _tiny_lm(dtype, seed=3):
    from transformers import Qwen2Config, Qwen2ForCausalLM

    torch.manual_seed(seed)
    cfg = Qwen2Config(vocab_size=211, hidden_size=512, intermediate_size=1024, num_hidden_layers=2, num_attention_heads=4,
                      num_key_value_heads=2, max_position_embeddings=1024)
    cfg._attn_implementation = "sdpa"
    m = Qwen2ForCausalLM(cfg)
    with torch.no_grad():
        m.lm_head.weight.mul_(30.0)  # decisive argmax: greedy tokens are stable
    return m.to(dtype).to(DEV).eval()


def _generate(model, engine, ids, steps):
    K = _k()
    cache = K.INT8CacheWrapperContainer(engine, 2)
    K.apply_int8_fused_patch(model)
    try:
        with torch.no_grad():
            out = model(input_ids=ids, past_key_values=cache, use_cache=True)
            toks = [out.logits[:, -1].argmax(-1)]
            for _ in range(steps - 1):
                out = model(input_ids=toks[-1].view(-1, 1), past_key_values=cache, use_cache=True)
                toks.append(out.logits[:, -1].argmax(-1))
    finally:
        K.remove_int8_fused_patch(model)
    return torch.stack(toks, 1)


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_hook_generates_the_models_tokens(dtype):
    """Prompt and decode steps through the patched model over fp16 / bf16 pages give the unpatched model's tokens,
    and so do a window and a budget that the sequence stays within."""
    K = _k()
    print(f"[hook] {dtype}", flush=True)
    m = _tiny_lm(dtype)
    ids = torch.randint(0, 211, (2, 40), generator=torch.Generator().manual_seed(9)).to(DEV)
    with torch.no_grad():
        toks, cur = [], ids
        for _ in range(8):
            toks.append(m(input_ids=cur).logits[:, -1].argmax(-1))
            cur = torch.cat([cur, toks[-1].view(-1, 1)], 1)
    want = torch.stack(toks, 1)
    for kw in (dict(), dict(window=100, sinks=4), dict(budget=100)):
        engine = K.PagedKVCache(2, device=DEV, dtype=dtype, page_size=16, **kw)
        got = _generate(m, engine, ids, 8)
        assert torch.equal(got, want), (kw, got.tolist(), want.tolist())
        assert engine.get_seq_len() == 47 and engine.get_decode_stats()["fused_decode_calls"] == 14


def test_hook_bounded_generation():
    """A window and a budget shorter than the sequence: positions go on, what is held stays bounded."""
    K = _k()
    m = _tiny_lm(F16)
    ids = torch.randint(0, 211, (1, 120), generator=torch.Generator().manual_seed(9)).to(DEV)
    for kw in (dict(window=32, sinks=4), dict(budget=32, sinks=4)):
        for dt in (F16, torch.int8):
            engine = K.PagedKVCache(2, device=DEV, dtype=dt, page_size=16, **kw)
            out = _generate(m, engine, ids, 40)
            assert out.shape == (1, 40) and engine.get_seq_len() == 159
            assert sum(p >= 0 for p in engine._rows[0]) <= 5, engine._rows
            if "budget" in kw:
                assert engine.get_seq_lens()[0] <= 32 + 16


def test_hook_refuses_padding():
    K = _k()
    m = _tiny_lm(F16)
    ids = torch.randint(0, 211, (2, 20), generator=torch.Generator().manual_seed(9)).to(DEV)
    mask = torch.ones_like(ids)
    mask[0, :5] = 0
    K.apply_int8_fused_patch(m)
    try:
        with torch.no_grad(), pytest.raises(ValueError, match="padding"):
            m(input_ids=ids, attention_mask=mask, use_cache=True,
              past_key_values=K.INT8CacheWrapperContainer(K.PagedKVCache(2, device=DEV), 2))
    finally:
        K.remove_int8_fused_patch(m)
