"""Several answers from one prompt, as they are used together: PagedKVCache.fork with shared attention against caches that
share nothing, the hook, sample_from_ids and generate_from_ids with log probabilities.

Attention over a shared prefix and each by itself round their results once each and their probabilities once a token: two
results differ by at most twice the tolerance that test_gpu_paged derives, and both are held to it."""
import math

import pytest
import torch

from test_gpu_paged import BF16, D, DEV, F16, SM, check, reference, visible
from test_gpu_paged_engine import _tiny_lm

pytestmark = pytest.mark.gpu


def _k():
    import llm_kvcache_quantization_amd as K

    return K


def randn(*shape, dtype, g):
    return torch.randn(shape, generator=g).to(dtype).to(DEV)


@pytest.mark.parametrize("dtype,pages", [(F16, F16), (BF16, BF16), (F16, torch.int8), (BF16, torch.int8)])
@pytest.mark.parametrize("page", [16, 64])
def test_forked_steps(dtype, pages, page, monkeypatch):
    """Prompts, a fork into samples, steps, an uneven fork, steps: every step's attention against float64 over what get_kv
    says is held, and what is held against a cache that was given each sequence's tokens by itself."""
    K = _k()
    import llm_kvcache_quantization_amd.paged_cache as M

    print(f"[fork] {dtype} {pages} page {page}", flush=True)
    monkeypatch.setattr(M, "_MIN_SAVED", 1)
    monkeypatch.setattr(M, "_PATCHED", 1)
    monkeypatch.setattr(M, "_DEARER", dict.fromkeys(M._DEARER, 1.0))
    shared = []
    real = M.decode_attn_shared
    monkeypatch.setattr(M, "decode_attn_shared", lambda *a, **kw: (shared.append(a[5]), real(*a, **kw))[1])
    g = torch.Generator().manual_seed(page)
    hq, h, layers = 12, 2, 2
    cache = K.PagedKVCache(layers, device=DEV, dtype=pages, page_size=page)
    said = [[[] for _ in range(layers)] for _ in range(2)]  # k, v of each sequence, layer by layer
    seq = 333
    for layer in range(layers):
        k, v, q = (randn(2, n, seq, D, dtype=dtype, g=g) for n in (h, h, hq))
        cache.prefill_attn(layer, q, k, v, SM, lens=[seq, 290])
        for b, n in enumerate((seq, 290)):
            said[b][layer].append((k[b, :, :n], v[b, :, :n]))

    def fork(parents):
        cache.fork(parents)
        return [[list(x) for x in said[p]] for p in parents]

    def steps(n):
        for _ in range(n):
            for layer in range(layers):
                rows = len(said)
                k, v, q = (randn(rows, m, 1, D, dtype=dtype, g=g) for m in (h, h, hq))
                out = cache.append_decode_attn(layer, q.squeeze(2), k, v, SM)
                for b in range(rows):
                    said[b][layer].append((k[b], v[b]))
                kd, vd = cache.get_kv(layer)
                for b, held in enumerate(cache.get_seq_lens(layer)):
                    kk, vv = kd[b].double().cpu(), vd[b].double().cpu()
                    if pages == torch.int8:  # K's values are used as they are, not rounded to fp16
                        kp, _, ks, _, table, _ = cache.get_paged_tensors(layer)
                        t = torch.arange(kk.shape[1])
                        pg, sl = table[b].cpu()[(t // page).clamp(max=table.shape[1] - 1)].long(), t % page
                        kk = (kp.cpu()[pg, :, sl].double().unflatten(-1, (-1, 32)) * ks.cpu()[pg, :, sl].double().unsqueeze(-1)).flatten(-2).transpose(0, 1)
                        kk[:, held:] = 0
                    ref, tol, _, _ = reference(q[b, :, 0].cpu(), kk, vv, visible(held, kk.shape[1], None, 0), SM, dtype if pages == torch.int8 else pages,
                                               F16 if pages == torch.int8 else dtype, 0)
                    check(out[b], ref, tol, ("row", b, layer))

    said = fork([0, 0, 0, 1, 1])
    steps(3)
    assert shared and shared[-1].sizes == (3, 2) and shared[-1].lens == (seq // page * page, 290 // page * page)
    said = fork([1, 2, 4, 1])
    steps(page + 2)
    cache.compact()
    said = fork([3, 0, 2])
    steps(2)
    for layer in range(layers):
        kd, vd = cache.get_kv(layer)
        for b in range(len(said)):
            alone = K.PagedKVCache(1, device=DEV, dtype=pages, page_size=page)
            for k, v in said[b][layer]:
                alone.append(0, k[None], v[None])
            ka, va = alone.get_kv(0)
            n = ka.shape[2]
            assert torch.equal(kd[b, :, :n], ka[0]) and torch.equal(vd[b, :, :n], va[0]), (layer, b)


def test_fork_then_a_chunk():
    """A chunk of tokens behind a forked prompt: each sequence attends its own past."""
    K = _k()
    g = torch.Generator().manual_seed(4)
    c = K.PagedKVCache(1, device=DEV, dtype=F16, page_size=16)
    k, v, q = (randn(1, n, 70, D, dtype=F16, g=g) for n in (2, 2, 12))
    c.prefill_attn(0, q, k, v, SM)
    c.fork([0, 0, 0])
    k2, v2, q2 = (randn(3, n, 20, D, dtype=F16, g=g) for n in (2, 2, 12))
    out = c.prefill_attn(0, q2, k2, v2, SM)
    kk, vv = torch.cat([k.expand(3, -1, -1, -1), k2], 2).double().cpu(), torch.cat([v.expand(3, -1, -1, -1), v2], 2).double().cpu()
    for b in range(3):
        for i in (0, 7, 19):
            ref, tol, _, _ = reference(q2[b, :, i].cpu(), kk[b], vv[b], visible(71 + i, 90, None, 0), SM, F16, F16, 0)
            check(out[b, :, i], ref, tol, (b, i))


def test_budget_and_window_forks():
    """Forks of bounded caches go on like caches of their own."""
    K = _k()
    for kw in (dict(budget=40, sinks=2, recent=8, slack=4), dict(window=24, sinks=4)):
        g = torch.Generator().manual_seed(5)
        k, v, q = (randn(1, n, 60, D, dtype=F16, g=g) for n in (2, 2, 12))
        new = [[(randn(1, 2, 1, D, dtype=F16, g=g), randn(1, 2, 1, D, dtype=F16, g=g), randn(1, 12, D, dtype=F16, g=g)) for _ in range(2)]
               for _ in range(30)]
        c = K.PagedKVCache(1, device=DEV, dtype=F16, page_size=16, **kw)
        c.prefill_attn(0, q, k, v, SM)
        c.fork([0, 0])
        outs = []
        for step in new:
            kn, vn, qn = (torch.cat([s[i] for s in step]) for i in range(3))
            outs.append(c.append_decode_attn(0, qn, kn, vn, SM))
        for b in range(2):
            one = K.PagedKVCache(1, device=DEV, dtype=F16, page_size=16, **kw)
            one.prefill_attn(0, q, k, v, SM)
            for step, out in zip(new, outs):
                kn, vn, qn = step[b]
                want = one.append_decode_attn(0, qn, kn, vn, SM)
                # the same tokens in another split: both within the tolerance, of 60 values about 1 that is 2^-9 and less
                assert (want[0].float() - out[b].float()).abs().max() <= 2.0 ** -8, (kw, b)
            assert one.get_seq_lens() == [c.get_seq_lens()[b]]


# ---------------------------------------------------------------- through the model


class Tok:
    def __init__(self, eos):
        self.eos_token_id = eos


@pytest.mark.parametrize("dtype,kv", [(F16, None), (BF16, None), (F16, torch.int8)])
def test_samples_have_their_log_probabilities(dtype, kv, monkeypatch):
    """sample_from_ids: the samples' log probabilities, entropies and alternatives are those of the unpatched model run over
    prompt and sample; samples of one prompt differ; a seed draws the same again."""
    K = _k()
    import llm_kvcache_quantization_amd.paged_cache as M

    monkeypatch.setattr(M, "_MIN_SAVED", 1)
    monkeypatch.setattr(M, "_PATCHED", 1)
    monkeypatch.setattr(M, "_DEARER", dict.fromkeys(M._DEARER, 1.0))
    used = []
    real = M.decode_attn_shared
    monkeypatch.setattr(M, "decode_attn_shared", lambda *a, **kw: (used.append(a[5]), real(*a, **kw))[1])
    m = _tiny_lm(dtype)
    with torch.no_grad():
        m.lm_head.weight.div_(20.0)  # not so decisive
    ids = torch.randint(0, 211, (2, 70), generator=torch.Generator().manual_seed(9)).to(DEV)
    out = K.sample_from_ids(m, None, ids, num_samples=4, max_new_tokens=9, temperature=0.8, seed=3, top_logprobs=5, kv_dtype=kv, page_size=16)
    assert out.generated_ids.shape == (8, 9) and out.lengths == [9] * 8 and out.top_tokens.shape == (8, 9, 5)
    assert used and used[-1].sizes == (4, 4) and used[-1].lens == (64, 64)
    assert len({tuple(r) for r in out.generated_ids.tolist()}) > 2
    again = K.sample_from_ids(m, None, ids, num_samples=4, max_new_tokens=9, temperature=0.8, seed=3, top_logprobs=5, kv_dtype=kv, page_size=16)
    assert torch.equal(again.generated_ids, out.generated_ids) and torch.equal(again.logprobs, out.logprobs)
    with torch.no_grad():
        full = torch.cat([ids.repeat_interleave(4, 0), out.generated_ids], 1)
        logits = m(input_ids=full).logits[:, 69:-1].double() / 0.8
    lp = torch.log_softmax(logits, -1)
    want = lp.gather(-1, out.generated_ids.unsqueeze(-1)).squeeze(-1)
    # The model's own attention and the cache's differ by roundings of the type (and, INT8, of the cache) in two layers; logits
    # are of size 10 in the type: a few of its steps
    step = {F16: 2.0 ** -10, BF16: 2.0 ** -7}[dtype] * 16 * (4 if kv is not None else 1)
    assert (out.logprobs.double() - want).abs().max() <= step, (out.logprobs.double() - want).abs().max()
    H = -(lp.exp() * lp).sum(-1)
    assert (out.entropy.double() - H).abs().max() <= 2 * step * 6  # d H <= sum p |lp + H| |d lp|, sum p |lp + H| below 6
    assert (out.top_logprobs.double() - lp.gather(-1, out.top_tokens)).abs().max() <= step
    assert (out.top_logprobs.diff(dim=-1) <= 0).all()


def test_samples_end_and_leave(monkeypatch):
    """A sample ends with its eos; the others go on as they would have; behind the end there are eos and zeros."""
    K = _k()
    m = _tiny_lm(F16)
    with torch.no_grad():
        m.lm_head.weight.div_(20.0)
    ids = torch.randint(0, 211, (1, 40), generator=torch.Generator().manual_seed(2)).to(DEV)
    free = K.sample_from_ids(m, None, ids, num_samples=6, max_new_tokens=12, seed=1)
    eos = int(free.generated_ids[2, 4])
    out = K.sample_from_ids(m, Tok(eos), ids, num_samples=6, max_new_tokens=12, seed=1)
    for row, n in enumerate(out.lengths):
        got = out.generated_ids[row].tolist()
        assert eos not in got[: n - 1] and (n == 12 or got[n - 1] == eos)
        assert all(x == eos for x in got[n:]) and not out.logprobs[row, n:].any() and (out.logprobs[row, :n] <= 0).all()
    assert min(out.lengths) <= 5
    with torch.no_grad():
        for row, n in enumerate(out.lengths):
            full = torch.cat([ids, out.generated_ids[row : row + 1, :n]], 1)
            lp = torch.log_softmax(m(input_ids=full).logits[0, 39:-1].double(), -1)
            want = lp.gather(-1, out.generated_ids[row, :n].unsqueeze(-1)).squeeze(-1)
            assert (out.logprobs[row, :n].double() - want).abs().max() <= 2.0 ** -10 * 16, row
    assert K.sample_from_ids(m, Tok(eos), ids, num_samples=6, max_new_tokens=12, seed=1, stop_on_eos=False).lengths == [12] * 6


def test_samples_of_a_model_without_numbers():
    """Logits that are NaN draw some token each, whose log probability is NaN."""
    K = _k()
    m = _tiny_lm(F16)
    with torch.no_grad():
        m.lm_head.weight.fill_(math.nan)
    ids = torch.randint(0, 211, (1, 20), generator=torch.Generator().manual_seed(2)).to(DEV)
    out = K.sample_from_ids(m, None, ids, num_samples=3, max_new_tokens=4)
    assert ((out.generated_ids >= 0) & (out.generated_ids < 211)).all() and out.logprobs.isnan().all()


@pytest.mark.parametrize("temperature", [1e-29, 0.05, 1.0, 1e29])
def test_draws_follow_the_temperature(temperature):
    """4096 samples of one token: cold ones are the likeliest, others as often as their probability says, within 6
    deviations and 36 (Bernstein: one of 211 tokens beyond that by chance, below 1e-5)."""
    K = _k()
    m = _tiny_lm(F16)
    with torch.no_grad():
        m.lm_head.weight.div_(20.0)
    ids = torch.randint(0, 211, (1, 20), generator=torch.Generator().manual_seed(2)).to(DEV)
    n = 4096
    out = K.sample_from_ids(m, None, ids, num_samples=n, max_new_tokens=1, temperature=temperature)
    with torch.no_grad():
        logits = m(input_ids=ids).logits[0, -1].double()
    off = 2.0 ** -10 * 16  # by the attention's roundings (above), so that logits differ by twice that more or less
    if temperature < 0.01:
        assert (logits[out.generated_ids] >= logits.max() - 2 * off).all()
        return
    p = torch.softmax(logits / temperature, -1)
    seen = torch.bincount(out.generated_ids[:, 0], minlength=211).double()
    assert ((seen - n * p).abs() <= 6 * (n * p * (1 - p)).sqrt() + 36 + n * p * math.expm1(2 * off / temperature)).all()


def test_greedy_samples_are_the_models_tokens():
    K = _k()
    m = _tiny_lm(F16)
    ids = torch.randint(0, 211, (2, 40), generator=torch.Generator().manual_seed(9)).to(DEV)
    out = K.sample_from_ids(m, None, ids, num_samples=2, max_new_tokens=8, temperature=0.0)
    want = K.generate_from_ids(m, None, ids, max_new_tokens=8, kv_mode="fp16", top_logprobs=3)
    assert torch.equal(out.generated_ids, want.generated_ids.repeat_interleave(2, 0))
    assert torch.equal(want.top_tokens[..., 0], want.generated_ids)
    assert torch.equal(want.top_logprobs[..., 0], want.logprobs) and want.entropy.shape == (2, 8)
    assert (out.logprobs - want.logprobs.repeat_interleave(2, 0)).abs().max() <= 2.0 ** -10 * 320  # logits 20 times those above
    plain = K.generate_from_ids(m, None, ids, max_new_tokens=8, kv_mode="fp16")
    assert plain.logprobs is None and plain.top_tokens is None and torch.equal(plain.generated_ids, want.generated_ids)


def test_refusals():
    K = _k()
    m = _tiny_lm(F16)
    ids = torch.zeros(1, 4, dtype=torch.long, device=DEV)
    for kw in (dict(num_samples=0), dict(max_new_tokens=0), dict(temperature=-1.0), dict(temperature=math.inf), dict(top_logprobs=33),
               dict(top_logprobs=-1), dict(max_new_tokens=2000), dict(kv_dtype=torch.float32)):
        with pytest.raises(ValueError):
            K.sample_from_ids(m, None, ids, **kw)
    for t in (1e-31, 1e-320, 1e31, math.nan):
        with pytest.raises(ValueError):
            K.sample_from_ids(m, None, ids, temperature=t)
    with pytest.raises(TypeError):
        K.sample_from_ids(m, None, [[1, 2]])
    with pytest.raises(ValueError):
        K.sample_from_ids(m, None, ids[0])
    with pytest.raises(ValueError):
        K.generate_from_ids(m, None, ids, top_logprobs=33)
