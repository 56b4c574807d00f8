"""PagedKVCache on the GPU: refused calls, layers in every order, bounds that bind in several layers, types.

Attention is compared with float64 over what the cache should hold, with the tolerances derived in
test_gpu_paged.py."""
import math

import pytest
import torch

from test_gpu_paged import BF16, F16, SM

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
D = 128


def _k():
    import llm_kvcache_quantization_amd as K

    return K


@pytest.mark.parametrize("budget", [None, 40])
@pytest.mark.parametrize("dtype", [F16, torch.int8])
def test_refused_prompts_and_steps_change_nothing(budget, dtype):
    """A retry after a refusal gives what a cache that never saw the refused call gives, bit for bit."""
    K = _k()
    print(f"[refusals] {budget} {dtype}", flush=True)
    g = torch.Generator(device=DEV).manual_seed(2)
    c, clean = (K.PagedKVCache(1, device=DEV, dtype=dtype, page_size=16, budget=budget) for _ in range(2))
    draw = lambda *s: torch.randn(*s, generator=g, device=DEV).half()  # noqa: E731
    for S in (30, 25):
        q, k, v = draw(2, 4, S, D), draw(2, 2, S, D), draw(2, 2, S, D)
        bad = [dict(q=q.bfloat16()), dict(q=q.float()), dict(q=q.cpu()), dict(q=q[:, :3]), dict(q=q[..., :64]), dict(k=k[:, :1]),
               dict(inv_tau=torch.ones(3, device=DEV)), dict(q=q.clone().requires_grad_()), dict(k=k.clone().requires_grad_()),
               dict(lens=[S, S + 1]), dict(lens=[S]), dict(v=v.float()), dict(v=v[:, :, :-1])]
        if budget:
            bad.append(dict(q=torch.zeros(2, 34, S, D, device=DEV, dtype=F16)))
        for kw in bad:
            with pytest.raises((ValueError, NotImplementedError)):
                c.prefill_attn(0, **dict(dict(q=q, k=k, v=v), **kw))
            assert c.get_seq_lens() == clean.get_seq_lens() and c.get_seq_len() == clean.get_seq_len(), kw.keys()
        assert torch.equal(c.prefill_attn(0, q, k, v, SM), clean.prefill_attn(0, q, k, v, SM))
        for step in range(12):
            q, k, v = draw(2, 4, D), draw(2, 2, 1, D), draw(2, 2, 1, D)
            bad = [dict(q=q.float()), dict(q=q[:, :3]), dict(q=q.clone().requires_grad_()), dict(inv_tau=torch.ones(3, device=DEV)),
                   dict(q=torch.zeros(2, 34, D, device=DEV, dtype=F16)), dict(inv_tau=torch.ones(4, device=DEV).requires_grad_()),
                   dict(k=k.clone().requires_grad_()), dict(v=v[:, :1])]
            with pytest.raises((ValueError, NotImplementedError)):
                c.append_decode_attn(0, **dict(dict(q=q, k=k, v=v), **bad[step % len(bad)]))
            assert c.get_seq_lens() == clean.get_seq_lens() and c.get_seq_len() == clean.get_seq_len(), step
            assert torch.equal(c.append_decode_attn(0, q, k, v, SM), clean.append_decode_attn(0, q, k, v, SM)), step
    for a, b in zip(c.get_kv(0), clean.get_kv(0)):
        assert torch.equal(a, b)


def test_refused_batch_of_too_many_rows():
    K = _k()
    c = K.PagedKVCache(1, device=DEV, page_size=16)
    one = torch.zeros(4097, 1, 1, D, device=DEV, dtype=F16)
    with pytest.raises(NotImplementedError, match="4096"):
        c.append_decode_attn(0, one[:, :, 0], one, one)
    assert c.get_seq_len() == 0
    c.append(0, one[:2], one[:2])
    assert c.get_seq_lens() == [1, 1]


@pytest.mark.parametrize("pages", [BF16, torch.int8])
def test_bf16_queries_of_a_step_beyond_fp16(pages):
    """Queries of 2^20 against keys of 2^-20: a step attends as a prompt of the same token does."""
    K = _k()
    g = torch.Generator(device=DEV).manual_seed(3)
    f = 2.0 ** 20 if pages == BF16 else 2.0 ** 10  # INT8 scales are fp16
    q, k, v = (torch.randn(2, h, 40, D, generator=g, device=DEV) for h in (4, 2, 2))
    q, k, v = (q * f * 2.0 ** 7).to(BF16), (k / f * 2.0 ** -7).to(BF16), v.to(BF16)
    assert q.abs().max() > 65504
    c = K.PagedKVCache(1, device=DEV, dtype=pages, page_size=16)
    for i in range(40):
        out = c.append_decode_attn(0, q[:, :, i], k[:, :, i : i + 1], v[:, :, i : i + 1], SM)
    kd, vd = (x.double() for x in c.get_kv(0))
    for h in range(4):
        s = (kd[:, h // 2] * q[:, h, 39:40].double()).sum(-1) * SM
        p = torch.softmax(s, -1)
        want = (p.unsqueeze(-1) * vd[:, h // 2]).sum(1)
        # the output's rounding (2^-8), P's in bf16 or fp16 and V's in fp16 (2^-8 at most each), all below |v| < 5
        assert (out[:, h].double() - want).abs().max() <= 3 * 5 * 2.0 ** -8


def test_lengths_in_64_bits():
    """Lengths and positions of 2^32 and more are behind the table, not at their low 32 bits."""
    K = _k()
    g = torch.Generator(device=DEV).manual_seed(1)
    k, v = (torch.randn(3, 2, 16, D, generator=g, device=DEV).half() for _ in range(2))
    q = torch.randn(2, 4, D, generator=g, device=DEV).half()
    table = torch.tensor([[2, 0], [1, 2]], dtype=torch.int32, device=DEV)
    lens = torch.tensor([32, 9], device=DEV)
    want = K.decode_attn_paged(q, k, v, table, lens.int())
    far = torch.tensor([2 ** 32 + 5, 9], device=DEV)
    assert torch.equal(K.decode_attn_paged(q, k, v, table, far), want)
    assert not K.decode_attn_paged(q, k, v, table, far - 2 ** 40)[0].any()
    x = torch.randn(2, 2, 4, D, generator=g, device=DEV).half()
    was = k.clone()
    K.append_paged(x, x, k, v, table, torch.tensor([2 ** 32, 2 ** 32 + 9], device=DEV))
    assert torch.equal(k, was)
    out = K.prefill_attn_window(x, x, x, q_lens=torch.tensor([2 ** 33, 2], device=DEV), kv_lens=torch.tensor([2 ** 32, 2], device=DEV))
    assert torch.equal(out, K.prefill_attn_window(x, x, x, q_lens=torch.tensor([4, 2], device=DEV), kv_lens=torch.tensor([4, 2], device=DEV)))


@pytest.mark.parametrize("dtype", [F16, torch.int8])
def test_a_windowed_chunk_takes_memory_for_the_window(dtype):
    """A chunk after 40000 tokens gives what it gives after the last of them alone, in memory that does not follow the
    history."""
    K = _k()
    g = torch.Generator(device=DEV).manual_seed(5)
    c, short = (K.PagedKVCache(1, device=DEV, dtype=dtype, page_size=64, window=200) for _ in range(2))
    k, v = (torch.randn(2, 2, 40000, D, generator=g, device=DEV).half() for _ in range(2))
    c.append(0, k, v)
    short.append(0, k[:, :, 39936 - 256 :], v[:, :, 39936 - 256 :])  # a whole number of pages fewer
    for S in (70, 300):
        q, kn, vn = (torch.randn(2, h, S, D, generator=g, device=DEV).half() for h in (4, 2, 2))
        want = short.prefill_attn(0, q, kn, vn, SM)
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        out = c.prefill_attn(0, q, kn, vn, SM)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        # K and V of 200 + 63 + S tokens in a few copies (INT8: one in fp32), and what the attention itself takes
        rows = 2 * 2 * (264 + S) * D
        assert torch.cuda.max_memory_allocated() - before <= 16 * 4 * rows + (8 << 20), S
