"""The attention hook over an engine that attends prompts itself, on the CPU: which masks it takes, and what it hands
to the engine."""
import types

import pytest
import torch

from llm_kvcache_quantization_amd import patch as P

D, HQ, HKV = 16, 4, 2


class Engine:
    """Records what it is given; attends to nothing."""

    decode_attn_impl = "hip_fused"
    use_attn_temperature = True

    def __init__(self, past=0, inv_tau=None):
        self._layer_seq_lens = [past]
        self.inv_tau = inv_tau
        self.calls = []

    def get_seq_len(self):
        return self._layer_seq_lens[0]

    def get_paged_tensors(self, layer_id):
        raise AssertionError("not needed")

    def prefill_attn(self, layer_id, q, k, v, sm_scale=None, inv_tau=None):
        self.calls.append((q, k, v, inv_tau))
        return torch.zeros_like(q)

    def append_decode_attn(self, layer_id, q, k, v, sm_scale=None, inv_tau=None):
        self.calls.append((q, k, v, inv_tau))
        return torch.zeros_like(q)


def attention(dtype=torch.float32):
    torch.manual_seed(0)
    m = torch.nn.Module()
    m.head_dim, m.num_heads, m.num_key_value_heads, m.layer_idx = D, HQ, HKV, 0
    for name, out in (("q_proj", HQ * D), ("k_proj", HKV * D), ("v_proj", HKV * D)):
        setattr(m, name, torch.nn.Linear(32, out, bias=False))
    m.o_proj = torch.nn.Linear(HQ * D, 32, bias=False)
    return m.to(dtype)


def prompt(mask, q_len, past=0, batch=2, **kw):
    engine = Engine(past)
    x = torch.randn(batch, q_len, 32)
    rope = torch.ones(q_len, D), torch.zeros(q_len, D)
    wrapper = types.SimpleNamespace(engine=engine, layer_idx=0)
    out, _ = P._prefill_forward_impl(attention(), x, wrapper, attention_mask=mask, position_embeddings=rope)
    assert out.shape == x.shape and len(engine.calls) == 1


def causal(q_len, past=0, batch=2):
    return torch.ones(q_len, past + q_len, dtype=torch.bool).tril(past).expand(batch, 1, -1, -1)


def bias(seen, low):
    return torch.zeros(seen.shape).masked_fill(~seen, low)


@pytest.mark.parametrize("past", [0, 5])
def test_causal_masks_are_taken(past):
    seen = causal(7, past)
    lowest = torch.finfo(torch.float32).min
    for mask in (None, seen, seen[:1], seen[:, 0], bias(seen, lowest), bias(seen, -float("inf")), bias(seen, -65504.0).half(),
                 bias(seen, -1e4), torch.ones(2, past + 7, dtype=torch.long), torch.ones(2, past + 7, dtype=torch.bool)):
        prompt(mask, 7, past)


@pytest.mark.parametrize("past", [0, 5])
def test_other_masks_are_refused(past):
    """Whatever closes a key that causal attention sees, or opens one that it does not, in any row."""
    seen, low = causal(7, past), torch.finfo(torch.float32).min
    prefix = seen.clone()
    prefix[..., : past + 3] = True  # the first tokens see each other: the last row looks like a causal one's
    inner = seen.clone()
    inner[0, 0, 4, 1] = False
    window = seen & ~torch.ones(7, past + 7, dtype=torch.bool).tril(past - 3)
    left = seen.clone()
    left[1, ..., :2] = False
    last = seen.clone()
    last[..., -1, 0] = False
    everything = torch.ones_like(seen)
    slope = bias(seen, low) - 0.1 * torch.arange(past + 7)
    masks = [m if dtype else bias(m, low) for m in (prefix, inner, window, left, last, everything) for dtype in (True, False)]
    masks += [slope, bias(seen, -5.0), torch.nn.functional.pad(seen, (0, 2), value=True), causal(7, past + 2), seen[..., 1:, :],
              seen.long(), torch.full((2, past + 7), 2), torch.zeros(7)]
    if past:
        masks.append(causal(7))  # the tokens before are not in it
    pads = torch.ones(2, past + 7)
    pads[0, 1] = 0
    masks.append(pads)
    for i, mask in enumerate(masks):
        with pytest.raises(ValueError, match="padding"):
            prompt(mask, 7, past)
            raise AssertionError(f"mask {i} was taken")


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_steps_hand_over_what_prompts_do(dtype):
    """q in the model's type, beyond fp16's range too, and the temperature beside it in fp32."""
    tau = torch.rand(1, HQ) + 0.5
    m = attention(dtype)
    with torch.no_grad():
        m.q_proj.weight.mul_(1e4 if dtype == torch.float16 else 1e6)
    x = torch.randn(2, 1, 32).to(dtype)
    rope = torch.ones(1, D), torch.zeros(1, D)
    got = []
    for forward in (P._prefill_forward_impl, P._fused_forward_impl):
        engine = Engine(inv_tau=tau)
        forward(m, x, types.SimpleNamespace(engine=engine, layer_idx=0), position_embeddings=rope)
        got.append(engine.calls[0])
    (q0, k0, v0, t0), (q1, k1, v1, t1) = got
    assert q1.shape == (2, HQ, D) and q1.dtype == dtype and torch.equal(q1, q0[:, :, 0])
    assert dtype == torch.float16 or q1.abs().max() > 65504 and torch.isfinite(q1).all()
    assert torch.equal(k0, k1) and torch.equal(v0, v1)
    assert t0.dtype == t1.dtype == torch.float32 and torch.equal(t0, tau[0]) and torch.equal(t1, tau[0])


def test_an_unpatched_model_gets_no_windowed_cache():
    """`update` hands out all that is held, which a window does not see: refused before anything is appended."""
    import llm_kvcache_quantization_amd as K

    x = torch.zeros(1, 2, 3, 128, dtype=torch.float16)
    for kw, refused in ((dict(window=20), True), (dict(), False), (dict(budget=20), False)):
        engine = K.PagedKVCache(1, device="cpu", **kw)
        log = []
        engine.append = lambda layer, k, v: log.append(layer)
        engine.get_kv = lambda layer: (x, x)
        for cache in (P.INT8CacheWrapper(engine, 0), P.INT8CacheWrapperContainer(engine, 1)):
            if refused:
                with pytest.raises(ValueError, match="window"):
                    cache.update(x, x, 0)
            else:
                assert cache.update(x, x, 0) == (x, x)
        assert len(log) == (0 if refused else 2)
