"""The draw of sample_from_ids: temperatures down to the coldest, rows without numbers, and how often each token comes."""
import ctypes
import math

import pytest
import torch

from llm_kvcache_quantization_amd.modes import _draw


def draw(x, temperature, seed=1, device="cpu"):
    return _draw(x.to(device), temperature, torch.Generator(device=device).manual_seed(seed)).cpu()


@pytest.mark.parametrize("temperature", [1.0000001e-30, 1e-29, 1e-20, 1e-3])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_cold_draws_are_the_likeliest(temperature, dtype):
    """Logits of several thousand, of either sign, with one that leads by 32 and more: 32000 temperatures."""
    x, best = leading(4096.0, dtype)
    assert torch.equal(draw(x, temperature), best)


@pytest.mark.parametrize("dtype,top,temperature", [(torch.float32, 2.0 ** 33, 1e-29), (torch.bfloat16, 2.0 ** 40, 1e-29),
                                                   (torch.bfloat16, 2.0 ** 127, 0.125), (torch.float32, 2.0 ** 127, 0.1)])
def test_logits_whose_quotient_passes_fp32(dtype, top, temperature):
    x, best = leading(top, dtype)
    assert torch.equal(draw(x, temperature), best)


def test_temperatures_that_are_taken():
    """The same from 1e-30 to 1e30 everywhere: sample_from_ids looks before the prompt runs, kvq_token_logprobs at the inverse in
    fp32 (rows of 0: nothing is launched)."""
    from llm_kvcache_quantization_amd import sample_from_ids
    from test_shared_cpu import _lib, _logprobs

    C, L = _lib()
    ends = [1e-30, math.nextafter(1e-30, 1), 1.00000002e-30, 1.0, 9.9999998e29, math.nextafter(1e30, 0), 1e30]
    for t in ends:
        assert L.kvq_token_logprobs(ctypes.byref(_logprobs(C, rows=0, inv_temperature=1.0 / t)), None) == 0, t
    for t in (0.99e-30, 1.01e30, 1e37):
        assert L.kvq_token_logprobs(ctypes.byref(_logprobs(C, rows=0, inv_temperature=1.0 / t)), None) == 1, t
        with pytest.raises(ValueError, match="temperature"):
            sample_from_ids(None, None, torch.zeros(1, 4, dtype=torch.long), temperature=t)
    if not torch.cuda.is_available():
        for t in ends:
            with pytest.raises(RuntimeError, match="GPU"):
                sample_from_ids(None, None, torch.zeros(1, 4, dtype=torch.long), temperature=t)


def leading(top, dtype):
    """Rows of whole multiples of top / 512, of which one is above all others: some rows all positive or none, some masked."""
    g = torch.Generator().manual_seed(2)
    x = torch.randint(-100, 100, (64, 211), generator=g).float()
    best = torch.randint(211, (64,), generator=g)
    x[1::4] -= 112
    x[2::4] += 112
    x = x / 256 * (top / 2)
    x[3::4, :7] = -math.inf
    others = x.scatter(1, best[:, None], -math.inf).amax(1)
    x.scatter_(1, best[:, None], (others + top / 64)[:, None])
    return x.to(dtype), best


def test_rows_without_numbers_draw_a_token():
    x = torch.zeros(4, 211)
    x[0] = math.nan
    x[1] = -math.inf
    x[2, 5] = math.inf
    x[3, 5] = math.nan
    for t in (0.0, 1e-29, 1.0, 1e29):
        got = draw(x, t)
        assert ((got >= 0) & (got < 211)).all()


def chi_square(seen, p):
    """(sum of (seen - n p)^2 / n p, its degrees of freedom); tokens expected fewer than 50 times are counted with the last of
    the others."""
    want, order = (seen.sum() * p).sort(descending=True)
    seen, cells = seen[order], int((want >= 50).sum())
    seen, want = (torch.cat([x[: cells - 1], x[cells - 1 :].sum(0, keepdim=True)]) for x in (seen, want))
    return float(((seen - want) ** 2 / want).sum()), cells - 1


@pytest.mark.parametrize("temperature", [0.3, 1.0, 1.7, 1e29])
@pytest.mark.parametrize("device,n", [("cpu", 1 << 16), pytest.param("cuda:0", 1 << 20, marks=pytest.mark.gpu)])
def test_every_token_comes_as_often_as_its_probability_says(device, n, temperature):
    """A chi-square of k degrees of freedom is above k + 2 sqrt(20 k) + 40 with a probability below e^-20.  (A draw from a third
    of 211 tokens alike would have 2 n, one that never draws one of them n / 211.)"""
    logits = torch.randn(211, generator=torch.Generator().manual_seed(3)) * 1.5
    p = torch.softmax(logits.double() / temperature, 0)
    seen = torch.bincount(draw(logits.expand(n, -1), temperature, 5, device), minlength=211).double()
    value, k = chi_square(seen, p)
    assert value <= k + 2 * math.sqrt(20 * k) + 40, (value, k)


def test_the_chi_square_sees_a_wrong_draw():
    p = torch.softmax(torch.randn(211, generator=torch.Generator().manual_seed(3)).double(), 0)
    n = 1 << 16
    for wrong in (lambda x: x % 70, lambda x: torch.where(x == 100, 101, x)):
        value, k = chi_square(torch.bincount(wrong(torch.multinomial(p, n, replacement=True, generator=torch.Generator().manual_seed(1))), minlength=211).double(), p)
        assert value > k + 2 * math.sqrt(20 * k) + 40


def test_more_rows_than_a_step_takes_are_refused_before_the_prompt_runs():
    from llm_kvcache_quantization_amd import sample_from_ids

    for batch, n in ((1, 4097), (2, 2049), (4097, 1)):
        with pytest.raises(ValueError, match="4096"):
            sample_from_ids(None, None, torch.zeros(batch, 4, dtype=torch.long), num_samples=n, max_new_tokens=2)
    if not torch.cuda.is_available():  # no step comes after the first token
        with pytest.raises(RuntimeError, match="GPU"):
            sample_from_ids(None, None, torch.zeros(1, 4, dtype=torch.long), num_samples=4097, max_new_tokens=1)
        with pytest.raises(RuntimeError, match="GPU"):
            sample_from_ids(None, None, torch.zeros(2, 4, dtype=torch.long), num_samples=2048)
