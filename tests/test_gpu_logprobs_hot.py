"""token_logprobs at the ends of the temperatures that it takes, with logits as large as their type has them, and what it refuses
beyond them."""
import math

import pytest
import torch

from test_gpu_logprobs import TYPES, DEV, _k, check

pytestmark = pytest.mark.gpu


def extremes(rows, v, dtype, temperature):
    """Rows half of one lowest value, half of numbers up to as much above 0: differences, and their quotients with the
    temperature, are as large as fp32 has them."""
    g = torch.Generator().manual_seed(v)
    top = min(torch.finfo(dtype).max, 1.6e38 * min(temperature, 1.0))
    x = (torch.rand(rows, v, generator=g, dtype=torch.float64) * 2 - 1) * top
    x[torch.rand(rows, v, generator=g) < 0.5] = -top
    return x.to(dtype), torch.randint(v, (rows,), generator=g)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("temperature", [1e-30, 1e-20, 1.0, 1e20, 1e30])
@pytest.mark.parametrize("rows,v", [(3, 5003), (2, 100001)])
def test_temperatures_from_end_to_end(dtype, temperature, rows, v):
    check(*extremes(rows, v, dtype, temperature), 7, temperature)


def test_hot_and_cold_are_refused():
    x, t = extremes(3, 5003, torch.float32, 1.0)
    for temperature in (1e-31, 0.999e-30, 1.001e30, 1e31, 1e38, 1e300):
        with pytest.raises(ValueError):
            _k().token_logprobs(x.to(DEV), t.to(DEV), temperature=temperature)


def test_lowest_values_below_a_highest():
    """Logits further than fp32 goes below the row's largest have log probability -Inf, and add nothing to the rest."""
    x = torch.randn(3, 5003, generator=torch.Generator().manual_seed(1))
    x[:, ::3] = torch.finfo(torch.float32).min
    x[:, 5] = 1e38
    got = _k().token_logprobs(x.to(DEV), torch.tensor([5, 3, 4], device=DEV), 2, temperature=1e30)
    assert got.logprobs.tolist() == [0.0, -math.inf, pytest.approx(-1e8)] and not got.entropy.any()
    assert got.top_tokens[:, 0].tolist() == [5, 5, 5]
