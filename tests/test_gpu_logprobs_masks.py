"""token_logprobs of rows that a grammar masks at random, a few tokens of a hundred left: rows of several work-groups, of one,
and rows that no vector load divides, against float64 as in test_gpu_logprobs (whose tolerances hold for any logits).  Inputs
are made on the CPU."""
import math

import pytest
import torch

from test_gpu_logprobs import TYPES, check

pytestmark = pytest.mark.gpu


def masked(rows, v, dtype, seed, share, lowest=False):
    """Logits of which a share is masked at random, by -Inf or the type's lowest value, with 24 likely tokens a row."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, v, generator=g) * 2
    x.masked_fill_(torch.rand(rows, v, generator=g) < share, torch.finfo(dtype).min if lowest else -math.inf)
    likely = torch.rand(rows, v, generator=g).argsort(1)[:, :24]
    x.scatter_(1, likely, torch.rand(likely.shape, generator=g) * 8)
    return x.to(dtype), torch.where(torch.rand(rows, generator=g) < 0.7, likely[:, 0], torch.randint(v, (rows,), generator=g))


@pytest.mark.parametrize("seed", range(4))
def test_random_masks_over_unaligned_rows(seed):
    check(*masked(77, 50257, torch.float32, seed, 0.95), 5)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,v", [(1, 32000), (3, 151936), (500, 4099)])
@pytest.mark.parametrize("share", [0.5, 0.95, 0.9999])
@pytest.mark.parametrize("lowest", [False, True])
def test_random_masks(dtype, rows, v, share, lowest):
    check(*masked(rows, v, dtype, rows, share, lowest), 20)
