"""The paged operators at values that a softmax has none for, and at those far below its largest, against float64."""
import math

import pytest
import torch

from test_gpu_paged import BF16, F16, SM, Pool, visible

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
D = 128


def _k():
    import llm_kvcache_quantization_amd as K

    return K


@pytest.mark.parametrize("int8", [0, 64])
@pytest.mark.parametrize("slots", [None, 4000])  # one work-group a row, and split
def test_weights_of_tokens_that_are_not_seen(int8, slots):
    """A row whose softmax is none (a NaN, an infinite score) gives NaN weights to the tokens it sees; those outside its window
    and on pages that are not there get nothing, in its tiles too."""
    K = _k()
    print(f"[unseen] {int8} {slots}", flush=True)
    lens, window, sinks = [90, 90, 90, 90], 50, 3
    pool = Pool(lens, 2, 16, F16, int8, seed=3, slots=slots)
    T = pool.cols * 16
    vis = [visible(n, T, window, sinks) for n in lens]
    pool.fill(lambda b: vis[b])
    vis[2][48:64] = False  # its page is gone
    pool.table[2, 3] = -1
    q = torch.randn(4, 6, D, generator=torch.Generator().manual_seed(4)).half()
    q[0, 1, 5] = math.nan   # one head of a row
    q[1] = math.inf
    q[2, :, 7] = -math.inf
    pool.cuda()
    w = torch.rand(4, 2, T + 4, generator=torch.Generator().manual_seed(5)).to(DEV)
    was = w.clone()
    K.decode_attn_paged(q.to(DEV), *pool.args(), torch.tensor(lens, device=DEV), SM, **pool.scales(), window=window, sinks=sinks, weights=w)
    torch.cuda.synchronize()
    for b in range(4):
        seen = torch.nn.functional.pad(vis[b], (0, 4)).to(DEV)
        assert torch.equal(w[b][:, ~seen], was[b][:, ~seen]), b
        nan = torch.isnan(w[b][:, seen])
        if b == 0:  # query heads 0 to 2 are KV head 0's
            assert nan[0].all() and not nan[1].any()
        elif b == 3:
            assert not nan.any() and (w[b][:, seen] > was[b][:, seen]).all()
        else:
            assert nan.all()
