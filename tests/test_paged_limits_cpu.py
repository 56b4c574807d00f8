"""Limits of the paged operators that are refused on the host, on the CPU: sizes whose counters would leave 32 bits,
lengths that do not fit int32, and what would carry a derivative."""
import pytest
import torch

from test_paged_cpu import _append, _cache, _evict, _lib, _refused


class OnGpu(torch.Tensor):
    """A CPU tensor that passes for one of a GPU: what is refused before anything is enqueued."""

    is_cuda = True


def gpu(x):
    return x.as_subclass(OnGpu)


def pages():
    return gpu(torch.zeros(4, 2, 16, 128, dtype=torch.float16))


def test_budgets_and_weights_past_2_30():
    """A work-group's places pass the end by its share: they are counted in 32 bits."""
    import llm_kvcache_quantization_amd as K

    C, L = _lib()
    c = _cache(C)
    for over in (dict(budget=2 ** 31 - 1), dict(budget=2 ** 30 + 1), dict(w_tokens=2 ** 31 - 1), dict(w_tokens=2 ** 30 + 1)):
        _refused(L, "kvq_paged_evict", _evict(C, c, **over))
    k, table, lens = pages(), gpu(torch.zeros(1, 2, dtype=torch.int32)), gpu(torch.ones(1, dtype=torch.int32))
    w = gpu(torch.zeros(1, 2, 32))
    for budget in (2 ** 30 + 1, 2 ** 31 - 1, 2 ** 31, 2 ** 40):
        with pytest.raises(ValueError, match="2.30"):
            K.evict_paged(k, k, table, lens, w, budget)


def test_more_new_tokens_than_2_30():
    """One row repeated 2^31 - 1 times is a view of 256 bytes: the places past its end wrapped to negative ones."""
    C, L = _lib()
    for n in (2 ** 30 + 1, 2 ** 31 - 1):
        p = _append(C, _cache(C, batch=1, kv_heads=1), seq_new=n, k_stride_s=0, v_stride_s=0)
        _refused(L, "kvq_paged_append", p)
        assert b"2^30" in L.kvq_last_error()


def test_lengths_that_do_not_fit_int32():
    """They stand for what they say: behind every table, or in front of it."""
    from llm_kvcache_quantization_amd.paged import _i32

    cpu, far = torch.device("cpu"), [2 ** 32 + 5, -2 ** 40, 7, 2 ** 31, -2 ** 31 - 1, 2 ** 63 - 1]
    got = _i32(torch.tensor(far), "lens", 6, cpu)
    assert got.dtype == torch.int32 and got.tolist() == [2 ** 31 - 1, -2 ** 31, 7, 2 ** 31 - 1, -2 ** 31, 2 ** 31 - 1]
    assert _i32(torch.tensor([2 ** 32 - 1, 5], dtype=torch.int64).to(torch.uint32), "lens", 2, cpu).tolist() == [2 ** 31 - 1, 5]
    for t in (torch.int8, torch.uint8, torch.int16, torch.int32):
        assert _i32(torch.tensor([3, 100], dtype=t), "lens", 2, cpu).tolist() == [3, 100]
    for t in (torch.float32, torch.bool, torch.uint64, torch.complex64):
        with pytest.raises(ValueError, match="integers"):
            _i32(torch.zeros(2).to(t), "lens", 2, cpu)


def test_tensors_with_a_tangent():
    """Forward differentiation, whether or not gradients are recorded."""
    from torch.autograd import forward_ad

    import llm_kvcache_quantization_amd as K

    k, table, lens = pages(), gpu(torch.zeros(1, 2, dtype=torch.int32)), gpu(torch.ones(1, dtype=torch.int32))
    q, x, w, tau = (torch.randn(s) for s in ((1, 4, 128), (1, 2, 3, 128), (1, 2, 32), (4,)))
    q, x = q.half(), x.half()
    with forward_ad.dual_level():
        dual = lambda t: gpu(forward_ad.make_dual(t, torch.ones_like(t)))  # noqa: E731
        x0, q0 = gpu(x), gpu(q)
        for call in (lambda: K.append_paged(dual(x), x0, k, k, table, lens),
                     lambda: K.decode_attn_paged(dual(q), k, k, table, lens),
                     lambda: K.decode_attn_paged(q0, k, k, table, lens, inv_tau=dual(tau)),
                     lambda: K.decode_attn_paged(q0, dual(torch.zeros(4, 2, 16, 128).half()), k, table, lens),
                     lambda: K.prefill_attn_window(gpu(x.repeat(1, 2, 1, 1)), dual(x), x0),
                     lambda: K.evict_paged(k, k, table, lens, dual(w), 1)):
            for recorded in (True, False):
                with torch.set_grad_enabled(recorded), pytest.raises(NotImplementedError, match="tangent"):
                    call()


def test_scales_that_want_a_gradient():
    import llm_kvcache_quantization_amd as K

    i8 = gpu(torch.zeros(4, 2, 16, 128, dtype=torch.int8))
    table, lens = gpu(torch.zeros(1, 2, dtype=torch.int32)), gpu(torch.ones(1, dtype=torch.int32))
    q, x, w = (gpu(torch.zeros(s).half()) for s in ((1, 4, 128), (1, 2, 3, 128), (1, 2, 32)))
    for side in ("k_scale", "v_scale"):
        sc = {n: gpu(torch.ones(4, 2, 16, 4).half().requires_grad_(n == side)) for n in ("k_scale", "v_scale")}
        for call in (lambda: K.append_paged(x, x, i8, i8, table, lens, **sc), lambda: K.decode_attn_paged(q, i8, i8, table, lens, **sc),
                     lambda: K.evict_paged(i8, i8, table, lens, w.float(), 1, **sc)):
            with pytest.raises(NotImplementedError, match="backward"):
                call()


def test_written_pages_have_memory_of_their_own():
    """Expanded pages or heads may be read; who writes them would write one place from several work-groups."""
    C, L = _lib()
    for over in (dict(k_stride_p=0), dict(v_stride_p=0), dict(k_stride_h=0), dict(v_stride_h=0)):
        for int8 in (False, True):
            c = _cache(C, int8, **over)
            _refused(L, "kvq_paged_append", _append(C, c))
            assert b"stride of 0" in L.kvq_last_error()
            _refused(L, "kvq_paged_evict", _evict(C, c))
            assert b"stride of 0" in L.kvq_last_error()
    for over in (dict(ks_stride_p=0), dict(vs_stride_p=0), dict(ks_stride_h=0), dict(vs_stride_h=0)):
        _refused(L, "kvq_paged_append", _append(C, _cache(C, True, **over)))
        assert b"stride of 0" in L.kvq_last_error()
    # one page, one head: their strides mean nothing
    c = _cache(C, num_pages=1, kv_heads=1, k_stride_p=0, v_stride_p=0, k_stride_h=0, v_stride_h=0)
    import ctypes

    assert L.kvq_paged_append(ctypes.byref(_append(C, c, seq_new=0)), None) == 0
