"""The boundary of copies, shared attention and log probabilities, on the CPU: include/kvq_shared.h and kvq_logprobs.h
against their ctypes mirrors, what the entry points refuse before anything is enqueued (made-up addresses: nothing reads
them), and the plan of a shared prefix."""
import ctypes
import re
import subprocess
from pathlib import Path

import pytest
import torch

from test_paged_cpu import AT, CACHE_FAULTS, INT8_FAULTS, _cache, _lib

ROOT = Path(__file__).resolve().parents[1]
STRUCTS = {"kvq_shared.h": {"kvq_page_pool": "PagePool", "kvq_copy_pages_params": "CopyPagesParams",
                            "kvq_shared_plan_info": "SharedPlanInfo", "kvq_shared_decode_params": "SharedDecodeParams"},
           "kvq_logprobs.h": {"kvq_token_logprobs_params": "TokenLogprobsParams"}}


def test_headers_and_exports():
    C, L = _lib()
    for header, symbols in (("kvq_shared.h", C.SHARED_SYMBOLS), ("kvq_logprobs.h", C.LOGPROBS_SYMBOLS)):
        names = set(re.findall(r"^\s*(?:int|int64_t)\s+(kvq_\w+)\(", (ROOT / "include" / header).read_text(), re.M))
        assert names == set(symbols)
        assert all(hasattr(L, n) for n in names)


@pytest.mark.parametrize("header", STRUCTS)
def test_struct_layouts(tmp_path, header):
    from llm_kvcache_quantization_amd import _capi as C

    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{header}"', "int main(void){"]
    for s, py in STRUCTS[header].items():
        lines.append(f'printf("{s} size %zu\\n", sizeof({s}));')
        lines += [f'printf("{s} {f} %zu\\n", offsetof({s}, {f.rstrip("_")}));' for f, _ in getattr(C, py)._fields_]
    (tmp_path / "p.c").write_text("\n".join(lines + ["return 0;}"]))
    subprocess.run(["gcc", "-I", str(ROOT / "include"), str(tmp_path / "p.c"), "-o", str(tmp_path / "p")], check=True)
    out = subprocess.run([str(tmp_path / "p")], capture_output=True, text=True, check=True).stdout
    got = {tuple(x.split()[:2]): int(x.split()[2]) for x in out.splitlines()}
    for s, py in STRUCTS[header].items():
        cls = getattr(C, py)
        assert got[(s, "size")] == ctypes.sizeof(cls)
        for f, _ in cls._fields_:
            assert got[(s, f)] == getattr(cls, f).offset, (s, f)


def test_packed_blocks_are_the_structs():
    from llm_kvcache_quantization_amd import _capi as C
    from llm_kvcache_quantization_amd import paged, scoring, shared

    for cls, packer in ((C.CopyPagesParams, shared._COPY), (C.SharedDecodeParams, shared._SHARED), (C.TokenLogprobsParams, scoring._LOGPROBS)):
        values = list(range(1, len(list(paged._leaves(cls))) + 1))
        block = cls.from_buffer_copy(packer.pack(*values))

        def flat(s):
            for name, t in s._fields_:
                x = getattr(s, name)
                if isinstance(x, ctypes.Structure):
                    yield from flat(x)
                else:
                    yield x

        assert [int(x) for x in flat(block)] == values


def _refused(L, fn, p):
    rc = getattr(L, fn)(ctypes.byref(p), None)
    assert rc in (1, 2), rc
    assert L.kvq_last_error()


def _pool(C, **over):
    x = C.PagePool()
    x.base, x.stride_p, x.stride_h, x.stride_t, x.row_bytes = AT, 4 * 16 * 256, 16 * 256, 256, 256
    for k, v in over.items():
        setattr(x, k, v)
    return x


def _copy(C, pools=None, into=None, **over):
    p = C.CopyPagesParams()
    keep = [(C.PagePool * 1)(pools or _pool(C)), (C.PagePool * 1)(into or pools or _pool(C))]
    p.from_, p.to = (ctypes.addressof(k) for k in keep)
    p.src = p.dst = AT
    p.n_pools, p.pairs, p.page_size, p.heads, p.from_pages, p.to_pages = 1, 3, 16, 4, 10, 10
    for k, v in over.items():
        setattr(p, k, v)
    p.keep = keep
    return p


def test_bad_copies_are_refused():
    C, L = _lib()
    for over in (dict(n_pools=-1), dict(pairs=-1), dict(heads=0), dict(heads=4097), dict(page_size=8), dict(page_size=48),
                 dict(page_size=512), dict(from_pages=-1), dict(to_pages=-1), dict(src=None), dict(dst=None), dict(from_=None), dict(to=None)):
        _refused(L, "kvq_copy_pages", _copy(C, **over))
    for over in (dict(base=None), dict(base=AT + 8), dict(stride_p=100), dict(stride_h=8), dict(stride_t=240), dict(stride_t=260),
                 dict(row_bytes=0), dict(row_bytes=1), dict(row_bytes=96), dict(row_bytes=2048), dict(stride_p=-4096),
                 dict(row_bytes=8), dict(stride_p=1 << 40)):
        _refused(L, "kvq_copy_pages", _copy(C, _pool(C, **over)))
    for over in (dict(stride_p=0), dict(stride_h=0), dict(row_bytes=128, stride_t=128)):  # of what is written
        _refused(L, "kvq_copy_pages", _copy(C, _pool(C), _pool(C, **over)))
    for over in (dict(n_pools=0), dict(pairs=0), dict(from_pages=0), dict(to_pages=0)):  # nothing to do
        assert L.kvq_copy_pages(ctypes.byref(_copy(C, **over)), None) == 0
    assert L.kvq_copy_pages(None, None) == 1


def _decode(C, cache, **over):
    p = C.SharedDecodeParams()
    p.cache = cache
    p.q = p.out = p.context_lens = p.workspace = p.plan_words = AT
    p.q_stride_b, p.q_stride_h, p.q_heads = 8 * 128, 128, 8
    p.workspace_bytes = 1 << 40
    p.sm_scale = 0.1
    p.plan = C.SharedPlanInfo(cache.batch, 2, 48, 40)
    for k, v in over.items():
        setattr(p, k, v)
    return p


@pytest.mark.parametrize("fault", CACHE_FAULTS + [dict(k_stride_p=1 << 33)], ids=str)
def test_a_bad_cache_is_refused(fault):
    C, L = _lib()
    _refused(L, "kvq_shared_decode", _decode(C, _cache(C, **fault)))


@pytest.mark.parametrize("fault", INT8_FAULTS, ids=str)
def test_a_bad_int8_cache_is_refused(fault):
    C, L = _lib()
    _refused(L, "kvq_shared_decode", _decode(C, _cache(C, True, **fault)))


def test_bad_shared_calls_are_refused():
    C, L = _lib()
    c = _cache(C)
    for over in (dict(q_type=7), dict(q_type=C.KVQ_PAGED_BF16), dict(q_heads=6), dict(q_heads=0), dict(q_heads=4 * 129), dict(q=None),
                 dict(out=None), dict(context_lens=None), dict(plan_words=None), dict(q=AT + 8), dict(q_stride_h=132), dict(workspace=None),
                 dict(workspace_bytes=64), dict(workspace=AT + 4), dict(plan=C.SharedPlanInfo(2, 2, 48, 32)),
                 dict(plan=C.SharedPlanInfo(3, -1, 48, 32)), dict(plan=C.SharedPlanInfo(3, 1 << 24, 48, 32)),
                 dict(plan=C.SharedPlanInfo(3, 2, 1 << 30, 32))):
        _refused(L, "kvq_shared_decode", _decode(C, c, **over))
    big = _cache(C, batch=4097)
    _refused(L, "kvq_shared_decode", _decode(C, big))
    assert L.kvq_shared_decode_workspace_bytes(ctypes.byref(_decode(C, c))) > 0
    assert L.kvq_shared_decode_workspace_bytes(ctypes.byref(_decode(C, big))) == 0
    assert L.kvq_shared_decode(None, None) == 1


def _words(K, *args):
    p = K.SharedPrefix(*args, device="cpu")
    return p, p._words.view(-1, 8).tolist()


@pytest.mark.parametrize("sizes,lens", [([16], [8176]), ([1], [5]), ([3, 1, 7], [0, 64, 1000]), ([100, 29], [65, 4096]), ([4096], [16]),
                                        ([2, 2], [0, 0]), ([64], [32768]), ([1, 33, 5], [100000, 63, 64])])
@pytest.mark.parametrize("q_heads,kv_heads", [(28, 4), (12, 2), (128, 1), (1, 1), (40, 8)])
def test_plan_covers_every_column_and_token_once(sizes, lens, q_heads, kv_heads):
    import llm_kvcache_quantization_amd as K

    p, words = _words(K, sizes, lens, q_heads, kv_heads)
    rep = q_heads // kv_heads
    rows, units, slots, n = p._info
    assert rows == sum(sizes) == p.rows and n == 8 * (rows + units) == p._words.numel()
    plan, work = words[:rows], words[rows:]
    seen, taken = {}, set()
    row = 0
    for size, length in zip(sizes, lens):
        for i in range(size):
            assert plan[row + i][:2] == [row, length] and plan[row + i][5] == size * rep
        row += size
    for row0, col0, cols, t0, t1, length, slot, _ in work:
        assert 0 < cols <= 128 and t0 < t1 and plan[row0][1] == length
        for t in range(t0, t1):
            for c0 in range(col0, col0 + cols, 32):  # blocks of whole waves' columns
                assert (row0, c0, t) not in seen
                seen[(row0, c0, t)] = 1
        places = set(range(slot, slot + cols))
        assert not places & taken
        taken |= places
    assert len(taken) == slots and (not taken or taken == set(range(slots)))
    row = 0
    for size, length in zip(sizes, lens):
        tiles, blocks = -(-length // 64), -(-size * rep // 32)
        mine = [k for k in seen if k[0] == row]
        assert len(mine) == tiles * blocks
        # where the join looks for a column's parts
        _, _, slot, splits, per, cols = plan[row][:6]
        for c in {0, cols // 2, cols - 1} if splits else ():
            c0 = c // per * per
            width = min(per, cols - c0)
            units_of = sorted((w[3], w[6] + c - w[1]) for w in work if w[0] == row and w[1] == c0)
            assert [s for _, s in units_of] == [slot + c0 * splits + s * width + c - c0 for s in range(splits)]
        row += size


def test_plans_are_refused():
    import llm_kvcache_quantization_amd as K

    _lib()
    for args in (([1], [1, 2], 4, 2), ([0], [1], 4, 2), ([1], [-1], 4, 2), ([1], [1], 5, 2), ([1], [1], 0, 2), ([1], [1], 4, 0),
                 ([1 << 40], [1], 4, 2)):
        with pytest.raises(ValueError):
            K.SharedPrefix(*args, device="cpu")
    for args in (([4097], [1], 4, 2), ([1], [(1 << 30) + 1], 4, 2), ([1], [1], 129, 1)):
        with pytest.raises(NotImplementedError):
            K.SharedPrefix(*args, device="cpu")


def _logprobs(C, **over):
    p = C.TokenLogprobsParams()
    p.logits = p.tokens = p.logprobs = p.entropy = p.top_logprobs = p.top_tokens = p.workspace = AT
    p.row_stride, p.rows, p.vocab, p.top, p.logits_type, p.inv_temperature = 200000, 3, 200000, 5, C.KVQ_LOGITS_BF16, 1.0
    p.workspace_bytes = 1 << 40
    for k, v in over.items():
        setattr(p, k, v)
    return p


def test_bad_log_probability_calls_are_refused():
    C, L = _lib()
    for over in (dict(rows=-1), dict(vocab=0), dict(vocab=(1 << 28) + 1), dict(top=-1), dict(top=33), dict(top=5, vocab=4), dict(logits_type=3),
                 dict(logits_type=-1), dict(inv_temperature=0.0), dict(inv_temperature=-1.0), dict(inv_temperature=float("nan")),
                 dict(inv_temperature=float("inf")), dict(logits=None), dict(entropy=None), dict(logprobs=None), dict(top_logprobs=None),
                 dict(top_tokens=None), dict(logits=AT + 1), dict(logits=AT + 2, logits_type=C.KVQ_LOGITS_F32), dict(workspace=None),
                 dict(workspace_bytes=8), dict(workspace=AT + 4), dict(rows=1 << 24)):
        _refused(L, "kvq_token_logprobs", _logprobs(C, **over))
    assert L.kvq_token_logprobs(ctypes.byref(_logprobs(C, rows=0)), None) == 0
    assert L.kvq_token_logprobs(None, None) == 1
    assert L.kvq_token_logprobs_workspace_bytes(ctypes.byref(_logprobs(C))) > 0
    assert L.kvq_token_logprobs_workspace_bytes(ctypes.byref(_logprobs(C, rows=5000))) == 0  # a work-group a row: nothing to join


def test_the_operators_need_a_gpu():
    import llm_kvcache_quantization_amd as K

    with pytest.raises(ValueError):
        K.PagePools([torch.zeros(4, 2, 16, 128, dtype=torch.float16)])
    with pytest.raises(ValueError):
        K.token_logprobs(torch.zeros(2, 10))
    with pytest.raises(ValueError):
        K.PagePools([])
