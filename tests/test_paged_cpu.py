"""The paged cache's boundary, on the CPU: include/kvq_paged.h against its ctypes mirrors, and what the entry
points refuse before anything is enqueued (made-up addresses: nothing reads them)."""
import ctypes
import re
import subprocess
from pathlib import Path

import pytest
import torch

ROOT = Path(__file__).resolve().parents[1]
HEADER = ROOT / "include" / "kvq_paged.h"
AT = 1 << 20


def _lib():
    from llm_kvcache_quantization_amd import _capi as C

    if not C.LIB_PATH.exists():
        pytest.skip("libkvq.so not built (run __graft_entry__.build())")
    return C, C.lib()


STRUCTS = {"kvq_paged_cache": "PagedCache", "kvq_paged_append_params": "PagedAppendParams",
           "kvq_paged_decode_params": "PagedDecodeParams", "kvq_prefill_params": "PrefillParams",
           "kvq_paged_evict_params": "PagedEvictParams"}


def test_header_and_exports():
    C, L = _lib()
    names = set(re.findall(r"^\s*(?:int|int64_t)\s+(kvq_\w+)\(", HEADER.read_text(), re.M))
    assert names == set(C.PAGED_SYMBOLS)
    assert all(hasattr(L, n) for n in names)


def test_struct_layouts(tmp_path):
    from llm_kvcache_quantization_amd import _capi as C

    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "kvq_paged.h"', "int main(void){"]
    for s, py in STRUCTS.items():
        lines.append(f'printf("{s} size %zu\\n", sizeof({s}));')
        lines += [f'printf("{s} {f} %zu\\n", offsetof({s}, {f}));' for f, _ in getattr(C, py)._fields_]
    (tmp_path / "p.c").write_text("\n".join(lines + ["return 0;}"]))
    subprocess.run(["gcc", "-I", str(ROOT / "include"), str(tmp_path / "p.c"), "-o", str(tmp_path / "p")], check=True)
    out = subprocess.run([str(tmp_path / "p")], capture_output=True, text=True, check=True).stdout
    got = {tuple(x.split()[:2]): int(x.split()[2]) for x in out.splitlines()}
    for s, py in STRUCTS.items():
        cls = getattr(C, py)
        assert got[(s, "size")] == ctypes.sizeof(cls)
        for f, _ in cls._fields_:
            assert got[(s, f)] == getattr(cls, f).offset, (s, f)


def test_packed_blocks_are_the_structs():
    """One pack() of the fields in order gives the struct's bytes."""
    from llm_kvcache_quantization_amd import _capi as C
    from llm_kvcache_quantization_amd import paged as P

    for py, packer in (("PagedAppendParams", P._APPEND), ("PagedDecodeParams", P._DECODE), ("PrefillParams", P._PREFILL),
                       ("PagedEvictParams", P._EVICT)):
        cls = getattr(C, py)
        values = list(range(1, len(list(P._leaves(cls))) + 1))
        block = cls.from_buffer_copy(packer.pack(*values))

        def flat(s):
            for name, t in s._fields_:
                x = getattr(s, name)
                if isinstance(x, ctypes.Structure):
                    yield from flat(x)
                else:
                    yield x

        assert [int(x) for x in flat(block)] == values


def _cache(C, int8=False, **over):
    c = C.PagedCache()
    row = 128 if int8 else 256
    c.k = c.v = AT
    c.k_stride_t = c.v_stride_t = row
    c.k_stride_h = c.v_stride_h = 16 * row
    c.k_stride_p = c.v_stride_p = 64 * row
    c.table, c.table_stride = AT, 8
    c.num_pages, c.max_pages, c.page_size = 100, 8, 16
    c.batch, c.kv_heads = 3, 4
    if int8:
        c.format, c.group_size = C.KVQ_PAGED_INT8, 32
        c.k_scale = c.v_scale = AT
        c.ks_stride_h = c.vs_stride_h = 128
        c.ks_stride_p = c.vs_stride_p = 512
    for k, v in over.items():
        setattr(c, k, v)
    return c


CACHE_FAULTS = [dict(page_size=8), dict(page_size=48), dict(page_size=512), dict(format=3), dict(format=-1), dict(k=None),
                dict(table=None), dict(k=AT + 8), dict(v_stride_t=264), dict(k_stride_t=128), dict(v_stride_p=100),
                dict(k_stride_t=1 << 23), dict(kv_heads=0), dict(batch=-1), dict(num_pages=-1), dict(max_pages=-2),
                dict(max_pages=1 << 28)]
INT8_FAULTS = [dict(group_size=16), dict(group_size=0), dict(k_scale=None), dict(v_scale=AT + 2), dict(ks_stride_p=100),
               dict(v_stride_h=2052)]


def _append(C, cache, **over):
    p = C.PagedAppendParams()
    p.cache = cache
    p.k = p.v = p.write_pos = AT
    p.seq_new = 5
    p.k_stride_b = p.v_stride_b = 4 * 5 * 128
    p.k_stride_h = p.v_stride_h = 5 * 128
    p.k_stride_s = p.v_stride_s = 128
    for k, v in over.items():
        setattr(p, k, v)
    return p


def _decode(C, cache, **over):
    p = C.PagedDecodeParams()
    p.cache = cache
    p.q = p.out = p.context_lens = p.workspace = AT
    p.q_stride_b, p.q_stride_h, p.q_heads = 8 * 128, 128, 8
    p.workspace_bytes = 1 << 40
    p.sm_scale = 0.1
    for k, v in over.items():
        setattr(p, k, v)
    return p


def _evict(C, cache, **over):
    p = C.PagedEvictParams()
    p.cache = cache
    p.context_lens = p.weights = p.new_lens = p.kept = p.new_weights = AT
    p.w_tokens, p.budget, p.sinks, p.recent = 128, 50, 4, 10
    for k, v in over.items():
        setattr(p, k, v)
    return p


def _prefill(C, **over):
    p = C.PrefillParams()
    p.q = p.k = p.v = p.out = p.workspace = AT
    p.batch, p.q_heads, p.kv_heads, p.seq_q, p.seq_kv = 2, 8, 4, 100, 200
    for n, s, h in (("q", 100, 8), ("o", 100, 8), ("k", 200, 4), ("v", 200, 4)):
        setattr(p, n + "_stride_b", h * s * 128)
        setattr(p, n + "_stride_h", s * 128)
        setattr(p, n + "_stride_s", 128)
    p.workspace_bytes = 1 << 40
    p.sm_scale = 0.1
    for k, v in over.items():
        setattr(p, k, v)
    return p


def _refused(L, fn, p):
    rc = getattr(L, fn)(ctypes.byref(p), None)
    assert rc in (1, 2), rc
    assert L.kvq_last_error()


@pytest.mark.parametrize("fault", CACHE_FAULTS, ids=str)
def test_a_bad_cache_is_refused_everywhere(fault):
    C, L = _lib()
    c = _cache(C, **fault)
    _refused(L, "kvq_paged_append", _append(C, c))
    _refused(L, "kvq_paged_decode", _decode(C, c))
    _refused(L, "kvq_paged_evict", _evict(C, c, w_tokens=1 << 30))


@pytest.mark.parametrize("fault", INT8_FAULTS, ids=str)
def test_a_bad_int8_cache_is_refused_everywhere(fault):
    C, L = _lib()
    c = _cache(C, True, **fault)
    _refused(L, "kvq_paged_append", _append(C, c))
    _refused(L, "kvq_paged_decode", _decode(C, c))
    _refused(L, "kvq_paged_evict", _evict(C, c))


def test_bad_calls_are_refused():
    C, L = _lib()
    c = _cache(C)
    for over in (dict(seq_new=-1), dict(x_type=2), dict(x_type=C.KVQ_PAGED_BF16), dict(k=None), dict(write_pos=None),
                 dict(v=AT + 2), dict(k_stride_s=130), dict(v_stride_h=4)):
        _refused(L, "kvq_paged_append", _append(C, c, **over))
    for over in (dict(q_type=7), dict(q_type=C.KVQ_PAGED_BF16), dict(q_heads=6), dict(q_heads=0), dict(q_heads=68),
                 dict(q=None), dict(out=None), dict(context_lens=None), dict(q=AT + 8), dict(q_stride_h=132)):
        _refused(L, "kvq_paged_decode", _decode(C, c, **over))
    for over in (dict(workspace=None), dict(workspace_bytes=8), dict(workspace=AT + 4)):  # rows that are shared out
        _refused(L, "kvq_paged_decode", _decode(C, _cache(C, max_pages=1000), **over))
    _refused(L, "kvq_paged_decode", _decode(C, _cache(C, batch=4097)))
    for over in (dict(budget=0), dict(sinks=-1), dict(recent=-1), dict(recent=47), dict(w_tokens=127), dict(weights=None),
                 dict(kept=None), dict(new_lens=None), dict(sinks=2 ** 31 - 1, recent=2 ** 31 - 1)):
        _refused(L, "kvq_paged_evict", _evict(C, c, **over))
    for over in (dict(batch=-1), dict(q_heads=6), dict(kv_heads=0), dict(seq_q=-1), dict(type=2), dict(q=None), dict(v=None),
                 dict(k=AT + 8), dict(o_stride_s=132), dict(k_stride_s=-128), dict(v_stride_s=1 << 24), dict(seq_kv=2 ** 31 - 1)):
        _refused(L, "kvq_prefill_attn", _prefill(C, **over))
    small = _prefill(C, batch=1, q_heads=1, kv_heads=1, seq_q=1, seq_kv=4096)
    assert L.kvq_prefill_workspace_bytes(ctypes.byref(small)) > 0
    small.workspace_bytes = 8
    _refused(L, "kvq_prefill_attn", small)
    for fn in ("kvq_paged_append", "kvq_paged_decode", "kvq_paged_evict", "kvq_prefill_attn"):
        assert getattr(L, fn)(None, None) == 1


def test_calls_with_nothing_to_do_return():
    C, L = _lib()
    assert L.kvq_paged_append(ctypes.byref(_append(C, _cache(C), seq_new=0)), None) == 0
    assert L.kvq_paged_append(ctypes.byref(_append(C, _cache(C, batch=0))), None) == 0
    assert L.kvq_paged_decode(ctypes.byref(_decode(C, _cache(C, batch=0))), None) == 0
    assert L.kvq_paged_evict(ctypes.byref(_evict(C, _cache(C, batch=0))), None) == 0
    assert L.kvq_prefill_attn(ctypes.byref(_prefill(C, seq_q=0)), None) == 0


def test_workspace_covers_what_a_call_writes():
    """The decode workspace of any cache holds its parts: two a work-group, at most four work-groups a CU and
    never more than there are tiles to give eight each; and the scores where weights are kept."""
    C, L = _lib()
    for batch, heads, rep, pages, size in ((1, 1, 1, 1, 16), (1, 2, 6, 40, 16), (8, 8, 5, 1024, 64), (300, 4, 7, 8, 256)):
        for weights in (None, AT):
            p = _decode(C, _cache(C, batch=batch, kv_heads=heads, max_pages=pages, page_size=size), q_heads=heads * rep, weights=weights)
            n = L.kvq_paged_decode_workspace_bytes(ctypes.byref(p))
            tiles = -(-pages * size // 32)
            assert n >= 4 * (batch + 2) or (n == 0 and tiles <= 32 and not weights)
            if weights:
                assert n >= 4 * heads * batch * tiles * rep * 32 + 4 * batch * heads * rep
            assert n <= (4 << 20) + 2 * 1088 * 16 * 520 + (0 if not weights else 5 * heads * batch * (tiles + 1) * rep * 32)
    bad = _decode(C, _cache(C, page_size=7))
    assert L.kvq_paged_decode_workspace_bytes(ctypes.byref(bad)) == 0


def _pages(dtype=torch.float16, pages=4, heads=2, size=16):
    return torch.zeros(pages, heads, size, 128, dtype=dtype)


def test_python_refusals():
    import llm_kvcache_quantization_amd as K

    k, v = _pages(), _pages()
    table, lens = torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    q = torch.zeros(1, 4, 128, dtype=torch.float16)
    with pytest.raises(ValueError, match="GPU"):
        K.decode_attn_paged(q, k, v, table, lens)
    with pytest.raises(ValueError, match=r"\[B, Hq, 128\]"):
        K.decode_attn_paged(q[0], k, v, table, lens)
    with pytest.raises(ValueError, match=r"\[B, Hq, 128\]"):
        K.decode_attn_paged(q[..., :64], k, v, table, lens)
    with pytest.raises(ValueError, match="pages must be"):
        K.decode_attn_paged(q, k[0], v[0], table, lens)
    with pytest.raises(ValueError, match="differ in shape"):
        K.decode_attn_paged(q, k, v[:2], table, lens)
    x = torch.zeros(1, 2, 5, 128, dtype=torch.float16)
    with pytest.raises(ValueError, match="alike"):
        K.append_paged(x, x[:, :, :3], k, v, table, lens)
    with pytest.raises(ValueError, match="GPU"):
        K.append_paged(x, x, k, v, table, lens)
    with pytest.raises(ValueError, match="GPU"):
        K.evict_paged(k, v, table, lens, torch.zeros(1, 2, 32), 4)
    qq = torch.zeros(1, 4, 5, 128, dtype=torch.float16)
    with pytest.raises(ValueError, match="one GPU"):
        K.prefill_attn_window(qq, x, x)
    with pytest.raises(ValueError, match=r"\[B, Hq, S, 128\]"):
        K.prefill_attn_window(qq[0], x, x)
    with pytest.raises(ValueError, match="alike"):
        K.prefill_attn_window(qq, x, x[:, :, :2])
