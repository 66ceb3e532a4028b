"""Refusals of the paged key/value cache calls: every check answers before
any device work, so they run without a GPU."""
from __future__ import annotations

import ctypes as C

import pytest
import torch

from flash_moe_b200 import _lib
from flash_moe_b200.formats import BF16, F16, F32, Q4_K, Q8_0
from flash_moe_b200.paged_kv import KVBatch, PagedKVCache

A = 0x10000  # an aligned stand-in address: no refused call follows it


def cache(**kw):
    f = dict(type=F16, num_pages=4, page_size=16, kv_heads=2, head_dim=64, k=A, v=A,
             k_scales=None, v_scales=None)
    f.update(kw)
    return _lib.KVCacheStruct(f["type"], f["num_pages"], f["page_size"], f["kv_heads"],
                              f["head_dim"], 0, f["k"], f["v"], f["k_scales"], f["v_scales"])


def batch(**kw):
    f = dict(sequences=2, tokens=3, max_pages=4, table_stride=4, q_start=A, kv_lens=A,
             page_table=A)
    f.update(kw)
    return _lib.KVBatchStruct(f["sequences"], f["tokens"], f["max_pages"], 0, f["table_stride"],
                              f["q_start"], f["kv_lens"], f["page_table"])


def rows(lib, name, c, b, type_id=F16, k=A, kts=128, khs=64, v=A, vts=128, vhs=64, status=None):
    return getattr(lib, name)(C.byref(c) if c else None, C.byref(b) if b else None, type_id, k, kts,
                              khs, v, vts, vhs, status, None)


def attend(lib, c, b, type_id=F16, q=A, qts=256, qhs=64, heads=4, out=A, ots=256, ohs=64, lse=None,
           scale=0.125, causal=1, window=0, ws=A, ws_bytes=1 << 40, status=None):
    return lib.moe_b200_attend(C.byref(c) if c else None, C.byref(b) if b else None, type_id, q,
                               qts, qhs, heads, out, ots, ohs, lse, scale, causal, window, ws,
                               ws_bytes, status, None)


CACHE_BAD = [
    (dict(k=None), -1), (dict(v=None), -1), (dict(num_pages=0), -1), (dict(kv_heads=0), -1),
    (dict(kv_heads=1025), -1), (dict(type=Q4_K), -2), (dict(type=F32), -2), (dict(head_dim=16), -2),
    (dict(head_dim=72), -2), (dict(head_dim=288), -2), (dict(page_size=8), -1),
    (dict(page_size=48), -1), (dict(page_size=512), -1), (dict(num_pages=1 << 30, kv_heads=4), -1),
    (dict(type=Q8_0), -1), (dict(type=Q8_0, k_scales=A), -1), (dict(k_scales=A, v_scales=A), -1),
    (dict(k=A + 8), -7), (dict(type=Q8_0, k_scales=A, v_scales=A + 2), -7),
]
BATCH_BAD = [
    (dict(sequences=-1), -1), (dict(tokens=-1), -1), (dict(max_pages=-1), -1),
    (dict(q_start=None), -1), (dict(kv_lens=None), -1), (dict(page_table=None), -1),
    (dict(table_stride=3), -1), (dict(q_start=A + 2), -7), (dict(page_table=A + 1), -7),
]


@pytest.mark.parametrize("kw,code", CACHE_BAD)
def test_bad_cache(lib, kw, code):
    for name in ("moe_b200_kv_write", "moe_b200_kv_read"):
        assert rows(lib, name, cache(**kw), batch()) == code
    assert attend(lib, cache(**kw), batch()) == code
    n = C.c_size_t(0)
    assert lib.moe_b200_attend_workspace(C.byref(cache(**kw)), C.byref(batch()), 4,
                                         C.byref(n)) == code


@pytest.mark.parametrize("kw,code", BATCH_BAD)
def test_bad_batch(lib, kw, code):
    for name in ("moe_b200_kv_write", "moe_b200_kv_read"):
        assert rows(lib, name, cache(), batch(**kw)) == code
    assert attend(lib, cache(), batch(**kw)) == code


@pytest.mark.parametrize("kw,code", [
    (dict(type_id=Q8_0), -2), (dict(type_id=7), -2), (dict(k=None), -1), (dict(v=None), -1),
    (dict(k=A + 2), -7), (dict(kts=132), -7), (dict(vhs=68), -7), (dict(type_id=F32, kts=130), -7),
    (dict(status=A + 2), -7),
])
def test_bad_rows(lib, kw, code):
    for name in ("moe_b200_kv_write", "moe_b200_kv_read"):
        assert rows(lib, name, cache(), batch(), **kw) == code


@pytest.mark.parametrize("kw,code", [
    (dict(type_id=F32), -2), (dict(type_id=BF16), -2), (dict(heads=0), -1), (dict(heads=5), -1),
    (dict(heads=65538), -1), (dict(causal=2), -1), (dict(window=-1), -1),
    (dict(causal=0, window=8), -1), (dict(scale=float("nan")), -1), (dict(scale=float("inf")), -1),
    (dict(q=None), -1), (dict(out=None), -1), (dict(ws=None), -1), (dict(q=A + 8), -7),
    (dict(ots=260), -7), (dict(lse=A + 2), -7), (dict(ws=A + 128), -7), (dict(ws_bytes=0), -8),
])
def test_bad_attend(lib, kw, code):
    assert attend(lib, cache(), batch(), **kw) == code


def test_null_structs_and_workspace(lib):
    for name in ("moe_b200_kv_write", "moe_b200_kv_read"):
        assert rows(lib, name, None, batch()) == -1
        assert rows(lib, name, cache(), None) == -1
    assert attend(lib, None, batch()) == -1
    assert attend(lib, cache(), None) == -1
    n = C.c_size_t(0)
    assert lib.moe_b200_attend_workspace(C.byref(cache()), C.byref(batch()), 3, C.byref(n)) == -1
    assert lib.moe_b200_attend_workspace(C.byref(cache()), C.byref(batch()), 4, None) == -1
    assert lib.moe_b200_attend_workspace(C.byref(cache()), C.byref(batch()), 4, C.byref(n)) == 0
    assert n.value > 0


def test_too_many_rows(lib):
    assert attend(lib, cache(), batch(tokens=1 << 30)) == -1


def test_nothing_to_do_is_no_error(lib):
    for b in (batch(tokens=0), batch(sequences=0, q_start=None, kv_lens=None, page_table=None,
                                     max_pages=0, table_stride=0)):
        for name in ("moe_b200_kv_write", "moe_b200_kv_read"):
            assert rows(lib, name, cache(), b) == 0
        assert attend(lib, cache(), b) == 0


def test_python_refuses_host_tensors():
    z = torch.zeros(4, 2, 16, 64, dtype=torch.float16)
    with pytest.raises(ValueError, match="CUDA"):
        PagedKVCache(z, z.clone())
    i = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(ValueError, match="int32 CUDA"):
        KVBatch(i, i[:2], torch.zeros(2, 4, dtype=torch.int32))


@pytest.mark.parametrize("shape,dtype,match", [
    ((4, 2, 16, 48), torch.float16, "head_dim"), ((4, 2, 16, 288), torch.float16, "head_dim"),
    ((4, 2, 24, 64), torch.float16, "page_size"), ((4, 2, 8, 64), torch.bfloat16, "page_size"),
    ((4, 2, 16, 64), torch.float32, "dtype"), ((4, 2, 16, 64), torch.int8, "scales"),
    ((2, 16, 64), torch.float16, "one shape"), ((0, 2, 16, 64), torch.float16, "one page"),
])
def test_python_refuses_caches(shape, dtype, match):
    z = torch.zeros(shape, dtype=dtype)
    with pytest.raises(ValueError, match=match):
        PagedKVCache(z, z.clone())


def test_python_refuses_scales_and_types():
    z = torch.zeros(4, 2, 16, 64, dtype=torch.float16)
    s = torch.zeros(4, 2, 16, 2, dtype=torch.float16)
    with pytest.raises(ValueError, match="only a Q8_0"):
        PagedKVCache(z, z.clone(), s, s.clone())
    with pytest.raises(ValueError, match="scales of shape"):
        PagedKVCache(z.to(torch.int8), z.to(torch.int8), s, s[..., :1])
    with pytest.raises(ValueError, match="cache type"):
        PagedKVCache.empty(4, 16, 2, 64, Q4_K, "cpu")
