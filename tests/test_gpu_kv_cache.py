"""Writing and reading the paged key/value cache.

16-bit caches round once, so they are compared bit for bit.  Q8_0: for 16-bit
rows max|x| / 127 and x / d are quotients of 11-bit by 7- and 11-bit numbers,
which differ from every binary16 value and every tie by more than 2^-20
relative, so fp32 division gives the codes and scales of exact arithmetic bit
for bit.  fp32 rows are held to |x - d code| <= d / 2 plus the fp32 rounding of
the quotient (127 * 2^-24 steps) and to a scale within one binary16 step.
"""
from __future__ import annotations

import pytest
import torch

import kv_cases as K
from flash_moe_b200 import _lib
from flash_moe_b200.formats import BF16, F16, Q8_0
from flash_moe_b200.paged_kv import KVBatch, PagedKVCache

pytestmark = pytest.mark.gpu
DEV = "cuda"

# new rows, cached lengths, page size, heads, head_dim
SHAPES = {
    "one": ([1], [1], 16, 1, 32),
    "page_end": ([1, 1, 2], [16, 17, 33], 16, 2, 64),
    "ragged": ([5, 0, 37, 1], [5, 9, 100, 64], 16, 3, 96),
    "wide": ([70, 3], [300, 3], 256, 2, 256),
    "many": ([1] * 67, list(range(1, 68)), 32, 8, 128),
    "long": ([2000], [2111], 64, 5, 160),
}
DTYPES = [torch.float16, torch.bfloat16, torch.float32]


def filled_cache(type_id, pool, page, heads, dim):
    c = PagedKVCache.empty(pool, page, heads, dim, type_id, DEV)
    for t in (c.k, c.v):
        t.fill_(7)
    if type_id == Q8_0:
        c.k_scales.fill_(0.5)
        c.v_scales.fill_(0.25)
    return c


def slots(batch, new, kv, page):
    """(page, row) of every new row, in order."""
    out = []
    table = batch.page_table.cpu()
    for b, (n, length) in enumerate(zip(new, kv)):
        for p in range(length - n, length):
            out.append((int(table[b, p // page]), p % page))
    return out


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("type_id", [F16, BF16, Q8_0])
@pytest.mark.parametrize("name", SHAPES)
def test_write_and_read(name, type_id, dtype):
    new, kv, page, heads, dim = SHAPES[name]
    start, lens, table, pool = K.make_batch(new, kv, page, device=DEV)
    batch = KVBatch(start, lens, table)
    T = sum(new)
    g = torch.Generator().manual_seed(3)
    both = (torch.randn(T, 2, heads, dim, generator=g) * 3).to(dtype).to(DEV)
    cache = filled_cache(type_id, pool, page, heads, dim)
    want_k, want_v = cache.k.clone(), cache.v.clone()
    status = torch.full((1,), 99, dtype=torch.int32, device=DEV)
    cache.write(batch, both[:, 0], both[:, 1], status=status)
    assert status.item() == 0
    where = slots(batch, new, kv, page)
    pages = torch.tensor([p for p, _ in where], device=DEV)
    rows = torch.tensor([r for _, r in where], device=DEV)
    if type_id != Q8_0:
        want_k[pages, :, rows] = both[:, 0].to(want_k.dtype)
        want_v[pages, :, rows] = both[:, 1].to(want_v.dtype)
        assert torch.equal(cache.k, want_k) and torch.equal(cache.v, want_v)
    else:
        for i, (codes, scales, want) in enumerate(((cache.k, cache.k_scales, want_k),
                                                   (cache.v, cache.v_scales, want_v))):
            n, d = K.quantise(both[:, i])
            got_n, got_d = codes[pages, :, rows], scales[pages, :, rows]
            if dtype != torch.float32:
                assert torch.equal(got_n.double(), n)
                assert torch.equal(got_d.double(), d)
            else:
                step = got_d.double().repeat_interleave(32, -1)
                err = (both[:, i].double() - got_n.double() * step).abs()
                assert (err <= step * (0.5 + 127 * 2.0 ** -24)).all()
                assert ((got_d.double() - d).abs() <= d * 2.0 ** -10).all()
            codes[pages, :, rows] = 7      # nothing else was touched
            assert torch.equal(codes, want)
            codes[pages, :, rows] = got_n
    for out_dtype in DTYPES:
        k, v = cache.read(batch, tokens=T, dtype=out_dtype)
        for got, codes, scales in ((k, cache.k, cache.k_scales), (v, cache.v, cache.v_scales)):
            x = codes[pages, :, rows]
            if type_id == Q8_0:
                want = K.values(x, scales[pages, :, rows]).float().to(out_dtype)
            else:
                want = x.float().to(out_dtype)
            assert torch.equal(got, want)


def test_rows_without_a_place_are_skipped():
    """Negative positions, rows behind the last sequence, bad pages and
    lengths past the table: skipped in a write, zeros or untouched in a read,
    and named by the status word."""
    page, heads, dim = 16, 2, 64
    start = torch.tensor([0, 3, 5, 7], dtype=torch.int32, device=DEV)
    lens = torch.tensor([1, 18, 34], dtype=torch.int32, device=DEV)
    #       two rows before 0 | second page out of the cache | length past the table
    table = torch.tensor([[0, 1], [2, 9], [3, 4]], dtype=torch.int32, device=DEV)
    batch = KVBatch(start, lens, table)
    cache = filled_cache(F16, 6, page, heads, dim)
    before = cache.k.clone()
    x = torch.randn(9, heads, dim, device=DEV).half()
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    cache.write(batch, x, x, status=status)
    assert status.item() == _lib.KV_BAD_PAGE | _lib.KV_BAD_LENGTH
    want = before
    want[0, :, 0] = x[2]
    assert torch.equal(cache.k, want) and torch.equal(cache.v, want)
    out = [torch.full((9, heads, dim), 5.0, device=DEV, dtype=torch.float16) for _ in range(2)]
    cache.read(batch, out=tuple(out), status=status)
    assert status.item() == _lib.KV_BAD_PAGE | _lib.KV_BAD_LENGTH
    for o in out:
        assert torch.equal(o[2], x[2])
        assert (o[[0, 1, 3, 4, 5, 6]] == 0).all()
        assert (o[7:] == 5).all()


def test_special_values_quantised():
    """Zeros, the smallest and largest values, NaN and infinities."""
    start, lens, table, pool = K.make_batch([8], [8], 16, device=DEV)
    batch = KVBatch(start, lens, table)
    x = torch.zeros(8, 1, 64, device=DEV)
    x[1] = 2.0 ** -24
    x[2, 0, 3], x[2, 0, 40] = 3e38, -1e6
    x[3, 0, 5] = float("nan")
    x[4, 0, 6] = float("inf")
    x[5, 0, 7] = -float("inf")
    x[6] = 127.0
    x[7, 0] = torch.arange(64, device=DEV) * 1e-7
    cache = PagedKVCache.empty(pool, 16, 1, 64, Q8_0, DEV)
    cache.write(batch, x, x)
    k, v = cache.read(batch, tokens=8, dtype=torch.float32)
    assert torch.equal(k.nan_to_num(1e9), v.nan_to_num(1e9))
    assert (k[0] == 0).all()
    assert ((k[1] - 2.0 ** -24).abs() <= 2.0 ** -25).all()
    assert k[2, 0, 3] == 127 * 515.5 and k[2, 0, 40] == -127 * 515.5
    for row, at in ((3, 5), (4, 6), (5, 7)):
        assert k[row, 0, :32].isnan().all() and (k[row, 0, 32:] == 0).all(), (row, at)
    assert (k[6] == 127).all()
    n, d = K.quantise(x[7].cpu())
    step = d.repeat_interleave(32, -1)
    assert ((k[7].cpu().double() - x[7].cpu().double()).abs() <= step * 0.5001).all()
    half = cache.read(batch, tokens=8, dtype=torch.float16)[0]
    assert half[2].isfinite().all()


def test_unaligned_and_strided_rows():
    """Rows that are not 16-byte aligned are copied first; outputs must be
    aligned."""
    start, lens, table, pool = K.make_batch([6], [20], 16, device=DEV)
    batch = KVBatch(start, lens, table)
    cache = filled_cache(F16, pool, 16, 3, 32)
    wide = torch.randn(6, 3, 33, device=DEV).half()
    moved = torch.randn(32, 3, 6, device=DEV).half().permute(2, 1, 0)
    cache.write(batch, wide[..., 1:], moved)
    out = torch.zeros(6, 2, 3, 32, device=DEV, dtype=torch.float16)
    k, v = cache.read(batch, out=(out[:, 0], out[:, 1]))
    assert torch.equal(out[:, 0], wide[..., 1:]) and torch.equal(out[:, 1], moved)
    with pytest.raises(ValueError, match="aligned"):
        cache.read(batch, out=(wide[..., 1:], wide[..., 1:]))


def test_other_stream():
    start, lens, table, pool = K.make_batch([50], [50], 16, device=DEV)
    batch = KVBatch(start, lens, table)
    cache = filled_cache(Q8_0, pool, 16, 2, 64)
    x = torch.randn(50, 2, 64, device=DEV)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    cache.write(batch, x, x, stream=s)
    k, _ = cache.read(batch, tokens=50, stream=s)
    s.synchronize()
    cache.write(batch, x, x)
    assert torch.equal(k, cache.read(batch, tokens=50)[0])
