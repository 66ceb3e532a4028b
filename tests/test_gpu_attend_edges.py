"""Calls of the attention at the edges of what its documentation allows.  The
allowed errors are those of test_gpu_attend.py."""
from __future__ import annotations

import pytest
import torch

from kv_cases import gather
from flash_moe_b200.formats import Q8_0
from flash_moe_b200.paged_kv import KVBatch
from test_gpu_attend import CASES, DEV, KINDS, build, check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("window", [0, 300])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim,heads,q_heads,wide", [(64, 1, 4, False), (128, 2, 8, False),
                                                    (160, 1, 4, False), (256, 2, 8, False),
                                                    (256, 1, 4, True)])
def test_maxima_that_grow_in_every_unit(dim, heads, q_heads, wide, kind, window):
    """Keys whose scores rise by 12 powers of two from one 128-key unit to the
    next, so that every unit replaces every row's maximum and rescales its
    sums; a window adds rows that meet their first key in a later unit.  Every
    run gives the same bits."""
    new, kv = [300, 40, 129], [2600, 1500, 129]
    cache, batch, q = build(new, kv, 32, heads, dim, q_heads, kind, seed=40)
    if wide:   # a table too wide for expanded pages: codes decoded on their way
        table = torch.full((3, 70000 // heads), -1, dtype=torch.int32, device=DEV)
        table[:, :batch.max_pages] = batch.page_table
        batch = KVBatch(batch.q_start, batch.kv_lens, table)
    scale = 0.125
    g = torch.Generator(device=DEV).manual_seed(47)
    q = (1 + 0.1 * torch.randn(q.shape, generator=g, device=DEV)).to(q.dtype)
    for b, length in enumerate(kv):
        pos = torch.arange(length, device=DEV)
        # q . k * scale * log2(e) = 12 per 128 keys
        rise = pos * (12 / 128) / (dim * scale * 1.4427)
        pages, rows = batch.page_table[b].long()[pos // 32], pos % 32
        noise = 0.05 * torch.randn((length, heads, dim), generator=g, device=DEV)
        k = rise[:, None, None] + noise
        if cache.type == Q8_0:
            blocks = k.unflatten(-1, (-1, 32))
            step = (blocks.abs().amax(-1) / 120).clamp(min=1e-4).half()
            cache.k[pages, :, rows] = (blocks / step[..., None]).round().flatten(-2).to(torch.int8)
            cache.k_scales[pages, :, rows] = step
        else:
            cache.k[pages, :, rows] = k.to(cache.k.dtype)
    lse = torch.empty(q.shape[:2], device=DEV)
    first = cache.attend(batch, q, scale=scale, window=window, lse=lse)
    check(cache, batch, q, first, lse, new, kv, scale, window=window)
    for _ in range(30):
        assert torch.equal(cache.attend(batch, q, scale=scale, window=window), first)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("new,kv,given", [([5], [40], 3), ([3, 4], [70, 90], 4),
                                          ([200], [500], 130), ([40, 300], [60, 900], 170)])
def test_fewer_rows_than_the_batch(new, kv, given, kind):
    """Rows that are not given are not computed; the others stay at the
    positions that the batch gives them."""
    cache, batch, q = build(new, kv, 16, 2, 128, 8, kind, seed=41)
    left, part, length = given, [], []
    for n, k in zip(new, kv):
        part.append(min(n, left))
        length.append(k - (n - part[-1]))   # a causal row sees no further
        left -= part[-1]
    for window in (0, 50):
        out = cache.attend(batch, q[:given], window=window)
        check(cache, batch, q[:given], out, None, part, length, 128 ** -0.5, window=window)
    out = cache.attend(batch, q[:given], causal=False)
    check(cache, batch, q[:given], out, None, part, kv, 128 ** -0.5, causal=False)


@pytest.mark.parametrize("kind", ["f16", "q8_bf16"])
@pytest.mark.parametrize("dim,new", [(64, 1), (128, 5), (128, 60), (128, 200),
                                     (256, 1), (256, 20), (256, 200)])
def test_pages_behind_the_window(dim, new, kind):
    """Table entries of pages that lie before every row's window may name no
    page."""
    kv, window = [new + 300, new + 411], 100
    cache, batch, q = build([new, new], kv, 16, 2, dim, 8, kind, seed=42)
    status = torch.full((1,), 99, dtype=torch.int32, device=DEV)
    want = cache.attend(batch, q, window=window)
    for b, length in enumerate(kv):
        batch.page_table[b, :(length - new - window + 1) // 16] = -1
    out = cache.attend(batch, q, window=window, status=status)
    assert status.item() == 0
    assert torch.equal(out, want)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("scale,size", [(0.0, 1e-9), (1e-38, 1e-20), (3e38, 0.0), (-3e38, 0.0)])
@pytest.mark.parametrize("name", ["drafts", "chunk", "chunk_256"])
def test_vanishing_scores(name, scale, size, kind):
    """Scores of zero, or so small that they do not matter: the mean of the
    attended values, whatever the scale and the size of the queries."""
    new, kv, page, heads, dim, q_heads = CASES[name]
    cache, batch, q = build(new, kv, page, heads, dim, q_heads, kind, seed=43)
    q = (q.float().clamp(-3, 3) * size).to(q.dtype)
    out = cache.attend(batch, q, scale=scale)
    check(cache, batch, q, out, None, new, kv, 0.0)


@pytest.mark.parametrize("top", [2.0 ** 112, 2.0 ** 113, 2.0 ** 126, 2.0 ** 127])
@pytest.mark.parametrize("name", ["drafts", "chunk", "chunk_256"])
def test_large_queries_over_codes(name, top):
    """bf16 queries up to the largest finite ones over a Q8_0 cache."""
    new, kv, page, heads, dim, q_heads = CASES[name]
    cache, batch, q = build(new, kv, page, heads, dim, q_heads, "q8_bf16", seed=44)
    cache.k_scales.fill_(2.0 ** -20)
    q = (q.float().clamp(-1.9, 1.9) * top).bfloat16()
    scale = 2.0 ** 10 / top
    out = cache.attend(batch, q, scale=scale)
    check(cache, batch, q, out, None, new, kv, scale)


def test_the_longest_sequence_with_many_heads():
    """The units of all heads of one tile pass 2^31.  The long sequence's table
    names its last page only, so that the rest is passed over quickly; that
    page is all that its rows get, and the next sequence is as ever."""
    heads, dim, length = 272, 32, (1 << 31) - 65536
    cache, small, q = build([1, 1], [256, 77], 256, heads, dim, heads, "f16", seed=48)
    table = torch.full((2, 1 << 23), -1, dtype=torch.int32, device=DEV)
    table[0, length // 256 - 1] = small.page_table[0, 0]
    table[1, 0] = small.page_table[1, 0]
    lens = torch.tensor([length, 77], dtype=torch.int32, device=DEV)
    lse = torch.empty(q.shape[:2], device=DEV)
    out = cache.attend(KVBatch(small.q_start, lens, table), q, lse=lse)
    check(cache, small, q, out, lse, [1, 1], [256, 77], dim ** -0.5)


@pytest.mark.parametrize("kind", ["f16", "q8_f16"])
@pytest.mark.parametrize("window", [1 << 31, 1 << 32, (1 << 32) + 5])
def test_windows_wider_than_any_sequence(window, kind):
    cache, batch, q = build([3, 100], [40, 300], 16, 2, 64, 4, kind, seed=45)
    assert torch.equal(cache.attend(batch, q, window=window), cache.attend(batch, q))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("size", [1e3, 1e6, 1e9])
@pytest.mark.parametrize("name", ["decode", "decode_256", "drafts", "chunk", "chunk_256"])
def test_large_scores(name, size, kind):
    """One key's score stands out by so much that it takes all the weight, at
    sizes where neighbouring fp32 numbers are far apart."""
    new, kv, page, heads, dim, q_heads = CASES[name]
    cache, batch, q = build(new, kv, page, heads, dim, q_heads, kind, seed=46)
    q = torch.ones_like(q)
    target = cache.k if cache.k_scales is None else cache.k_scales
    target.abs_()
    if cache.type == Q8_0:
        cache.k.fill_(100)
    out = cache.attend(batch, q, scale=size)
    assert out.isfinite().all()
    lo = 0
    for b, (n, length) in enumerate(zip(new, kv)):
        k = gather(cache.k, cache.k_scales, batch.page_table[b], length, page)
        v = gather(cache.v, cache.v_scales, batch.page_table[b], length, page)
        s = k.sum(-1)                       # [length, heads]
        for i in range(n):
            hi = length - n + i + 1
            if hi < 2:
                continue
            top = s[:hi].topk(2, dim=0)
            # sums of dim terms in fp32, and the rounding of score and maximum
            sure = (top.values[0] - top.values[1]) * size > 40 + (dim + 4) * 2.0 ** -22 * top.values[0] * size
            want = v[top.indices[0], torch.arange(heads, device=DEV)]
            got = out[lo + i].view(heads, -1, dim).double()
            err = (got - want[:, None]).abs().amax(-1).amax(-1)
            assert (err[sure] <= 2.0 ** -7 * want.abs().amax(-1)[sure]).all(), (b, i)
        lo += n


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("largest", [1e5, 1e7, 4e7])
@pytest.mark.parametrize("name", ["decode", "decode_256", "drafts", "chunk", "chunk_256"])
def test_large_scores(name, largest, kind):
    """Scores up to the largest documented ones: a key whose score stands out
    takes all the weight, and every row stays finite."""
    new, kv, page, heads, dim, q_heads = CASES[name]
    cache, batch, q = build(new, kv, page, heads, dim, q_heads, kind, seed=46)
    q = torch.ones_like(q)
    target = cache.k if cache.k_scales is None else cache.k_scales
    target.abs_()
    if cache.type == Q8_0:
        cache.k.fill_(100)
    kv_rows = [[gather(c, s, batch.page_table[b], n, page) for c, s in
                ((cache.k, cache.k_scales), (cache.v, cache.v_scales))] for b, n in enumerate(kv)]
    scale = largest / max(k.sum(-1).max().item() for k, _ in kv_rows)
    for sign in (1, -1):
        out = cache.attend(batch, q, scale=sign * scale)
        assert out.isfinite().all()
        at = torch.arange(heads, device=DEV)
        lo = 0
        for b, (n, length) in enumerate(zip(new, kv)):
            k, v = kv_rows[b]
            s = k.sum(-1) * sign * scale                 # [length, heads]
            for i in range(n):
                hi = length - n + i + 1
                if hi < 2:
                    continue
                top = s[:hi].topk(2, dim=0)
                # sums of dim fp32 terms, two roundings to the maximum's magnitude
                slack = (dim + 4) * 2.0 ** -22 * s[:hi].abs().amax(0)
                sure = top.values[0] - top.values[1] > 40 + slack
                want = v[top.indices[0], at]
                err = (out[lo + i].view(heads, -1, dim).double() - want[:, None]).abs()
                tol = 2.0 ** -7 * want.abs().amax(-1)
                assert (err.amax(-1).amax(-1)[sure] <= tol[sure]).all(), (b, i)
            lo += n
