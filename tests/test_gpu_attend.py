"""Attention over the paged cache against its definition in 64 bits.

The allowed error of an output, per element (mass = sum_j p_j |v_j|):
* its own rounding, eps/2 |o|;
* the 16-bit probabilities, eps_p/2 mass (eps_p of the cache's type, binary16
  for Q8_0);
* the fp32 scores: every product sum of D terms is off by at most
  D 2^-23 sum|q k| (the tensor cores may cut instead of round), plus 2^-21 for
  the exponential and the running rescales; numerator and denominator both
  move by that, so 2 delta mass;
* the fp32 sums over n keys, n 2^-23 mass;
* probabilities below binary16's normal range: the row's largest one is held
  as at least 2^7 (2^15, or up to 2^8 less while a larger maximum has not been
  taken over yet), so a smallest binary16 step, 2^-24, is 2^-31 of it, half of
  that 2^-32 per key: 2^-32 sum_j |v_j|.
"""
from __future__ import annotations

import math

import pytest
import torch

import kv_cases as K
from flash_moe_b200 import _lib
from flash_moe_b200.formats import BF16, F16, Q8_0
from flash_moe_b200.paged_kv import KVBatch, PagedKVCache

pytestmark = pytest.mark.gpu
DEV = "cuda"
KINDS = {"f16": (F16, torch.float16), "bf16": (BF16, torch.bfloat16),
         "q8_f16": (Q8_0, torch.float16), "q8_bf16": (Q8_0, torch.bfloat16)}


def build(new, kv, page, heads, dim, q_heads, kind, seed=0, spread=1.0, **kw):
    type_id, dtype = KINDS[kind]
    start, lens, table, pool = K.make_batch(new, kv, page, seed, DEV, **kw)
    g = torch.Generator(device=DEV).manual_seed(seed + 1)
    cache = PagedKVCache.empty(pool, page, heads, dim, type_id, DEV)
    for codes, scales in ((cache.k, cache.k_scales), (cache.v, cache.v_scales)):
        if type_id == Q8_0:
            codes.copy_(torch.randint(-127, 128, codes.shape, generator=g, device=DEV,
                                      dtype=torch.int8))
            scales.copy_((0.5 + torch.rand(scales.shape, generator=g, device=DEV)) * 2.5 / 127)
        else:
            codes.copy_(torch.randn(codes.shape, generator=g, device=DEV))
    q = (torch.randn(sum(new), q_heads, dim, generator=g, device=DEV) * spread).to(dtype)
    return cache, KVBatch(start, lens, table), q


def check(cache, batch, q, out, lse, new, kv, scale, causal=True, window=0, skip=()):
    kind = torch.float16 if cache.type == Q8_0 else cache.k.dtype
    eps_o, eps_p = K.HALF[q.dtype], K.HALF[kind]
    lo = 0
    for b, (n, length) in enumerate(zip(new, kv)):
        if b not in skip and n:
            k = K.gather(cache.k, cache.k_scales, batch.page_table[b], length, cache.page_size)
            v = K.gather(cache.v, cache.v_scales, batch.page_table[b], length, cache.page_size)
            want, want_lse, mass = K.attend(q[lo:lo + n], k, v, length - n, scale, causal, window)
            group = q.shape[1] // k.shape[1]
            if length:
                qk = torch.einsum("nhd,khd->nhk", q[lo:lo + n].double().abs(),
                                  k.abs().repeat_interleave(group, 1)).amax(-1) * abs(scale)
            else:
                qk = torch.zeros(q[lo:lo + n].shape[:2], device=DEV, dtype=torch.float64)
            delta = (q.shape[2] * 2.0 ** -23 * qk + 2.0 ** -21)[..., None]
            tol = eps_o * want.abs() + (eps_p + 2 * delta + length * 2.0 ** -23) * mass * 1.01
            if kind == torch.float16:
                total = v.abs().sum(0).repeat_interleave(group, 0) if length else 0.0
                tol = tol + 2.0 ** -32 * total
            # a 16-bit output below its smallest normal rounds to half of its smallest step
            tol = tol + (2.0 ** -25 if q.dtype == torch.float16 else 1e-40)
            err = (out[lo:lo + n].double() - want).abs()
            assert out[lo:lo + n].isfinite().all()
            worst = (err / tol).max().item()
            assert worst <= 1, f"sequence {b}: {worst} of the allowed error"
            if lse is not None:
                gone = want_lse == -math.inf
                assert torch.equal(lse[lo:lo + n] == -math.inf, gone)
                e = (lse[lo:lo + n].double() - want_lse)[~gone].abs()
                t = (delta[..., 0] + eps_p + length * 2.0 ** -23 + 2.0 ** -21 * (1 + want_lse.abs()))[~gone]
                assert (e <= t).all()
        lo += n


# new, kv, page, kv heads, head_dim, query heads
CASES = {
    "one_key": ([1], [1], 16, 1, 64, 1),
    "decode": ([1, 1, 1], [17, 300, 1], 16, 2, 128, 16),
    "decode_256": ([1, 1], [1000, 64], 64, 2, 256, 16),
    "decode_group5": ([1] * 9, [40 * i + 1 for i in range(9)], 32, 3, 96, 15),
    "decode_mqa": ([1, 1], [513, 30], 128, 1, 128, 48),
    "drafts": ([5, 3, 1, 4], [5, 130, 1, 67], 16, 4, 64, 8),
    "empty_rows": ([4, 0, 2, 3], [2, 5, 0, 3], 16, 2, 32, 2),
    "mha_chunk": ([130], [130], 16, 3, 64, 3),
    "chunk": ([200, 1, 65], [500, 70, 65], 16, 2, 128, 8),
    "chunk_256": ([129, 40], [700, 41], 64, 1, 256, 8),
    "chunk_odd": ([77, 260], [90, 261], 32, 1, 192, 7),
    "chunk_160": ([50], [333], 256, 2, 160, 4),
    "chunk_group3": ([300], [1000], 128, 2, 96, 6),
}


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("name", CASES)
def test_matches_definition(name, kind):
    new, kv, page, heads, dim, q_heads = CASES[name]
    cache, batch, q = build(new, kv, page, heads, dim, q_heads, kind)
    lse = torch.empty(q.shape[:2], device=DEV)
    status = torch.full((1,), 99, dtype=torch.int32, device=DEV)
    out = cache.attend(batch, q, lse=lse, status=status)
    assert status.item() == 0
    check(cache, batch, q, out, lse, new, kv, dim ** -0.5)


@pytest.mark.parametrize("kind", ["f16", "q8_bf16"])
@pytest.mark.parametrize("window", [1, 16, 100])
@pytest.mark.parametrize("name", ["decode", "drafts", "empty_rows", "chunk", "chunk_256"])
def test_window(name, window, kind):
    new, kv, page, heads, dim, q_heads = CASES[name]
    cache, batch, q = build(new, kv, page, heads, dim, q_heads, kind, seed=5)
    lse = torch.empty(q.shape[:2], device=DEV)
    out = cache.attend(batch, q, window=window, lse=lse, scale=0.2)
    check(cache, batch, q, out, lse, new, kv, 0.2, window=window)


@pytest.mark.parametrize("kind", ["bf16", "q8_f16"])
@pytest.mark.parametrize("name", ["decode", "drafts", "empty_rows", "chunk", "chunk_odd"])
def test_not_causal(name, kind):
    new, kv, page, heads, dim, q_heads = CASES[name]
    cache, batch, q = build(new, kv, page, heads, dim, q_heads, kind, seed=6)
    lse = torch.empty(q.shape[:2], device=DEV)
    out = cache.attend(batch, q, causal=False, lse=lse)
    check(cache, batch, q, out, lse, new, kv, dim ** -0.5, causal=False)


@pytest.mark.parametrize("kind", ["f16", "bf16", "q8_f16"])
@pytest.mark.parametrize("new,kv", [([1, 1], [20000, 333]), ([16], [9000]), ([300], [6000])])
def test_long_contexts(new, kv, kind):
    """Contexts long enough to be split over the GPU and joined again."""
    cache, batch, q = build(new, kv, 64, 2, 128, 8, kind, seed=7, spread=2.0)
    lse = torch.empty(q.shape[:2], device=DEV)
    out = cache.attend(batch, q, lse=lse)
    check(cache, batch, q, out, lse, new, kv, 128 ** -0.5)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("name", ["decode", "drafts", "chunk", "chunk_256"])
def test_poison_outside_the_rows_keys(name, kind):
    """NaN and infinities in unused pages, behind the sequences and at
    tokens that only some rows attend: the other rows do not see them."""
    new, kv, page, heads, dim, q_heads = CASES[name]
    cache, batch, q = build(new, kv, page, heads, dim, q_heads, kind, seed=8)
    clean = cache.attend(batch, q)
    used = torch.zeros(cache.num_pages, page, dtype=torch.bool, device=DEV)
    newest = torch.zeros_like(used)
    for b, length in enumerate(kv):
        pos = torch.arange(length, device=DEV)
        used[batch.page_table[b].long()[pos // page], pos % page] = True
        last = length - 1
        newest[int(batch.page_table[b, last // page]), last % page] = True
    for poison in (float("nan"), float("inf"), -float("inf")):
        for t, s in ((cache.k, cache.k_scales), (cache.v, cache.v_scales)):
            target = t if s is None else s
            m = (~used)[:, None, :, None].expand(target.shape)
            target[m] = poison
        assert torch.equal(cache.attend(batch, q), clean)
    # the newest token of each sequence holds poison: only its own row shows it
    starts = batch.q_start.tolist()
    for t, s in ((cache.v, cache.v_scales), (cache.k, cache.k_scales)):
        target = t if s is None else s
        m = newest[:, None, :, None].expand(target.shape)
        keep = target[m].clone()
        target[m] = float("nan")
        out = cache.attend(batch, q)
        for b, n in enumerate(new):
            rows = out[starts[b]:starts[b + 1]]
            assert torch.equal(rows[:-1], clean[starts[b]:starts[b + 1] - 1])
            assert rows[-1].isnan().all()
        target[m] = keep


@pytest.mark.parametrize("kind", ["f16", "bf16", "q8_f16"])
@pytest.mark.parametrize("name", ["drafts", "chunk", "chunk_256"])
def test_poisoned_value_within_a_chunk(name, kind):
    """One value of a token in the middle of the new rows is infinite: rows
    before it are untouched, rows from it on have that one column infinite."""
    new, kv, page, heads, dim, q_heads = CASES[name]
    cache, batch, q = build(new, kv, page, heads, dim, q_heads, kind, seed=9)
    clean = cache.attend(batch, q)
    b, i, col = 0, new[0] // 2, 37
    pos = kv[0] - new[0] + i
    pg, row = int(batch.page_table[b, pos // page]), pos % page
    if cache.type == Q8_0:
        cache.v_scales[pg, 0, row, col // 32] = float("nan")
        cols = slice(col // 32 * 32, col // 32 * 32 + 32)
    else:
        cache.v[pg, 0, row, col] = float("inf")
        cols = slice(col, col + 1)
    out = cache.attend(batch, q)
    group = q_heads // heads
    assert torch.equal(out[:i], clean[:i]) and torch.equal(out[new[0]:], clean[new[0]:])
    hit = out[i:new[0], :group]
    assert not hit[..., cols].isfinite().any()
    rest = torch.ones(dim, dtype=torch.bool)
    rest[cols] = False
    assert torch.equal(hit[..., rest], clean[i:new[0], :group][..., rest])
    assert torch.equal(out[i:new[0], group:], clean[i:new[0], group:])


@pytest.mark.parametrize("n", [1, 40])
def test_padded_batch_and_bad_pages(n):
    """Rows behind the last sequence stay; bad pages and lengths are named by
    the status word and disturb no other sequence."""
    new, kv = [n, n, n], [n + 30, n + 30, n + 30]
    cache, batch, q = build(new, kv, 16, 2, 64, 8, "f16", seed=10)
    wide = torch.cat([q, q[:5]])
    out = torch.full_like(wide, 3.0)
    lse = torch.full(wide.shape[:2], 4.0, device=DEV)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    cache.attend(batch, wide, out=out, lse=lse, status=status)
    assert status.item() == 0
    check(cache, batch, q, out, lse, new, kv, 64 ** -0.5)
    assert (out[3 * n:] == 3).all() and (lse[3 * n:] == 4).all()
    batch.page_table[1, 1] = cache.num_pages
    batch.kv_lens[2] = 1 << 30
    cache.attend(batch, wide, out=out, lse=lse, status=status)
    assert status.item() == _lib.KV_BAD_PAGE | _lib.KV_BAD_LENGTH
    check(cache, batch, q, out, lse, new, kv, 64 ** -0.5, skip=(1, 2))
    assert (out[3 * n:] == 3).all()


def test_strided_and_unaligned_queries():
    new, kv = [3, 20], [40, 20]
    cache, batch, q = build(new, kv, 16, 2, 64, 4, "bf16", seed=11)
    want = cache.attend(batch, q)
    fused = torch.zeros(23, 8, 64, device=DEV, dtype=torch.bfloat16)
    fused[:, 2:6] = q
    out = torch.zeros(23, 4, 128, device=DEV, dtype=torch.bfloat16)
    cache.attend(batch, fused[:, 2:6], out=out[..., 64:])
    assert torch.equal(out[..., 64:], want) and (out[..., :64] == 0).all()
    odd = torch.zeros(23 * 4 * 64 + 1, device=DEV, dtype=torch.bfloat16)[1:].view(23, 4, 64)
    odd.copy_(q)
    assert torch.equal(cache.attend(batch, odd), want)
    with pytest.raises(ValueError, match="aligned"):
        cache.attend(batch, q, out=odd)


def test_refusals():
    cache, batch, q = build([2], [20], 16, 2, 64, 4, "f16")
    bad = [dict(q=q[:, :3]), dict(q=q.bfloat16()), dict(q=q[..., :32]), dict(q=q[0]),
           dict(q=q, window=4, causal=False), dict(q=q, window=-1),
           dict(q=q, out=torch.empty_like(q)[:1]), dict(q=q, lse=torch.empty(2, 3, device=DEV)),
           dict(q=q, status=torch.zeros(1, device=DEV)), dict(q=q.cpu())]
    for kw in bad:
        with pytest.raises(ValueError):
            cache.attend(batch, **kw)
    with pytest.raises(ValueError):
        KVBatch(batch.q_start, batch.kv_lens, batch.page_table[:, :1].expand(1, 3).t())
    with pytest.raises(ValueError):
        KVBatch(batch.q_start[:1], batch.kv_lens, batch.page_table)
    with pytest.raises(RuntimeError, match="status -1"):
        cache.attend(batch, q, scale=float("nan"))


@pytest.mark.parametrize("kind,n", [("f16", 1), ("q8_bf16", 3), ("bf16", 90)])
def test_captured_and_replayed(kind, n):
    """A graph of write and attend reads the lengths of each replay; two
    graphs at once on two streams keep to themselves."""
    new, kv = [n, n], [n + 700, n + 50]
    cache, batch, q = build(new, kv, 16, 2, 128, 8, kind, seed=12, extra_pages=4)
    cache2, batch2, q2 = build(new, kv, 16, 2, 128, 8, kind, seed=13, extra_pages=4)
    x = torch.randn(2 * n, 2, 128, device=DEV).to(q.dtype)
    graphs = []
    for c, b, qq in ((cache, batch, q), (cache2, batch2, q2)):
        c.attend(b, qq)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            c.write(b, x, x)
            o = c.attend(b, qq)
        graphs.append((g, o))
    streams = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    for _ in range(3):
        for s, (g, _) in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for (g, o), (c, b, qq) in zip(graphs, ((cache, batch, q), (cache2, batch2, q2))):
        check(c, b, qq, o, None, new, kv, 128 ** -0.5)
        assert torch.equal(o, c.attend(b, qq))
    # other lengths, same graph
    batch.kv_lens -= 25
    graphs[0][0].replay()
    check(cache, batch, q, graphs[0][1], None, new, [k - 25 for k in kv], 128 ** -0.5)


def test_repeats_are_equal():
    cache, batch, q = build([1] * 20 + [70], [900 * (i % 5) + 7 for i in range(20)] + [4000], 16, 2,
                            128, 16, "f16", seed=14)
    first = cache.attend(batch, q)
    for _ in range(3):
        assert torch.equal(cache.attend(batch, q), first)


@pytest.mark.parametrize("kind", ["f16", "bf16", "q8_f16"])
@pytest.mark.parametrize("dim,new,kv", [(256, [64], [2560]), (256, [129], [700]),
                                        (128, [300], [2560]), (64, [400, 3], [900, 800])])
def test_split_tiles_repeat(dim, new, kv, kind):
    """Short stretches of many tiles per CTA: every start and end of a tile
    meets every phase of the pipeline; twenty runs, one result."""
    cache, batch, q = build(new, kv, 64, 1, dim, 8, kind, seed=21)
    first = cache.attend(batch, q)
    check(cache, batch, q, first, None, new, kv, dim ** -0.5)
    for _ in range(20):
        assert torch.equal(cache.attend(batch, q), first)


@pytest.mark.parametrize("kind", ["q8_f16", "q8_bf16"])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_quantised_chunk_under_a_wide_table(dim, kind):
    """A page table so wide that the pages are not expanded in the workspace:
    the kernel decodes the codes of several tiles itself, to the same bits."""
    new, kv = [200, 90], [700, 95]
    cache, batch, q = build(new, kv, 256, 2, dim, 8, kind, seed=22)
    narrow = cache.attend(batch, q)
    check(cache, batch, q, narrow, None, new, kv, dim ** -0.5)
    wide = torch.full((2, 1100 * 256 // dim), -1, dtype=torch.int32, device=DEV)
    wide[:, :batch.max_pages] = batch.page_table
    out = cache.attend(KVBatch(batch.q_start, batch.kv_lens, wide), q)
    assert torch.equal(out, narrow)


@pytest.mark.parametrize("scale", [0.0, -0.3])
@pytest.mark.parametrize("kind", ["f16", "bf16", "q8_bf16"])
@pytest.mark.parametrize("name", ["decode", "drafts", "chunk", "chunk_256"])
def test_unusual_scales(name, kind, scale):
    """Zero: the mean of the attended values; negative: the smallest products
    weigh most."""
    new, kv, page, heads, dim, q_heads = CASES[name]
    cache, batch, q = build(new, kv, page, heads, dim, q_heads, kind, seed=15)
    out = cache.attend(batch, q, scale=scale, window=(1 << 31) - 1)
    check(cache, batch, q, out, None, new, kv, scale)


def test_many_short_sequences():
    """More sequences than threads, empty ones among them (at both ends), and
    one long; rows of one sequence reaching other tiles than their neighbours."""
    new = [0, 0] + [i % 3 for i in range(700)] + [40] + [1] * 50 + [0]
    kv = [n + (7 * i) % 90 for i, n in enumerate(new)]
    for kind in ("bf16", "q8_f16"):
        cache, batch, q = build(new, kv, 16, 2, 64, 4, kind, seed=16)
        lse = torch.empty(q.shape[:2], device=DEV)
        out = cache.attend(batch, q, lse=lse)
        check(cache, batch, q, out, lse, new, kv, 0.125)


@pytest.mark.parametrize("n", [1, 70])
def test_shared_pages(n):
    """Two sequences whose tables share the pages of a common beginning."""
    kv = [64 + n, 64 + n]
    cache, batch, q = build([n, n], kv, 16, 2, 128, 8, "f16", seed=17)
    batch.page_table[1, :4] = batch.page_table[0, :4]
    out = cache.attend(batch, q)
    check(cache, batch, q, out, None, [n, n], kv, 128 ** -0.5)


@pytest.mark.parametrize("n", [1, 100])
def test_other_stream(n):
    cache, batch, q = build([n], [900], 16, 2, 128, 8, "q8_bf16", seed=18)
    want = cache.attend(batch, q)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    outs = [cache.attend(batch, q, stream=s) for _ in range(4)]
    s.synchronize()
    assert all(torch.equal(o, want) for o in outs)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows", [8, 9, 16, 17, 48, 49, 64, 65])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_numbers_of_rows_between_the_kernels(dim, rows, kind):
    """Every tile height on both sides of the sizes at which it changes."""
    new, kv = [rows, rows - 3, rows + 3], [rows + 600, rows - 3, 900]
    cache, batch, q = build(new, kv, 32, 1, dim, 1, kind, seed=34)
    lse = torch.empty(q.shape[:2], device=DEV)
    check(cache, batch, q, cache.attend(batch, q, lse=lse), lse, new, kv, dim ** -0.5)


@pytest.mark.parametrize("kind", ["f16", "q8_bf16"])
@pytest.mark.parametrize("n", [1, 5, 300])
def test_two_streams_at_once(n, kind):
    """Calls that run side by side have workspaces of their own."""
    parts = []
    for seed in (31, 32):
        cache, batch, q = build([n, 2], [n + 900 + seed, 40], 16, 2, 128, 8, kind, seed=seed)
        parts.append((cache, batch, q, cache.attend(batch, q), torch.cuda.Stream()))
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(10):
        for i, (cache, batch, q, _, stream) in enumerate(parts):
            outs[i].append(cache.attend(batch, q, stream=stream))
    torch.cuda.synchronize()
    for i, (_, _, _, want, _) in enumerate(parts):
        assert all(torch.equal(o, want) for o in outs[i])


@pytest.mark.parametrize("kind", ["f16", "q8_bf16"])
@pytest.mark.parametrize("dim,n", [(64, 1), (128, 4), (128, 700), (256, 300)])
def test_output_in_place_of_the_queries(dim, n, kind):
    cache, batch, q = build([n, 1, 3], [n + 1500, 700, 3], 32, 2, dim, 8, kind, seed=33)
    want = cache.attend(batch, q)
    got = cache.attend(batch, q, out=q)
    assert got.data_ptr() == q.data_ptr() and torch.equal(got, want)


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("n", [1, 3, 90])
def test_infinite_scores(n, kind):
    """Rows whose scores are all minus infinity have no softmax: NaN, as in
    the definition; a single such key gets no weight."""
    cache, batch, q = build([n, n], [n + 200, n + 200], 16, 1, 64, 4, kind, seed=19)
    q.abs_()
    cache.k[batch.page_table[0].long()] = -float("inf")
    pg = int(batch.page_table[1, 2])
    cache.k[pg, 0, 5] = -float("inf")
    out = cache.attend(batch, q)
    assert out[:n].isnan().all()
    assert out[n:].isfinite().all()
    clean = cache.k.clone()
    cache.k[pg, 0, 5] = torch.finfo(cache.k.dtype).min / 64
    assert torch.equal(cache.attend(batch, q)[n:], out[n:])
    cache.k.copy_(clean)


@pytest.mark.parametrize("kind", ["f16", "q8_bf16"])
def test_serving_run(kind):
    """A prompt in chunks, then single tokens: write and attend step by step,
    every output equal to attention over the values read back."""
    type_id, dtype = KINDS[kind]
    page, heads, dim, q_heads = 16, 2, 64, 8
    g = torch.Generator(device=DEV).manual_seed(1)
    cache = PagedKVCache.empty(40, page, heads, dim, type_id, DEV)
    table = torch.randperm(40, generator=g, device=DEV).to(torch.int32).view(2, 20)
    length = [0, 0]
    for step in ([100, 33], [60, 1], [1, 0], [1, 1], [1, 1], [4, 2], [1, 1]):
        length = [a + b for a, b in zip(length, step)]
        start = torch.tensor([0, step[0], sum(step)], dtype=torch.int32, device=DEV)
        batch = KVBatch(start, torch.tensor(length, dtype=torch.int32, device=DEV), table)
        T = sum(step)
        k, v = (torch.randn(T, heads, dim, generator=g, device=DEV).to(dtype) for _ in range(2))
        q = torch.randn(T, q_heads, dim, generator=g, device=DEV).to(dtype)
        cache.write(batch, k, v)
        out = cache.attend(batch, q)
        check(cache, batch, q, out, None, step, length, dim ** -0.5)
        rk, rv = cache.read(batch, tokens=T, dtype=torch.float32)
        if type_id != Q8_0:
            assert torch.equal(rk, k.float()) and torch.equal(rv, v.float())


def test_offsets_past_32_bits():
    """A cache of more than 2^31 values (and 2^32 bytes): the last pages."""
    if torch.cuda.mem_get_info()[0] < (24 << 30):
        pytest.skip("not enough free memory")
    pages, page, heads, dim = 70000, 64, 2, 256
    cache = PagedKVCache.empty(pages, page, heads, dim, F16, DEV)
    table = torch.arange(pages - 3, pages, dtype=torch.int32, device=DEV).view(1, 3)
    for n in (1, 100):
        batch = KVBatch(torch.tensor([0, n], dtype=torch.int32, device=DEV),
                        torch.tensor([150], dtype=torch.int32, device=DEV), table)
        first = KVBatch(torch.tensor([0, 150], dtype=torch.int32, device=DEV), batch.kv_lens, table)
        k = torch.randn(150, heads, dim, device=DEV).half()
        v = torch.randn(150, heads, dim, device=DEV).half()
        cache.write(first, k, v)
        rk, rv = cache.read(first, tokens=150)
        assert torch.equal(rk, k) and torch.equal(rv, v)
        q = torch.randn(n, 16, dim, device=DEV).half()
        check(cache, batch, q, cache.attend(batch, q), None, [n], [150], dim ** -0.5)


def test_the_longest_sequence():
    """2^31 - 65536 cached tokens, all in one page that the table names eight
    million times: what attention over that page once gives.  A thread adds up
    226k probabilities and 113k products in fp32, each off by at most 2^-23 of
    the sum.  One token more is refused."""
    cache = PagedKVCache.empty(1, 256, 1, 32, F16, DEV)
    g = torch.Generator(device=DEV).manual_seed(36)
    cache.k.copy_(torch.randn(cache.k.shape, generator=g, device=DEV))
    cache.v.copy_(torch.randn(cache.v.shape, generator=g, device=DEV) + 1)
    q = torch.randn((1, 1, 32), generator=g, device=DEV).half()
    table = torch.zeros((1, 1 << 23), dtype=torch.int32, device=DEV)
    start = torch.tensor([0, 1], dtype=torch.int32, device=DEV)
    lens = torch.tensor([(1 << 31) - 65536], dtype=torch.int32, device=DEV)
    status = torch.full((1,), 99, dtype=torch.int32, device=DEV)
    out = cache.attend(KVBatch(start, lens, table), q, status=status)
    assert status.item() == 0
    w = torch.softmax(cache.k[0, 0].double() @ q[0, 0].double() * 32 ** -0.5, 0)
    want = w @ cache.v[0, 0].double()
    tol = ((226e3 + 113e3) * 2 ** -23 + 2 * K.HALF[torch.float16]) * want.abs().max()
    assert (out[0, 0].double() - want).abs().max() <= tol
    lens += 1
    cache.attend(KVBatch(start, lens, table), q, status=status)
    assert status.item() == _lib.KV_BAD_LENGTH


def test_overlapping_outputs_are_refused():
    cache, batch, q = build([2], [20], 16, 2, 64, 4, "f16")
    one = torch.empty(1, 4, 64, device=DEV, dtype=torch.float16)
    rows = torch.empty(2, 1, 64, device=DEV, dtype=torch.float16)
    for out in (one.expand(2, 4, 64), rows.expand(2, 4, 64)):
        with pytest.raises(ValueError, match="overlap"):
            cache.attend(batch, q, out=out)
        with pytest.raises(ValueError, match="overlap"):
            cache.read(batch, out=(out[:, :2], torch.empty_like(out[:, :2])))
