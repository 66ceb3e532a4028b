"""Inputs and 64-bit definitions for the paged key/value cache tests."""
from __future__ import annotations

import math

import torch

# How far a result may be off, in the units of its own rounding: half a step
# relative to the value is eps / 2.
HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def make_batch(new, kv, page, seed=0, device="cpu", spare=2, extra_pages=0):
    """q_start, kv_lens, page_table of sequences with `new` rows and `kv`
    cached tokens; the pages lie anywhere in a pool of the returned size."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // page) for n in kv]
    pool = sum(need) + spare
    order = torch.randperm(pool, generator=g).to(torch.int32)
    width = max([1, *need]) + extra_pages
    table = torch.full((len(kv), width), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    start = torch.tensor([0, *torch.tensor(new).cumsum(0).tolist()], dtype=torch.int32)
    return (start.to(device), torch.tensor(kv, dtype=torch.int32).to(device), table.to(device),
            pool)


def quantise(x):
    """Q8_0 codes and scales of x [..., dim] (float64 arithmetic)."""
    b = x.double().unflatten(-1, (-1, 32))
    want = b.abs().amax(-1) / 127
    d = want.half()
    # one binary16 step above d (2^-24 above zero and the smallest values)
    step = torch.exp2((torch.frexp(d.float()).exponent.double() - 11).clamp(min=-24))
    up = d.double() + torch.where(d > 0, step, 2.0 ** -24)
    d = torch.where(d.double() < want, up, d.double()).clamp(max=515.5)
    n = torch.where(d[..., None] > 0, b / torch.where(d > 0, d, 1.0)[..., None], 0.0)
    return n.round().clamp(-127, 127).flatten(-2), d


def values(codes, scales):
    return (codes.double().unflatten(-1, (-1, 32)) * scales.double()[..., None]).flatten(-2)


def gather(cache, scales, table, length, page):
    """[length, heads, dim] float64 rows of one sequence; Q8_0 values rounded
    to binary16, as the attention takes them."""
    pos = torch.arange(length, device=cache.device)
    ids = table.long()[pos // page]
    x = cache[ids, :, pos % page].double()
    if scales is not None:
        x = values(x, scales[ids, :, pos % page]).half().double()
    return x


def attend(q, k, v, first, scale, causal=True, window=0):
    """q [n, Hq, D] over k, v [length, H, D] in 64 bits, the rows at positions
    first, first + 1, ...: outputs, log-sum-exp, and per row and head the sum
    of p |v| (what a relative error of the probabilities can move)."""
    n, hq, dim = q.shape
    length, h, _ = k.shape
    group = hq // h
    out = torch.zeros(n, hq, dim, dtype=torch.float64, device=q.device)
    lse = torch.full((n, hq), -math.inf, dtype=torch.float64, device=q.device)
    mass = torch.zeros_like(out)
    for i in range(n):
        hi = min(first + i + 1, length) if causal else length
        lo = max(0, first + i - window + 1) if window else 0
        if hi <= lo:
            continue
        for g in range(h):
            s = q[i, g * group:(g + 1) * group].double() @ k[lo:hi, g].T * scale
            p = torch.softmax(s, -1)
            out[i, g * group:(g + 1) * group] = p @ v[lo:hi, g]
            mass[i, g * group:(g + 1) * group] = p @ v[lo:hi, g].abs()
            lse[i, g * group:(g + 1) * group] = torch.logsumexp(s, -1)
    return out, lse, mass
