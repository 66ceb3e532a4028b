"""The paged key/value cache and the attention that reads it, as measured cases.

Three operators, reached through ``flash_moe_b200.paged_kv``:

* ``store``   ``PagedKVCache.write``: new keys and values scattered into the
  pages of their sequences; a Q8_0 cache quantises them on the way (32 values
  share a binary16 scale) and ``PagedKVCache.read`` gives back the values the
  codes stand for;
* ``read``    ``PagedKVCache.read``: whole sequences gathered out of the pages;
* ``attend``  ``PagedKVCache.attend``: the new tokens of every sequence (a chunk
  of a prompt, a few drafted tokens, a single decoded token) over their cached
  keys, causal, with shared key/value heads and an optional window.

A batch is ``q_start`` [B + 1] (rows of each sequence among the new tokens),
``kv_lens`` [B] (cached length with the new tokens) and ``page_table``
[B, max_pages]: row i of sequence b stands at position
``kv_lens[b] - (q_start[b+1] - q_start[b]) + i``.
"""
import math
import random
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "intel-optimized-moe-streaming_b200"))

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
SIZES = {"f16": 2, "bf16": 2, "f32": 4}
BLOCK = 32            # values that share one scale in a Q8_0 row
SCALE_MAX = 515.5     # largest scale: 127 * 515.5 stays inside binary16


def listed():
    return [
        # one decoded token's keys and values into a quantised cache: latency
        {"name": "store_one_q8", "op": "store", "kind": "q8_0", "dtype": "f16", "seqs": 1,
         "new": 1, "past": 900, "heads": 2, "dim": 256, "page": 16, "lens": 1},
        # a ragged batch of prompts into a 16-bit cache of small pages
        {"name": "store_prompts_bf16", "op": "store", "kind": "bf16", "dtype": "bf16", "seqs": 37,
         "new": 611, "past": 1200, "heads": 8, "dim": 128, "page": 16, "lens": 2},
        # long prompts quantised as they are written, and read back
        {"name": "store_prompts_q8", "op": "store", "kind": "q8_0", "dtype": "bf16", "seqs": 16,
         "new": 8192, "past": 0, "heads": 8, "dim": 128, "page": 64, "lens": 3},
        # one short sequence gathered out of a 16-bit cache
        {"name": "read_short_f16", "op": "read", "kind": "f16", "dtype": "f16", "seqs": 1,
         "new": 333, "past": 0, "heads": 2, "dim": 256, "page": 32, "lens": 4},
        # a batch of long quantised sequences gathered as bf16
        {"name": "read_long_q8", "op": "read", "kind": "q8_0", "dtype": "bf16", "seqs": 24,
         "new": 20000, "past": 0, "heads": 4, "dim": 128, "page": 64, "lens": 5},
        # one token of one short sequence: the smallest decode step
        {"name": "decode_one_f16", "op": "attend", "kind": "f16", "dtype": "f16", "seqs": 1,
         "new": 1, "past": 1000, "q_heads": 16, "heads": 2, "dim": 256, "page": 16, "window": 0,
         "lens": 6},
        # a serving batch of single tokens over ragged contexts
        {"name": "decode_batch_bf16", "op": "attend", "kind": "bf16", "dtype": "bf16", "seqs": 64,
         "new": 1, "past": 8000, "q_heads": 32, "heads": 8, "dim": 128, "page": 16, "window": 0,
         "lens": 7},
        # single tokens over long quantised contexts
        {"name": "decode_long_q8", "op": "attend", "kind": "q8_0", "dtype": "bf16", "seqs": 24,
         "new": 1, "past": 32768, "q_heads": 16, "heads": 2, "dim": 256, "page": 64, "window": 0,
         "lens": 8},
        # drafted tokens of a batch checked in one pass
        {"name": "draft_f16", "op": "attend", "kind": "f16", "dtype": "f16", "seqs": 33,
         "new": 5, "past": 3000, "q_heads": 16, "heads": 8, "dim": 64, "page": 32, "window": 0,
         "lens": 9},
        # a chunk of a long prompt behind its cached beginning
        {"name": "chunk_long_bf16", "op": "attend", "kind": "bf16", "dtype": "bf16", "seqs": 1,
         "new": 4096, "past": 12288, "q_heads": 16, "heads": 2, "dim": 256, "page": 64,
         "window": 0, "lens": 10},
        # ragged chunks of several prompts, each row seeing a window
        {"name": "chunk_ragged_f16", "op": "attend", "kind": "f16", "dtype": "f16", "seqs": 9,
         "new": 1700, "past": 2500, "q_heads": 32, "heads": 8, "dim": 128, "page": 16,
         "window": 1024, "lens": 11},
        # chunks of prompts over a quantised cache
        {"name": "chunk_q8", "op": "attend", "kind": "q8_0", "dtype": "bf16", "seqs": 2,
         "new": 2048, "past": 8192, "q_heads": 32, "heads": 8, "dim": 128, "page": 64,
         "window": 0, "lens": 12},
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    largest = {}
    for c in listed():
        w = work(c)
        for k in ("bytes", "flops"):
            largest[c["op"], k] = max(largest.get((c["op"], k), 0), w[k])
    op = rng.choice(["store", "read", "attend", "attend", "attend"])
    while True:
        kind = rng.choice(["f16", "bf16", "q8_0"])
        c = {"op": op, "kind": kind,
             "dtype": rng.choice(["f16", "bf16"]) if kind == "q8_0" else kind,
             "seqs": _log_int(rng, 1, 64), "heads": rng.choice([1, 2, 3, 4, 8]),
             "dim": rng.choice([64, 96, 128, 192, 256]), "page": rng.choice([16, 32, 64, 128]),
             "lens": rng.randrange(1 << 30)}
        if op == "attend":
            c["q_heads"] = c["heads"] * rng.choice([1, 2, 4, 5, 8])
            c["new"] = rng.choice([1, 1, _log_int(rng, 2, 16), _log_int(rng, 17, 4096)])
            c["past"] = _log_int(rng, 1, 32768)
            c["window"] = rng.choice([0, 0, 0, _log_int(rng, 16, 4096)])
        elif op == "store":
            c["new"] = rng.choice([1, _log_int(rng, 2, 8192)])
            c["past"] = _log_int(rng, 1, 4096)
        else:
            c["new"] = _log_int(rng, 1, 20000)
            c["past"] = 0
        w = work(c)
        if all(w[k] <= largest[op, k] for k in ("bytes", "flops")):
            return c


def _lengths(case):
    """New tokens and cached length of every sequence.  One sequence has
    exactly the case's sizes; of several, the first has them and the others
    spread below (down to a half for new tokens, anywhere for the past)."""
    rng = random.Random(case["lens"])
    new, kv = [], []
    for b in range(case["seqs"]):
        n = case["new"] if b == 0 or case["new"] < 8 else rng.randint(case["new"] // 2, case["new"])
        p = case["past"] if b == 0 else rng.randint(0, case["past"])
        new.append(n)
        kv.append(n + p)
    return new, kv


def _pairs(n, length, window):
    """Attended (row, key) pairs and touched keys of one sequence."""
    first = length - n
    if not window:
        return n * first + n * (n + 1) // 2, length
    pairs = sum(min(first + i + 1, window) for i in range(n))
    return pairs, min(length, n + window - 1)


def work(case):
    new, kv = _lengths(case)
    T, H, D = sum(new), case["heads"], case["dim"]
    row = D + D // BLOCK * 2 if case["kind"] == "q8_0" else D * SIZES[case["kind"]]
    val = D * SIZES[case["dtype"]]
    if case["op"] == "store":
        back = val if case["kind"] == "q8_0" else 0
        return {"bytes": 2 * T * H * (val + row + back), "flops": 0}
    if case["op"] == "read":
        return {"bytes": 2 * T * H * (row + val), "flops": 0}
    pairs = keys = 0
    for n, length in zip(new, kv):
        p, k = _pairs(n, length, case["window"])
        pairs += p
        keys += k
    return {"bytes": 2 * T * case["q_heads"] * val + 2 * keys * H * row,
            "flops": 4 * D * case["q_heads"] * pairs}


# --------------------------------------------------------------------- inputs

def _inputs(case, seed):
    """Tensors of a case: the batch, the cache with every page filled, the new
    rows.  The pages of a sequence lie anywhere in the pool."""
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    new, kv = _lengths(case)
    H, D, P = case["heads"], case["dim"], case["page"]
    need = [-(-length // P) for length in kv]
    pool = sum(need) + 3
    order = torch.randperm(pool, generator=g, device=dev).to(torch.int32)
    width = max(need)
    table = torch.zeros((len(kv), width), dtype=torch.int32, device=dev)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    st = {"q_start": torch.tensor(starts, dtype=torch.int32, device=dev),
          "kv_lens": torch.tensor(kv, dtype=torch.int32, device=dev), "page_table": table,
          "new": new, "kv": kv}

    def normal(*shape, dtype, spread=1.0):
        x = torch.randn(shape, generator=g, device=dev, dtype=torch.float16)
        return (x * spread).to(dtype)

    shape = (pool, H, P, D)
    if case["kind"] == "q8_0":
        for name in "kv":
            st[name] = torch.randint(-127, 128, shape, generator=g, device=dev, dtype=torch.int8)
            # scales of rows of unit variance: a block's maximum is near 2.1
            u = torch.rand((pool, H, P, D // BLOCK), generator=g, device=dev)
            st[name + "_scales"] = ((1.3 + 1.6 * u) / 127).half()
    else:
        for name in "kv":
            st[name] = normal(*shape, dtype=DTYPES[case["kind"]])
    T = sum(new)
    if case["op"] == "attend":
        st["q"] = normal(T, case["q_heads"], D, dtype=DTYPES[case["dtype"]])
    elif case["op"] == "store":
        # a projection's output holds keys and values side by side: strided rows
        both = normal(T, 2, H, D, dtype=DTYPES[case["dtype"]])
        st["new_k"], st["new_v"] = both[:, 0], both[:, 1]
    return st


def prepare(case, seed):
    st = _inputs(case, seed)
    st["case"] = case
    st["scale"] = case["dim"] ** -0.5
    if own:
        from flash_moe_b200.paged_kv import KVBatch, PagedKVCache
        st["cache"] = PagedKVCache(st["k"], st["v"], st.get("k_scales"), st.get("v_scales"))
        st["batch"] = KVBatch(st["q_start"], st["kv_lens"], st["page_table"])
    return st


# ---------------------------------------------------------------- plain forms

def _slots(st, page, b):
    """Page and row of each new token of sequence b."""
    n, length = st["new"][b], st["kv"][b]
    pos = torch.arange(length - n, length, device=st["page_table"].device)
    return st["page_table"][b].long()[pos // page], pos % page


def _quantise(x):
    """Q8_0 codes and scales of fp32 rows: d = max|x| / 127 rounded up to
    binary16, code = x / d to the nearest integer."""
    blocks = x.unflatten(-1, (-1, BLOCK))
    want = blocks.abs().amax(-1) / 127
    d = want.half()
    low = d.float() < want
    d = torch.where(low, (d.view(torch.int16) + 1).view(torch.float16), d)
    d = d.clamp(max=SCALE_MAX)
    step = torch.where(d > 0, d, torch.ones_like(d)).float()
    codes = torch.round(blocks / step[..., None]).clamp(-127, 127)
    codes = torch.where(d[..., None] > 0, codes, torch.zeros_like(codes))
    return codes.flatten(-2).to(torch.int8), d


def _values(codes, scales):
    return (codes.float().unflatten(-1, (-1, BLOCK)) * scales.float()[..., None]).flatten(-2)


def _gather(st, case, name, pages, rows):
    """fp32 rows [n, heads, dim] of a cache at (pages, rows)."""
    if case["kind"] == "q8_0":
        return _values(st[name][pages, :, rows], st[name + "_scales"][pages, :, rows])
    return st[name][pages, :, rows].float()


def _plain_store(st, case):
    out = {"k": [], "v": []}
    for b in range(case["seqs"]):
        pages, rows = _slots(st, case["page"], b)
        lo = sum(st["new"][:b])
        for name in "kv":
            x = st["new_" + name][lo:lo + st["new"][b]].float()
            if case["kind"] == "q8_0":
                codes, d = _quantise(x)
                st[name][pages, :, rows] = codes
                st[name + "_scales"][pages, :, rows] = d
                out[name].append(_values(codes, d).to(DTYPES[case["dtype"]]))
            else:
                st[name][pages, :, rows] = x.to(DTYPES[case["kind"]])
    if case["kind"] == "q8_0":
        return torch.cat(out["k"]), torch.cat(out["v"])
    return st["k"], st["v"]


def _plain_read(st, case):
    out = {"k": [], "v": []}
    for b in range(case["seqs"]):
        pages, rows = _slots(st, case["page"], b)
        for name in "kv":
            out[name].append(_gather(st, case, name, pages, rows).to(DTYPES[case["dtype"]]))
    return torch.cat(out["k"]), torch.cat(out["v"])


def _plain_attend(st, case):
    Hq, H, D, window = case["q_heads"], case["heads"], case["dim"], case["window"]
    group = Hq // H
    out = torch.empty_like(st["q"])
    dev = out.device
    lo = 0
    for n, length, table in zip(st["new"], st["kv"], st["page_table"].long()):
        pos = torch.arange(length, device=dev)
        pages, rows = table[pos // case["page"]], pos % case["page"]
        k = _gather(st, case, "k", pages, rows).permute(1, 2, 0)    # [H, D, keys]
        v = _gather(st, case, "v", pages, rows).permute(1, 0, 2)    # [H, keys, D]
        step = max(1, (1 << 28) // (Hq * length))
        for r in range(0, n, step):
            m = min(step, n - r)
            q = st["q"][lo + r:lo + r + m].float().view(m, H, group, D)
            q = q.permute(1, 0, 2, 3).reshape(H, m * group, D)
            s = (q @ k).view(H, m, group, length) * st["scale"]
            at = torch.arange(length - n + r, length - n + r + m, device=dev)[:, None]
            seen = pos[None] <= at
            if window:
                seen &= pos[None] > at - window
            s = s.masked_fill(~seen[None, :, None], float("-inf"))
            p = torch.exp(s - s.amax(-1, keepdim=True))
            o = (p.view(H, m * group, length) @ v) / p.sum(-1).view(H, m * group, 1)
            o = o.view(H, m, group, D).permute(1, 0, 2, 3).reshape(m, Hq, D)
            out[lo + r:lo + r + m] = o.to(out.dtype)
        lo += n
    return out


def run(st):
    case = st["case"]
    if own:
        cache, batch = st["cache"], st["batch"]
        if case["op"] == "attend":
            return cache.attend(batch, st["q"], scale=st["scale"], window=case["window"])
        if case["op"] == "read":
            return cache.read(batch, tokens=sum(st["new"]), dtype=DTYPES[case["dtype"]])
        cache.write(batch, st["new_k"], st["new_v"])
        if case["kind"] == "q8_0":
            return cache.read(batch, tokens=sum(st["new"]), dtype=DTYPES[case["dtype"]])
        return cache.k, cache.v
    return {"store": _plain_store, "read": _plain_read, "attend": _plain_attend}[case["op"]](st, case)


# ---------------------------------------------------------------------- exact

def exact(case, seed):
    """The definition in 64 bits: every key and value looked up one page at a
    time, sums over all of a row's keys at once."""
    st = _inputs(case, seed)
    P, D, H = case["page"], case["dim"], case["heads"]
    bounds = st["q_start"].tolist()
    tables = st["page_table"].tolist()

    def rows_of(name, b, first, last):
        parts = []
        for page in range(first // P, -(-last // P)):
            a, z = max(first - page * P, 0), min(last - page * P, P)
            x = st[name][tables[b][page], :, a:z].double()
            if case["kind"] == "q8_0":
                d = st[name + "_scales"][tables[b][page], :, a:z].double()
                x = x * d.repeat_interleave(BLOCK, dim=-1)
            parts.append(x)
        return torch.cat(parts, dim=1)             # [H, last - first, D]

    if case["op"] == "store":
        if case["kind"] != "q8_0":
            for b, length in enumerate(st["kv"]):
                first = length - st["new"][b]
                for i in range(st["new"][b]):
                    page, row = divmod(first + i, P)
                    for name in "kv":
                        st[name][tables[b][page], :, row] = st["new_" + name][bounds[b] + i]
            return st["k"].double(), st["v"].double()
        back = []
        for name in "kv":
            x = st["new_" + name].double().reshape(-1, H, D // BLOCK, BLOCK)
            top = x.abs().max(dim=-1, keepdim=True).values / 127
            d = top.half().double()
            # one binary16 step up where rounding to nearest went below
            up = d + torch.exp2((torch.frexp(d).exponent.double() - 11).clamp(min=-24))
            d = torch.where(d < top, up, d).clamp(max=SCALE_MAX)
            n = torch.where(d > 0, x / d, torch.zeros_like(x)).round()
            back.append((n * d).reshape(-1, H, D))
        return tuple(back)
    if case["op"] == "read":
        both = []
        for name in "kv":
            seqs = [rows_of(name, b, length - st["new"][b], length).transpose(0, 1)
                    for b, length in enumerate(st["kv"])]
            both.append(torch.cat(seqs))
        return tuple(both)
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device=st["q"].device)
    group = case["q_heads"] // H
    for b, length in enumerate(st["kv"]):
        n = st["new"][b]
        k, v = rows_of("k", b, 0, length), rows_of("v", b, 0, length)
        step = max(1, (1 << 27) // (group * length))
        for h in range(H):
            for r in range(0, n, step):
                m = min(step, n - r)
                q = st["q"][bounds[b] + r:bounds[b] + r + m, h * group:(h + 1) * group].double()
                s = torch.einsum("mgd,kd->mgk", q, k[h]) / math.sqrt(D)
                behind = (torch.arange(length - n + r, length - n + r + m, device=q.device)[:, None]
                          - torch.arange(length, device=q.device)[None])
                hidden = behind < 0
                if case["window"]:
                    hidden |= behind >= case["window"]
                s[hidden[:, None].expand_as(s)] = -math.inf
                w = torch.softmax(s, dim=-1)
                out[bounds[b] + r:bounds[b] + r + m, h * group:(h + 1) * group] = \
                    torch.einsum("mgk,kd->mgd", w, v[h])
    return out
