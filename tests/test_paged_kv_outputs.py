"""Outputs whose rows share memory are refused before any device work.  A cache
object without its tensors stands in for one on a device."""
from __future__ import annotations

import itertools

import pytest
import torch

from flash_moe_b200.paged_kv import PagedKVCache

DIM = 64


def rows(tokens, heads, ts, hs):
    cache = object.__new__(PagedKVCache)
    cache.head_dim, cache._index = DIM, -1   # torch's number for the host
    t = torch.empty(1 << 14, dtype=torch.float16).as_strided((tokens, heads, DIM), (ts, hs, 1))
    return cache._rows(t, heads, (torch.float16,), "out", output=True)


@pytest.mark.parametrize("tokens,heads", [(2, 2), (2, 4), (5, 3), (3, 1), (1, 3)])
def test_rows_that_overlap_are_refused(tokens, heads):
    """Strides in steps of eight values, against the addresses themselves."""
    for ts, hs in itertools.product(range(0, 6 * DIM, 24), range(0, 6 * DIM, 8)):
        at = sorted(i * ts + j * hs for i in range(tokens) for j in range(heads))
        if all(b - a >= DIM for a, b in zip(at, at[1:])):
            rows(tokens, heads, ts, hs)
        else:
            with pytest.raises(ValueError, match="overlap"):
                rows(tokens, heads, ts, hs)


@pytest.mark.parametrize("tokens,heads,ts,hs", [
    (7, 4, 4 * DIM, DIM), (7, 4, DIM, 7 * DIM), (7, 4, 8 * DIM, 2 * DIM), (1, 4, 0, DIM),
    (7, 1, DIM, 0)])
def test_usual_layouts_are_taken(tokens, heads, ts, hs):
    assert rows(tokens, heads, ts, hs)[3] is not None
