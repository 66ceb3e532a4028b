"""Sizes just past the documented ones are refused before any device work."""
from __future__ import annotations

import pytest

from test_kv_abi import attend, batch, cache


@pytest.mark.parametrize("kv_heads,q_heads,tokens", [
    (1, 1, (1 << 31) - 255), (1, 1, (1 << 31) - 1), (1, 3, ((1 << 31) - 256) // 3 + 1),
    (2, 4, (1 << 29) - 63)])
def test_rows_that_fill_no_whole_tiles_below_2_31(lib, kv_heads, q_heads, tokens):
    assert attend(lib, cache(kv_heads=kv_heads), batch(tokens=tokens), heads=q_heads) == -1
