"""The paged cache at the largest number of rows."""
from __future__ import annotations

import pytest
import torch

from flash_moe_b200.formats import F16
from flash_moe_b200.paged_kv import KVBatch, PagedKVCache

pytestmark = pytest.mark.gpu
DEV = "cuda"


def test_write_of_almost_2_31_rows():
    """The largest number of rows, all equal, written over one page that the
    table names eight million times."""
    n = (1 << 31) - 1
    cache = PagedKVCache.empty(1, 256, 1, 32, F16, DEV)
    cache.k.fill_(7)
    cache.v.fill_(7)
    table = torch.zeros((1, 1 << 23), dtype=torch.int32, device=DEV)
    start = torch.tensor([0, n], dtype=torch.int32, device=DEV)
    lens = torch.tensor([n], dtype=torch.int32, device=DEV)
    k = torch.randn(1, 1, 32, device=DEV).half()
    v = torch.randn(1, 1, 32, device=DEV).half()
    status = torch.full((1,), 99, dtype=torch.int32, device=DEV)
    cache.write(KVBatch(start, lens, table), k.expand(n, 1, 32), v.expand(n, 1, 32), status=status)
    assert status.item() == 0
    assert (cache.k == k[0]).all() and (cache.v == v[0]).all()
