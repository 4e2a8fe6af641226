"""Eviction as a call: the largest budgets, and tables that are the same memory."""

from __future__ import annotations

import pytest
import torch

from sglang_restomod_b200 import ops
from tests.test_gpu_evict import BF16, Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("budget", [(1 << 31) - 1, (1 << 31) - 300])
def test_largest_budgets(cuda_device, budget):
    """Nothing is over the budget: kept is the tokens, then -1 to its end (8 GB)."""
    c = Case(1, [37], 40, 0, 0, 1, 64, 16, BF16)
    kept, lens = ops.kv_cache_evict(c.cache, c.scores, c.table.cuda(),
                                    torch.tensor([37], dtype=torch.int32, device="cuda"), budget)
    assert kept.shape == (1, 1, budget) and lens.tolist() == [37]
    assert kept[0, 0, :37].tolist() == list(range(37))
    for at in range(37, budget, 1 << 28):
        assert bool((kept[0, 0, at:at + (1 << 28)] == -1).all())
    for got, was in zip(c.dev, c.data):
        assert torch.equal(got.cpu(), was)
    assert ops.attention_status() == 0


@pytest.mark.parametrize("lens", [[700], [700, 90, 333]])
def test_out_table_is_the_page_table(cuda_device, lens):
    """In place, also where one row's view has another stride."""
    c = Case(2, lens, 100, 9, 3, 2, 64, 16, BF16)
    table = c.table.cuda()
    out = table[0, :12][None] if len(lens) == 1 else table
    assert (out.stride(0) != table.stride(0)) == (len(lens) == 1)
    kept, new = ops.kv_cache_evict(c.cache, c.scores, table,
                                   torch.tensor(lens, dtype=torch.int32, device="cuda"), 100, recent=9,
                                   first=3, out_table=out)
    c.check(True, kept, new)
