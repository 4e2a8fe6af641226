"""What a row sees and what it does not."""

from __future__ import annotations

import pytest
import torch

from sglang_restomod_b200 import ops
from tests.test_gpu_attention import BF16, E4M3, F16, build

pytestmark = pytest.mark.gpu


def run(case, max_q, **kw):
    cache, q, table, kv_lens, starts = case[:5]
    return ops.paged_attention(q.cuda(), cache, table.cuda(), kv_lens.cuda(), starts.cuda(), max_q,
                               return_lse=True, **kw)


@pytest.mark.parametrize("store,q_dtype", [(BF16, BF16), (F16, F16), (E4M3, BF16)])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("page", [1, 8, 16, 24, 64])
@pytest.mark.parametrize("q_len", [1, 30])
def test_pages_before_the_window_may_be_gone(cuda_device, store, q_dtype, dim, page, q_len):
    window, kv = 53, 331
    case = build(dim + page, [q_len, 1], [kv, 77], 2, 4, dim, page, q_dtype, store)
    table = case[2]
    for s, n in ((0, kv - q_len), (1, 76)):
        table[s, :max(0, n - window + 1) // page] = -1
    want, want_lse = run(build(dim + page, [q_len, 1], [kv, 77], 2, 4, dim, page, q_dtype, store),
                         q_len, window=window)
    got, lse = run(case, q_len, window=window)
    assert ops.attention_status() == 0
    assert torch.equal(got, want) and torch.equal(lse, want_lse)
