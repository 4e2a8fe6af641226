"""What the attention tests' bound sees: an oracle that loses part of the context is
outside it."""

from __future__ import annotations

import pytest
import torch

from oracle import attention as ref
from tests.test_gpu_attention_values import column_bound

KV, DIM = 20011, 128


def setup():
    g = torch.Generator().manual_seed(1)
    q = torch.randn(1, 2, DIM, generator=g).to(torch.bfloat16)
    k = torch.randn(1, KV, 1, DIM, generator=g).double()
    table, lens = torch.zeros(1, 1, dtype=torch.int32), torch.tensor([KV])
    return g, (q, k), (table, lens, torch.tensor([0, 1], dtype=torch.int32), DIM ** -0.5)


@pytest.mark.parametrize("lost", [slice(KV // 2, KV), slice(0, 700), slice(9000, 9200)])
@pytest.mark.parametrize("kind", ["pieces", "normal"])
def test_lost_values_are_outside_the_bound(lost, kind):
    g, (q, k), (table, lens, starts, scale) = setup()
    if kind == "pieces":
        v = torch.zeros(1, KV, 1, DIM, dtype=torch.float64)
        t = torch.arange(KV)
        v[0, t, 0, t * DIM // KV] = 1.0
    elif lost.stop - lost.start < 10000:
        return  # a short run of random values is no more than a rounding of their mean
    else:
        v = torch.randn(1, KV, 1, DIM, generator=g).double()
    want, _ = ref.paged_attention_ref(q, k, v, table, lens, starts, scale)
    tol, _ = column_bound(q, k, v, table, lens, starts, scale, 0, torch.bfloat16, False)
    assert (tol < 0.02).all()
    less = v.clone()
    less[:, lost] = 0
    got, _ = ref.paged_attention_ref(q, k, less, table, lens, starts, scale)
    assert ((got - want).abs() > tol).any()
