"""Values outside a call's window or past its lengths may be anything, an
infinity or NaN too: no row that does not see them shows it. And calls at the
borders of the kernels' rules."""

from __future__ import annotations

import math

import pytest
import torch

from oracle import attention as ref
from sglang_restomod_b200 import ops
from tests.test_gpu_attention import BF16, E4M3, F16, bounds, build, check

pytestmark = pytest.mark.gpu


def poison(case, s, tokens, page):
    """Infinities and NaN at some cached tokens of sequence s (their float64
    values stay what they were: no row sees them)."""
    cache, table = case[0], case[2]
    for i, t in enumerate(tokens):
        at = (table[s, t // page].item(), t % page)
        if cache.k_scale is None:
            cache.k[at] = cache.v[at] = float("nan") if i % 2 else float("inf")
        else:
            cache.k_scale[at] = cache.v_scale[at] = 255


@pytest.mark.parametrize("store,q_dtype", [(BF16, BF16), (F16, F16), (E4M3, BF16)])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("page", [1, 16, 24, 64])
@pytest.mark.parametrize("q_len", [1, 4, 45, 150])
def test_not_finite_before_the_window(cuda_device, store, q_dtype, dim, page, q_len):
    window, kv = 37, 301
    case = build(dim + page + q_len, [q_len, 1], [kv, 20], 2, 3, dim, page, q_dtype, store)
    poison(case, 0, range(kv - q_len - window + 1), page)
    check(case, window=window)


def test_more_sequences_than_the_plan_keeps_on_chip(cuda_device):
    seqs = 4200
    check(build(3, [3] * seqs, [3 + s % 7 for s in range(seqs)], 1, 6, 64, 8, BF16, BF16))


@pytest.mark.parametrize("store,q_dtype", [(BF16, BF16), (F16, F16), (E4M3, BF16)])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("page", [8, 12])
@pytest.mark.parametrize("q_len,groups", [(1, 8), (2, 8), (1, 9), (2, 16), (33, 4), (129, 4), (171, 3)])
def test_rows_around_the_rules(cuda_device, store, q_dtype, dim, page, q_len, groups):
    check(build(dim + q_len, [q_len, 1, 0], [q_len + 150, 70, 3], 1, groups, dim, page, q_dtype, store))


def test_one_unit_over_all_blocks(cuda_device):
    check(build(5, [20], [20011], 1, 1, 128, 64, BF16, E4M3))
    check(build(6, [20, 2], [20011, 9000], 1, 1, 256, 16, F16, F16), window=15000)


@pytest.mark.parametrize("store,q_dtype", [(BF16, BF16), (F16, F16), (E4M3, BF16), (E4M3, F16)])
@pytest.mark.parametrize("page", [1, 16])
@pytest.mark.parametrize("scale", [0.0, -0.11, 1e-30])
@pytest.mark.parametrize("q_len,groups", [(1, 8), (40, 4), (150, 4)])
def test_scales_of_any_sign(cuda_device, store, q_dtype, page, scale, q_len, groups):
    case = build(q_len, [q_len, 2], [q_len + 190, 2], 1, groups, 128, page, q_dtype, store)
    cache, q, table, kv_lens, starts, kc, vc = case
    out, lse = ops.paged_attention(q.cuda(), cache, table.cuda(), kv_lens.cuda(), starts.cuda(),
                                   max(q_len, 2), scale=scale, return_lse=True)
    want, want_lse = ref.paged_attention_ref(q, kc, vc, table, kv_lens, starts, scale)
    # (the bound grows with the scores' magnitude, whatever their sign)
    tol, lse_tol = bounds(q, kc, vc, abs(scale), q_dtype, q_dtype)
    assert (out.cpu().double() - want).abs().max().item() <= tol
    assert (lse.cpu().double() - want_lse).abs().max().item() <= lse_tol


@pytest.mark.parametrize("page", [1, 16])
@pytest.mark.parametrize("q_len", [1, 40, 150])
@pytest.mark.parametrize("size", [2.0 ** -12, 2.0 ** 13])
def test_e4m3_of_small_and_large_values(cuda_device, page, q_len, size):
    """Values of V about `size`; K's are the usual ones."""
    cache, q, table, kv_lens, starts, kc, vc = build(q_len, [q_len], [q_len + 190], 1, 4, 128, page,
                                                     BF16, E4M3)
    shift = round(math.log2(size))
    scaled = cache.v_scale.cpu().int() + shift
    written = cache.v_scale.cpu() != 255
    # the bytes' powers of two moved alike: codes and float64 values follow
    cache.v_scale.copy_(torch.where(written, scaled.clamp(103, 134), 255).to(torch.uint8))
    assert (scaled[written] >= 103).all() and (scaled[written] <= 134).all()
    check((cache, q, table, kv_lens, starts, kc, vc * size))
