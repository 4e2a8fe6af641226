"""Offsets past 32 bits: caches, queries and norm inputs of more than 2^31 elements
(up to 11 GB on the device; nothing of it is copied to the host but samples)."""

from __future__ import annotations

import pytest
import torch

from oracle import attention as ref
from sglang_restomod_b200 import kv_cache, ops
from tests.test_gpu_attention import BF16, E4M3, F16, bounds

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("store,page", [(E4M3, 64), (BF16, 64), (BF16, 1)])
@pytest.mark.parametrize("q_len", [1, 50])
def test_cache_of_more_than_2_31_elements(cuda_device, store, page, q_len):
    heads, dim, kv = 8, 128, 300
    pages = (1 << 31) // (heads * dim * page) + 700
    cache = kv_cache.PagedKVCache.empty(pages, page, heads, dim, cuda_device, store)
    g = torch.Generator().manual_seed(page)
    need = -(-kv // page)
    order = torch.arange(need) + pages - need  # the last pages, backwards
    table = order.flip(0).int()[None]
    t = torch.arange(kv)
    slots = table[0].long()[t // page] * page + t % page
    k, v = (torch.randn(kv, heads, dim, generator=g).to(BF16) for _ in "kv")
    ops.kv_cache_write(cache, k.cuda(), v.cuda(), slots.cuda())
    got_k, got_v = ops.kv_cache_read(cache, slots.cuda(), BF16)
    values = [ref.kv_values_ref(*ref.kv_quantize_ref(x)) if store == E4M3 else x.double()
              for x in (k, v)]
    assert torch.equal(got_k.cpu().double(), values[0]) and torch.equal(got_v.cpu().double(), values[1])
    q = torch.randn(q_len, 4 * heads, dim, generator=g).to(BF16)
    lens = torch.tensor([kv], dtype=torch.int32)
    starts = torch.tensor([0, q_len], dtype=torch.int32)
    out = ops.paged_attention(q.cuda(), cache, table.cuda(), lens.cuda(), starts.cuda(), q_len)
    # the same values on the pages of a small cache
    kc, vc = (x.reshape(1, kv, heads, dim) for x in values)
    want, _ = ref.paged_attention_ref(q, kc, vc, torch.zeros(1, 1, dtype=torch.int32), lens, starts,
                                      dim ** -0.5)
    tol, _ = bounds(q, kc, vc, dim ** -0.5, BF16, BF16)
    assert (out.cpu().double() - want).abs().max().item() <= tol
    assert ops.attention_status() == 0


@pytest.mark.parametrize("q_len", [1, 20])
def test_queries_of_more_than_2_31_elements(cuda_device, q_len):
    """Every sequence sees one token, so that every row of its output is that token's value."""
    heads, groups, dim = 4, 8, 256
    seqs = (1 << 31) // (q_len * heads * groups * dim) + 300
    cache = kv_cache.PagedKVCache.empty(16, 16, heads, dim, cuda_device, F16)
    g = torch.Generator(device="cuda").manual_seed(1)
    kv = torch.randn(256, heads, dim, generator=g, device="cuda").to(F16)
    ops.kv_cache_write(cache, kv, kv, torch.arange(256, device="cuda"))
    i32 = dict(dtype=torch.int32, device="cuda")
    table = (torch.arange(seqs, **i32) % 16)[:, None].contiguous()
    starts = torch.arange(seqs + 1, **i32) * q_len
    q = torch.ones(seqs * q_len, heads * groups, dim, dtype=F16, device="cuda")
    out = ops.paged_attention(q, cache, table, torch.ones(seqs, **i32), starts, q_len, causal=False)
    first = kv[::16]  # each page's first token
    for s in (0, 17, seqs // 2, seqs - 1):
        rows = out[s * q_len:(s + 1) * q_len].view(q_len, heads, groups, dim)
        assert torch.equal(rows, first[s % 16][None, :, None].expand_as(rows))
    assert ops.attention_status() == 0


@pytest.mark.parametrize("fp8", [False, True])
def test_norm_of_more_than_2_31_elements(cuda_device, fp8):
    hidden = 7168
    rows = (1 << 31) // hidden + 500
    x = torch.ones(rows, hidden, dtype=BF16, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(2)
    x[-3:] = torch.randn(3, hidden, generator=g, device="cuda").to(BF16)
    w = torch.randn(hidden, generator=g, device="cuda")
    small, big = (ops.add_rms_norm_fp8 if fp8 else ops.add_rms_norm)(x[-3:].clone(), w), \
        (ops.add_rms_norm_fp8 if fp8 else ops.add_rms_norm)(x, w)
    assert torch.equal(big[0][-3:].view(torch.uint8), small[0].view(torch.uint8))
    if fp8:
        assert torch.equal(big[1][:, -3:], small[1])
