"""What a cached token does not see adds nothing to its score, whatever it holds: rows of
the next sequences, rows after the last sequence, later queries, log-sums, scale bytes.
All calls have more rows a sequence than the streaming kernel takes, and those that some
tokens see nothing of leave them the same bits."""

from __future__ import annotations

import math

import pytest
import torch

from sglang_restomod_b200 import ops
from tests.test_gpu_attention import BF16, E4M3, F16, TYPES
from tests.test_gpu_scores import Case

pytestmark = pytest.mark.gpu

STREAMED = 32  # rows a sequence that no cache type gives the streaming kernel more of
SHAPES = [(64, 16, 3), (128, 1, 4), (128, 64, 8), (256, 8, 2)]  # head_dim, page size, groups


def tiled(seed, q_lens, kv_lens, dim, page, groups, q_dtype, store, **kw):
    c = Case(seed, q_lens, kv_lens, 2, groups, dim, page, q_dtype, store, **kw)
    assert c.max_q * groups > STREAMED
    return c


def slots(c, s):
    at = torch.arange(int(c.kv_lens[s]))
    return c.table[s].long()[at // c.cache.page_size], at % c.cache.page_size


def compare(c, got, want, row, head):
    """`got` is `want` but for NaN at the tokens that see head `head` of row `row`."""
    got, want = got.cpu(), want.cpu()
    for s in range(len(c.kv_lens)):
        a, b = int(c.starts[s]), int(c.starts[s + 1])
        at = torch.arange(int(c.kv_lens[s]))
        nan = torch.zeros(len(at), c.cache.kv_heads, dtype=torch.bool)
        if a <= row < b:
            pos = int(c.kv_lens[s]) - b + row
            seen = at <= pos
            if c.window:
                seen &= at > pos - c.window
            nan[:, head // (c.q.shape[1] // c.cache.kv_heads)] = seen
        x, y = got[slots(c, s)], want[slots(c, s)]
        assert not y.isnan().any()
        assert torch.equal(x.isnan(), nan), (s, int(x.isnan().sum()), int(nan.sum()))
        assert torch.equal(x[~nan], y[~nan])


@pytest.mark.parametrize("q_dtype,store", TYPES)
@pytest.mark.parametrize("dim,page,groups", SHAPES)
@pytest.mark.parametrize("window", [0, 40])
def test_a_row_spoils_what_sees_it(cuda_device, q_dtype, store, dim, page, groups, window):
    """A query or a log-sum that is not finite: in the middle, first and last rows of sequences."""
    c = tiled(dim, [45, 33, 70], [45, 400, 290], dim, page, groups, q_dtype, store, window=window)
    want = c.run()
    q, lse = c.dev[0].clone(), c.lse.clone()
    for row, head, value in ((7, 0, math.nan), (45, 1, math.inf), (77, groups, math.nan),
                             (100, 2 * groups - 1, -math.inf), (147, groups, math.inf)):
        c.dev[0][row, head] = value
        compare(c, c.run(), want, row, head)
        c.dev[0].copy_(q)
        c.lse[row, head] = math.nan
        compare(c, c.run(), want, row, head)
        c.lse.copy_(lse)
    assert ops.attention_status() == 0


@pytest.mark.parametrize("q_dtype,store", TYPES)
@pytest.mark.parametrize("dim,page,groups", SHAPES)
@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_rows_after_the_last_sequence(cuda_device, q_dtype, store, dim, page, groups, value):
    """A padded batch: the tile of the last new tokens goes on into rows of no sequence."""
    c = tiled(dim + 1, [21, 37], [300, 165], dim, page, groups, q_dtype, store)
    want = c.run()
    pad = torch.full((40, *c.q.shape[1:]), value, dtype=q_dtype, device="cuda")
    c.dev = (torch.cat([c.dev[0], pad]), *c.dev[1:])
    c.lse = torch.cat([c.lse, torch.full((40, c.q.shape[1]), math.nan, device="cuda")])
    got = c.run()
    assert torch.equal(torch.nan_to_num(got, 3.0), torch.nan_to_num(want, 3.0))
    compare(c, got, want, -1, 0)


@pytest.mark.parametrize("q_dtype", [BF16, F16])
@pytest.mark.parametrize("dim,page,groups", SHAPES)
def test_a_token_that_no_row_sees(cuda_device, q_dtype, dim, page, groups):
    """Its key's scale byte is 255, or its codes are NaN: it keeps its score, in an item that
    rows do reach."""
    c = tiled(dim + 2, [40], [300], dim, page, groups, q_dtype, E4M3, window=20)
    # positions 260 .. 299: the first row sees 241 .. 260
    want = c.run()
    out = torch.full(c.old.shape, 5.0, device="cuda")
    c.run(out=out)
    pages, offsets = (t.cuda() for t in slots(c, 0))
    for token in (1, 200, 240):
        c.cache.k_scale[pages[token], offsets[token]] = 255
        c.cache.k.view(torch.uint8)[pages[token - 1], offsets[token - 1]] = 0x7f
    assert torch.equal(torch.nan_to_num(c.run(), 3.0), torch.nan_to_num(want, 3.0))
    there = torch.full(c.old.shape, 5.0, device="cuda")
    assert torch.equal(torch.nan_to_num(c.run(out=there), 3.0), torch.nan_to_num(out, 3.0))
    c.cache.k_scale[pages[241], offsets[241]] = 255
    got = c.run().cpu()[slots(c, 0)]
    assert got[241].isnan().all() and int(got.isnan().sum()) == 2


@pytest.mark.parametrize("q_dtype,store", TYPES)
@pytest.mark.parametrize("scale", [0.0, 1e-9, -1e-9, 1e-30])
def test_small_scales_and_small_queries(cuda_device, q_dtype, store, scale):
    """Factors that leave fp32's range: rows of zeros, tiny rows, a scale of zero."""
    c = Case(20, [40, 11], [300, 50], 2, 4, 128, 16, q_dtype, store, scale=scale)
    assert c.max_q * 4 > STREAMED
    q = c.q.clone()
    q[3] = 0
    q[20:] = 0
    q[9] *= 2.0 ** -20
    if q_dtype == BF16:
        q[10] *= 2.0 ** -110
    c.q = q
    c.dev = (q.cuda(), *c.dev[1:])
    _, c.lse = ops.paged_attention(*c.dev, scale=scale, return_lse=True)
    c.all()
