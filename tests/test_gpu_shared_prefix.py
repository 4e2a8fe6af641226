"""Attention of a batch that shares prefixes against 64 bits.

Tolerances as in test_gpu_attention: P is rounded to the products' 16-bit type
once, the output once, (u_p + u_out) max|v| beside the fp32 products. Adding the
two passes in fp32 takes each pass's log-sum-exp L to e^(L - m): L is off by
2^-23 |L| through its scaling to log2 and back, which moves weights, and the sum,
by that; |L| is at most A + ln(keys) here, below 2^7, so 2^-16 of max|v|."""

from __future__ import annotations

import pytest
import torch

from oracle import attention as ref
from sglang_restomod_b200 import ops
from tests.test_gpu_attention import BF16, E4M3, F16, TYPES, U, bounds, build

pytestmark = pytest.mark.gpu


def prefix_build(seed, group_sizes, prefix_lens, q_lens, kv_lens, heads, groups, dim, page, dtype,
                 store, **kw):
    assert sum(group_sizes) == len(q_lens) == len(kv_lens)
    n = len(q_lens)
    cache, q, table, lens, starts, kc, vc = build(seed, q_lens + [0] * len(prefix_lens),
                                                  kv_lens + prefix_lens, heads, groups, dim, page,
                                                  dtype, store, **kw)
    group_starts = torch.tensor([0] + group_sizes).cumsum(0).int()
    return dict(q=q, cache=cache, prefix_table=table[n:], prefix_lens=lens[n:],
                group_starts=group_starts, table=table[:n], kv_lens=lens[:n], starts=starts[:n + 1],
                kc=kc, vc=vc)


def args(c, max_q=None):
    if max_q is None:
        max_q = int((c["starts"][1:] - c["starts"][:-1]).max())
    return [c["q"].cuda(), c["cache"], *(c[n].cuda() for n in (
        "prefix_table", "prefix_lens", "group_starts", "table", "kv_lens", "starts")), max_q]


def reference(c, scale):
    return ref.shared_prefix_attention_ref(c["q"], c["kc"], c["vc"], c["prefix_table"],
                                           c["prefix_lens"], c["group_starts"], c["table"],
                                           c["kv_lens"], c["starts"], scale)


def compare(c, out, lse, scale, rows=None):
    want, want_lse = reference(c, scale)
    dtype = c["q"].dtype
    # e4m3 caches multiply in f16, whose rounding is the smaller one
    # (A is made of magnitudes: |scale| max|q| max|k|)
    tol, lse_tol = bounds(c["q"], c["kc"], c["vc"], abs(scale), dtype, dtype)
    top = float(torch.nan_to_num(c["vc"]).abs().max())
    tol, lse_tol = tol + 2.0 ** -16 * top, lse_tol + 2.0 ** -16
    out, lse = out.cpu(), lse.cpu()
    rows = torch.ones(len(out), dtype=torch.bool) if rows is None else rows
    seen = torch.isfinite(want_lse) & rows[:, None]
    assert torch.equal(torch.isinf(lse[rows]), torch.isinf(want_lse[rows]))
    assert (lse.double() - want_lse)[seen].abs().max().item() <= lse_tol if seen.any() else True
    assert (out.double() - want)[rows].abs().max().item() <= tol
    assert (out[rows[:, None] & ~seen] == 0).all()
    assert ops.attention_status() == 0


def check(c, *, scale=None, max_q=None):
    scale = c["q"].shape[-1] ** -0.5 if scale is None else scale
    out, lse = ops.shared_prefix_attention(*args(c, max_q), scale=scale, return_lse=True)
    compare(c, out, lse, scale)
    return out, lse


@pytest.mark.parametrize("q_dtype,store", TYPES)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("heads,groups,page", [(2, 8, 16), (1, 3, 1), (3, 1, 24), (1, 16, 64)])
def test_decode(cuda_device, q_dtype, store, dim, heads, groups, page):
    """Single tokens: groups of several sizes, one without a prefix, one of one sequence,
    sequences with nothing of their own, prefixes that end within a page."""
    check(prefix_build(dim + page, [4, 1, 3], [333, 65, 0], [1] * 8, [1, 0, 90, 17, 5, 40, 0, 200],
                       heads, groups, dim, page, q_dtype, store, token_major=page == 24))


@pytest.mark.parametrize("q_dtype,store", TYPES)
@pytest.mark.parametrize("dim,groups,page", [(64, 3, 1), (128, 4, 16), (256, 2, 64)])
def test_chunks(cuda_device, q_dtype, store, dim, groups, page):
    check(prefix_build(dim, [3, 2], [500, 130], [70, 0, 41, 9, 33], [70, 10, 300, 9, 64], 2, groups,
                       dim, page, q_dtype, store))


@pytest.mark.parametrize("store", [BF16, E4M3])
def test_large_groups(cuda_device, store):
    """Rows that fill several tiles, two in turn, prefixes of one token and of many; one
    key/value head over the whole GPU."""
    check(prefix_build(3, [90, 40], [1500, 1], [1] * 130, [1 + i % 37 for i in range(130)], 1, 8,
                       128, 16, BF16, store))
    check(prefix_build(4, [2], [9000], [1, 1], [30, 1], 1, 4, 128, 64, BF16, store))
    check(prefix_build(5, [2], [700], [300, 280], [300, 500], 2, 4, 128, 64, BF16, store))


@pytest.mark.parametrize("store", [BF16, E4M3])
@pytest.mark.parametrize("q_len", [1, 40])
def test_prefixes_far_above_and_below(cuda_device, store, q_len):
    """Scores of one pass outweigh the other's by e^hundreds, either way."""
    c = prefix_build(6, [2, 2], [200, 200], [q_len] * 4, [q_len + 60] * 4, 1, 2, 128, 16, BF16, store,
                     k_scale=20.0)
    check(c)
    check(c, scale=-0.09)
    check(c, scale=0.0)


def test_no_prefix_is_paged_attention(cuda_device):
    c = prefix_build(7, [3], [0], [1, 1, 1], [100, 40, 3], 2, 4, 128, 16, BF16, BF16)
    out, lse = check(c)
    a = args(c)
    want, want_lse = ops.paged_attention(a[0], a[1], a[5], a[6], a[7], 1, return_lse=True)
    assert (out.float() - want.float()).abs().max() <= 2 * U[BF16] * want.float().abs().max()
    assert (lse - want_lse).abs().max() <= 2.0 ** -16


@pytest.mark.parametrize("q_lens,max_q", [([1, 3, 1, 2], 1), ([40, 90, 33, 64], 40)])
def test_rows_past_max_q_and_of_no_sequence_stay(cuda_device, q_lens, max_q):
    """Further new tokens keep their positions and are left unwritten, as are rows after
    the last sequence."""
    c = prefix_build(8, [2, 2], [150, 70], q_lens, [n + 20 for n in q_lens], 2, 2, 64, 16, F16, F16)
    c["q"] = torch.cat([c["q"], c["q"][:5]])
    a = args(c, max_q)
    out = torch.full_like(a[0], 7.0)
    out, lse = ops.shared_prefix_attention(*a, out=out, return_lse=True)
    rows = torch.zeros(len(c["q"]), dtype=torch.bool)
    for s, n in enumerate(q_lens):
        rows[int(c["starts"][s]):int(c["starts"][s]) + min(n, max_q)] = True
    compare(c, out, lse, 64 ** -0.5, rows)
    assert (out.cpu()[~rows] == 7.0).all()


def test_strides(cuda_device):
    """Queries out of a fused projection, outputs into a wider row, heads first."""
    c = prefix_build(9, [3], [100], [1] * 3, [30, 7, 1], 2, 4, 128, 16, BF16, E4M3)
    a = args(c)
    wide = torch.zeros(3, 12, 128, dtype=BF16, device="cuda")
    wide[:, 2:10] = a[0]
    out = torch.zeros(8, 3, 256, dtype=BF16, device="cuda")
    want = ops.shared_prefix_attention(*a)
    a[0] = wide[:, 2:10]
    got = ops.shared_prefix_attention(*a, out=out.transpose(0, 1)[..., :128])
    assert torch.equal(got, want) and (out[..., 128:] == 0).all()


def test_bad_pages_read_as_zeros_and_are_reported(cuda_device):
    c = prefix_build(10, [2], [40], [1, 1], [20, 20], 1, 4, 128, 16, BF16, BF16)
    a = args(c)
    a[2][0, 1] = -5
    out, _ = ops.shared_prefix_attention(*a, return_lse=True)
    assert ops.attention_status() == 16 and torch.isfinite(out).all()
    a = args(c)
    a[5][1, 0] = 1 << 20
    out, _ = ops.shared_prefix_attention(*a, return_lse=True)
    assert ops.attention_status() == 16 and torch.isfinite(out).all()


@pytest.mark.parametrize("q_len", [1, 30])
@pytest.mark.parametrize("reserved", [False, True])
def test_captured(cuda_device, q_len, reserved):
    """Replays see new prefix lengths, groups and tables."""
    c = prefix_build(11, [3, 1], [300, 90], [q_len] * 4, [q_len + 50] * 4, 2, 4, 128, 16, BF16, BF16)
    d = dict(c, prefix_lens=torch.tensor([120, 0], dtype=torch.int32),
             group_starts=torch.tensor([0, 1, 4], dtype=torch.int32),
             kv_lens=torch.tensor([q_len, q_len + 50, q_len + 3, q_len + 50], dtype=torch.int32))
    a = args(c)
    side = torch.cuda.Stream()
    out = torch.empty_like(a[0])
    with torch.cuda.stream(side):
        if reserved:
            ops.reserve_shared_prefix_workspace(128, len(out), 8, 4, 2)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        _, lse = ops.shared_prefix_attention(*a, out=out, return_lse=True)
    graph.replay()
    compare(c, out, lse, 128 ** -0.5)
    for i, name in ((3, "prefix_lens"), (4, "group_starts"), (6, "kv_lens")):
        a[i].copy_(d[name])
    graph.replay()
    compare(d, out, lse, 128 ** -0.5)


def test_nothing_to_do(cuda_device):
    c = prefix_build(12, [1], [40], [1], [4], 1, 4, 128, 16, BF16, BF16)
    a = args(c)
    empty = [a[0][:0], a[1], a[2][:0], a[3][:0], a[4][:1], a[5][:0], a[6][:0], a[7][:1], 1]
    assert ops.shared_prefix_attention(*empty).shape == (0, 4, 128)
