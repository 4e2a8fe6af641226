"""Accumulated attention weight of cached tokens against 64 bits.

A weight e^x, x = scale q.k - lse, is off by what x is: the products' sum by at
most D 2^-22 A, A = scale max|q| max|k| (norms), as in test_gpu_attention (e4m3 keys:
queries hold to 2^-22 of their largest element, within the same), x's own
arithmetic in log2 by 2^-22 (A + |lse|), the exponential by 2^-21. fp32 sums of n
positive terms, 128 at a time, add (128 + n / 128) 2^-24. All relative to a token's
added weight; then one addition to the old score, 2^-24 of the result. Weights
below 2^-126 count as zero: n 2^-126."""

from __future__ import annotations

import math

import pytest
import torch

from oracle import attention as ref
from sglang_restomod_b200 import ops
from tests.test_gpu_attention import BF16, E4M3, F16, TYPES, build

pytestmark = pytest.mark.gpu


class Case:
    def __init__(self, *args, lse_from="attention", causal=True, window=0, scale=None, max_q=None,
                 **kw):
        self.cache, self.q, self.table, self.kv_lens, self.starts, self.kc, _ = build(*args, **kw)
        self.scale = self.q.shape[-1] ** -0.5 if scale is None else scale
        self.causal, self.window = causal, window
        n = self.starts[1:] - self.starts[:-1]
        self.max_q = int(n.max()) if max_q is None else max_q
        self.dev = (self.q.cuda(), self.cache, self.table.cuda(), self.kv_lens.cuda(),
                    self.starts.cuda(), self.max_q)
        lse = torch.full(self.q.shape[:2], math.nan, device="cuda")  # (rows past max_q)
        _, got = ops.paged_attention(*self.dev, scale=self.scale, causal=causal, window=window,
                                     return_lse=True)
        new = torch.zeros(len(self.q), dtype=torch.bool)
        for a, m in zip(self.starts[:-1].tolist(), n.tolist()):
            new[a:a + min(m, self.max_q)] = True
        lse[new.cuda()] = got[new.cuda()]
        self.lse = lse
        g = torch.Generator().manual_seed(17)
        # NaN in what must not be read: new tokens' old scores and free slots
        self.old = torch.full(self.cache.k.shape[:3], math.nan)
        for s, kv in enumerate(self.kv_lens.tolist()):
            at = torch.arange(max(0, kv - int(n[s])) if causal else kv)
            page = self.table[s].long()[at // self.cache.page_size]
            self.old[page, at % self.cache.page_size] = torch.rand(len(at), self.cache.kv_heads,
                                                                   generator=g)

    def scores(self):
        s = self.cache.empty_scores()
        return s.copy_(self.old)

    def run(self, **kw):
        return ops.kv_cache_scores(*self.dev, self.lse, kw.pop("scores", None)
                                   if "scores" in kw else self.scores(), scale=self.scale,
                                   causal=self.causal, window=self.window, **kw)

    def check(self, got, untouched=None):
        want, added = ref.kv_cache_scores_ref(self.q, self.kc, self.table, self.kv_lens, self.starts,
                                              self.lse.cpu(), self.old, self.scale, self.causal,
                                              self.window, self.max_q)
        a = abs(self.scale) * float(self.q.double().norm(dim=-1).max()) * \
            float(torch.nan_to_num(self.kc).norm(dim=-1).max())
        finite = self.lse[torch.isfinite(self.lse)]
        top = float(finite.abs().max()) if finite.numel() else 0.0
        n = self.q.shape[0] * self.q.shape[1] // self.cache.kv_heads
        rel = self.q.shape[-1] * 2.0 ** -22 * a + 2.0 ** -22 * (a + top) + 2.0 ** -21 + \
            (128 + n / 128) * 2.0 ** -24
        got = got.cpu().double()
        there = torch.zeros(got.shape, dtype=torch.bool)
        for s, kv in enumerate(self.kv_lens.tolist()):
            at = torch.arange(kv)
            there[self.table[s].long()[at // self.cache.page_size], at % self.cache.page_size] = True
        bound = rel * added + 2.0 ** -24 * want.abs() + n * 2.0 ** -126
        off = (got - want).abs()
        assert bool((off <= bound)[there].all()), (off / bound)[there].max()
        rest = self.old.double() if untouched is None else untouched.cpu().double()
        assert torch.equal(torch.nan_to_num(got[~there], 77.0), torch.nan_to_num(rest[~there], 77.0))
        assert ops.attention_status() == 0

    def all(self):
        self.check(self.run())
        out = torch.full(self.old.shape, 5.0, device="cuda")
        got = self.run(out=out)
        assert got is out
        self.check(out, torch.full(self.old.shape, 5.0))
        again = self.run()
        assert torch.equal(torch.nan_to_num(again, 3.0), torch.nan_to_num(self.run(), 3.0))


LENS = [1, 15, 128, 129, 0, 255, 256, 257, 130, 1000]


@pytest.mark.parametrize("q_dtype,store", TYPES)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("heads,groups,page", [(2, 8, 16), (1, 3, 1), (3, 1, 24), (2, 16, 64), (1, 64, 128)])
def test_single_tokens(cuda_device, q_dtype, store, dim, heads, groups, page):
    Case(dim + page, [1] * len(LENS), LENS, heads, groups, dim, page, q_dtype, store,
         token_major=page == 24).all()


@pytest.mark.parametrize("q_dtype,store", TYPES)
@pytest.mark.parametrize("dim,page", [(64, 16), (128, 1), (128, 64), (256, 8), (64, 12), (256, 24)])
@pytest.mark.parametrize("groups", [1, 3, 8])
def test_chunks(cuda_device, q_dtype, store, dim, page, groups):
    """Prompts, chunks on contexts, an idle sequence and one without new tokens."""
    Case(dim + page, [70, 300, 1, 0, 33, 129], [70, 700, 0, 90, 290, 513], 2, groups, dim, page,
         q_dtype, store).all()


@pytest.mark.parametrize("q_dtype,store", TYPES)
@pytest.mark.parametrize("window", [1, 16, 100, 300, 5000])
@pytest.mark.parametrize("q_lens,kv_lens", [([1, 2, 1], [700, 333, 50]), ([200, 90], [900, 90]),
                                            ([1], [5000])])
def test_windows(cuda_device, q_dtype, store, window, q_lens, kv_lens):
    Case(window, q_lens, kv_lens, 2, 4, 64, 16, q_dtype, store, window=window).all()


@pytest.mark.parametrize("store", [BF16, E4M3])
def test_not_causal(cuda_device, store):
    Case(1, [1, 40, 9], [300, 30, 500], 2, 4, 128, 16, BF16, store, causal=False).all()


@pytest.mark.parametrize("store", [BF16, E4M3])
def test_long_and_many(cuda_device, store):
    Case(2, [1], [20011], 1, 8, 128, 16, BF16, store).all()
    Case(3, [1] * 700, [(37 * i) % 290 for i in range(700)], 1, 2, 64, 16, BF16, store).all()
    Case(4, [1500], [1500], 1, 4, 128, 64, BF16, store).all()
    Case(5, [1], [9000], 1, 2, 64, 16, BF16, store, window=50).all()


@pytest.mark.parametrize("store", [BF16, F16, E4M3])
@pytest.mark.parametrize("scale", [-0.09, 0.0, 1.0])
def test_scales(cuda_device, store, scale):
    """Scores in the hundreds, of either sign; and uniform weights."""
    dtype = F16 if store == F16 else BF16
    Case(6, [1, 30], [400, 90], 2, 4, 128, 16, dtype, store, scale=scale).all()


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_queries_of_every_size(cuda_device, dtype):
    """e4m3 keys: rows whose elements span many powers of two, tiny and large rows, zeros."""
    c = Case(7, [40], [300], 1, 2, 128, 16, dtype, E4M3)
    g = torch.Generator().manual_seed(3)
    shape = c.q.shape
    q = torch.randn(shape, generator=g) * torch.exp2(torch.randint(-12, 3, shape, generator=g).float())
    q[0] = 0
    q[1] *= 2.0 ** -10
    q[2] = 0
    q[2, :, 5] = 1.0
    if dtype == BF16:
        q[3] *= 2.0 ** -120
        q[4] = 2.0 ** -133
    c.q = q.to(dtype)
    c.dev = (c.q.cuda(), *c.dev[1:])
    _, c.lse = ops.paged_attention(*c.dev, return_lse=True)
    c.all()


def test_rows_past_max_q_add_nothing(cuda_device):
    for q_lens, max_q in (([1, 3, 1, 2], 1), ([40, 90, 33, 64], 40)):
        Case(8, q_lens, [n + 20 for n in q_lens], 2, 2, 64, 16, F16, F16, max_q=max_q).all()


def test_weights_of_a_row_sum_to_one(cuda_device):
    c = Case(9, [64], [640], 2, 4, 128, 16, BF16, BF16)
    s = torch.zeros(c.old.shape, device="cuda")
    c.run(scores=s)
    assert abs(float(s.double().sum()) / (64 * 8) - 1) < 2.0 ** -12


def test_infinite_log_sums_and_nan(cuda_device):
    """A row of -inf adds nothing, one of +inf nothing either, NaN shows where it is seen."""
    c = Case(10, [3], [200], 1, 1, 64, 16, BF16, BF16)
    s0 = c.run()
    c.lse[0] = -math.inf
    c.lse[1] = math.inf
    c.check(c.run())
    c.lse[2] = math.nan
    got = c.run().cpu()
    at = torch.arange(200)
    page = c.table[0].long()[at // 16]
    assert got[page, at % 16].isnan().all() and not s0.cpu()[page, at % 16].isnan().any()
    # a key's NaN stays with its token
    c = Case(11, [1], [200], 1, 1, 64, 16, BF16, BF16)
    c.cache.k[int(c.table[0, 3]), 5] = math.nan
    got = c.run().cpu()[page := c.table[0].long()[at // 16], at % 16]
    assert got[3 * 16 + 5].isnan().all() and int(got.isnan().sum()) == 1


def test_next_sequences_nan_stays_there(cuda_device):
    """Rows of one tile belong to several sequences in memory."""
    c = Case(12, [5, 5], [90, 90], 1, 4, 128, 16, BF16, BF16)
    want = c.run().cpu()
    c.dev[0][5:] = math.nan
    got = c.run().cpu()
    at = torch.arange(90)
    for s, same in ((0, True), (1, False)):
        page = c.table[s].long()[at // 16]
        assert torch.equal(got[page, at % 16], want[page, at % 16]) == same


def test_strides(cuda_device):
    """Queries out of a fused projection, one query for all heads, token-major scores."""
    c = Case(13, [4, 2], [50, 20], 2, 4, 128, 16, BF16, E4M3)
    want = c.run()
    wide = torch.zeros(6, 12, 128, dtype=BF16, device="cuda")
    wide[:, 2:10] = c.dev[0]
    c.dev = (wide[:, 2:10], *c.dev[1:])
    flat = torch.full((*c.old.shape[:2], 5), 9.0, device="cuda")
    flat[..., 1:3] = c.old.cuda()
    got = c.run(scores=flat[..., 1:3])
    assert torch.equal(torch.nan_to_num(got, 3.0), torch.nan_to_num(want, 3.0))
    assert (flat[..., 0] == 9).all() and (flat[..., 3:] == 9).all()
    one = c.dev[0][:, :1].expand(6, 8, 128)
    c.dev = (one, *c.dev[1:])
    a = c.run()
    c.dev = (one.contiguous(), *c.dev[1:])
    assert torch.equal(torch.nan_to_num(a, 3.0), torch.nan_to_num(c.run(), 3.0))


def test_bad_pages(cuda_device):
    c = Case(14, [1], [100], 1, 4, 64, 16, BF16, BF16)
    table = c.dev[2].clone()
    table[0, 2] = -9
    c.dev = (*c.dev[:2], table, *c.dev[3:])
    want = c.run()
    assert ops.attention_status() == 16
    assert torch.isnan(want[int(c.table[0, 2])]).sum() == c.old[int(c.table[0, 2])].isnan().sum()


@pytest.mark.parametrize("q_len", [1, 30])
@pytest.mark.parametrize("store", [BF16, E4M3])
def test_captured(cuda_device, q_len, store):
    """Replays see new lengths, and add again."""
    c = Case(15, [q_len] * 3, [q_len + 300, q_len + 50, q_len], 2, 4, 128, 16, BF16, store)
    s = c.scores()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        c.run(scores=s)
    for _ in range(2):
        s.copy_(c.old)
        graph.replay()
        c.check(s)
    c.dev[3].copy_(torch.tensor([q_len + 100, q_len + 20, q_len], dtype=torch.int32))
    c.kv_lens = c.dev[3].cpu()
    _, lse = ops.paged_attention(*c.dev, return_lse=True)
    c.lse.copy_(lse)
    s.copy_(c.scores().nan_to_num(0.25))
    c.old = s.cpu()
    graph.replay()
    c.check(s)


def test_after_a_shared_prefix(cuda_device):
    """With the log-sum-exp over prefix and own tokens, a row's weights over both sum to one."""
    from tests.test_gpu_shared_prefix import args, prefix_build

    p = prefix_build(16, [3], [200], [1, 1, 1], [40, 7, 1], 2, 4, 128, 16, BF16, BF16)
    a = args(p)
    _, lse = ops.shared_prefix_attention(*a, return_lse=True)
    s = torch.zeros(p["cache"].k.shape[:3], device="cuda")
    ops.kv_cache_scores(a[0], p["cache"], a[5], a[6], a[7], 1, lse, s)
    own = float(s.double().sum())
    # the group's three tokens over the prefix, none masked
    starts = torch.tensor([0, 3], dtype=torch.int32, device="cuda")
    ops.kv_cache_scores(a[0], p["cache"], a[2], a[3], starts, 3, lse, s, causal=False)
    assert 0 < own < float(s.double().sum())
    prefix_pages = p["prefix_table"][0].long()[torch.arange(200) // 16]
    assert abs(float(s.double().sum()) / 24 - 1) < 2.0 ** -12
    assert s[prefix_pages.cuda(), torch.arange(200, device="cuda") % 16].min() > 0


def test_no_new_tokens(cuda_device):
    c = Case(17, [1], [20], 1, 1, 64, 16, BF16, BF16)
    q, cache, table, kv, starts, _ = c.dev
    s = c.scores()
    before = s.clone()
    ops.kv_cache_scores(q[:0], cache, table, kv, torch.zeros_like(starts), 1, c.lse[:0], s)
    assert torch.equal(torch.nan_to_num(s, 3.0), torch.nan_to_num(before, 3.0))


@pytest.mark.parametrize("store", [BF16, E4M3])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("page", [1, 16])
def test_many_items_a_block(cuda_device, store, dim, page):
    """Several items an SM, some of a single half: the halves' rings of keys come round."""
    kv = [700 - 29 * (i % 7) for i in range(25)]
    Case(dim + page, [5 - i % 3 for i in range(25)], kv, 8, 8, dim, page, BF16, store).all()


@pytest.mark.parametrize("q_dtype,store", [(BF16, BF16), (F16, F16), (BF16, E4M3), (F16, E4M3)])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("q_len,groups,window", [(4, 8, 0), (7, 3, 0), (17, 1, 9), (2, 16, 100), (32, 1, 0)])
def test_a_few_tokens(cuda_device, q_dtype, store, dim, q_len, groups, window):
    """17 to 32 rows: the most that the streaming kernel takes, and one more than half of it."""
    kv = [q_len + n for n in (0, 1, 30, 205, 999)]
    q_lens = [q_len, q_len, 1, q_len, q_len - 1]
    Case(dim + q_len, q_lens, kv, 2, groups, dim, 16, q_dtype, store, window=window).all()
