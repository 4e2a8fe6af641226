"""Eviction of cached tokens by score: which tokens stay, and every byte of the cache
afterwards, against a plain restatement. Nothing here is rounded: all must be equal."""

from __future__ import annotations

import math

import pytest
import torch

from sglang_restomod_b200 import kv_cache, ops

pytestmark = pytest.mark.gpu

BF16, F16, E4M3 = torch.bfloat16, torch.float16, torch.float8_e4m3fn


def choose(score, n, budget, recent, first):
    """The indices that stay, ascending, of one row of scores."""
    if n <= budget:
        return list(range(n))
    middle = range(first, n - recent)
    value = [-math.inf if math.isnan(score[i]) else score[i] for i in middle]
    # (NaN below -inf)
    order = sorted(range(len(value)), key=lambda i: (not math.isnan(score[first + i]), value[i]),
                   reverse=True)  # stable: equals keep their order
    return sorted([*range(first), *(first + i for i in order[:budget - first - recent]),
                   *range(n - recent, n)])


class Case:
    def __init__(self, seed, lens, budget, recent, first, heads, dim, page, store, *, wide=2,
                 token_major=False, scores=None):
        g = torch.Generator().manual_seed(seed)
        need = [-(-n // page) for n in lens]
        to = [-(-min(n, budget) // page) for n in lens]
        pages = sum(need) + sum(to) + 2
        order = torch.randperm(pages, generator=g)
        self.lens, self.budget, self.recent, self.first = lens, budget, recent, first
        self.heads, self.page = heads, page

        def table(need, at, extra):
            t = torch.full((len(lens), max(1, max(need)) + extra), 1 << 29, dtype=torch.int32)
            for s, n in enumerate(need):
                t[s, :n] = order[at:at + n].int()
                at += n
            return t

        self.table, self.out_table = table(need, 0, wide), table(to, sum(need), 1)
        shape = (pages, page, heads, dim) if token_major else (pages, heads, page, dim)

        def view(t):
            return t if token_major else t.transpose(1, 2)

        raw = torch.uint8 if store == E4M3 else torch.int16
        self.data = [view(torch.randint(-30000, 30000, shape, generator=g).to(raw)) for _ in range(2)]
        if store == E4M3:
            self.data += [view(torch.randint(0, 256, shape[:3], generator=g).to(torch.uint8))
                          for _ in range(2)]
        s = torch.exp(3 * torch.randn(pages, heads, page, generator=g)) if scores is None \
            else scores(pages, heads, page, g)
        self.data.append(s.float().transpose(1, 2))
        dev = [t.cuda() for t in self.data]
        # (a copy keeps its strides)
        assert all(a.stride() == b.stride() for a, b in zip(dev, self.data))
        self.dev = dev
        self.cache = kv_cache.PagedKVCache(dev[0].view(store), dev[1].view(store),
                                           *(dev[2:4] if store == E4M3 else ()))
        self.scores = dev[-1]

    def slots(self, table, s, n):
        at = torch.arange(n)
        return table[s].long()[at // self.page], at % self.page

    def check(self, in_place, kept, lens):
        want = [t.clone() for t in self.data]
        ids = torch.full((len(self.lens), self.heads, self.budget), -1, dtype=torch.int32)
        for s, n in enumerate(self.lens):
            page, offset = self.slots(self.table, s, n)
            m = min(n, self.budget)
            to_page, to_offset = self.slots(self.table if in_place else self.out_table, s, m)
            for h in range(self.heads):
                stay = torch.tensor(choose(self.data[-1][page, offset, h].tolist(), n, self.budget,
                                           self.recent, self.first), dtype=torch.long)
                ids[s, h, :m] = stay.int()
                for now, was in zip(want, self.data):
                    now[to_page, to_offset, h] = was[page[stay], offset[stay], h]
        assert lens.tolist() == [min(n, self.budget) for n in self.lens]
        assert torch.equal(kept.cpu(), ids)
        for got, now in zip(self.dev, want):
            got = got.cpu()
            if got.dtype == torch.float32:
                got, now = got.view(torch.int32), now.view(torch.int32)
            assert torch.equal(got, now)
        assert ops.attention_status() == 0

    def run(self, in_place):
        kept, lens = ops.kv_cache_evict(
            self.cache, self.scores, self.table.cuda(),
            torch.tensor(self.lens, dtype=torch.int32, device="cuda"), self.budget,
            recent=self.recent, first=self.first,
            out_table=None if in_place else self.out_table.cuda())
        self.check(in_place, kept, lens)


def ties(pages, heads, page, g):
    return torch.randint(0, 3, (pages, heads, page), generator=g).float() - 1.0


def odd_values(pages, heads, page, g):
    pick = torch.tensor([math.nan, -math.inf, math.inf, 0.0, -0.0, 1e-40, -1e-40, -5.0, 2.0])
    return pick[torch.randint(0, len(pick), (pages, heads, page), generator=g)]


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("store,dim,page,heads,token_major", [
    (BF16, 64, 1, 3, False), (BF16, 128, 16, 2, False), (F16, 256, 24, 1, True),
    (E4M3, 64, 16, 5, False), (E4M3, 128, 64, 2, True), (E4M3, 256, 8, 2, False)])
@pytest.mark.parametrize("budget,recent,first", [(1, 0, 0), (40, 0, 0), (40, 40, 0), (100, 30, 4),
                                                 (257, 100, 157), (1030, 1, 1)])
def test_evict(cuda_device, in_place, store, dim, page, heads, token_major, budget, recent, first):
    lens = [0, 1, 39, 40, 41, 100, 101, 300, 1500, 2047]
    Case(budget + dim, lens, budget, recent, first, heads, dim, page, store,
         token_major=token_major).run(in_place)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("scores", [ties, odd_values])
def test_equal_and_odd_scores(cuda_device, in_place, scores):
    """Ties go to the lowest index; NaN is below -inf, and -0 equals 0."""
    for budget in (1, 77, 700):
        Case(budget, [1000, 5, 701, 1200], budget, budget // 9, budget // 13, 2, 64, 16, BF16,
             scores=scores).run(in_place)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("n,budget,pairs", [(70001, 30000, 1), (70001, 69999, 2), (20000, 3, 2),
                                            (9000, 8999, 300)])
def test_long_and_many(cuda_device, in_place, n, budget, pairs):
    """One row over a cluster, and more rows than the GPU has blocks for."""
    lens = [n] if pairs < 3 else [n if i == 7 else 20 + i for i in range(pairs // 2)]
    Case(n, lens, budget, min(budget, 100), 0, min(pairs, 2), 64, 16, E4M3).run(in_place)


def test_more_scores_than_shared_memory(cuda_device):
    """A row whose blocks cannot hold their scores reads them again."""
    Case(1, [500003], 1000, 10, 3, 1, 64, 128, E4M3).run(False)
    Case(2, [60000] + [5] * 299, 500, 10, 3, 1, 64, 128, E4M3).run(True)


def test_rare_scales_of_score(cuda_device):
    """Scores that share all but the last bits."""
    def close(pages, heads, page, g):
        bits = torch.randint(0, 50, (pages, heads, page), generator=g).int() + 0x3f800000
        return bits.view(torch.float32)

    Case(3, [5000, 3000], 1234, 0, 0, 3, 64, 16, BF16, scores=close).run(False)


def test_twice_in_place(cuda_device):
    """What an eviction leaves is a sequence like any other."""
    c = Case(4, [900, 400], 300, 20, 2, 2, 128, 16, BF16)
    c.run(True)
    c.data = [t.cpu() for t in c.dev]
    c.lens, c.budget = [300, 300], 111
    c.run(True)


@pytest.mark.parametrize("in_place", [False, True])
def test_captured(cuda_device, in_place):
    """A replay sees new lengths and scores."""
    c = Case(5, [900, 400, 20], 100, 20, 2, 2, 128, 16, BF16)
    lens = torch.tensor([100, 50, 20], dtype=torch.int32, device="cuda")  # nothing to evict
    table, out_table = c.table.cuda(), None if in_place else c.out_table.cuda()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        kept, new = ops.kv_cache_evict(c.cache, c.scores, table, lens, 100, recent=20, first=2,
                                       out_table=out_table)
    if in_place:
        graph.replay()
        assert new.tolist() == [100, 50, 20] and kept[1, 0, :51].tolist() == [*range(50), -1]
    lens.copy_(torch.tensor(c.lens))
    graph.replay()
    c.check(in_place, kept, new)


def test_bad_pages_are_reported_and_not_moved(cuda_device):
    c = Case(6, [64], 20, 0, 0, 1, 64, 16, BF16)
    table = c.table.cuda()
    table[0, 1] = -3
    kept, lens = ops.kv_cache_evict(c.cache, c.scores, table,
                                    torch.tensor([64], dtype=torch.int32, device="cuda"), 20,
                                    out_table=c.out_table.cuda())
    assert ops.attention_status() == 16 and lens.tolist() == [20]
    assert not any(16 <= i < 32 for i in kept.flatten().tolist())  # other tokens have real scores


def test_the_table_itself_is_in_place(cuda_device):
    c = Case(7, [300, 90], 64, 8, 1, 2, 64, 16, E4M3)
    table = c.table.cuda()
    kept, lens = ops.kv_cache_evict(c.cache, c.scores, table,
                                    torch.tensor(c.lens, dtype=torch.int32, device="cuda"), 64,
                                    recent=8, first=1, out_table=table)
    c.check(True, kept, lens)


def test_no_sequences(cuda_device):
    c = Case(8, [3], 2, 0, 0, 1, 64, 16, BF16)
    kept, lens = ops.kv_cache_evict(c.cache, c.scores, c.table.cuda()[:0],
                                    torch.zeros(0, dtype=torch.int32, device="cuda"), 2)
    assert kept.shape == (0, 1, 2) and lens.shape == (0,)
