"""Integer linear, shared prefixes, scores and eviction as calls: threads, and offsets
past 32 bits (up to 30 GB on the device; nothing of it is copied to the host)."""

from __future__ import annotations

import threading

import pytest
import torch

from sglang_restomod_b200 import kv_cache, ops, synth
from tests.test_gpu_attention import BF16, E4M3
from tests.test_gpu_attention_calls import in_fresh_thread

pytestmark = pytest.mark.gpu
HEADS, DIM = 2, 128


def job(seed, q_len, store, page=16, tokens=37):
    """A run of all four on caches of its own; each call of it starts from the same state."""
    dev = torch.device("cuda")
    g = torch.Generator().manual_seed(seed)
    i32 = dict(dtype=torch.int32, device=dev)
    pages = -(-900 // page)
    shared = torch.randperm(4 * pages, generator=g)
    lens = [q_len, q_len + 200, q_len + 311]
    cache = kv_cache.PagedKVCache.empty(4 * pages, page, HEADS, DIM, dev, store)
    kv = torch.randn(4 * pages * page, 2 * HEADS, DIM, generator=g).to(BF16).to(dev)
    ops.kv_cache_write(cache, kv[:, :HEADS], kv[:, HEADS:], torch.arange(4 * pages * page, device=dev))
    table = shared[:3 * pages].view(3, pages).int().to(dev)
    prefix = (shared[3 * pages:][None].int().to(dev), torch.tensor([700], **i32),
              torch.tensor([0, 3], **i32))
    own = (table, torch.tensor(lens, **i32), torch.arange(4, **i32) * q_len, q_len)
    q = torch.randn(3 * q_len, 8 * HEADS, DIM, generator=g).to(BF16).to(dev)
    x = torch.randn(tokens, 1024, generator=g).to(BF16).to(dev)
    (w,), (ws,) = synth.int8_bank(1, 520, 1024, dev, seed)
    old = torch.rand(cache.k.shape[:3], generator=g).to(dev)

    def run():
        y = ops.int8_linear(x, w, ws)
        o, lse = ops.shared_prefix_attention(q, cache, *prefix, *own, return_lse=True)
        s = ops.kv_cache_scores(q, cache, *own, lse, old, out=torch.zeros_like(old))
        return y, o, lse, s, *ops.kv_cache_evict(cache, s, table, own[1], 100, recent=5, first=2,
                                                 out_table=spare)

    spare_pages = -(-100 // page)
    # pages past every sequence's tokens: the last of each row of the table
    spare = table[:, pages - spare_pages:].contiguous()
    assert (pages - spare_pages) * page >= max(lens)
    torch.cuda.synchronize()
    return run


def same(a, b):
    return all(torch.equal(torch.nan_to_num(x.float()), torch.nan_to_num(y.float()))
               for x, y in zip(a, b))


@pytest.mark.parametrize("q_len", [1, 50])
def test_first_call_of_a_thread(cuda_device, q_len):
    run = job(1, q_len, E4M3)
    want = run()
    torch.cuda.synchronize()
    assert same(want, in_fresh_thread(run))


def test_threads_on_one_stream(cuda_device):
    """Calls of several threads on one stream share its workspace; each call's
    launches stay together."""
    runs = [job(2, 1, BF16), job(3, 40, E4M3), job(4, 25, BF16, page=1, tokens=300), job(5, 2, E4M3)]
    wants = [run() for run in runs]
    torch.cuda.synchronize()
    wrong, gate = [], threading.Barrier(len(runs))

    def work(run, want):
        gate.wait(20)
        got = [run() for _ in range(40)]
        torch.cuda.current_stream().synchronize()
        wrong.extend(not same(g, want) for g in got)

    threads = [threading.Thread(target=work, args=pair) for pair in zip(runs, wants)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(120)
    assert len(wrong) == 4 * 40 and not any(wrong)
    assert ops.attention_status() == 0


def test_products_of_more_than_2_31_outputs(cuda_device):
    m, n, k = (1 << 31) // 4096 + 300, 4096, 16
    x = synth.activations(m, k, cuda_device, seed=1)
    (w,), (ws,) = synth.int8_bank(1, n, k, cuda_device, 2)
    y = ops.int8_linear(x, w, ws)
    for rows in (slice(0, 5), slice(m // 2, m // 2 + 7), slice(m - 301, m)):
        assert torch.equal(y[rows], ops.int8_linear(x[rows].contiguous(), w, ws))
    assert ops.attention_status() == 0


@pytest.mark.parametrize("store,page", [(E4M3, 64), (BF16, 64), (BF16, 1)])
@pytest.mark.parametrize("q_len", [1, 50])
def test_cache_and_scores_of_more_than_2_31_elements(cuda_device, store, page, q_len):
    """The last pages of a large cache against a small one: the same bits."""
    dev, heads, kv, far = cuda_device, 8, 300, 200
    need = [-(-n // page) for n in (kv, far, 120)]  # own tokens, prefix, evicted to
    g = torch.Generator().manual_seed(page)
    k, v = (torch.randn(kv + far, heads, DIM, generator=g).to(BF16).to(dev) for _ in "kv")
    q = torch.randn(q_len, 4 * heads, DIM, generator=g).to(BF16).to(dev)
    old = torch.rand(sum(need), page, heads, generator=g).to(dev)
    i32 = dict(dtype=torch.int32, device=dev)
    t = torch.arange(kv + far, device=dev)

    def run(pages, score_stride):
        cache = kv_cache.PagedKVCache.empty(pages, page, heads, DIM, dev, store)
        scores = torch.empty((pages - 1) * score_stride + page * heads, device=dev).as_strided(
            (pages, page, heads), (score_stride, heads, 1))
        last = torch.arange(pages - sum(need), pages, **i32).flip(0)
        own, prefix, to = (p[None].contiguous() for p in last.split(need))
        at = torch.cat([own[0].long()[t[:kv] // page] * page + t[:kv] % page,
                        prefix[0].long()[t[:far] // page] * page + t[:far] % page])
        ops.kv_cache_write(cache, k, v, at)
        scores[last.long()] = old
        lens = torch.tensor([kv], **i32)
        tables = (own, lens, torch.tensor([0, q_len], **i32), q_len)
        o, lse = ops.shared_prefix_attention(q, cache, prefix, torch.tensor([far], **i32),
                                             torch.tensor([0, 1], **i32), *tables, return_lse=True)
        ops.kv_cache_scores(q, cache, *tables, lse, scores)
        got = [o, lse, scores[last.long()].clone()]
        got += ops.kv_cache_evict(cache, scores, own, lens, 120, recent=9, first=3, out_table=to)
        got += ops.kv_cache_evict(cache, scores, own, lens, 120, recent=9, first=3)
        some = torch.arange(120, device=dev)
        for pages_of in (own, to):
            got += ops.kv_cache_read(cache, pages_of[0].long()[some // page] * page + some % page, BF16)
        got.append(scores[last.long()])
        return got

    small = run(sum(need) + 3, page * heads)
    pages = (1 << 31) // (heads * DIM * page) + 700
    large = run(pages, max(page * heads, (1 << 31) // pages + 1000))
    assert len(small) == len(large) == 12
    for i, (a, b) in enumerate(zip(small, large)):
        assert torch.equal(a, b), i
    assert torch.equal(small[3], small[5]) and torch.equal(small[7], small[9])
    assert ops.attention_status() == 0
