"""A serving loop on integer projections, a shared prefix, gathered attention weights
and eviction, against a plain float64 layer; the same operators as torch custom ops."""

from __future__ import annotations

import math
import subprocess
import sys
from pathlib import Path

import pytest
import torch

from oracle import attention as ref
from sglang_restomod_b200 import _lib, decoder, kv_cache, ops, serving_ops, synth
from tests.test_gpu_decoder import DIM, HEADS, HIDDEN, KV, PAGE, relative, rotary

B = torch.ops.b200_moe
META = torch.device("meta")
BF16, E4M3 = torch.bfloat16, torch.float8_e4m3fn
ROOT = Path(__file__).resolve().parent.parent


# ------------------------------------------------------------------ on a CPU
def test_batches_with_a_prefix():
    prefix = decoder.SharedPrefix.of([5, 0], [[7, 3], []], [2, 1], "cpu")
    assert prefix.page_table.tolist() == [[7, 3], [0, 0]] and prefix.lens.tolist() == [5, 0]
    assert prefix.group_starts.tolist() == [0, 2, 3]
    b = decoder.TokenBatch.of([1, 2, 1], [3, 2, 6], [[0], [1], [2, 4]], 4, "cpu", [5, 5, 9], prefix)
    assert b.positions.tolist() == [7, 5, 6, 14] and b.slots.tolist() == [2, 4, 5, 17]
    assert b.prefix is prefix
    with pytest.raises(ValueError, match="group sizes"):
        decoder.SharedPrefix.of([5], [[7]], [2, 1], "cpu")
    block = decoder.AttentionBlock(1, 1, 64, *[torch.zeros(0)] * 5, window=3)
    with pytest.raises(ValueError, match="window"):
        block.forward(torch.zeros(4, 8), None, None, b)


def test_integer_weights_fill_their_range():
    q, s = synth.int8_bank(2, 5, 64, "cpu", 3)
    assert q.shape == (2, 5, 64) and s.shape == (2, 5) and q.dtype == torch.int8
    assert (q.abs().amax(-1) == 127).all() and not torch.equal(q[0], q[1])


WRITTEN = {"kv_cache_scores": {"scores"},
           "kv_cache_evict": {"k_cache", "v_cache", "k_scale", "v_scale", "scores"}}


def test_ops_are_registered_and_mark_what_they_write():
    for name in serving_ops.names():
        schema = getattr(B, name).default._schema
        assert schema.name == f"b200_moe::{name}"
        assert {a.name for a in schema.arguments if a.alias_info is not None
                and a.alias_info.is_write} == WRITTEN.get(name, set())


def test_fake_implementations_propagate_shapes():
    x = torch.empty(5, 256, dtype=BF16, device=META)
    w, ws = torch.empty(48, 256, dtype=torch.int8, device=META), torch.empty(48, device=META)
    q, s = B.int8_act_quant(x)
    assert q.shape == x.shape and q.dtype == torch.int8
    assert s.shape == (5,) and s.dtype == torch.float32
    assert B.int8_linear(x[None], w, ws, torch.float16).shape == (1, 5, 48)
    y = B.int8_linear_quantized(q, s, w, ws, BF16)
    assert y.shape == (5, 48) and y.dtype == BF16
    i32 = dict(dtype=torch.int32, device=META)
    kv = torch.empty(9, PAGE, KV, DIM, dtype=BF16, device=META)
    q = torch.empty(5, HEADS, DIM, dtype=BF16, device=META)
    table, lens, starts = torch.empty(2, 3, **i32), torch.empty(2, **i32), torch.empty(3, **i32)
    out, lse = B.shared_prefix_attention(q, kv, kv, None, None, table[:1], lens[:1], starts[:2],
                                         table, lens, starts, 4)
    assert out.shape == q.shape and out.dtype == BF16
    assert lse.shape == (5, HEADS) and lse.dtype == torch.float32
    scores = torch.empty(9, PAGE, KV, device=META)
    assert B.kv_cache_scores(q, kv, kv, None, None, table, lens, starts, 4, lse, scores) is None
    kept, now = B.kv_cache_evict(kv, kv, None, None, scores, table, lens, 7)
    assert kept.shape == (2, KV, 7) and now.shape == (2,)
    assert kept.dtype == now.dtype == torch.int32


# ---------------------------------------------------------------- on a B200
class Plain:
    """The block in float64 on the CPU, without rounding: per sequence and head the
    cached keys, values and gathered weights; prefixes apart."""

    def __init__(self, block):
        self.block = block
        self.wq = block.w_qkv.cpu().double() * block.s_qkv.cpu().double()[:, None]
        self.wo = block.w_o.cpu().double() * block.s_o.cpu().double()[:, None]
        self.crest = 0.0  # of what is quantized: largest element by root mean square

    def project(self, x, residual, positions):
        y, _ = ref.add_rms_norm_ref(x.cpu(), self.block.norm.cpu(), self.block.eps,
                                    None if residual is None else residual.cpu())
        self.note(y)
        q, k, v = (y @ self.wq.T).view(len(x), HEADS + 2 * KV, DIM).split([HEADS, KV, KV], 1)
        return rotary(q, positions.cpu()), rotary(k, positions.cpu()), v

    def note(self, y):
        self.crest = max(self.crest, float((y.abs().amax(1) / y.square().mean(1).sqrt()).max()))

    def step(self, x, residual, batch, seqs):
        """seqs: per sequence a dict of prefix (k, v) or None and per-head lists k, v, w."""
        q, k, v = self.project(x, residual, batch.positions)
        out = torch.zeros(len(x), HEADS, DIM, dtype=torch.float64)
        starts = batch.q_starts.tolist()
        for s, (a, b) in enumerate(zip(starts, starts[1:])):
            one = seqs[s]
            for h in range(KV):
                one["k"][h] = torch.cat([one["k"][h], k[a:b, h]])
                one["v"][h] = torch.cat([one["v"][h], v[a:b, h]])
                one["w"][h] = torch.cat([one["w"][h], torch.zeros(b - a, dtype=torch.float64)])
                n = len(one["k"][h])
                keys, values = one["k"][h], one["v"][h]
                before = 0
                if one["prefix"] is not None:
                    pk, pv = one["prefix"]
                    before = len(pk)
                    keys, values = torch.cat([pk[:, h], keys]), torch.cat([pv[:, h], values])
                for t in range(a, b):
                    seen = before + n - (b - a) + t - a + 1
                    for g in range(HEADS // KV):
                        p = torch.softmax(keys[:seen] @ q[t, h * (HEADS // KV) + g] * DIM ** -0.5, 0)
                        out[t, h * (HEADS // KV) + g] = p @ values[:seen]
                        one["w"][h][:seen - before] += p[before:]
        flat = out.reshape(len(x), -1)
        self.note(flat)
        return flat @ self.wo.T


def tolerance(crest, store):
    """Between x and the output: two roundings to 8-bit integers, each off by at most
    half a step of crest / 127 of the root mean square, uniformly: 1 / sqrt(12) of it;
    K's and V's to the cache (e4m3: 2^-4 at most, 1 / sqrt(3) of it); 16-bit ones. Weights
    are e^x of such errors times logits of order one. They are independent, and
    random matrices hand a relative error on unchanged: added up, they bound its size."""
    of_cache = 2 * 2.0 ** -4 / math.sqrt(3) if store == E4M3 else 0.0
    return 2 * crest / 127 / math.sqrt(12) + of_cache + 0.01


@pytest.mark.gpu
@pytest.mark.parametrize("store", [BF16, E4M3])
def test_shared_prompt_scored_evicted_and_decoded(cuda_device, store):
    dev = cuda_device
    block = decoder.AttentionBlock.synthetic(HIDDEN, HEADS, KV, DIM, dev, int8=True, rotary=rotary)
    plain = Plain(block)
    cache = kv_cache.PagedKVCache.empty(24, PAGE, KV, DIM, dev, store)
    scores = cache.empty_scores().fill_(float("nan"))
    prefix_pages = [20, 3, 11, 0, 6]
    pages = [[7, 1, 9, 5], [2, 8], [23, 4, 10, 12]]

    # a prompt of 70 tokens, shared by the first two of three sequences
    x = synth.activations(70, HIDDEN, dev, seed=1)
    batch = decoder.TokenBatch.of([70], [70], [prefix_pages], PAGE, dev)
    out, _ = block.forward(x, None, cache, batch)
    none = lambda: [torch.zeros(0, DIM, dtype=torch.float64) for _ in range(KV)]
    fresh = lambda p: dict(prefix=p, k=none(), v=none(),
                           w=[torch.zeros(0, dtype=torch.float64) for _ in range(KV)])
    alone = fresh(None)
    want = plain.step(x, None, batch, [alone])
    assert relative(out, want) <= tolerance(plain.crest, store)
    shared = tuple(torch.stack(alone[n], 1) for n in "kv")
    prefix = decoder.SharedPrefix.of([70, 0], [prefix_pages, []], [2, 1], dev)
    seqs = [fresh(shared), fresh(shared), fresh(None)]
    before, lens = [70, 70, 0], [0, 0, 0]

    def step(q_lens, seed, cache, scores):
        for s, n in enumerate(q_lens):
            lens[s] += n
        x = synth.activations(sum(q_lens), HIDDEN, dev, seed=seed)
        residual = synth.activations(sum(q_lens), HIDDEN, dev, seed=seed + 100)
        batch = decoder.TokenBatch.of(q_lens, lens, pages, PAGE, dev, before, prefix)
        want = plain.step(x, residual, batch, seqs)
        out, _ = block.forward(x, residual, cache, batch, scores)
        assert relative(out, want) <= tolerance(plain.crest, store)

    def rows(s, h):  # a sequence's scores
        t = torch.arange(lens[s])
        return scores[torch.tensor(pages[s])[t // PAGE].to(dev), (t % PAGE).to(dev), h].cpu()

    def check_scores():
        got = torch.cat([rows(s, h) for s in range(3) for h in range(KV)])
        want = torch.cat([seqs[s]["w"][h] for s in range(3) for h in range(KV)])
        assert relative(got, want) <= tolerance(plain.crest, store)

    step([40, 9, 33], 2, cache, scores)   # the questions in chunks, then a token each
    step([15, 3, 20], 3, cache, scores)
    step([1, 1, 1], 4, cache, scores)
    check_scores()

    # the choice is the plain one on the same scores; the plain layer follows it
    budget, recent, first = 24, 5, 2
    was = [[rows(s, h) for h in range(KV)] for s in range(3)]
    batch = decoder.TokenBatch.of([0] * 3, lens, pages, PAGE, dev, before, prefix)
    kept, now = ops.kv_cache_evict(cache, scores, batch.page_table, batch.kv_lens, budget,
                                   recent=recent, first=first)
    for s in range(3):
        n = lens[s]
        assert int(now[s]) == min(n, budget)
        for h in range(KV):
            rank = was[s][h].clone()
            rank[:first], rank[max(0, n - recent):] = math.inf, math.inf
            chosen = torch.sort(rank, descending=True, stable=True).indices[:budget].sort().values
            assert kept[s, h, :len(chosen)].cpu().tolist() == chosen.tolist()
            for name in "kvw":
                seqs[s][name][h] = seqs[s][name][h][chosen]
        before[s] += n - min(n, budget)
        lens[s] = min(n, budget)
    check_scores()
    step([1, 1, 1], 5, cache, scores)  # positions go on, places in the cache do not
    step([4, 1, 2], 6, cache, scores)
    check_scores()

    # decode from one captured graph
    twin = kv_cache.PagedKVCache(cache.k.clone(), cache.v.clone(),
                                 *(t if t is None else t.clone() for t in (cache.k_scale, cache.v_scale)))
    twin_scores = scores.clone()
    buf = synth.activations(3, HIDDEN, dev, seed=7)
    batch = decoder.TokenBatch.of([1] * 3, [n + 1 for n in lens], pages, PAGE, dev, before, prefix)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, _ = block.forward(buf, None, twin, batch, twin_scores)
    for i in range(3):
        now = decoder.TokenBatch.of([1] * 3, [n + 1 + i for n in lens], pages, PAGE, dev, before, prefix)
        x = synth.activations(3, HIDDEN, dev, seed=8 + i)
        want, _ = block.forward(x, None, cache, now, scores)
        buf.copy_(x)
        for name in ("kv_lens", "slots", "positions"):
            getattr(batch, name).copy_(getattr(now, name))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    assert torch.equal(torch.nan_to_num(scores, 7.0), torch.nan_to_num(twin_scores, 7.0))
    assert torch.equal(cache.k.view(torch.uint8), twin.k.view(torch.uint8))
    assert ops.attention_status() == 0


@pytest.mark.gpu
def test_decoder_layer_on_integer_projections(cuda_device):
    dev = cuda_device
    layer = decoder.DecoderLayer.synthetic(synth.CONFIG0, _lib.QUANT_FP8_BLOCK, HEADS, KV, DIM, dev,
                                           int8=True)
    cache = kv_cache.PagedKVCache.empty(8, PAGE, KV, DIM, dev)
    scores = cache.empty_scores()
    x = synth.activations(30, HIDDEN, dev, seed=5)
    batch = decoder.TokenBatch.of([30], [30], [[3, 1]], PAGE, dev)
    y, stream = layer.forward(x, None, cache, batch, scores)
    h, _ = layer.attention.forward(x, None, cache, batch)
    _, want = ref.add_rms_norm_ref(h.cpu(), layer.norm.cpu(), layer.eps, x.cpu())
    assert (stream.double().cpu() - want).abs().max() <= 2.0 ** -8 * want.abs().max()
    assert torch.isfinite(y.float()).all()
    # every row's weights sum to one (e4m3-free: fp32 sums of 30 weights, each off by
    # a few 2^-24 of it and of its logits, of order one)
    used = scores[[3, 1]].reshape(2 * PAGE, KV)[:30]
    assert abs(float(used.double().sum()) / (30 * HEADS) - 1) <= 2.0 ** -15
    assert ops.attention_status() == 0 and ops.workspace_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("store", [BF16, E4M3])
def test_custom_ops_agree_with_the_calls(cuda_device, store):
    dev = cuda_device
    x = synth.activations(20, 512, dev, seed=1)
    (w,), (ws,) = synth.int8_bank(1, 72, 512, dev, 2)
    q8, s8 = B.int8_act_quant(x)
    r8, t8 = ops.int8_act_quant(x)
    assert torch.equal(q8, r8) and torch.equal(s8, t8)
    want = ops.int8_linear(x, w, ws)
    assert torch.equal(B.int8_linear(x, w, ws, BF16), want)
    assert torch.equal(B.int8_linear_quantized(q8, s8, w, ws, BF16), want)

    cache = kv_cache.PagedKVCache.empty(8, PAGE, KV, DIM, dev, store)
    kv = synth.activations(8 * PAGE, 2 * KV * DIM, dev, seed=2).view(8 * PAGE, 2 * KV, DIM)
    ops.kv_cache_write(cache, kv[:, :KV], kv[:, KV:], torch.arange(8 * PAGE, device=dev))
    four = (cache.k, cache.v, cache.k_scale, cache.v_scale)
    i32 = dict(dtype=torch.int32, device=dev)
    shared = (torch.tensor([[6, 7]], **i32), torch.tensor([29], **i32), torch.tensor([0, 2], **i32))
    own = (torch.tensor([[4, 1], [0, 3]], **i32), torch.tensor([30, 18], **i32),
           torch.tensor([0, 3, 5], **i32), 3)
    q = synth.activations(5, HEADS * DIM, dev, seed=3).view(5, HEADS, DIM)
    out, lse = B.shared_prefix_attention(q, *four, *shared, *own)
    want = ops.shared_prefix_attention(q, cache, *shared, *own, return_lse=True)
    assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
    a, b = (torch.zeros(cache.k.shape[:3], device=dev) for _ in range(2))
    B.kv_cache_scores(q, *four, *own, lse, a)
    ops.kv_cache_scores(q, cache, *own, lse, b)
    assert torch.equal(a, b) and float(a.sum()) > 0

    twin = kv_cache.PagedKVCache(*(t if t is None else t.clone() for t in four))
    got = B.kv_cache_evict(twin.k, twin.v, twin.k_scale, twin.v_scale, a, own[0], own[1], 9, 2, 1)
    want = ops.kv_cache_evict(cache, b, own[0], own[1], 9, recent=2, first=1)
    assert all(torch.equal(x, y) for x, y in zip(got, want)) and torch.equal(a, b)
    assert torch.equal(cache.k.view(torch.uint8), twin.k.view(torch.uint8))
    if store == BF16:  # opcheck's schema test multiplies the inputs: not for float8 tensors
        check = torch.library.opcheck
        check(B.int8_act_quant.default, (x,))
        check(B.int8_linear.default, (x, w, ws, BF16))
        check(B.int8_linear_quantized.default, (q8, s8, w, ws, BF16))
        check(B.shared_prefix_attention.default, (q, *four, *shared, *own))
        check(B.kv_cache_scores.default, (q, *four, *own, lse, a))
        check(B.kv_cache_evict.default, (*four, a, own[0], own[1], 9, 2, 1))


@pytest.mark.gpu
def test_first_calls_of_a_process_may_be_captured(cuda_device):
    code = """
import torch
from sglang_restomod_b200 import kv_cache, ops, synth
dev = torch.device("cuda", 0)
x = synth.activations(2, 2048, dev)
(w,), (ws,) = synth.int8_bank(1, 2048, 2048, dev, 2)
cache = kv_cache.PagedKVCache.empty(300, 64, 1, 128, dev)
cache.k.copy_(synth.activations(300 * 64, 128, dev, seed=3).view(cache.k.shape))
cache.v.copy_(synth.activations(300 * 64, 128, dev, seed=4).view(cache.v.shape))
scores = torch.rand(300, 64, 1, device=dev)
old = scores.clone()
i32 = dict(dtype=torch.int32, device=dev)
pages = torch.arange(300, **i32)[None]
prefix, own, to = pages[:, :9], pages[:, 9:200], pages[:, 200:]
plen, lens = torch.tensor([500], **i32), torch.tensor([191 * 64 - 5], **i32)
starts, groups = torch.tensor([0, 20], **i32), torch.tensor([0, 1], **i32)
q = synth.activations(20, 2 * 128, dev).view(20, 2, 128)

def run():
    y = ops.int8_linear(x, w, ws)
    o, lse = ops.shared_prefix_attention(q, cache, prefix, plen, groups, own, lens, starts, 20,
                                         return_lse=True)
    ops.kv_cache_scores(q, cache, own, lens, starts, 20, lse, scores)
    return (y, o, lse, *ops.kv_cache_evict(cache, scores, own, lens, 4000, out_table=to))

torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = run()
graph.replay()
torch.cuda.synchronize()
kept = scores.clone()
scores.copy_(old)
want = run()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(got, want)) and torch.equal(kept, scores)
assert ops.attention_status() == 0
"""
    env_root = str(ROOT / "sglang-restomod_b200")
    done = subprocess.run([sys.executable, "-c", f"import sys; sys.path.insert(0, {env_root!r})\n{code}"],
                          capture_output=True, text=True, timeout=240)
    assert done.returncode == 0, done.stderr[-2000:]


@pytest.mark.gpu
def test_streams_do_not_disturb_one_another(cuda_device):
    """The same calls on two streams at once give what they give alone."""
    dev = cuda_device
    (w,), (ws,) = synth.int8_bank(1, 4096, 2048, dev, 2)
    i32 = dict(dtype=torch.int32, device=dev)

    def job(seed, tokens):
        cache = kv_cache.PagedKVCache.empty(120, PAGE, KV, DIM, dev, E4M3)
        kv = synth.activations(120 * PAGE, 2 * KV * DIM, dev, seed=seed).view(-1, 2 * KV, DIM)
        ops.kv_cache_write(cache, kv[:, :KV], kv[:, KV:], torch.arange(120 * PAGE, device=dev))
        x = synth.activations(4 * tokens, 2048, dev, seed=seed)
        q = synth.activations(4 * tokens, HEADS * DIM, dev, seed=seed + 1).view(-1, HEADS, DIM)
        table = torch.arange(80, **i32).view(4, 20)
        shared = (torch.arange(80, 120, **i32)[None], torch.tensor([630], **i32),
                  torch.tensor([0, 4], **i32))
        own = (table, torch.tensor([300, 20 + tokens, 310, 200], **i32),
               torch.arange(5, **i32) * tokens, tokens)

        def run():
            s = torch.zeros(cache.k.shape[:3], device=dev)
            y = ops.int8_linear(x, w, ws)
            o, lse = ops.shared_prefix_attention(q, cache, *shared, *own, return_lse=True)
            ops.kv_cache_scores(q, cache, *own, lse, s)
            return y, o, lse, s

        return run

    jobs = [job(1, 1), job(2, 30)]
    alone = [run() for run in jobs]
    streams = [torch.cuda.Stream() for _ in jobs]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, (run, stream) in enumerate(zip(jobs, streams)):
            with torch.cuda.stream(stream):
                got[i].append(run())
    torch.cuda.synchronize()
    for want, several in zip(alone, got):
        for each in several:
            assert all(torch.equal(a, b) for a, b in zip(each, want))
    assert ops.attention_status() == 0
