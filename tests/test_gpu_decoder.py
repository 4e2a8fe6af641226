"""The attention half of a decoder layer as a serving loop uses it: one layer
over a paged cache, prefill in chunks, decode from a captured graph, against a
plain float64 layer; and the operators as torch custom ops."""

from __future__ import annotations

import math

import pytest
import torch

import oracle
from oracle import attention as ref
from sglang_restomod_b200 import _lib, attention_ops, decoder, kv_cache, ops, synth

B = torch.ops.b200_moe
META = torch.device("meta")
BF16, E4M3 = torch.bfloat16, torch.float8_e4m3fn
HIDDEN, HEADS, KV, DIM, PAGE = 1024, 8, 2, 128, 16


# ------------------------------------------------------------------ on a CPU
def test_token_batch_from_host_lists():
    b = decoder.TokenBatch.of([1, 3, 0], [5, 3, 0], [[2, 0], [1], []], 4, "cpu")
    assert b.slots.tolist() == [0, 4, 5, 6] and b.positions.tolist() == [4, 0, 1, 2]
    assert b.q_starts.tolist() == [0, 1, 4, 4] and b.kv_lens.tolist() == [5, 3, 0]
    assert b.page_table.tolist() == [[2, 0], [1, 0], [0, 0]] and b.max_q_len == 3
    with pytest.raises(ValueError, match="new tokens"):
        decoder.TokenBatch.of([2], [1], [[0]], 4, "cpu")
    with pytest.raises(IndexError):
        decoder.TokenBatch.of([1], [5], [[0]], 4, "cpu")
    empty = decoder.TokenBatch.of([], [], [], 4, "cpu")
    assert empty.q_starts.tolist() == [0] and empty.page_table.shape == (0, 1)


def test_ops_are_registered_and_mark_what_they_write():
    written = {"kv_cache_write": {"k_cache", "v_cache", "k_scale", "v_scale"}}
    for name in attention_ops.names():
        schema = getattr(B, name).default._schema
        assert schema.name == f"b200_moe::{name}"
        assert {a.name for a in schema.arguments if a.alias_info is not None
                and a.alias_info.is_write} == written.get(name, set())


def test_fake_implementations_propagate_shapes():
    x = torch.empty(5, 256, dtype=BF16, device=META)
    w = torch.empty(256, dtype=BF16, device=META)
    y, h = B.add_rms_norm(x, w, 1e-6, x)
    assert y.shape == h.shape == (5, 256) and y.dtype == BF16
    assert B.add_rms_norm(x, w, 1e-6)[1].numel() == 0
    q8, s8, h = B.add_rms_norm_fp8(x, w, 1e-6, None, 0.0, 128)
    assert q8.dtype == E4M3 and q8.shape == (5, 256) and s8.shape == (2, 128) and h.numel() == 0
    wq = torch.empty(512, 256, dtype=E4M3, device=META)
    ws = torch.empty(4, 2, device=META)
    assert B.w8a8_linear_quantized(q8, s8, wq, ws, _lib.GATED_FUSED, BF16).shape == (5, 256)
    kv = torch.empty(9, PAGE, KV, DIM, dtype=E4M3, device=META)
    sc = torch.empty(9, PAGE, KV, dtype=torch.uint8, device=META)
    slots = torch.empty(5, dtype=torch.int64, device=META)
    k = torch.empty(5, KV, DIM, dtype=BF16, device=META)
    assert B.kv_cache_write(kv, kv, sc, sc, k, k, slots) is None
    got = B.kv_cache_read(kv, kv, sc, sc, slots, BF16)
    assert got[0].shape == got[1].shape == (5, KV, DIM) and got[0].dtype == BF16
    i32 = dict(dtype=torch.int32, device=META)
    q = torch.empty(5, HEADS, DIM, dtype=BF16, device=META)
    out, lse = B.paged_attention(q, kv, kv, sc, sc, torch.empty(2, 3, **i32),
                                 torch.empty(2, **i32), torch.empty(3, **i32), 4)
    assert out.shape == q.shape and out.dtype == BF16
    assert lse.shape == (5, HEADS) and lse.dtype == torch.float32


# ---------------------------------------------------------------- on a B200
def rotary(x, positions):
    """Halves rotated by position, computed in fp32 and returned in x's type."""
    half = x.shape[-1] // 2
    freq = 10000.0 ** (-torch.arange(half, device=x.device, dtype=torch.float64) / half)
    angle = positions.double()[:, None, None] * freq
    a, b = x[..., :half].double(), x[..., half:].double()
    return torch.cat([a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin()],
                     -1).to(x.dtype)


def attention_plain(block, x, residual, batch, window):
    """The block without a cache and without rounding, in float64 on the CPU:
    every sequence's tokens are all new."""
    wq = oracle.dequant_block_fp8(block.w_qkv.cpu(), block.s_qkv.cpu()).double()
    wo = oracle.dequant_block_fp8(block.w_o.cpu(), block.s_o.cpu()).double()
    y, h = ref.add_rms_norm_ref(x.cpu(), block.norm.cpu(), block.eps,
                                None if residual is None else residual.cpu())
    qkv = (y @ wq.T).view(x.shape[0], HEADS + 2 * KV, DIM)
    q, k, v = qkv.split([HEADS, KV, KV], 1)
    at = batch.positions.cpu()
    q, k = rotary(q, at), rotary(k, at)
    starts = batch.q_starts.tolist()
    longest = max(b - a for a, b in zip(starts, starts[1:]))
    kc, vc = (torch.zeros(len(starts) - 1, longest, KV, DIM, dtype=torch.float64) for _ in "kv")
    for s, (a, b) in enumerate(zip(starts, starts[1:])):
        kc[s, :b - a], vc[s, :b - a] = k[a:b], v[a:b]
    table = torch.arange(len(starts) - 1)[:, None]
    out, _ = ref.paged_attention_ref(q, kc, vc, table, batch.kv_lens.cpu(), batch.q_starts.cpu(),
                                     DIM ** -0.5, True, window)
    return out.reshape(x.shape[0], -1) @ wo.T, h


def relative(got, want):
    return float((got.double().cpu() - want.double().cpu()).norm() / want.double().norm())


# An e4m3 rounding is off by 2^-4 of the element at most, by at most 2^-4 /
# sqrt(3) in the root mean square; a product with random weights hands such a
# relative error on unchanged. Between x and the block's output the values pass
# four of them (norm output, K or V, attention output; K's and the norm's once
# more through scores of order one), and bf16's are 16 times smaller.
FOUR_ROUNDINGS = math.sqrt(4) * 2.0 ** -4 / math.sqrt(3) + 0.01


@pytest.mark.gpu
@pytest.mark.parametrize("window", [0, 40])
@pytest.mark.parametrize("store", [BF16, E4M3])
def test_attention_block_whole_chunked_and_decoded(cuda_device, store, window):
    dev = cuda_device
    block = decoder.AttentionBlock.synthetic(HIDDEN, HEADS, KV, DIM, dev, window=window,
                                             rotary=rotary)
    lens = [70, 1, 33]
    pages = [[7, 0, 3, 9, 5], [2], [8, 1, 4]]
    x = synth.activations(sum(lens), HIDDEN, dev, seed=3)
    residual = synth.activations(sum(lens), HIDDEN, dev, seed=4)
    whole = decoder.TokenBatch.of(lens, lens, pages, PAGE, dev)
    want, want_h = attention_plain(block, x, residual, whole, window)

    def cache():
        return kv_cache.PagedKVCache.empty(10, PAGE, KV, DIM, dev, store)

    stream = residual.clone()
    out, h = block.forward(x, stream, cache(), whole)
    assert h is stream
    assert (h.double().cpu() - want_h).abs().max() <= 2.0 ** -8 * want_h.abs().max()
    assert relative(out, want) <= FOUR_ROUNDINGS

    # the same tokens a chunk at a time, the last ones one by one
    kept, got = cache(), torch.empty_like(out)
    starts = whole.q_starts.tolist()
    at = [0, 0, 0]
    for step in ([40, 0, 20], [27, 1, 10], [1, 0, 1], [1, 0, 1], [1, 0, 1]):
        rows = [r for s, n in enumerate(step) for r in range(starts[s] + at[s], starts[s] + at[s] + n)]
        at = [a + n for a, n in zip(at, step)]
        part = decoder.TokenBatch.of(step, at, pages, PAGE, dev)
        got[rows], _ = block.forward(x[rows], residual[rows], kept, part)
    assert at == lens
    assert relative(got, want) <= FOUR_ROUNDINGS
    assert ops.attention_status() == 0


@pytest.mark.gpu
def test_decoder_layer_and_captured_decode(cuda_device):
    dev = cuda_device
    layer = decoder.DecoderLayer.synthetic(synth.CONFIG0, _lib.QUANT_FP8_BLOCK, HEADS, KV, DIM, dev)
    cache = kv_cache.PagedKVCache.empty(16, PAGE, KV, DIM, dev)
    pages = [[3, 1, 5], [0, 2, 4]]
    x = synth.activations(41, HIDDEN, dev, seed=5)
    kept = x.clone()
    first = decoder.TokenBatch.of([30, 11], [30, 11], pages, PAGE, dev)
    y, stream = layer.forward(x, None, cache, first)
    assert torch.equal(x, kept)  # the caller's rows stay
    h, _ = layer.attention.forward(x, None, cache, first)
    _, want_stream = ref.add_rms_norm_ref(h.cpu(), layer.norm.cpu(), layer.eps, x.cpu())
    assert (stream.double().cpu() - want_stream).abs().max() <= 2.0 ** -8 * want_stream.abs().max()
    assert y.shape == x.shape and torch.isfinite(y.float()).all()

    # a layer's two results are the next one's inputs; decode from a graph
    buf_x, buf_r = (synth.activations(2, HIDDEN, dev, seed=s) for s in (6, 7))
    batch = decoder.TokenBatch.of([1, 1], [31, 12], pages, PAGE, dev)
    layer.forward(buf_x, buf_r.clone(), cache, batch)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, out_stream = layer.forward(buf_x, buf_r, cache, batch)
    for step in range(3):
        now = decoder.TokenBatch.of([1, 1], [31 + step, 12 + step], pages, PAGE, dev)
        nx, nr = (synth.activations(2, HIDDEN, dev, seed=s + 2 * step) for s in (8, 9))
        want, want_stream = layer.forward(nx, nr.clone(), cache, now)
        buf_x.copy_(nx), buf_r.copy_(nr)
        batch.kv_lens.copy_(now.kv_lens), batch.slots.copy_(now.slots)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out_stream, want_stream) and torch.equal(out, want)
    assert ops.attention_status() == 0 and ops.workspace_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("store", [BF16, E4M3])
def test_custom_ops_agree_with_the_calls(cuda_device, store):
    dev = cuda_device
    x = synth.activations(20, 512, dev, seed=1)
    w = torch.ones(512, dtype=BF16, device=dev)
    for a, b in zip(B.add_rms_norm(x, w, 1e-6, x), ops.add_rms_norm(x, w, residual=x)):
        assert torch.equal(a, b)
    q8, s8, h = B.add_rms_norm_fp8(x, w, 1e-6, x, 0.0, 128)
    r8, t8, g = ops.add_rms_norm_fp8(x, w, residual=x, scales_ld=128)
    assert torch.equal(q8.view(torch.uint8), r8.view(torch.uint8)) and torch.equal(h, g)
    assert torch.equal(s8[:, :20], t8[:, :20])
    cache = kv_cache.PagedKVCache.empty(4, PAGE, KV, DIM, dev, store)
    args = (cache.k, cache.v, cache.k_scale, cache.v_scale)
    kv = synth.activations(20, 2 * KV * DIM, dev, seed=2).view(20, 2 * KV, DIM)
    slots = torch.randperm(4 * PAGE, generator=torch.Generator().manual_seed(1))[:20].to(dev)
    B.kv_cache_write(*args, kv[:, :KV], kv[:, KV:], slots)
    for a, b in zip(B.kv_cache_read(*args, slots, BF16), ops.kv_cache_read(cache, slots)):
        assert torch.equal(a, b)
    ops.kv_cache_write(cache, torch.zeros(64, KV, DIM, dtype=BF16, device=dev),
                       torch.ones(64, KV, DIM, dtype=BF16, device=dev),
                       torch.arange(64, device=dev))
    i32 = dict(dtype=torch.int32, device=dev)
    table, lens = torch.arange(4, **i32)[None], torch.tensor([50], **i32)
    starts = torch.tensor([0, 20], **i32)
    q = synth.activations(20, HEADS * DIM, dev, seed=3).view(20, HEADS, DIM)
    out, lse = B.paged_attention(q, *args, table, lens, starts, 20)
    want, want_lse = ops.paged_attention(q, cache, table, lens, starts, 20, return_lse=True)
    assert torch.equal(out, want) and torch.equal(lse, want_lse)
    if store == BF16:  # opcheck's schema test multiplies the inputs: not for float8 tensors
        torch.library.opcheck(B.add_rms_norm.default, (x, w, 1e-6, x))
        torch.library.opcheck(B.kv_cache_write.default, (*args, kv[:, :KV], kv[:, KV:], slots))
        torch.library.opcheck(B.kv_cache_read.default, (*args, slots, BF16))
        torch.library.opcheck(B.paged_attention.default, (q, *args, table, lens, starts, 20))
