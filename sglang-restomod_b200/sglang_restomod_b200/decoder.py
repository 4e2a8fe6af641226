"""A decoder layer around the quantized experts.

:class:`AttentionBlock` is the half that :mod:`.layer` does not have: the
residual-add RMS norm with its e4m3 output, the W8A8 query/key/value and output
projections, the paged key/value cache and attention over it.
:class:`DecoderLayer` puts it in front of a :class:`~.layer.QuantMoELayer`.

A serving loop holds one :class:`~.kv_cache.PagedKVCache` per layer and one
:class:`TokenBatch` per step; prefill chunks, decode steps and mixtures of both
are the same call. Nothing in it synchronizes with the host.

``python -m sglang_restomod_b200.decoder`` runs one layer of the benchmark's
512-expert shape: a prompt in chunks, then decode steps from a captured graph.
"""

from __future__ import annotations

from dataclasses import dataclass
from typing import Callable

import torch

from . import ops, synth
from .kv_cache import PagedKVCache
from .layer import QuantMoELayer


@dataclass
class TokenBatch:
    """The new tokens of one step: sequence s has rows ``q_starts[s] :
    q_starts[s + 1]``, ``kv_lens[s]`` cached tokens with them included, and the
    pages ``page_table[s]``; token t goes to slot ``slots[t]`` of the cache."""

    page_table: torch.Tensor
    kv_lens: torch.Tensor
    q_starts: torch.Tensor
    slots: torch.Tensor
    positions: torch.Tensor
    max_q_len: int

    @classmethod
    def of(cls, q_lens: list[int], kv_lens: list[int], pages: list[list[int]], page_size: int,
           device) -> "TokenBatch":
        """From host lists: ``pages[s]`` holds at least ``ceil(kv_lens[s] / page_size)`` pages."""
        width = max(1, max((len(p) for p in pages), default=1))
        table = torch.tensor([p + [0] * (width - len(p)) for p in pages],
                             dtype=torch.int32).reshape(len(pages), width)
        positions, slots, starts = [], [], [0]
        for s, (q, kv) in enumerate(zip(q_lens, kv_lens)):
            if q > kv:
                raise ValueError(f"sequence {s}: {q} new tokens in {kv} cached ones")
            for at in range(kv - q, kv):
                positions.append(at)
                slots.append(pages[s][at // page_size] * page_size + at % page_size)
            starts.append(starts[-1] + q)
        i32 = dict(dtype=torch.int32, device=device)
        return cls(table.to(device), torch.tensor(kv_lens, **i32), torch.tensor(starts, **i32),
                   torch.tensor(slots, dtype=torch.int64, device=device),
                   torch.tensor(positions, dtype=torch.int64, device=device), max(q_lens, default=0))


Rotary = Callable[[torch.Tensor, torch.Tensor], torch.Tensor]


@dataclass
class AttentionBlock:
    """norm -> W8A8 q/k/v -> cache write -> attention -> W8A8 output projection.

    ``w_qkv`` e4m3 ``[(q_heads + 2 kv_heads) * head_dim, hidden]`` and ``w_o``
    ``[hidden, q_heads * head_dim]``, row-major, with fp32 scales per 128 x 128
    block. ``rotary(x, positions)``, if given, is applied to queries and keys
    ``[tokens, heads, head_dim]`` and returns them."""

    q_heads: int
    kv_heads: int
    head_dim: int
    norm: torch.Tensor
    w_qkv: torch.Tensor
    s_qkv: torch.Tensor
    w_o: torch.Tensor
    s_o: torch.Tensor
    eps: float = 1e-6
    norm_bias: float = 0.0
    window: int = 0
    rotary: Rotary | None = None

    def forward(self, x: torch.Tensor, residual: torch.Tensor | None, cache: PagedKVCache,
                batch: TokenBatch) -> tuple[torch.Tensor, torch.Tensor]:
        """(attention output, residual stream) of ``x`` ``[tokens, hidden]``: the
        stream is ``x + residual``, updated in place when ``residual`` is given."""
        tokens = x.shape[0]
        q8, scales, stream = ops.add_rms_norm_fp8(
            x, self.norm, self.eps, residual=residual, residual_out=residual,
            weight_bias=self.norm_bias, scales_ld=ops.w8a8_scales_ld(tokens))
        qkv = ops.w8a8_linear_quantized(q8, scales, self.w_qkv, self.s_qkv, out_dtype=x.dtype)
        qkv = qkv.view(tokens, self.q_heads + 2 * self.kv_heads, self.head_dim)
        q, k, v = qkv.split([self.q_heads, self.kv_heads, self.kv_heads], dim=1)
        if self.rotary is not None:
            q, k = self.rotary(q, batch.positions), self.rotary(k, batch.positions)
        ops.kv_cache_write(cache, k, v, batch.slots)
        o = ops.paged_attention(q, cache, batch.page_table, batch.kv_lens, batch.q_starts,
                                batch.max_q_len, window=self.window)
        return ops.w8a8_linear(o.view(tokens, -1), self.w_o, self.s_o), \
            x if stream is None else stream

    @classmethod
    def synthetic(cls, hidden: int, q_heads: int, kv_heads: int, head_dim: int, device,
                  seed: int = 20, **kw) -> "AttentionBlock":
        """Random-init block (weights N(0, 0.02), block FP8)."""
        wq, sq = synth.fp8_bank(1, (q_heads + 2 * kv_heads) * head_dim, hidden, device, seed)
        wo, so = synth.fp8_bank(1, hidden, q_heads * head_dim, device, seed + 1)
        norm = torch.ones(hidden, dtype=torch.bfloat16, device=device)
        return cls(q_heads, kv_heads, head_dim, norm, wq[0], sq[0], wo[0], so[0], **kw)


@dataclass
class DecoderLayer:
    """Attention block, then norm -> router -> quantized experts."""

    attention: AttentionBlock
    moe: QuantMoELayer
    norm: torch.Tensor
    router: torch.Tensor  # [experts, hidden]
    eps: float = 1e-6

    def forward(self, x: torch.Tensor, residual: torch.Tensor | None, cache: PagedKVCache,
                batch: TokenBatch) -> tuple[torch.Tensor, torch.Tensor]:
        """(the experts' output, residual stream); the next layer adds them."""
        h, stream = self.attention.forward(x, residual, cache, batch)
        # without a residual the stream is the caller's x, which stays as it is
        own = torch.empty_like(stream) if residual is None else stream
        y, stream = ops.add_rms_norm(h, self.norm, self.eps, residual=stream, residual_out=own)
        return self.moe.forward_logits(y, torch.matmul(y, self.router.t()).float()), stream

    @classmethod
    def synthetic(cls, shape: synth.MoEShape, quant: int, q_heads: int, kv_heads: int,
                  head_dim: int, device, seed: int = 20, **kw) -> "DecoderLayer":
        g = torch.Generator(device=device).manual_seed(seed + 7)
        router = torch.randn(shape.experts, shape.hidden, generator=g, device=device) * synth.WEIGHT_STD
        return cls(
            AttentionBlock.synthetic(shape.hidden, q_heads, kv_heads, head_dim, device, seed, **kw),
            QuantMoELayer.synthetic(shape, quant, device),
            torch.ones(shape.hidden, dtype=torch.bfloat16, device=device),
            router.to(torch.bfloat16))


def main(prompt: int = 4096, chunk: int = 2048, seqs: int = 8, steps: int = 32,
         page_size: int = 64) -> None:
    """Prefill of one prompt per sequence in chunks, then ``steps`` decode steps."""
    from . import _lib

    dev = torch.device("cuda", torch.cuda.current_device())
    shape = synth.CONFIG2
    layer = DecoderLayer.synthetic(shape, _lib.QUANT_FP8_BLOCK, q_heads=16, kv_heads=2,
                                   head_dim=128, device=dev)
    per = -(-(prompt + steps) // page_size)
    pages = [list(range(s * per, (s + 1) * per)) for s in range(seqs)]
    cache = PagedKVCache.empty(seqs * per, page_size, 2, 128, dev)

    def timed(fn):
        a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        torch.cuda.synchronize()
        a.record()
        fn()
        b.record()
        b.synchronize()
        return a.elapsed_time(b)

    for at in range(0, prompt, chunk):
        n = min(chunk, prompt - at)
        batch = TokenBatch.of([n] * seqs, [at + n] * seqs, pages, page_size, dev)
        x = synth.activations(n * seqs, shape.hidden, dev, seed=at)
        if at == 0:
            layer.forward(x, None, cache, batch)  # loads the kernels; the same tokens again below
        ms = timed(lambda: layer.forward(x, None, cache, batch))
        print(f"prefill: {seqs} x {n} tokens on {at} cached, {ms:.3f} ms")

    # One captured graph serves every step: only the buffers' contents change.
    batch = TokenBatch.of([1] * seqs, [prompt + 1] * seqs, pages, page_size, dev)
    x = synth.activations(seqs, shape.hidden, dev, seed=1)
    residual = torch.zeros_like(x)
    layer.forward(x, residual, cache, batch)  # sizes the workspaces
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        ops.reserve_attention_workspace(128, seqs, seqs)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        layer.forward(x, residual, cache, batch)
    total = 0.0
    for i in range(steps):
        now = TokenBatch.of([1] * seqs, [prompt + 1 + i] * seqs, pages, page_size, dev)
        for name in ("kv_lens", "slots", "positions"):
            getattr(batch, name).copy_(getattr(now, name))
        residual.zero_()
        total += timed(graph.replay)
    print(f"decode: {seqs} sequences of {prompt} tokens, {total / steps:.3f} ms a step")
    if ops.attention_status(dev) or ops.workspace_status(dev):
        raise RuntimeError("a kernel reported an error")


if __name__ == "__main__":
    main()
