"""A decoder layer around the quantized experts.

:class:`AttentionBlock` is the half that :mod:`.layer` does not have: the
residual-add RMS norm, the query/key/value and output projections (block-FP8 W8A8,
or 8-bit integers with a scale per token and channel), the paged key/value cache and
attention over it, with a :class:`SharedPrefix` for sequences that begin alike.
:class:`DecoderLayer` puts it in front of a :class:`~.layer.QuantMoELayer`.

A serving loop holds one :class:`~.kv_cache.PagedKVCache` per layer and one
:class:`TokenBatch` per step; prefill chunks, decode steps and mixtures of both
are the same call. Given ``scores``, a step also adds up the attention weights that
cached tokens get, by which :func:`.ops.kv_cache_evict` then shortens the sequences.
Nothing in it synchronizes with the host.

``python -m sglang_restomod_b200.decoder`` runs one layer of the benchmark's
512-expert shape: a prompt in chunks, then decode steps from a captured graph; and
questions behind a shared prompt, whose caches are cut before they are answered.
"""

from __future__ import annotations

from dataclasses import dataclass
from typing import Callable

import torch

from . import ops, synth
from .kv_cache import PagedKVCache
from .layer import QuantMoELayer


@dataclass
class SharedPrefix:
    """Prefixes that several sequences of a batch share: the sequences
    ``group_starts[g] : group_starts[g + 1]`` come after the first ``lens[g]`` tokens of
    the pages ``page_table[g]``. A :class:`TokenBatch` with one describes each
    sequence's own tokens only."""

    page_table: torch.Tensor
    lens: torch.Tensor
    group_starts: torch.Tensor

    @classmethod
    def of(cls, lens: list[int], pages: list[list[int]], group_sizes: list[int],
           device) -> "SharedPrefix":
        """From host lists: a prefix of ``lens[g]`` tokens on ``pages[g]`` before each of the
        next ``group_sizes[g]`` sequences (no prefix: length 0, no pages)."""
        if not len(lens) == len(pages) == len(group_sizes):
            raise ValueError(f"{len(lens)} lengths, {len(pages)} page lists and "
                             f"{len(group_sizes)} group sizes")
        starts = [0]
        for n in group_sizes:
            starts.append(starts[-1] + n)
        i32 = dict(dtype=torch.int32, device=device)
        return cls(_page_table(pages, device), torch.tensor(lens, **i32),
                   torch.tensor(starts, **i32))


def _page_table(pages: list[list[int]], device) -> torch.Tensor:
    width = max(1, max((len(p) for p in pages), default=1))
    return torch.tensor([p + [0] * (width - len(p)) for p in pages],
                        dtype=torch.int32).reshape(len(pages), width).to(device)


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
    prefix: SharedPrefix | None = None

    @classmethod
    def of(cls, q_lens: list[int], kv_lens: list[int], pages: list[list[int]], page_size: int,
           device, before: list[int] | None = None,
           prefix: SharedPrefix | None = None) -> "TokenBatch":
        """From host lists: ``pages[s]`` holds at least ``ceil(kv_lens[s] / page_size)`` pages.
        ``before[s]`` is how many positions come before the sequence's cached tokens: the
        length of its shared prefix, and the tokens that an eviction took out."""
        positions, slots, starts = [], [], [0]
        for s, (q, kv) in enumerate(zip(q_lens, kv_lens)):
            if q > kv:
                raise ValueError(f"sequence {s}: {q} new tokens in {kv} cached ones")
            for at in range(kv - q, kv):
                positions.append(at + (before[s] if before else 0))
                slots.append(pages[s][at // page_size] * page_size + at % page_size)
            starts.append(starts[-1] + q)
        i32 = dict(dtype=torch.int32, device=device)
        return cls(_page_table(pages, device), torch.tensor(kv_lens, **i32),
                   torch.tensor(starts, **i32),
                   torch.tensor(slots, dtype=torch.int64, device=device),
                   torch.tensor(positions, dtype=torch.int64, device=device), max(q_lens, default=0),
                   prefix)


Rotary = Callable[[torch.Tensor, torch.Tensor], torch.Tensor]


@dataclass
class AttentionBlock:
    """norm -> 8-bit q/k/v -> cache write -> attention -> 8-bit output projection.

    ``w_qkv`` ``[(q_heads + 2 kv_heads) * head_dim, hidden]`` and ``w_o``
    ``[hidden, q_heads * head_dim]``, row-major: e4m3 with fp32 scales per 128 x 128
    block, or int8 with an fp32 scale per row. ``rotary(x, positions)``, if given, is
    applied to queries and keys ``[tokens, heads, head_dim]`` and returns them."""

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
                batch: TokenBatch,
                scores: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
        """(attention output, residual stream) of ``x`` ``[tokens, hidden]``: the
        stream is ``x + residual``, updated in place when ``residual`` is given.
        ``scores`` (:meth:`~.kv_cache.PagedKVCache.empty_scores`) gather the attention
        weights of the sequences' cached tokens (not of a shared prefix's)."""
        if batch.prefix is not None and self.window:
            raise ValueError("a shared prefix is seen whole: the block's window must be 0")
        tokens = x.shape[0]
        norm = dict(residual=residual, residual_out=residual, weight_bias=self.norm_bias)
        if self.w_qkv.dtype == torch.int8:
            y, stream = ops.add_rms_norm(x, self.norm, self.eps, **norm)
            qkv = ops.int8_linear(y, self.w_qkv, self.s_qkv)
        else:
            q8, scales, stream = ops.add_rms_norm_fp8(
                x, self.norm, self.eps, scales_ld=ops.w8a8_scales_ld(tokens), **norm)
            qkv = ops.w8a8_linear_quantized(q8, scales, self.w_qkv, self.s_qkv, out_dtype=x.dtype)
        qkv = qkv.view(tokens, self.q_heads + 2 * self.kv_heads, self.head_dim)
        q, k, v = qkv.split([self.q_heads, self.kv_heads, self.kv_heads], dim=1)
        if self.rotary is not None:
            q, k = self.rotary(q, batch.positions), self.rotary(k, batch.positions)
        ops.kv_cache_write(cache, k, v, batch.slots)
        own = (batch.page_table, batch.kv_lens, batch.q_starts, batch.max_q_len)
        want_lse = scores is not None
        if (shared := batch.prefix) is not None:
            o = ops.shared_prefix_attention(q, cache, shared.page_table, shared.lens,
                                            shared.group_starts, *own, return_lse=want_lse)
        else:
            o = ops.paged_attention(q, cache, *own, window=self.window, return_lse=want_lse)
        if want_lse:
            o, lse = o
            ops.kv_cache_scores(q, cache, *own, lse, scores, window=self.window)
        linear = ops.int8_linear if self.w_o.dtype == torch.int8 else ops.w8a8_linear
        return linear(o.view(tokens, -1), self.w_o, self.s_o), x if stream is None else stream

    @classmethod
    def synthetic(cls, hidden: int, q_heads: int, kv_heads: int, head_dim: int, device,
                  seed: int = 20, int8: bool = False, **kw) -> "AttentionBlock":
        """Random-init block (weights N(0, 0.02), block FP8 or int8)."""
        bank = synth.int8_bank if int8 else synth.fp8_bank
        wq, sq = bank(1, (q_heads + 2 * kv_heads) * head_dim, hidden, device, seed)
        wo, so = bank(1, hidden, q_heads * head_dim, device, seed + 1)
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
                batch: TokenBatch,
                scores: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
        """(the experts' output, residual stream); the next layer adds them."""
        h, stream = self.attention.forward(x, residual, cache, batch, scores)
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


def _timed(fn) -> float:
    a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    torch.cuda.synchronize()
    a.record()
    fn()
    b.record()
    b.synchronize()
    return a.elapsed_time(b)


def _decode(layer: DecoderLayer, cache: PagedKVCache, scores: torch.Tensor | None, steps: int,
            batch_of: Callable[[int], TokenBatch], reserve: Callable[[], object]) -> float:
    """Mean milliseconds of ``steps`` steps. One captured graph serves them all: only
    the buffers' contents change."""
    batch = batch_of(0)
    x = synth.activations(batch.slots.shape[0], layer.norm.shape[0], batch.slots.device, seed=1)
    residual = torch.zeros_like(x)
    layer.forward(x, residual, cache, batch, scores)  # sizes the workspaces
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        reserve()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        layer.forward(x, residual, cache, batch, scores)
    total = 0.0
    for i in range(steps):
        now = batch_of(i)
        for name in ("kv_lens", "slots", "positions"):
            getattr(batch, name).copy_(getattr(now, name))
        residual.zero_()
        total += _timed(graph.replay)
    return total / steps


def shared_prompt(prompt: int = 4096, question: int = 1024, budget: int = 512, seqs: int = 16,
                  steps: int = 32, page_size: int = 64) -> None:
    """Sequences that share a prompt, with int8 projections: the prompt once, a question
    each on it, the questions' caches cut to ``budget`` tokens by the weights they got,
    then ``steps`` decode steps."""
    from . import _lib

    dev = torch.device("cuda", torch.cuda.current_device())
    shape = synth.CONFIG2
    layer = DecoderLayer.synthetic(shape, _lib.QUANT_FP8_BLOCK, q_heads=16, kv_heads=2,
                                   head_dim=128, device=dev, int8=True)
    common = -(-prompt // page_size)
    per = -(-(question + steps) // page_size)
    prefix_pages = list(range(common))
    pages = [list(range(common + s * per, common + (s + 1) * per)) for s in range(seqs)]
    cache = PagedKVCache.empty(common + seqs * per, page_size, 2, 128, dev)
    scores = cache.empty_scores()
    x = synth.activations(prompt, shape.hidden, dev, seed=2)
    batch = TokenBatch.of([prompt], [prompt], [prefix_pages], page_size, dev)
    layer.forward(x, None, cache, batch)

    prefix = SharedPrefix.of([prompt], [prefix_pages], [seqs], dev)
    x = synth.activations(question * seqs, shape.hidden, dev, seed=3)
    batch = TokenBatch.of([question] * seqs, [question] * seqs, pages, page_size, dev,
                          [prompt] * seqs, prefix)
    layer.forward(x, None, cache, batch, scores)  # loads the kernels; the same again below
    ms = _timed(lambda: layer.forward(x, None, cache, batch, scores))
    print(f"prefill: {seqs} x {question} tokens behind a shared prompt of {prompt}, {ms:.3f} ms")
    tables = (batch.page_table, batch.kv_lens)
    ops.kv_cache_evict(cache, scores, *tables, question)  # loads the kernels; nothing to do
    ms = _timed(lambda: ops.kv_cache_evict(cache, scores, *tables, budget, recent=budget // 4,
                                           first=4))
    print(f"eviction: {question} to {budget} tokens each, {ms:.3f} ms")

    kept = min(budget, question)
    before = [prompt + question - kept] * seqs
    ms = _decode(layer, cache, scores, steps, lambda i: TokenBatch.of(
        [1] * seqs, [kept + 1 + i] * seqs, pages, page_size, dev, before, prefix),
        lambda: ops.reserve_shared_prefix_workspace(128, seqs, 16, seqs, 1))
    print(f"decode: {seqs} sequences of {kept} tokens on the shared prompt, {ms:.3f} ms a step")
    if ops.attention_status(dev) or ops.workspace_status(dev):
        raise RuntimeError("a kernel reported an error")


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

    for at in range(0, prompt, chunk):
        n = min(chunk, prompt - at)
        batch = TokenBatch.of([n] * seqs, [at + n] * seqs, pages, page_size, dev)
        x = synth.activations(n * seqs, shape.hidden, dev, seed=at)
        if at == 0:
            layer.forward(x, None, cache, batch)  # loads the kernels; the same tokens again below
        ms = _timed(lambda: layer.forward(x, None, cache, batch))
        print(f"prefill: {seqs} x {n} tokens on {at} cached, {ms:.3f} ms")

    ms = _decode(layer, cache, None, steps, lambda i: TokenBatch.of(
        [1] * seqs, [prompt + 1 + i] * seqs, pages, page_size, dev),
        lambda: ops.reserve_attention_workspace(128, seqs, seqs))
    print(f"decode: {seqs} sequences of {prompt} tokens, {ms:.3f} ms a step")
    if ops.attention_status(dev) or ops.workspace_status(dev):
        raise RuntimeError("a kernel reported an error")


if __name__ == "__main__":
    main()
    shared_prompt()
