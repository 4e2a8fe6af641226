"""The 8-bit integer linear, shared-prefix attention, and a cache's scores and eviction
as torch custom ops, beside those of :mod:`.attention_ops`, in the same form:
``torch.ops.b200_moe.int8_linear`` and so on. Importing the module registers them once.
"""

from __future__ import annotations

import torch

from . import ops
from .kv_cache import PagedKVCache
from .torch_ops import NAMESPACE

_LIBRARY = torch.library.Library(NAMESPACE, "FRAGMENT")

_CACHE = "Tensor k_cache, Tensor v_cache, Tensor? k_scale, Tensor? v_scale"
_SCHEMAS = {
    "int8_act_quant": "int8_act_quant(Tensor x) -> (Tensor, Tensor)",
    "int8_linear":
        "int8_linear(Tensor x, Tensor w, Tensor w_scales, ScalarType out_dtype) -> Tensor",
    "int8_linear_quantized":
        "int8_linear_quantized(Tensor q, Tensor scales, Tensor w, Tensor w_scales,"
        " ScalarType out_dtype) -> Tensor",
    "shared_prefix_attention":
        f"shared_prefix_attention(Tensor q, {_CACHE}, Tensor prefix_table, Tensor prefix_lens,"
        " Tensor group_starts, Tensor page_table, Tensor kv_lens, Tensor q_starts, int max_q_len,"
        " float? scale=None) -> (Tensor, Tensor)",
    "kv_cache_scores":
        f"kv_cache_scores(Tensor q, {_CACHE}, Tensor page_table, Tensor kv_lens, Tensor q_starts,"
        " int max_q_len, Tensor lse, Tensor(a!) scores, float? scale=None, bool causal=True,"
        " int window=0) -> ()",
    "kv_cache_evict":
        "kv_cache_evict(Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor(c!)? k_scale,"
        " Tensor(d!)? v_scale, Tensor(e!) scores, Tensor page_table, Tensor kv_lens, int budget,"
        " int recent=0, int first=0, Tensor? out_table=None) -> (Tensor, Tensor)",
}

for _schema in _SCHEMAS.values():
    _LIBRARY.define(_schema)


def _impl(name):
    def deco(fn):
        _LIBRARY.impl(name, fn, "CUDA")
        return fn

    return deco


def _fake(name):
    return torch.library.register_fake(f"{NAMESPACE}::{name}", lib=_LIBRARY)


@_impl("int8_act_quant")
def _quant_cuda(x):
    return ops.int8_act_quant(x)


@_fake("int8_act_quant")
def _quant_fake(x):
    return (x.new_empty(x.shape, dtype=torch.int8),
            x.new_empty(x.shape[:1], dtype=torch.float32))


@_impl("int8_linear")
def _linear_cuda(x, w, w_scales, out_dtype):
    return ops.int8_linear(x, w, w_scales, out_dtype=out_dtype)


@_fake("int8_linear")
def _linear_fake(x, w, w_scales, out_dtype):
    return x.new_empty((*x.shape[:-1], w.shape[0]), dtype=out_dtype)


@_impl("int8_linear_quantized")
def _linear_quantized_cuda(q, scales, w, w_scales, out_dtype):
    return ops.int8_linear_quantized(q, scales, w, w_scales, out_dtype=out_dtype)


@_fake("int8_linear_quantized")
def _linear_quantized_fake(q, scales, w, w_scales, out_dtype):
    return q.new_empty(q.shape[0], w.shape[0], dtype=out_dtype)


@_impl("shared_prefix_attention")
def _prefix_cuda(q, k_cache, v_cache, k_scale, v_scale, prefix_table, prefix_lens, group_starts,
                 page_table, kv_lens, q_starts, max_q_len, scale=None):
    return ops.shared_prefix_attention(q, PagedKVCache(k_cache, v_cache, k_scale, v_scale),
                                       prefix_table, prefix_lens, group_starts, page_table, kv_lens,
                                       q_starts, max_q_len, scale=scale, return_lse=True)


@_fake("shared_prefix_attention")
def _prefix_fake(q, k_cache, v_cache, k_scale, v_scale, prefix_table, prefix_lens, group_starts,
                 page_table, kv_lens, q_starts, max_q_len, scale=None):
    return q.new_empty(q.shape), q.new_empty(q.shape[:2], dtype=torch.float32)


@_impl("kv_cache_scores")
def _scores_cuda(q, k_cache, v_cache, k_scale, v_scale, page_table, kv_lens, q_starts, max_q_len,
                 lse, scores, scale=None, causal=True, window=0):
    ops.kv_cache_scores(q, PagedKVCache(k_cache, v_cache, k_scale, v_scale), page_table, kv_lens,
                        q_starts, max_q_len, lse, scores, scale=scale, causal=causal, window=window)


@_fake("kv_cache_scores")
def _scores_fake(q, k_cache, v_cache, k_scale, v_scale, page_table, kv_lens, q_starts, max_q_len,
                 lse, scores, scale=None, causal=True, window=0):
    return None


@_impl("kv_cache_evict")
def _evict_cuda(k_cache, v_cache, k_scale, v_scale, scores, page_table, kv_lens, budget, recent=0,
                first=0, out_table=None):
    return ops.kv_cache_evict(PagedKVCache(k_cache, v_cache, k_scale, v_scale), scores, page_table,
                              kv_lens, budget, recent=recent, first=first, out_table=out_table)


@_fake("kv_cache_evict")
def _evict_fake(k_cache, v_cache, k_scale, v_scale, scores, page_table, kv_lens, budget, recent=0,
                first=0, out_table=None):
    seqs = kv_lens.shape[0]
    return (kv_lens.new_empty(seqs, k_cache.shape[2], budget), kv_lens.new_empty(seqs))


def names() -> list[str]:
    return list(_SCHEMAS)
