"""The attention half's operations as torch custom ops, beside those of
:mod:`.torch_ops`: ``torch.ops.b200_moe.add_rms_norm`` and so on, each with a
schema, a CUDA implementation on the current stream and a fake one.

A paged cache is given by its four tensors (no scales for a 16-bit cache), so
the dispatcher sees that a write changes them. Importing the module registers
the ops once.
"""

from __future__ import annotations

import torch

from . import ops
from .kv_cache import PagedKVCache
from .torch_ops import NAMESPACE

_LIBRARY = torch.library.Library(NAMESPACE, "FRAGMENT")

_SCHEMAS = {
    "add_rms_norm":
        "add_rms_norm(Tensor x, Tensor weight, float eps, Tensor? residual=None,"
        " float weight_bias=0.0) -> (Tensor, Tensor)",
    "add_rms_norm_fp8":
        "add_rms_norm_fp8(Tensor x, Tensor weight, float eps, Tensor? residual=None,"
        " float weight_bias=0.0, int? scales_ld=None) -> (Tensor, Tensor, Tensor)",
    "w8a8_linear_quantized":
        "w8a8_linear_quantized(Tensor q, Tensor scales, Tensor w, Tensor w_scales,"
        " int gated_mode, ScalarType out_dtype) -> Tensor",
    "kv_cache_write":
        "kv_cache_write(Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor(c!)? k_scale,"
        " Tensor(d!)? v_scale, Tensor k, Tensor v, Tensor slots) -> ()",
    "kv_cache_read":
        "kv_cache_read(Tensor k_cache, Tensor v_cache, Tensor? k_scale, Tensor? v_scale,"
        " Tensor slots, ScalarType dtype) -> (Tensor, Tensor)",
    "paged_attention":
        "paged_attention(Tensor q, Tensor k_cache, Tensor v_cache, Tensor? k_scale,"
        " Tensor? v_scale, Tensor page_table, Tensor kv_lens, Tensor q_starts, int max_q_len,"
        " float? scale=None, bool causal=True, int window=0) -> (Tensor, Tensor)",
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


# Without a residual the stream is x itself, which an op may not return: the
# second result is then empty.
@_impl("add_rms_norm")
def _norm_cuda(x, weight, eps, residual=None, weight_bias=0.0):
    y, h = ops.add_rms_norm(x, weight, eps, residual=residual, weight_bias=weight_bias)
    return y, x.new_empty(0) if h is None else h


@_fake("add_rms_norm")
def _norm_fake(x, weight, eps, residual=None, weight_bias=0.0):
    return x.new_empty(x.shape), x.new_empty(0 if residual is None else x.shape)


@_impl("add_rms_norm_fp8")
def _norm_fp8_cuda(x, weight, eps, residual=None, weight_bias=0.0, scales_ld=None):
    q, scales, h = ops.add_rms_norm_fp8(x, weight, eps, residual=residual,
                                        weight_bias=weight_bias, scales_ld=scales_ld)
    return q, scales, x.new_empty(0) if h is None else h


@_fake("add_rms_norm_fp8")
def _norm_fp8_fake(x, weight, eps, residual=None, weight_bias=0.0, scales_ld=None):
    rows, hidden = x.shape
    return (x.new_empty(x.shape, dtype=torch.float8_e4m3fn),
            x.new_empty(hidden // 128, rows if scales_ld is None else scales_ld,
                        dtype=torch.float32),
            x.new_empty(0 if residual is None else x.shape))


@_impl("w8a8_linear_quantized")
def _linear_cuda(q, scales, w, w_scales, gated_mode, out_dtype):
    return ops.w8a8_linear_quantized(q, scales, w, w_scales, gated_mode=gated_mode,
                                     out_dtype=out_dtype)


@_fake("w8a8_linear_quantized")
def _linear_fake(q, scales, w, w_scales, gated_mode, out_dtype):
    n = w.shape[-2]
    return q.new_empty(q.shape[0], n // 2 if gated_mode == ops._lib.GATED_FUSED else n,
                       dtype=out_dtype)


@_impl("kv_cache_write")
def _write_cuda(k_cache, v_cache, k_scale, v_scale, k, v, slots):
    ops.kv_cache_write(PagedKVCache(k_cache, v_cache, k_scale, v_scale), k, v, slots)


@_fake("kv_cache_write")
def _write_fake(k_cache, v_cache, k_scale, v_scale, k, v, slots):
    return None


@_impl("kv_cache_read")
def _read_cuda(k_cache, v_cache, k_scale, v_scale, slots, dtype):
    return ops.kv_cache_read(PagedKVCache(k_cache, v_cache, k_scale, v_scale), slots, dtype)


@_fake("kv_cache_read")
def _read_fake(k_cache, v_cache, k_scale, v_scale, slots, dtype):
    shape = (slots.shape[0], *k_cache.shape[2:])
    return k_cache.new_empty(shape, dtype=dtype), k_cache.new_empty(shape, dtype=dtype)


@_impl("paged_attention")
def _attention_cuda(q, k_cache, v_cache, k_scale, v_scale, page_table, kv_lens, q_starts,
                    max_q_len, scale=None, causal=True, window=0):
    return ops.paged_attention(q, PagedKVCache(k_cache, v_cache, k_scale, v_scale), page_table,
                               kv_lens, q_starts, max_q_len, scale=scale, causal=causal,
                               window=window, return_lse=True)


@_fake("paged_attention")
def _attention_fake(q, k_cache, v_cache, k_scale, v_scale, page_table, kv_lens, q_starts,
                    max_q_len, scale=None, causal=True, window=0):
    return q.new_empty(q.shape), q.new_empty(q.shape[:2], dtype=torch.float32)


def names() -> list[str]:
    return list(_SCHEMAS)
