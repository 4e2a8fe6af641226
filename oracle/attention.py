"""Norm, key/value cache and paged attention in 64 bits (test infrastructure only).

The reference leaves norms and attention to upstream SGLang, so there is
nothing of its own to pin these against: they are the operators' formulas,
written plainly, in float64 on the CPU.
"""

from __future__ import annotations

import math

import torch


def add_rms_norm_ref(x, weight, eps, residual=None, weight_bias=0.0):
    """(y, h) in float64."""
    h = x.double()
    if residual is not None:
        h = h + residual.double()
    y = h / torch.sqrt((h * h).mean(-1, keepdim=True) + eps) * (weight.double() + weight_bias)
    return y, h


def kv_quantize_ref(x):
    """(codes e4m3, scale bytes uint8) of the vectors along the last axis: the
    smallest 2^e, e in [-24, 7], with max|x| <= 448 * 2^e; 255 where a vector
    holds an infinity or a NaN (codes 0)."""
    flat = x.reshape(-1, x.shape[-1]).double()
    codes = torch.zeros(flat.shape, dtype=torch.float8_e4m3fn)
    scale = torch.zeros(flat.shape[0], dtype=torch.uint8)
    for i, row in enumerate(flat):
        if not torch.isfinite(row).all():
            scale[i] = 255
            continue
        top = float(row.abs().max())
        e = -24
        while e < 7 and top > 448.0 * 2.0 ** e:
            e += 1
        scale[i] = 127 + e
        codes[i] = (row * 2.0 ** -e).clamp(-448.0, 448.0).float().to(torch.float8_e4m3fn)
    return codes.reshape(x.shape), scale.reshape(x.shape[:-1])


def kv_values_ref(codes, scale):
    """float64 values of codes and scale bytes."""
    v = codes.double() * torch.pow(2.0, scale.double() - 127.0)[..., None]
    return torch.where((scale == 255)[..., None], torch.full_like(v, math.nan), v)


def paged_attention_ref(q, k_cache, v_cache, table, kv_lens, q_starts, scale, causal=True, window=0):
    """(out, lse) in float64; k_cache / v_cache are values [pages, page_size, heads, dim]."""
    page = k_cache.shape[1]
    groups = q.shape[1] // k_cache.shape[2]
    out = torch.zeros(q.shape, dtype=torch.float64)
    lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64)
    for s, kv in enumerate(kv_lens.tolist()):
        a, b = int(q_starts[s]), int(q_starts[s + 1])
        if kv == 0 or a == b:
            continue
        at = torch.arange(kv)
        pages = table[s].long()[at // page]
        k = k_cache[pages, at % page].double()
        v = v_cache[pages, at % page].double()
        pos = kv - (b - a) + torch.arange(b - a)[:, None]
        seen = torch.ones(b - a, kv, dtype=torch.bool)
        if causal:
            seen = at[None, :] <= pos
            if window:
                seen &= at[None, :] > pos - window
        for h in range(q.shape[1]):
            x = q[a:b, h].double() @ k[:, h // groups].T * scale
            x = x.masked_fill(~seen, -math.inf)
            lse[a:b, h] = torch.logsumexp(x, -1)
            p = torch.exp(x - torch.where(lse[a:b, h] > -math.inf, lse[a:b, h], 0.0)[:, None])
            # a masked token weighs nothing, whatever its value holds
            out[a:b, h] = p @ torch.where(seen.any(0)[:, None], v[:, h // groups], 0.0)
    return out, lse
