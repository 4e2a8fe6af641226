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


def _cached(cache, table, n):
    """The first n tokens of a page table's row: [n, heads, dim]."""
    at = torch.arange(n)
    return cache[table.long()[at // cache.shape[1]], at % cache.shape[1]].double()


def shared_prefix_attention_ref(q, k_cache, v_cache, prefix_table, prefix_lens, group_starts, table,
                                kv_lens, q_starts, scale):
    """(out, lse) in float64: each sequence's new tokens over its group's prefix, whole,
    and its own tokens, causally."""
    groups = q.shape[1] // k_cache.shape[2]
    out = torch.zeros(q.shape, dtype=torch.float64)
    lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64)
    for g, far in enumerate(prefix_lens.tolist()):
        for s in range(int(group_starts[g]), int(group_starts[g + 1])):
            a, b, kv = int(q_starts[s]), int(q_starts[s + 1]), int(kv_lens[s])
            k, v = (torch.cat([_cached(c, prefix_table[g], far), _cached(c, table[s], kv)])
                    for c in (k_cache, v_cache))
            if a == b or not len(k):
                continue
            at = torch.cat([torch.full((far,), -1 << 31), torch.arange(kv)])
            seen = at[None, :] <= kv - (b - a) + torch.arange(b - a)[:, None]
            for h in range(q.shape[1]):
                x = (q[a:b, h].double() @ k[:, h // groups].T * scale).masked_fill(~seen, -math.inf)
                lse[a:b, h] = torch.logsumexp(x, -1)
                p = torch.exp(x - torch.where(lse[a:b, h] > -math.inf, lse[a:b, h], 0.0)[:, None])
                out[a:b, h] = p @ torch.where(seen.any(0)[:, None], v[:, h // groups], 0.0)
    return out, lse


def kv_cache_scores_ref(q, k_cache, table, kv_lens, q_starts, lse, scores, scale, causal=True,
                        window=0, max_q=1 << 30):
    """float64 scores [pages, page_size, heads] after adding each cached token's weights;
    ``scores`` (same shape) is what they were. Also each token's added sum alone."""
    groups, page = q.shape[1] // k_cache.shape[2], k_cache.shape[1]
    out, added = scores.double().clone(), torch.zeros(scores.shape, dtype=torch.float64)
    for s, kv in enumerate(kv_lens.tolist()):
        a, b = int(q_starts[s]), int(q_starts[s + 1])
        if kv == 0:
            continue
        at = torch.arange(kv)
        pages = table[s].long()[at // page]
        k = k_cache[pages, at % page].double()
        pos = (kv - (b - a) + torch.arange(b - a)[:, None])[:max_q]
        n = len(pos)
        seen = torch.ones(n, kv, dtype=torch.bool)
        if causal:
            seen = at[None, :] <= pos
            if window:
                seen &= at[None, :] > pos - window
        old = scores[pages, at % page].double()
        if causal:
            old[max(0, kv - (b - a)):] = 0.0
        total = torch.zeros(kv, k_cache.shape[2], dtype=torch.float64)
        for h in range(q.shape[1]):
            z = lse[a:a + n, h].double()[:, None]
            x = (q[a:a + n, h].double() @ k[:, h // groups].T * scale).masked_fill(~seen, -math.inf)
            p = torch.where((z == -math.inf) | ~seen, 0.0, torch.exp(x - z))
            total[:, h // groups] += p.sum(0)
        out[pages, at % page] = old + total
        added[pages, at % page] = total
    return out, added
