"""Measured cases of the attention half of a decoder layer: the residual-add
RMS norm (with the e4m3 output the W8A8 linears read), the paged key/value
cache (quantized as it is written, and read back), and attention of new tokens
over that cache (single-token decode, chunks on a context, whole prompts).

``own`` chooses between the plain form (elementary torch operations in fp32,
rounded once at the end) and the library's own entry points. ``listed`` gives
the fixed cases, ``draw`` more of the same ranges, ``prepare`` what a serving
loop has in hand before the call, ``run`` one pass, ``work`` the bytes and
operations a pass cannot do without, and ``exact`` the definition in 64 bits.

The quantized cache holds, per token and key/value head, ``head_dim`` e4m3
codes and one power-of-two scale 2^e stored as the byte 127 + e, with e the
smallest exponent in [-24, 7] for which the vector's largest magnitude is at
most 448 * 2^e; a code stands for ``code * 2^e``.
"""

import math
import random
import sys
from pathlib import Path

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
EPS = 1e-6


def _library():
    root = str(Path(__file__).resolve().parents[1] / "sglang-restomod_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    from sglang_restomod_b200 import kv_cache, ops

    return ops, kv_cache


# ------------------------------------------------------------------- cases
def _norm(name, rows, hidden, dtype, fp8, residual, weight_bias):
    return {"name": name, "op": "norm", "rows": rows, "hidden": hidden, "dtype": dtype,
            "fp8": fp8, "residual": residual, "weight_bias": weight_bias}


def _cache(name, tokens, heads, dim, page, dtype, fp8):
    return {"name": name, "op": "cache", "tokens": tokens, "heads": heads, "dim": dim,
            "page": page, "dtype": dtype, "fp8": fp8}


def _attn(name, seqs, q, kv, heads, groups, dim, page, dtype, fp8, *, causal=True, window=0,
          empty=0, ragged=True, lens_seed=1):
    return {"name": name, "op": "attention", "seqs": seqs, "q": q, "kv": kv, "heads": heads,
            "groups": groups, "dim": dim, "page": page, "dtype": dtype, "fp8": fp8,
            "causal": causal, "window": window, "empty": empty, "ragged": ragged,
            "lens_seed": lens_seed}


def listed():
    return [
        # one decoded token in front of a W8A8 projection: pure launch latency
        _norm("norm 1x7168 to fp8", 1, 7168, "bf16", True, True, 0.0),
        # a plain norm of an odd row count, f16, weights stored as offsets from one
        _norm("norm 1021x2048 f16", 1021, 2048, "f16", False, False, 1.0),
        # a long prefill batch in front of a W8A8 projection: bandwidth
        _norm("norm 16384x7168 to fp8", 16384, 7168, "bf16", True, True, 0.0),
        # one decode step of 131 sequences written into 16-token pages
        _cache("cache 131 tokens fp8", 131, 8, 128, 16, "bf16", True),
        # an unquantized f16 cache of single-token pages, odd token and head counts
        _cache("cache 3001 tokens f16", 3001, 5, 64, 1, "f16", False),
        # the keys and values of a long prefill batch, quantized on the way
        _cache("cache 32768 tokens fp8", 32768, 8, 128, 64, "bf16", True),
        # one user, one token, a short context: latency
        _attn("decode 1x4099 bf16", 1, 1, 4099, 8, 4, 128, 16, "bf16", False),
        # a serving batch of uneven contexts over the quantized cache
        _attn("decode 64x8192 fp8", 64, 1, 8192, 8, 8, 128, 64, "bf16", True),
        # long contexts, wide heads, two key/value heads
        _attn("decode 16x32768 d256", 16, 1, 32768, 2, 8, 256, 16, "bf16", False),
        # a chunk of a prompt on top of a long context, quantized cache
        _attn("chunk 512 on 16384 fp8", 1, 512, 16384, 8, 4, 128, 64, "bf16", True),
        # a whole prompt
        _attn("prefill 8192 bf16", 1, 8192, 8192, 8, 4, 128, 64, "bf16", False),
        # mixed chunks of up to 300 tokens, f16, three queries a head, a window,
        # single-token pages, and two idle slots whose rows see nothing
        _attn("mixed 16x300 f16 window", 16, 300, 4096, 8, 3, 64, 1, "f16", False, window=1000,
              empty=2),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "cache", "attention", "attention"])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    if op == "norm":
        fp8 = rng.random() < 0.6
        # odd multiples of the quantization group, or of one 16-byte access
        hidden = 128 * (2 * rng.randint(0, 31) + 1) if fp8 else 8 * (_log(rng, 8, 1023) | 1)
        rows = _log(rng, 1, min(131072, 16384 * 7168 // hidden))
        c = _norm("", rows, hidden, dtype, fp8, rng.random() < 0.7, rng.choice([0.0, 1.0]))
    elif op == "cache":
        dim = rng.choice([64, 128, 256])
        heads = rng.choice([1, 2, 3, 4, 5, 8, 16])
        tokens = _log(rng, 1, 32768 * 8 * 128 // (heads * dim))
        c = _cache("", tokens, heads, dim, rng.choice([1, 8, 16, 24, 64, 256]), dtype,
                   rng.random() < 0.7)
    else:
        dim = rng.choice([64, 128, 128, 256])
        heads = rng.choice([1, 2, 4, 8])
        groups = rng.choice([1, 2, 3, 4, 6, 8, 16])
        page = rng.choice([1, 16, 24, 64, 128])
        q = 1 if rng.random() < 0.5 else _log(rng, 2, 4096)
        kv = q + _log(rng, 1, 32768)
        # no more than the largest listed cases: scores, cached elements
        most = min(64, 8192 * 8192 * 32 // (heads * groups * q * kv),
                   64 * 8192 * 8 * 128 // (heads * dim * kv))
        if most < 1:
            kv = max(q, 8192 * 8192 * 32 // (heads * groups * q))
            most = 1
        c = _attn("", _log(rng, 1, most), q, kv, heads, groups, dim, page, dtype,
                  rng.random() < 0.5, causal=rng.random() < 0.85,
                  window=_log(rng, 16, 4096) if rng.random() < 0.25 else 0,
                  ragged=rng.random() < 0.8, lens_seed=rng.randint(1, 1 << 20))
        c["empty"] = rng.randint(0, 2) if c["seqs"] > 4 else 0
        if not c["causal"]:
            c["window"] = 0
    del c["name"]
    return c


def _lens(c):
    """(new tokens, cached tokens) of each sequence; the new ones are the last
    of the cached ones. The first sequence has the largest of both, and an
    idle slot has one new token and nothing cached."""
    rng = random.Random(c["lens_seed"])
    qs, kvs = [], []
    for i in range(c["seqs"]):
        q, kv = c["q"], c["kv"]
        if c["ragged"] and i:
            q = rng.randint(1, q)
            kv = rng.randint(q, kv)
        if i and i >= c["seqs"] - c["empty"]:
            q, kv = 1, 0
        qs.append(q)
        kvs.append(kv)
    return qs, kvs


# ----------------------------------------------------------------- prepare
def _randn(g, *shape, dtype, scale=1.0, step=1 << 27):
    """Seeded normal values, made in pieces so that the fp32 they pass through stays small."""
    out = torch.empty(*shape, dtype=dtype, device="cuda")
    flat = out.view(-1)
    for a in range(0, flat.numel(), step):
        b = min(a + step, flat.numel())
        flat[a:b] = torch.randn(b - a, generator=g, device="cuda").mul_(scale).to(dtype)
    return out


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    if case["op"] == "norm":
        rows, hidden = case["rows"], case["hidden"]
        s = {"case": case, "x": _randn(g, rows, hidden, dtype=dt),
             "residual": _randn(g, rows, hidden, dtype=dt, scale=3.0) if case["residual"] else None,
             "weight": (1.0 - case["weight_bias"]
                        + 0.1 * torch.randn(hidden, generator=g, device="cuda")).to(dt)}
        # the residual stream's new value goes to the other of two buffers
        s["residual_out"] = torch.empty_like(s["x"]) if case["residual"] else None
        return s
    heads, dim, page = case["heads"], case["dim"], case["page"]
    if case["op"] == "cache":
        n = case["tokens"]
        pages = -(-n // page) + 3
        # sequences' pages lie anywhere in the pool
        order = torch.randperm(pages, generator=g, device="cuda")
        at = torch.arange(n, device="cuda")
        slots = order[at // page] * page + at % page
        store = torch.float8_e4m3fn if case["fp8"] else dt
        kv = [torch.zeros(pages, heads, page, dim, dtype=torch.uint8 if case["fp8"] else dt,
                          device="cuda").view(store).transpose(1, 2) for _ in range(2)]
        sc = [torch.zeros(pages, heads, page, dtype=torch.uint8, device="cuda").transpose(1, 2)
              if case["fp8"] else None for _ in range(2)]
        # a fused projection's output: keys and values are slices of one row
        both = _randn(g, n, 2 * heads, dim, dtype=dt)
        both[:, :heads] *= 2.0
        return {"case": case, "k": both[:, :heads], "v": both[:, heads:], "slots": slots,
                "cache": (kv[0], kv[1], sc[0], sc[1])}
    qs, kvs = _lens(case)
    need = [-(-n // page) for n in kvs]
    width = max(1, max(need))
    pages = sum(need) + 2
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.zeros(len(kvs), width, dtype=torch.int32)
    at = 0
    rows = torch.arange(width)[None, :] < torch.tensor(need)[:, None]
    table[rows] = torch.arange(sum(need), dtype=torch.int32)
    table = table.cuda()
    table = torch.where(rows.cuda(), order[table.long()], torch.zeros_like(table))
    kv, sc = [], []
    for _ in range(2):
        raw = _randn(g, pages, heads, page, dim, dtype=dt)
        if case["fp8"]:
            codes = torch.empty(raw.shape, dtype=torch.uint8, device="cuda")
            scale = torch.empty(raw.shape[:-1], dtype=torch.uint8, device="cuda")
            step = max(1, (1 << 27) // (heads * page * dim))
            for a in range(0, pages, step):
                q8, sb = _plain_quantize(raw[a:a + step])
                codes[a:a + step] = q8.view(torch.uint8)
                scale[a:a + step] = sb
            kv.append(codes.view(torch.float8_e4m3fn).transpose(1, 2))
            sc.append(scale.transpose(1, 2))
            del raw
        else:
            kv.append(raw.transpose(1, 2))
            sc.append(None)
    starts = [0]
    for n in qs:
        starts.append(starts[-1] + n)
    i32 = dict(dtype=torch.int32, device="cuda")
    return {"case": case, "q": _randn(g, starts[-1], heads * case["groups"], dim, dtype=dt, scale=1.5),
            "cache": (kv[0], kv[1], sc[0], sc[1]), "table": table,
            "kv_lens": torch.tensor(kvs, **i32), "q_starts": torch.tensor(starts, **i32),
            "max_q": max(qs), "max_kv": max(1, max(kvs))}


# --------------------------------------------------------------- plain form
def _plain_norm(s):
    c = s["case"]
    h = s["x"].float()
    if s["residual"] is not None:
        h = h + s["residual"].float()
    y = h * torch.rsqrt((h * h).mean(dim=-1, keepdim=True) + EPS)
    y = y * (s["weight"].float() + c["weight_bias"])
    out = {}
    if s["residual"] is not None:
        out["residual"] = s["residual_out"].copy_(h)
    if c["fp8"]:
        groups = y.view(c["rows"], c["hidden"] // 128, 128)
        scale = (groups.abs().amax(dim=-1) / 448.0).clamp(min=1e-8)
        q = (groups / scale[..., None]).clamp(-448.0, 448.0)
        out["q"] = q.view(c["rows"], c["hidden"]).to(torch.float8_e4m3fn)
        out["scales"] = scale.t().contiguous()
    else:
        out["y"] = y.to(s["x"].dtype)
    return out


def _plain_quantize(x):
    """(e4m3 codes, scale bytes) of the vectors along the last axis."""
    x = x.float()
    top = x.abs().amax(dim=-1)
    mantissa, exponent = torch.frexp(top)  # top = mantissa * 2^exponent, mantissa in [0.5, 1)
    e = torch.where(mantissa <= 0.875, exponent - 9, exponent - 8)  # 448 = 0.875 * 2^9
    e = torch.where(top > 0, e, torch.full_like(e, -24)).clamp(-24, 7)
    codes = torch.ldexp(x, -e[..., None]).clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
    return codes, (e + 127).to(torch.uint8)


def _plain_values(cache, scale, page, offset):
    """fp32 values of the cached tokens (page, offset): [..., heads, dim]."""
    if scale is None:
        return cache[page, offset].float()
    codes = cache.view(torch.uint8)[page, offset].view(torch.float8_e4m3fn).float()
    return torch.ldexp(codes, scale[page, offset].to(torch.int32)[..., None] - 127)


def _plain_cache(s):
    c, (kc, vc, ks, vs) = s["case"], s["cache"]
    page, offset = s["slots"] // c["page"], s["slots"] % c["page"]
    out = {}
    for name, x, cache, scale in (("k", s["k"], kc, ks), ("v", s["v"], vc, vs)):
        if scale is None:
            cache[page, offset] = x
        else:
            codes, e = _plain_quantize(x)
            cache.view(torch.uint8)[page, offset] = codes.view(torch.uint8)
            scale[page, offset] = e
            out[name + "_scale"] = scale
        out[name + "_cache"] = cache
        out[name] = _plain_values(cache, scale, page, offset).to(x.dtype)
    return out


def _plain_attention(s):
    c, (kc, vc, ks, vs) = s["case"], s["cache"]
    heads, groups, dim, seqs = c["heads"], c["groups"], c["dim"], c["seqs"]
    lens, starts = s["kv_lens"].long(), s["q_starts"].long()
    at = torch.arange(s["max_kv"], device="cuda")
    page, offset = s["table"].long()[:, at // c["page"]], at % c["page"]
    there = at[None, :] < lens[:, None]
    k = _plain_values(kc, ks, page, offset).permute(0, 2, 3, 1)  # [seqs, heads, dim, kv]
    v = _plain_values(vc, vs, page, offset).permute(0, 2, 1, 3)
    v = torch.where(there[:, None, :, None], v, torch.zeros((), device="cuda"))
    new = torch.arange(s["max_q"], device="cuda")
    q = s["q"].float()[(starts[:-1, None] + new).clamp(max=s["q"].shape[0] - 1)]
    q = q.view(seqs, -1, heads, groups, dim).permute(0, 2, 3, 1, 4)
    score = torch.matmul(q.reshape(seqs, heads, -1, dim), k) * dim ** -0.5
    score = score.view(seqs, heads, groups, -1, s["max_kv"])
    seen = there[:, None, :].expand(-1, s["max_q"], -1)
    if c["causal"]:
        where = (lens - (starts[1:] - starts[:-1]))[:, None] + new  # each new token's position
        seen = seen & (at <= where[:, :, None])
        if c["window"]:
            seen = seen & (at > where[:, :, None] - c["window"])
    score = score.masked_fill_(~seen[:, None, None], -math.inf)
    top = score.amax(dim=-1, keepdim=True)
    top = torch.where(top > -math.inf, top, torch.zeros_like(top))
    p = score.sub_(top).exp_()
    total = p.sum(dim=-1, keepdim=True)
    o = torch.matmul(p.view(seqs, heads, -1, s["max_kv"]), v).view(seqs, heads, groups, -1, dim)
    o = torch.where(total > 0, o / total, torch.zeros_like(o))
    lse = (total.log() + top).squeeze(-1)  # -inf where nothing is seen
    token = torch.arange(s["q"].shape[0], device="cuda")
    seq = torch.searchsorted(starts[1:], token, right=True)
    row = token - starts[seq]
    o = o.permute(0, 3, 1, 2, 4)[seq, row].reshape(-1, heads * groups, dim)
    return {"out": o.to(s["q"].dtype),
            "lse": lse.permute(0, 3, 1, 2)[seq, row].reshape(-1, heads * groups)}


# ---------------------------------------------------------------------- run
def run(state):
    c = state["case"]
    if not own:
        return {"norm": _plain_norm, "cache": _plain_cache, "attention": _plain_attention}[c["op"]](state)
    ops, kv_cache = _library()
    if c["op"] == "norm":
        if c["fp8"]:
            q, scales, residual = ops.add_rms_norm_fp8(
                state["x"], state["weight"], EPS, residual=state["residual"],
                weight_bias=c["weight_bias"], residual_out=state["residual_out"])
            out = {"q": q, "scales": scales}
        else:
            y, residual = ops.add_rms_norm(
                state["x"], state["weight"], EPS, residual=state["residual"],
                weight_bias=c["weight_bias"], residual_out=state["residual_out"])
            out = {"y": y}
        if residual is not None:
            out["residual"] = residual
        return out
    if "handle" not in state:  # the cache object that a serving loop keeps
        state["handle"] = kv_cache.PagedKVCache(*state["cache"])
    cache = state["handle"]
    if c["op"] == "cache":
        ops.kv_cache_write(cache, state["k"], state["v"], state["slots"])
        k, v = ops.kv_cache_read(cache, state["slots"], state["k"].dtype)
        out = {"k": k, "v": v, "k_cache": cache.k, "v_cache": cache.v}
        if c["fp8"]:
            out["k_scale"], out["v_scale"] = cache.k_scale, cache.v_scale
        return out
    out, lse = ops.paged_attention(state["q"], cache, state["table"], state["kv_lens"],
                                   state["q_starts"], state["max_q"], causal=c["causal"],
                                   window=c["window"], return_lse=True)
    return {"out": out, "lse": lse}


# --------------------------------------------------------------------- work
def work(case):
    if case["op"] == "norm":
        n = case["rows"] * case["hidden"]
        b = 2 * n + 2 * case["hidden"] + (4 * n if case["residual"] else 0)
        b += n + 4 * (n // 128) if case["fp8"] else 2 * n
        return {"bytes": b, "flops": 6 * n}
    vector = case["dim"] + 1 if case["fp8"] else 2 * case["dim"]  # a cached key or value
    if case["op"] == "cache":
        n = 2 * case["tokens"] * case["heads"]
        return {"bytes": n * (4 * case["dim"] + 2 * vector) + 16 * case["tokens"],
                "flops": 2 * n * case["dim"]}
    qs, kvs = _lens(case)
    h = case["heads"] * case["groups"]
    pairs = read = 0
    for q, kv in zip(qs, kvs):
        if not kv:
            continue
        if not case["causal"]:
            pairs, read = pairs + q * kv, read + kv
            continue
        w = case["window"] or kv
        first = kv - q  # position of the first new token; position p sees min(p + 1, w) tokens
        short = max(0, min(q, w - 1 - first))  # new tokens that see all that is before them
        pairs += short * (first + 1) + short * (short - 1) // 2 + (q - short) * w
        read += min(kv, q - 1 + w)
    b = 2 * read * case["heads"] * vector + sum(qs) * h * (4 * case["dim"] + 4)
    b += 4 * sum(-(-n // case["page"]) for n in kvs) + 8 * case["seqs"]
    return {"bytes": b, "flops": 4 * pairs * h * case["dim"]}


# -------------------------------------------------------------------- exact
def _exact_vectors(cache, scale, page, offset):
    if scale is None:
        return cache[page, offset].double()
    codes = cache.view(torch.uint8)[page, offset].view(torch.float8_e4m3fn).double()
    return codes * torch.pow(2.0, scale[page, offset].double() - 127.0)[..., None]


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        h = s["x"].double() + (s["residual"].double() if case["residual"] else 0.0)
        y = h / torch.sqrt(h.pow(2).sum(-1, keepdim=True) / case["hidden"] + EPS)
        y = y * (s["weight"].double() + case["weight_bias"])
        out = {"residual": h} if case["residual"] else {}
        if not case["fp8"]:
            return {**out, "y": y}
        scales = torch.clamp_min(y.reshape(case["rows"], -1, 128).abs().max(-1).values / 448, 1e-8)
        return {**out, "q": y / scales.repeat_interleave(128, -1), "scales": scales.T.contiguous()}
    if case["op"] == "cache":
        out = {}
        page, offset = s["slots"] // case["page"], s["slots"] % case["page"]
        for name, cache in (("k", s["cache"][0]), ("v", s["cache"][1])):
            x = s[name].double()
            full = torch.zeros(cache.shape, dtype=torch.float64, device="cuda")
            if case["fp8"]:
                # a largest magnitude of exactly 448 * 2^e keeps e: the margin is far
                # below the spacing of 16-bit values and far above log2's rounding
                e = torch.log2(x.abs().max(-1, keepdim=True).values / 448)
                e = torch.ceil(e - 1e-9).clamp(-24, 7)
                full[page, offset] = x / torch.pow(2.0, e)
                out[name + "_scale"] = None
            else:
                full[page, offset] = x
            out[name], out[name + "_cache"] = x, full
        return out
    heads, groups, dim = case["heads"], case["groups"], case["dim"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.full(s["q"].shape[:2], -math.inf, dtype=torch.float64, device="cuda")
    qs, kvs = _lens(case)
    first = 0
    for i, (nq, nk) in enumerate(zip(qs, kvs)):
        at = torch.arange(nk, device="cuda")
        page, offset = s["table"][i].long()[at // case["page"]], at % case["page"]
        if nk:
            k = _exact_vectors(s["cache"][0], s["cache"][2], page, offset)
            v = _exact_vectors(s["cache"][1], s["cache"][3], page, offset)
            pos = nk - nq + torch.arange(nq, device="cuda")[:, None]
            hide = torch.zeros(nq, nk, dtype=torch.bool, device="cuda")
            if case["causal"]:
                hide |= at > pos
                if case["window"]:
                    hide |= at <= pos - case["window"]
            for h in range(heads * groups):
                q = s["q"][first:first + nq, h].double()
                x = (q @ k[:, h // groups].T / math.sqrt(dim)).masked_fill(hide, -math.inf)
                lse[first:first + nq, h] = torch.logsumexp(x, -1)
                out[first:first + nq, h] = torch.softmax(x, -1) @ v[:, h // groups]
        first += nq
    return {"out": out, "lse": lse}
