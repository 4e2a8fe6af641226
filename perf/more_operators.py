"""Measured cases of serving operators around the paged key/value cache: the
8-bit integer linear (a scale per token and per output channel), attention of a
batch whose sequences share a long prefix, the accumulated attention weight of
cached tokens, and the eviction of cached tokens by it.

``own`` chooses between the plain form (elementary torch operations in fp32,
rounded once at the end) and the library's own entry points. ``listed`` gives
the fixed cases, ``draw`` more of the same ranges, ``prepare`` what a serving
loop has in hand before the call, ``run`` one pass, ``work`` the bytes and
operations a pass cannot do without, and ``exact`` the definition in 64 bits.

The linear quantizes a token's row x by the scale s = max|x| / 127 to the whole
numbers rint(x / s), multiplies them by the weight's in whole numbers and the sum
by both scales. The quantized cache is that of ``operators.py``: e4m3 codes, and a
byte 127 + e per vector for the power of two they are multiplied by.
"""

import math
import random
import sys
from pathlib import Path

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


def _library():
    root = str(Path(__file__).resolve().parents[1] / "sglang-restomod_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    from sglang_restomod_b200 import kv_cache, ops

    return ops, kv_cache


# ------------------------------------------------------------------- cases
def _linear(name, tokens, out, inner, dtype):
    return {"name": name, "op": "linear", "tokens": tokens, "out": out, "inner": inner,
            "dtype": dtype}


def _prefix(name, seqs, q, kv, prefix, sharing, heads, groups, dim, page, dtype, fp8, *,
            bare=False, lens_seed=1):
    return {"name": name, "op": "prefix", "seqs": seqs, "q": q, "kv": kv, "prefix": prefix,
            "sharing": sharing, "heads": heads, "groups": groups, "dim": dim, "page": page,
            "dtype": dtype, "fp8": fp8, "bare": bare, "lens_seed": lens_seed}


def _scores(name, seqs, q, kv, heads, groups, dim, page, dtype, fp8, *, window=0, empty=0,
            lens_seed=1):
    return {"name": name, "op": "scores", "seqs": seqs, "q": q, "kv": kv, "heads": heads,
            "groups": groups, "dim": dim, "page": page, "dtype": dtype, "fp8": fp8,
            "window": window, "empty": empty, "lens_seed": lens_seed}


def _evict(name, seqs, kv, budget, recent, first, heads, dim, page, dtype, fp8, *, lens_seed=1):
    return {"name": name, "op": "evict", "seqs": seqs, "kv": kv, "budget": budget,
            "recent": recent, "first": first, "heads": heads, "dim": dim, "page": page,
            "dtype": dtype, "fp8": fp8, "lens_seed": lens_seed}


def listed():
    return [
        # one decoded token through a wide down projection: the weight's bytes
        _linear("linear 1 token 5120x25600", 1, 5120, 25600, "bf16"),
        # a decode batch of odd size, f16, an output width of no tile's multiple
        _linear("linear 77 tokens 7164x2048 f16", 77, 7164, 2048, "f16"),
        # a long prefill batch: the tensor cores' rate
        _linear("linear 8192 tokens 7168x4096", 8192, 7168, 4096, "bf16"),
        # four users in the first tokens of their answers on one short system prompt: latency
        _prefix("prefix 4 on 515", 4, 1, 60, 515, 4, 8, 4, 128, 16, "bf16", False),
        # a serving batch on one long document, quantized cache, uneven answers
        _prefix("prefix 64 on 8192 fp8", 64, 1, 1024, 8192, 64, 8, 8, 128, 64, "bf16", True),
        # questions of up to 300 tokens on three prompts of different lengths, f16,
        # three queries a head, single-token pages, and sequences that share nothing
        _prefix("prefix 16x300 on 4000 f16", 16, 300, 900, 4000, 6, 8, 3, 64, 1, "f16", False,
                bare=True),
        # a decode step's weights over a serving batch's uneven quantized contexts
        _scores("scores 64x8192 fp8", 64, 1, 8192, 8, 8, 128, 64, "bf16", True),
        # a whole prompt's weights
        _scores("scores prompt 8192", 1, 8192, 8192, 8, 4, 128, 64, "bf16", False),
        # mixed chunks, f16, three queries a head, a window, single-token pages, two idle slots
        _scores("scores 16x300 f16 window", 16, 300, 4096, 8, 3, 64, 1, "f16", False, window=1000,
                empty=2),
        # one user's context cut to half: latency of the choice
        _evict("evict 1x4099 to 2048", 1, 4099, 2048, 64, 4, 8, 128, 16, "bf16", False),
        # a serving batch's quantized contexts cut to 1024 tokens
        _evict("evict 64x8192 to 1024 fp8", 64, 8192, 1024, 128, 4, 8, 128, 64, "bf16", True),
        # long contexts, wide heads, two key/value heads
        _evict("evict 8x65536 to 16384 d256", 8, 65536, 16384, 1000, 0, 2, 256, 16, "bf16", False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["linear", "prefix", "prefix", "scores", "evict"])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    seed = rng.randint(1, 1 << 20)
    if op == "linear":
        inner = 16 * _log(rng, 4, 1600)
        out = _log(rng, 32, 5120 * 25600 // inner if inner > 5120 else 25600)
        tokens = _log(rng, 1, max(1, min(32768, 8192 * 7168 * 4096 // (inner * out))))
        c = _linear("", tokens, out, inner, dtype)
    else:
        dim = rng.choice([64, 128, 128, 256])
        heads = rng.choice([1, 2, 4, 8])
        groups = rng.choice([1, 2, 3, 4, 6, 8, 16])
        page = rng.choice([1, 16, 24, 64, 128])
        fp8 = rng.random() < 0.5
        if op == "prefix":
            q = 1 if rng.random() < 0.6 else _log(rng, 2, 500)
            kv = q + _log(rng, 1, 2048)
            prefix = _log(rng, 16, 16384)
            # no more than the largest listed case's operations, keys and values
            most = min(128, 16 * 300 * 24 * 64 * 5000 * 4 // (heads * groups * dim * q * (prefix + kv)),
                       64 * 9216 * 8 * 128 // (heads * dim * (prefix + kv)))
            seqs = _log(rng, 1, max(1, most))
            c = _prefix("", seqs, q, kv, prefix, rng.randint(1, seqs), heads, groups, dim, page,
                        dtype, fp8, bare=rng.random() < 0.2, lens_seed=seed)
        elif op == "scores":
            q = 1 if rng.random() < 0.5 else _log(rng, 2, 4096)
            kv = q + _log(rng, 1, 32768)
            most = min(64, 8192 * 8192 * 32 // (2 * heads * groups * q * kv),
                       64 * 8192 * 8 * 128 // (2 * heads * dim * kv))
            if most < 1:
                kv = max(q, 8192 * 8192 * 16 // (heads * groups * q))
            seqs = _log(rng, 1, max(1, most))
            c = _scores("", seqs, q, kv, heads, groups, dim, page, dtype, fp8,
                        window=_log(rng, 16, 4096) if rng.random() < 0.25 else 0,
                        empty=rng.randint(0, 2) if seqs > 4 else 0, lens_seed=seed)
        else:
            kv = _log(rng, 64, 65536)
            budget = _log(rng, 16, kv)
            recent = rng.randint(0, budget // 2)
            most = min(64, 8 * 65536 * 2 * 256 // (heads * dim * kv))
            c = _evict("", _log(rng, 1, max(1, most)), kv, budget, recent,
                       rng.randint(0, min(8, budget - recent)), heads, dim, page, dtype, fp8,
                       lens_seed=seed)
    del c["name"]
    largest = [work(x) for x in listed()]
    if any(work(c)[what] > max(w[what] for w in largest) for what in ("bytes", "flops")):
        return draw(rng)
    return c


def _lens(c):
    """(new tokens, cached tokens) of each sequence; the new ones are the last
    of the cached ones. The first sequence has the largest of both, and an
    idle slot has one new token and nothing cached."""
    rng = random.Random(c["lens_seed"])
    qs, kvs = [], []
    for i in range(c["seqs"]):
        q, kv = c.get("q", 1), c["kv"]
        if i:
            q = rng.randint(1, q)
            kv = rng.randint(q, kv)
        if i and i >= c["seqs"] - c.get("empty", 0):
            q, kv = 1, 0
        qs.append(q)
        kvs.append(kv)
    return qs, kvs


def _sharing(c):
    """(first sequence of each group, and the end; each group's prefix length)."""
    rng = random.Random(c["lens_seed"] + 1)
    starts, lens = [0], []
    while starts[-1] < c["seqs"]:
        lens.append(c["prefix"] if not lens else rng.randint(max(1, c["prefix"] // 4), c["prefix"]))
        starts.append(min(c["seqs"], starts[-1] + c["sharing"]))
    if c["bare"] and len(lens) > 1:
        lens[-1] = 0
    return starts, lens


# ----------------------------------------------------------------- prepare
def _randn(g, *shape, dtype, scale=1.0, step=1 << 27):
    """Seeded normal values, made in pieces so that the fp32 they pass through stays small."""
    out = torch.empty(*shape, dtype=dtype, device="cuda")
    flat = out.view(-1)
    for a in range(0, flat.numel(), step):
        b = min(a + step, flat.numel())
        flat[a:b] = torch.randn(b - a, generator=g, device="cuda").mul_(scale).to(dtype)
    return out


def _quantized(x):
    """(e4m3 codes, scale bytes) of the vectors along the last axis."""
    x = x.float()
    top = x.abs().amax(dim=-1)
    mantissa, exponent = torch.frexp(top)
    e = torch.where(mantissa <= 0.875, exponent - 9, exponent - 8)
    e = torch.where(top > 0, e, torch.full_like(e, -24)).clamp(-24, 7)
    codes = torch.ldexp(x, -e[..., None]).clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
    return codes, (e + 127).to(torch.uint8)


def _cache(g, c, pages):
    heads, dim, page, dt = c["heads"], c["dim"], c["page"], DTYPES[c["dtype"]]
    kv, sc = [], []
    for _ in range(2):
        raw = _randn(g, pages, heads, page, dim, dtype=dt)
        if not c["fp8"]:
            kv.append(raw.transpose(1, 2))
            sc.append(None)
            continue
        codes = torch.empty(raw.shape, dtype=torch.uint8, device="cuda")
        scale = torch.empty(raw.shape[:-1], dtype=torch.uint8, device="cuda")
        step = max(1, (1 << 27) // (heads * page * dim))
        for a in range(0, pages, step):
            q8, sb = _quantized(raw[a:a + step])
            codes[a:a + step] = q8.view(torch.uint8)
            scale[a:a + step] = sb
        kv.append(codes.view(torch.float8_e4m3fn).transpose(1, 2))
        sc.append(scale.transpose(1, 2))
        del raw
    return kv[0], kv[1], sc[0], sc[1]


def _table(order, need):
    """Page tables of rows of `need` pages each, taken from `order` in turn."""
    width = max(1, max(need))
    rows = torch.arange(width)[None, :] < torch.tensor(need)[:, None]
    table = torch.zeros(len(need), width, dtype=torch.int32)
    table[rows] = torch.arange(sum(need), dtype=torch.int32)
    rows = rows.cuda()
    return torch.where(rows, order[table.cuda().long()], torch.zeros_like(table).cuda())


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    i32 = dict(dtype=torch.int32, device="cuda")
    if case["op"] == "linear":
        tokens, out, inner = case["tokens"], case["out"], case["inner"]
        # activations with a few large channels; a weight's rows use the whole range
        spread = torch.exp(0.5 * torch.randn(inner, generator=g, device="cuda"))
        x = (torch.randn(tokens, inner, generator=g, device="cuda") * spread).to(dt)
        w = torch.randint(-127, 128, (out, inner), generator=g, device="cuda", dtype=torch.int8)
        ws = (0.5 + torch.rand(out, generator=g, device="cuda")) * 0.03 / 127
        return {"case": case, "x": x, "w": w, "w_scales": ws}
    heads, dim, page = case["heads"], case["dim"], case["page"]
    qs, kvs = _lens(case)
    need = [-(-n // page) for n in kvs]
    if case["op"] == "evict":
        budget = case["budget"]
        to = [-(-min(n, budget) // page) for n in kvs]
        pages = sum(need) + sum(to) + 2
        order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
        # weights as they accumulate: a few tokens have most of them, many next to none
        scores = torch.exp(3.0 * torch.randn(pages, heads, page, generator=g, device="cuda"))
        scores = torch.where(scores < 0.05, torch.zeros_like(scores), scores).transpose(1, 2)
        return {"case": case, "cache": _cache(g, case, pages), "scores": scores,
                "table": _table(order, need), "out_table": _table(order[sum(need):], to),
                "kv_lens": torch.tensor(kvs, **i32), "max_kv": max(kvs)}
    starts = [0]
    for n in qs:
        starts.append(starts[-1] + n)
    s = {"case": case, "kv_lens": torch.tensor(kvs, **i32), "q_starts": torch.tensor(starts, **i32),
         "max_q": max(qs), "max_kv": max(1, max(kvs))}
    shape = (starts[-1], heads * case["groups"], dim)
    s["q"] = _randn(g, *shape, dtype=dt, scale=1.5)
    if case["op"] == "prefix":
        group_starts, lens = _sharing(case)
        shared = [-(-n // page) for n in lens]
        pages = sum(need) + sum(shared) + 2
        order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
        s.update(cache=_cache(g, case, pages), table=_table(order, need),
                 prefix_table=_table(order[sum(need):], shared),
                 prefix_lens=torch.tensor(lens, **i32), max_prefix=max(lens),
                 group_starts=torch.tensor(group_starts, **i32))
        return s
    pages = sum(need) + 2
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    s.update(cache=_cache(g, case, pages), table=_table(order, need))
    scores = torch.rand(pages, heads, page, generator=g, device="cuda")
    # the attention call before left each query's log-sum-exp; the scores' new
    # values go to the other of two buffers
    s.update(scores=scores.transpose(1, 2), out=torch.zeros_like(scores).transpose(1, 2))
    s["lse"] = _plain_attention(s)["lse"]
    return s


# --------------------------------------------------------------- plain form
def _plain_linear(s):
    x = s["x"].float()
    scale = x.abs().amax(dim=-1, keepdim=True) / 127.0
    q = torch.round(x / torch.where(scale > 0, scale, torch.ones_like(scale))).clamp(-127.0, 127.0)
    y = torch.matmul(q, s["w"].float().t()) * scale * s["w_scales"]
    return {"y": y.to(s["x"].dtype)}


def _plain_values(cache, scale, page, offset):
    """fp32 values of the cached tokens (page, offset): [..., heads, dim]."""
    if scale is None:
        return cache[page, offset].float()
    codes = cache.view(torch.uint8)[page, offset].view(torch.float8_e4m3fn).float()
    return torch.ldexp(codes, scale[page, offset].to(torch.int32)[..., None] - 127)


def _plain_weights(s):
    """Scores [seqs, heads, groups, new, keys] of the new tokens, -inf where nothing is
    seen, and where the keys lie: (page, offset, there) [seqs, keys]. The keys are the
    prefix's, if there is one, and the sequence's own."""
    c, seqs = s["case"], s["case"]["seqs"]
    lens, starts = s["kv_lens"].long(), s["q_starts"].long()
    at = torch.arange(s["max_kv"], device="cuda")
    page, offset = s["table"].long()[:, at // c["page"]], (at % c["page"]).expand(seqs, -1)
    there = at[None, :] < lens[:, None]
    new = torch.arange(s["max_q"], device="cuda")
    where = (lens - (starts[1:] - starts[:-1]))[:, None] + new  # each new token's position
    seen = there[:, None, :] & (at <= where[:, :, None])
    if c.get("window"):
        seen = seen & (at > where[:, :, None] - c["window"])
    if "prefix_table" in s:
        group = torch.searchsorted(s["group_starts"][1:], torch.arange(seqs, device="cuda"), right=True)
        far = torch.arange(s["max_prefix"], device="cuda")
        has = far[None, :] < s["prefix_lens"].long()[group][:, None]
        page = torch.cat([s["prefix_table"].long()[group][:, far // c["page"]], page], dim=1)
        offset = torch.cat([(far % c["page"]).expand(seqs, -1), offset], dim=1)
        there = torch.cat([has, there], dim=1)
        seen = torch.cat([has[:, None, :].expand(-1, s["max_q"], -1), seen], dim=2)
    k = _plain_values(s["cache"][0], s["cache"][2], page, offset).permute(0, 2, 3, 1)
    q = s["q"].float()[(starts[:-1, None] + new).clamp(max=s["q"].shape[0] - 1)]
    q = q.view(seqs, -1, c["heads"], c["groups"], c["dim"]).permute(0, 2, 3, 1, 4)
    score = torch.matmul(q.reshape(seqs, c["heads"], -1, c["dim"]), k) * c["dim"] ** -0.5
    score = score.view(seqs, c["heads"], c["groups"], s["max_q"], -1)
    return score.masked_fill_(~seen[:, None, None], -math.inf), page, offset, there


def _plain_attention(s):
    c, (kc, vc, ks, vs) = s["case"], s["cache"]
    score, page, offset, there = _plain_weights(s)
    v = _plain_values(vc, vs, page, offset).permute(0, 2, 1, 3)
    v = torch.where(there[:, None, :, None], v, torch.zeros((), device="cuda"))
    top = score.amax(dim=-1, keepdim=True)
    top = torch.where(top > -math.inf, top, torch.zeros_like(top))
    p = score.sub_(top).exp_()
    total = p.sum(dim=-1, keepdim=True)
    o = torch.matmul(p.view(c["seqs"], c["heads"], -1, p.shape[-1]), v)
    o = o.view(c["seqs"], c["heads"], c["groups"], -1, c["dim"])
    o = torch.where(total > 0, o / total, torch.zeros_like(o))
    lse = (total.log() + top).squeeze(-1)  # -inf where nothing is seen
    starts = s["q_starts"].long()
    token = torch.arange(s["q"].shape[0], device="cuda")
    seq = torch.searchsorted(starts[1:], token, right=True)
    row = token - starts[seq]
    o = o.permute(0, 3, 1, 2, 4)[seq, row].reshape(s["q"].shape)
    return {"out": o.to(s["q"].dtype),
            "lse": lse.permute(0, 3, 1, 2)[seq, row].reshape(s["q"].shape[:2])}


def _plain_scores(s):
    c = s["case"]
    score, page, offset, there = _plain_weights(s)
    starts, lens = s["q_starts"].long(), s["kv_lens"].long()
    count = starts[1:] - starts[:-1]
    new = torch.arange(s["max_q"], device="cuda")
    lse = s["lse"][(starts[:-1, None] + new).clamp(max=s["q"].shape[0] - 1)]
    lse = lse.masked_fill((lse == -math.inf) | (new >= count[:, None])[:, :, None], math.inf)
    lse = lse.view(c["seqs"], -1, c["heads"], c["groups"]).permute(0, 2, 3, 1)
    weight = score.sub_(lse[..., None]).exp_().sum(dim=(2, 3))  # [seqs, heads, keys]
    old = s["scores"][page, offset].permute(0, 2, 1)  # of tokens that were there before
    before = torch.arange(s["max_kv"], device="cuda") < (lens - count)[:, None]
    weight = weight + torch.where(before[:, None], old, torch.zeros_like(old))
    s["out"][page[there], offset[there]] = weight.permute(0, 2, 1)[there]
    return {"scores": s["out"]}


def _plain_evict(s):
    c, budget, lens = s["case"], s["case"]["budget"], s["kv_lens"].long()
    at = torch.arange(s["max_kv"], device="cuda")
    page, offset = s["table"].long()[:, at // c["page"]], at % c["page"]
    score = s["scores"][page, offset].permute(0, 2, 1)  # [seqs, heads, keys]
    kept = (at < c["first"]) | (at >= lens[:, None] - c["recent"])
    score = torch.where(kept[:, None], torch.full_like(score, math.inf), score)
    score = torch.where((at < lens[:, None])[:, None], score, torch.full_like(score, -math.inf))
    best = torch.argsort(score, dim=-1, descending=True, stable=True)[..., :budget]
    new = lens.clamp(max=budget)
    to = torch.arange(best.shape[-1], device="cuda")
    there = to < new[:, None]
    best = torch.where(there[:, None], best, torch.full_like(best, s["max_kv"])).sort(dim=-1).values
    ids = torch.full((c["seqs"], c["heads"], budget), -1, dtype=torch.int32, device="cuda")
    ids[..., :best.shape[-1]] = torch.where(there[:, None], best, torch.full_like(best, -1))
    from_token = best.clamp(max=s["max_kv"] - 1).transpose(1, 2)[there]  # [moved, heads]
    seq = torch.arange(c["seqs"], device="cuda")[:, None].expand_as(there)[there]
    head = torch.arange(c["heads"], device="cuda")
    to_page = s["out_table"].long()[:, to // c["page"]][there]
    to_offset = (to % c["page"]).expand_as(there)[there]
    page = s["table"].long()[seq[:, None], from_token // c["page"]]
    offset = from_token % c["page"]
    for x in (*s["cache"], s["scores"]):
        if x is not None:
            x = x.view(torch.uint8) if x.dtype == torch.float8_e4m3fn else x
            x[to_page, to_offset] = x[page, offset, head]
    return _evicted(s, ids, new.to(torch.int32))


def _evicted(s, kept, lens):
    out = {"kept": kept, "lens": lens, "k": s["cache"][0], "v": s["cache"][1], "scores": s["scores"]}
    if s["case"]["fp8"]:
        out["k_scale"], out["v_scale"] = s["cache"][2], s["cache"][3]
    return out


# ---------------------------------------------------------------------- run
def run(state):
    c = state["case"]
    if not own:
        return {"linear": _plain_linear, "prefix": _plain_attention, "scores": _plain_scores,
                "evict": _plain_evict}[c["op"]](state)
    ops, kv_cache = _library()
    if c["op"] == "linear":
        return {"y": ops.int8_linear(state["x"], state["w"], state["w_scales"])}
    if "handle" not in state:  # the cache object that a serving loop keeps
        state["handle"] = kv_cache.PagedKVCache(*state["cache"])
    cache = state["handle"]
    if c["op"] == "prefix":
        out, lse = ops.shared_prefix_attention(
            state["q"], cache, state["prefix_table"], state["prefix_lens"], state["group_starts"],
            state["table"], state["kv_lens"], state["q_starts"], state["max_q"], return_lse=True)
        return {"out": out, "lse": lse}
    if c["op"] == "scores":
        return {"scores": ops.kv_cache_scores(
            state["q"], cache, state["table"], state["kv_lens"], state["q_starts"], state["max_q"],
            state["lse"], state["scores"], window=c["window"], out=state["out"])}
    kept, lens = ops.kv_cache_evict(cache, state["scores"], state["table"], state["kv_lens"],
                                    c["budget"], recent=c["recent"], first=c["first"],
                                    out_table=state["out_table"])
    return _evicted(state, kept, lens)


# --------------------------------------------------------------------- work
def work(case):
    if case["op"] == "linear":
        m, n, k = case["tokens"], case["out"], case["inner"]
        return {"bytes": 2 * m * k + n * k + 4 * n + 2 * m * n, "flops": 2 * m * n * k}
    vector = case["dim"] + 1 if case["fp8"] else 2 * case["dim"]  # a cached key or value
    heads = case["heads"]
    qs, kvs = _lens(case)
    tables = 4 * sum(-(-n // case["page"]) for n in kvs) + 8 * case["seqs"]
    if case["op"] == "evict":
        moved = heads * sum(min(n, case["budget"]) for n in kvs)
        b = 4 * heads * sum(kvs) + moved * (2 * 2 * vector + 4 + 4) + tables
        return {"bytes": b, "flops": heads * sum(kvs)}
    h = heads * case["groups"]
    pairs = read = 0
    for q, kv in zip(qs, kvs):
        if not kv:
            continue
        w = case.get("window") or kv
        first = kv - q  # position of the first new token; position p sees min(p + 1, w) tokens
        short = max(0, min(q, w - 1 - first))  # new tokens that see all that is before them
        pairs += short * (first + 1) + short * (short - 1) // 2 + (q - short) * w
        read += min(kv, q - 1 + w)
    if case["op"] == "scores":
        b = read * heads * vector + sum(qs) * h * (2 * case["dim"] + 4) + 8 * heads * sum(kvs)
        return {"bytes": b + tables, "flops": 2 * pairs * h * case["dim"]}
    starts, lens = _sharing(case)
    for g, n in enumerate(lens):
        pairs += n * sum(qs[starts[g]:starts[g + 1]])
    read += sum(lens)
    tables += 4 * sum(-(-n // case["page"]) for n in lens) + 8 * len(lens)
    b = 2 * read * heads * vector + sum(qs) * h * (4 * case["dim"] + 4)
    return {"bytes": b + tables, "flops": 4 * pairs * h * case["dim"]}


# -------------------------------------------------------------------- exact
def _exact_vectors(cache, scale, page, offset):
    if scale is None:
        return cache[page, offset].double()
    codes = cache.view(torch.uint8)[page, offset].view(torch.float8_e4m3fn).double()
    return codes * torch.pow(2.0, scale[page, offset].double() - 127.0)[..., None]


def _exact_keys(s, i, n, table="table"):
    at = torch.arange(n, device="cuda")
    return s[table][i].long()[at // s["case"]["page"]], at % s["case"]["page"]


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "linear":
        x = s["x"].double()
        scale = x.abs().max(-1, keepdim=True).values / 127
        q = torch.where(scale > 0, x / scale, 0.0).round()
        return {"y": (q @ s["w"].double().T) * scale * s["w_scales"].double()}
    qs, kvs = _lens(case)
    heads = case["heads"]
    if case["op"] == "evict":
        # nothing is computed but the choice: each row's own order, by (weight, index)
        for i, n in enumerate(kvs):
            m = min(n, case["budget"])
            page, offset = _exact_keys(s, i, n)
            to_page, to_offset = _exact_keys(s, i, m, "out_table")
            late = n - case["recent"]
            for h in range(heads):
                value = s["scores"][page, offset, h].double()
                value[:case["first"]] = math.inf
                value[max(0, late):] = math.inf
                ids = torch.sort(torch.sort(-value, stable=True).indices[:m]).values
                for x in (*s["cache"], s["scores"]):
                    if x is not None:
                        x = x.view(torch.uint8) if x.dtype == torch.float8_e4m3fn else x
                        x[to_page, to_offset, h] = x[page[ids], offset[ids], h]
        return {"kept": None, "lens": None, "k": s["cache"][0].double(), "v": s["cache"][1].double(),
                "scores": s["scores"].double(),
                **({"k_scale": None, "v_scale": None} if case["fp8"] else {})}
    groups, dim = case["groups"], case["dim"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.full(s["q"].shape[:2], -math.inf, dtype=torch.float64, device="cuda")
    scores = s["out"].double() if case["op"] == "scores" else None
    starts, lens = _sharing(case) if case["op"] == "prefix" else ([0, case["seqs"]], [0])
    first = group = 0
    for i, (nq, nk) in enumerate(zip(qs, kvs)):
        while i >= starts[group + 1]:
            group += 1
        page, offset = _exact_keys(s, i, nk)
        at = torch.arange(nk, device="cuda")
        if lens[group]:
            more = _exact_keys(s, group, lens[group], "prefix_table")
            page, offset = torch.cat([more[0], page]), torch.cat([more[1], offset])
            at = torch.cat([torch.full((lens[group],), -1, device="cuda"), at])
        if len(page):
            k = _exact_vectors(s["cache"][0], s["cache"][2], page, offset)
            pos = nk - nq + torch.arange(nq, device="cuda")[:, None]
            hide = at > pos
            if case.get("window"):
                hide = hide | (at <= pos - case["window"])
            v = None if scores is not None else _exact_vectors(s["cache"][1], s["cache"][3], page, offset)
            if scores is not None:
                was = s["scores"][page, offset].double()
                was[max(0, nk - nq):] = 0.0
            for h in range(heads * groups):
                q = s["q"][first:first + nq, h].double()
                x = (q @ k[:, h // groups].T / math.sqrt(dim)).masked_fill(hide, -math.inf)
                if scores is None:
                    lse[first:first + nq, h] = torch.logsumexp(x, -1)
                    out[first:first + nq, h] = torch.softmax(x, -1) @ v[:, h // groups]
                else:
                    z = s["lse"][first:first + nq, h].double()
                    z = torch.where(z > -math.inf, z, math.inf)
                    was[:, h // groups] += torch.exp(x - z[:, None]).sum(0)
            if scores is not None:
                scores[page, offset] = was
        first += nq
    return {"scores": scores} if scores is not None else {"out": out, "lse": lse}
