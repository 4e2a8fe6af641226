"""Refusals of the C entry points of the 8-bit integer linear, shared-prefix attention,
scores and eviction, all made on the host before anything touches a GPU."""

from __future__ import annotations

import ctypes

import pytest

from sglang_restomod_b200 import _lib
from tests.test_attention_capi import BF16, E4M3, F16, F32, P, desc, err

ODD = ctypes.c_void_p(4096 + 2)  # aligned for 16-bit elements only


def call(name, defaults, kw, cache=None):
    assert set(kw) <= set(defaults)
    args = {**defaults, **kw}
    if cache is not None:
        args["cache"] = ctypes.addressof(cache)
    return getattr(_lib.load(), name)(*args.values())


# ------------------------------------------------------------ 8-bit integers
QUANT = dict(x=P, dtype=BF16, m=3, k=64, q=P, scales=P, stream=None)
QUANTIZED = dict(q=P, scales=P, m=3, k=64, w=P, w_scales=P, n=5, y=P, dtype=BF16, stream=None)
LINEAR = dict(x=P, dtype=BF16, m=3, k=64, w=P, w_scales=P, n=5, q=P, scales=P, y=P, y_dtype=F16,
              stream=None)
EACH = [("b200_int8_act_quant", QUANT), ("b200_int8_linear_quantized", QUANTIZED),
        ("b200_int8_linear", LINEAR)]


@pytest.mark.parametrize("name,defaults", EACH)
def test_integer_sizes_types_and_pointers(name, defaults):
    for k in (0, -16, 8, 72, 131088):
        assert "multiple of 16" in err(call(name, defaults, dict(k=k)), _lib.ERR_INVALID)
    for m in (-1, 1 << 31):
        assert "bad M" in err(call(name, defaults, dict(m=m)), _lib.ERR_INVALID)
    if "n" in defaults:
        for n in (0, -3, 1 << 31):
            assert "bad N" in err(call(name, defaults, dict(n=n)), _lib.ERR_INVALID)
    for dtype in ("dtype", "y_dtype"):
        for bad in (F32, E4M3):
            if dtype in defaults:
                assert "bf16 or f16" in err(call(name, defaults, {dtype: bad}), _lib.ERR_UNSUPPORTED)
    for p in ("x", "q", "scales", "w", "w_scales", "y"):
        if p not in defaults:
            continue
        assert "null pointer" in err(call(name, defaults, {p: None}), _lib.ERR_INVALID)
        wrong = ctypes.c_void_p(4097) if p == "y" else ODD
        assert "aligned" in err(call(name, defaults, {p: wrong}), _lib.ERR_INVALID)
    nothing = {p: None for p in ("x", "q", "scales", "w", "w_scales", "y") if p in defaults}
    assert call(name, defaults, dict(nothing, m=0)) == 0


# ---------------------------------------------------------- a shared prefix
PREFIX = dict(cache=None, q=P, dtype=BF16, q_tokens=3, q_heads=4, q_ts=512, q_hs=128, prefix_table=P,
              prefix_stride=2, prefix_width=2, prefix_lens=P, group_starts=P, groups=2, table=P,
              table_stride=2, table_width=2, kv_lens=P, q_starts=P, seqs=3, max_q_len=1, scale=0.1,
              out=P, out_ts=512, out_hs=128, lse=None, ws=P, ws_bytes=1 << 40, stream=None)


def prefix(cache=None, **kw):
    return call("b200_shared_prefix_attention", PREFIX, kw, cache or desc())


@pytest.mark.parametrize("kw,text", [
    # as every attention call's
    (dict(dtype=F32), "bf16 or f16"),
    (dict(dtype=F16), "own type"),
    (dict(q_heads=3), "cannot share"),
    (dict(q_heads=258), "at most 128"),
    (dict(seqs=-1), "count"),
    (dict(q_tokens=-1), "count"),
    (dict(scale=float("nan")), "finite"),
    (dict(q=None), "null pointer"),
    (dict(q_ts=513), "q: every vector"),
    (dict(out_hs=64), "overlap"),
    (dict(kv_lens=None), "null pointer"),
    (dict(lse=ctypes.c_void_p(4097)), "4-byte aligned"),
    # and its own
    (dict(groups=-1), "count"),
    (dict(groups=0), "no group"),
    (dict(groups=0x7fffffff), "count"),
    (dict(prefix_width=-1), "count"),
    (dict(prefix_table=None), "null pointer"),
    (dict(prefix_lens=None), "null pointer"),
    (dict(group_starts=None), "null pointer"),
    (dict(prefix_table=ODD), "4-byte aligned"),
    (dict(prefix_lens=ODD), "4-byte aligned"),
    (dict(group_starts=ODD), "4-byte aligned"),
    (dict(prefix_stride=-2), "negative strides"),
    (dict(ws=None), "workspace"),
    (dict(ws=ctypes.c_void_p(4096 + 128)), "workspace"),
    (dict(ws_bytes=4096), "workspace"),
])
def test_prefix_refusals(kw, text):
    assert text in err(prefix(**kw))


def test_prefix_over_nothing_is_no_error():
    for kw in (dict(seqs=0, groups=0), dict(q_tokens=0, q=None), dict(max_q_len=0, out=None)):
        assert prefix(**kw) == 0


def test_prefix_workspace_sizes():
    size = _lib.load().b200_shared_prefix_attention_workspace_bytes
    for bad in ((96, 1, 8, 1, 1), (128, -1, 8, 1, 1), (128, 1, 0, 1, 1), (128, 1, 8, -1, 1),
                (128, 1, 8, 1, -1)):
        assert size(*bad) == -1
    for dim in (64, 128, 256):  # a workspace for more serves fewer
        sizes = [size(dim, *n) for n in ((1, 8, 1, 1), (64, 8, 64, 1), (64, 32, 64, 1),
                                         (8192, 32, 64, 1), (8192, 32, 9000, 1), (8192, 32, 9000, 9000))]
        assert 0 < sizes[0] and sizes == sorted(sizes)
        # both passes' rows in fp32
        assert sizes[3] >= 8 * 8192 * 32 * dim


# ------------------------------------------------------------------ scores
SCORES = dict(cache=None, q=P, dtype=BF16, q_tokens=3, q_heads=4, q_ts=512, q_hs=128, table=P,
              table_stride=2, table_width=2, kv_lens=P, q_starts=P, seqs=3, max_q_len=1, scale=0.1,
              causal=1, window=0, lse=P, scores=P, in_page=32, in_token=1, in_head=16,
              out=ctypes.c_void_p(65536), out_page=32, out_token=2, out_head=1, ws=P,
              ws_bytes=1 << 40, stream=None)


def scores(cache=None, **kw):
    return call("b200_kv_cache_scores", SCORES, kw, cache or desc())


@pytest.mark.parametrize("kw,text", [
    (dict(dtype=F32), "bf16 or f16"),
    (dict(dtype=F16), "own type"),
    (dict(q_heads=3), "cannot share"),
    (dict(q_heads=130, q_ts=130 * 128), "at most 64"),
    (dict(max_q_len=-1), "count"),
    (dict(window=3, causal=0), "window"),
    (dict(scale=float("inf")), "finite"),
    (dict(q=None), "null pointer"),
    (dict(q_hs=0), "overlap"),  # one vector for all heads
    (dict(table=None), "null pointer"),
    (dict(lse=None), "null pointer"),
    (dict(scores=None), "null pointer"),
    (dict(out=None), "null pointer"),
    (dict(lse=ODD), "4-byte aligned"),
    (dict(scores=ODD), "4-byte aligned"),
    (dict(out=ODD), "4-byte aligned"),
    (dict(in_page=-1), "negative strides"),
    (dict(out_head=-1), "negative strides"),
    (dict(out=P), "same strides"),
    (dict(out_head=0), "overlap"),
    (dict(out_page=31), "overlap"),
    (dict(q_tokens=0), "another place"),
    (dict(max_q_len=0), "another place"),
    (dict(ws=None), "workspace"),
    (dict(ws_bytes=4096), "workspace"),
])
def test_scores_refusals(kw, text):
    assert text in err(scores(**kw))


def test_scores_over_nothing_is_no_error():
    same = dict(out=P, out_page=32, out_token=1, out_head=16)
    for kw in (dict(seqs=0), dict(same, q_tokens=0, q=None), dict(same, max_q_len=0)):
        assert scores(**kw) == 0


def test_scores_workspace_sizes():
    size = _lib.load().b200_kv_cache_scores_workspace_bytes
    assert size(96, 1, 8) == -1 and size(128, -1, 8) == -1 and size(128, 1, 0) == -1
    for dim in (64, 128, 256):
        assert 0 < size(dim, 1, 1) <= size(dim, 1, 64) <= size(dim, 8192, 64)


# ---------------------------------------------------------------- eviction
EVICT = dict(cache=None, scores=P, page=32, token=1, head=16, table=P, table_stride=2, table_width=2,
             kv_lens=P, seqs=3, budget=20, recent=4, first=2, out_table=ctypes.c_void_p(8192),
             out_stride=2, out_width=2, kept=P, lens=P, stream=None)


def evict(cache=None, **kw):
    return call("b200_kv_cache_evict", EVICT, kw, cache or desc())


@pytest.mark.parametrize("kw,text", [
    (dict(seqs=-1), "count"),
    (dict(table_width=-1), "count"),
    (dict(out_width=-1), "count"),
    (dict(budget=0, recent=0, first=0), "budget"),
    (dict(recent=-1), "budget"),
    (dict(first=-1), "budget"),
    (dict(recent=19), "budget"),
    (dict(recent=0x7fffffff, first=0x7fffffff), "budget"),
    (dict(seqs=0x7fffffff), "2^28 rows"),
    (dict(scores=None), "null pointer"),
    (dict(table=None), "null pointer"),
    (dict(kv_lens=None), "null pointer"),
    (dict(kept=None), "null pointer"),
    (dict(lens=None), "null pointer"),
    (dict(scores=ODD), "4-byte aligned"),
    (dict(table=ODD), "4-byte aligned"),
    (dict(kept=ODD), "4-byte aligned"),
    (dict(out_table=ODD), "4-byte aligned"),
    (dict(token=-1), "negative strides"),
    (dict(table_stride=-1), "negative strides"),
    (dict(out_stride=-1), "negative strides"),
    (dict(head=0), "scores overlap"),
    (dict(page=16), "scores overlap"),
    (dict(table_width=1 << 28), "tokens"),
    (dict(budget=1 << 30, table_width=1 << 20), "tokens stay"),
    (dict(out_width=1), "do not hold the budget"),
])
def test_evict_refusals(kw, text):
    assert text in err(evict(**kw))


@pytest.mark.parametrize("kw", [
    dict(head_stride=0), dict(head_stride=64), dict(token_stride=128), dict(page_stride=256),
    dict(dtype=E4M3, k_scale=4096, v_scale=8192, scale_page_stride=32, scale_token_stride=1)])
def test_evict_refuses_a_cache_whose_vectors_overlap(kw):
    assert "vectors overlap" in err(evict(desc(**kw)))


def test_evict_of_no_sequences_is_no_error():
    assert evict(seqs=0, scores=None, table=None, kv_lens=None, kept=None, lens=None) == 0


@pytest.mark.parametrize("kw,text", [
    (dict(k=None), "null pointer"),
    (dict(dtype=F32), "bf16, f16 or e4m3"),
    (dict(head_dim=96), "64, 128 or 256"),
    (dict(num_pages=0), "positive pages"),
    (dict(k_scale=4096, v_scale=8192), "scales belong"),
    (dict(token_stride=252), "16-byte aligned"),
    (dict(page_stride=-4096), "negative strides"),
])
def test_cache_descriptions(kw, text):
    for entry in (prefix, scores, evict):
        assert text in err(entry(desc(**kw)))


# --------------------------------------------------------- the package's calls
def test_operands_off_the_gpu_are_refused(monkeypatch):
    torch = pytest.importorskip("torch")
    from sglang_restomod_b200 import kv_cache, ops

    monkeypatch.setattr(ops, "_current_device", lambda: 0)
    x = torch.zeros(2, 64, dtype=torch.bfloat16)
    w, ws = torch.zeros(5, 64, dtype=torch.int8), torch.ones(5)
    cache = kv_cache.PagedKVCache.empty(4, 16, 2, 64, "cpu")
    q = torch.zeros(3, 4, 64, dtype=torch.bfloat16)
    i32 = dict(dtype=torch.int32)
    table, lens, starts = torch.zeros(3, 2, **i32), torch.ones(3, **i32), torch.arange(4, **i32)
    groups = torch.tensor([0, 3], **i32)
    for fn, args in ((ops.int8_act_quant, (x,)), (ops.int8_linear, (x, w, ws)),
                     (ops.int8_linear_quantized, (w[:2], ws[:2], w, ws)),
                     (ops.shared_prefix_attention, (q, cache, table[:1], lens[:1], groups, table, lens,
                                                    starts, 1)),
                     (ops.kv_cache_scores, (q, cache, table, lens, starts, 1, torch.zeros(3, 4),
                                            cache.empty_scores())),
                     (ops.kv_cache_evict, (cache, cache.empty_scores(), table, lens, 1))):
        with pytest.raises(ValueError, match="must be CUDA tensors"):
            fn(*args)


def test_empty_scores_have_the_cache_layout():
    from sglang_restomod_b200 import kv_cache

    s = kv_cache.PagedKVCache.empty(4, 16, 2, 64, "cpu").empty_scores()
    assert s.shape == (4, 16, 2) and s.stride() == (32, 1, 16)


def refused(error, text, fn, *args, **kw):
    with pytest.raises(error, match=text):
        fn(*args, **kw)


def test_wrappers_refuse_shapes_and_types(monkeypatch):
    torch = pytest.importorskip("torch")
    from sglang_restomod_b200 import kv_cache, ops

    monkeypatch.setattr(ops, "_on_device", lambda *a: 0)
    monkeypatch.setattr(ops, "_raw_stream", lambda index: 0)
    bf16, i32 = dict(dtype=torch.bfloat16), dict(dtype=torch.int32)
    x, w, ws = torch.zeros(2, 64, **bf16), torch.zeros(5, 64, dtype=torch.int8), torch.ones(5)
    refused(TypeError, "bf16 or f16", ops.int8_act_quant, x.float())
    refused(ValueError, "contiguous", ops.int8_act_quant, x[:, ::2])
    refused(ValueError, "contiguous", ops.int8_act_quant, x[0])
    refused(TypeError, "int8 and its scales float32", ops.int8_linear, x, w.float(), ws)
    refused(TypeError, "int8 and its scales float32", ops.int8_linear, x, w, ws.double())
    refused(ValueError, r"\[N, 64\]", ops.int8_linear, x, w[:, :48].contiguous(), ws)
    refused(ValueError, r"\[N, 64\]", ops.int8_linear, x, w, ws[:4])
    refused(ValueError, "contiguous", ops.int8_linear, x, torch.zeros(64, 5, dtype=torch.int8).t(), ws)
    refused(ValueError, "contiguous", ops.int8_linear, torch.zeros(2, 128, **bf16)[:, :64], w, ws)
    refused(ValueError, r"\[2, 5\]", ops.int8_linear, x, w, ws, out=torch.zeros(2, 6, **bf16))
    quantized = ops.int8_linear_quantized
    refused(TypeError, "q must be int8", quantized, x, ws[:2], w, ws)
    refused(ValueError, r"contiguous \[2\]", quantized, w[:2], ws, w, ws)

    cache = kv_cache.PagedKVCache.empty(4, 16, 2, 64, "cpu")
    q, scores, lse = torch.zeros(3, 4, 64, **bf16), cache.empty_scores(), torch.zeros(3, 4)
    table, lens, starts = torch.zeros(3, 2, **i32), torch.ones(3, **i32), torch.arange(4, **i32)
    groups = torch.tensor([0, 3], **i32)

    def prefix(**kw):
        a = dict(q=q, cache=cache, prefix_table=table[:1], prefix_lens=lens[:1], group_starts=groups,
                 page_table=table, kv_lens=lens, q_starts=starts, max_q_len=1)
        return lambda: ops.shared_prefix_attention(**{**a, **kw})

    refused(TypeError, "bf16 or f16", prefix(q=q.float()))
    refused(ValueError, "heads, 64", prefix(q=q[..., :32]))
    refused(ValueError, "prefix_table must be int32", prefix(prefix_table=table[:1].long()))
    refused(ValueError, "prefix_lens must be int32", prefix(prefix_lens=lens[:1].long()))
    refused(ValueError, "1 groups need", prefix(group_starts=starts))
    refused(ValueError, "1 groups need", prefix(prefix_table=table))
    refused(ValueError, "3 sequences need", prefix(page_table=table[:2]))
    refused(ValueError, "out must be", prefix(out=q[:2]))
    refused(TypeError, "uint8", prefix(workspace=torch.zeros(8)))

    def gather(**kw):
        a = dict(q=q, cache=cache, page_table=table, kv_lens=lens, q_starts=starts, max_q_len=1,
                 lse=lse, scores=scores)
        return lambda: ops.kv_cache_scores(**{**a, **kw})

    refused(ValueError, "lse must be", gather(lse=lse[:2]))
    refused(ValueError, "lse must be", gather(lse=lse.double()))
    refused(ValueError, "lse must be", gather(lse=torch.zeros(4, 3).t()))
    refused(TypeError, "scores must be float32", gather(scores=scores.half()))
    refused(ValueError, r"scores must be \(4, 16, 2\)", gather(scores=scores[:3]))
    refused(ValueError, r"out must be \(4, 16, 2\)", gather(out=scores.transpose(1, 2)))

    def evict(**kw):
        a = dict(cache=cache, scores=scores, page_table=table, kv_lens=lens, budget=2)
        return lambda: ops.kv_cache_evict(**{**a, **kw})

    refused(TypeError, "scores must be float32", evict(scores=scores.double()))
    refused(ValueError, r"scores must be \(4, 16, 2\)", evict(scores=scores[:, :8]))
    refused(ValueError, "page_table must be int32", evict(page_table=table.long()))
    refused(ValueError, "kv_lens must be", evict(kv_lens=lens[:2]))
    refused(ValueError, "out_table must be", evict(out_table=table[:2]))
    for budget in (0, -1, 1 << 31):
        refused(ValueError, "budget", evict(budget=budget))
    for kept in (dict(recent=-1), dict(first=-1), dict(recent=1, first=2), dict(recent=1 << 32)):
        refused(ValueError, "budget", evict(**kept))
