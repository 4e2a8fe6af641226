"""Refusals of the attention half's C entry points, all made on the host before
anything touches a GPU."""

from __future__ import annotations

import ctypes

import pytest

from sglang_restomod_b200 import _lib

P = ctypes.c_void_p(4096)
BF16, F16, F32, E4M3 = _lib.DTYPE_BF16, _lib.DTYPE_F16, _lib.DTYPE_F32, _lib.DTYPE_E4M3


def err(status, code=None):
    assert status != 0 and (code is None or status == code)
    return _lib.load().b200_last_error().decode()


def desc(**kw):
    """A 16-bit cache of 10 pages of 16 tokens, 2 heads of 128, token-major."""
    d = dict(k=4096, v=8192, k_scale=None, v_scale=None, num_pages=10, page_size=16, kv_heads=2,
             head_dim=128, dtype=BF16, page_stride=16 * 256, token_stride=256, head_stride=128,
             scale_page_stride=0, scale_token_stride=0, scale_head_stride=0)
    d.update(kw)
    return _lib.KVCacheDesc(**d)


def norm(**kw):
    a = dict(x=P, dtype=BF16, x_ld=256, rows=4, hidden=256, residual=None, residual_ld=0, weight=P,
             weight_dtype=BF16, weight_bias=0.0, eps=1e-6, residual_out=None, residual_out_ld=0,
             y=P, y_ld=256, q=None, scales=None, scales_ld=0, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return _lib.load().b200_add_rms_norm(*a.values())


@pytest.mark.parametrize("kw,text", [
    (dict(dtype=F32), "bf16 or f16"),
    (dict(weight_dtype=E4M3), "weight must be"),
    (dict(rows=-1), "row count"),
    (dict(hidden=0, x_ld=0), "multiple of 8"),
    (dict(hidden=252), "multiple of 8"),
    (dict(hidden=32776, x_ld=32776, y_ld=32776), "at most 32768"),
    (dict(y=None), "neither y nor q"),
    (dict(q=P), "belong together"),
    (dict(scales=P), "belong together"),
    (dict(hidden=200, q=P, scales=P, scales_ld=4), "128-wide"),
    (dict(q=P, scales=P, scales_ld=3), "scales_ld"),
    (dict(residual_out=P, residual_out_ld=256), "without a residual"),
    (dict(x=None), "null pointer"),
    (dict(weight=None), "null pointer"),
    (dict(x=ctypes.c_void_p(4104)), "16-byte aligned"),
    (dict(x_ld=260), "leading dimensions"),
    (dict(x_ld=128), "leading dimensions"),
    (dict(y_ld=0), "leading dimensions"),
    (dict(residual=P, residual_ld=8), "leading dimensions"),
])
def test_norm_refusals(kw, text):
    assert text in err(norm(**kw))


def test_norm_of_no_rows_is_no_error():
    assert norm(rows=0, x=None, y=None) == 0


CACHE_CASES = [
    (dict(k=None), "null pointer"),
    (dict(v=None), "null pointer"),
    (dict(dtype=F32), "bf16, f16 or e4m3"),
    (dict(head_dim=96), "head_dim"),
    (dict(num_pages=0), "positive pages"),
    (dict(page_size=0), "positive pages"),
    (dict(kv_heads=-1), "positive pages"),
    (dict(num_pages=1 << 28), "2^31 - 1"),
    (dict(k_scale=4096), "scales belong"),
    (dict(dtype=E4M3), "scales belong"),
    (dict(dtype=E4M3, k_scale=4096), "scales belong"),
    (dict(k=4104), "16-byte aligned"),
    (dict(head_stride=132), "16-byte aligned"),
    (dict(dtype=E4M3, k_scale=64, v_scale=64, token_stride=264), "16-byte aligned"),
    (dict(token_stride=-256), "negative strides"),
]


@pytest.mark.parametrize("kw,text", CACHE_CASES)
def test_cache_descriptions_refused_by_every_entry(kw, text):
    lib = _lib.load()
    d = desc(**kw)
    c = ctypes.addressof(d)
    assert text in err(lib.b200_kv_cache_write(c, P, P, BF16, 256, 128, 256, 128, P, 3, None))
    assert text in err(lib.b200_kv_cache_read(c, P, 3, P, P, BF16, 256, 128, None))
    assert text in err(attention(c))


def test_cache_copies_refused():
    lib = _lib.load()
    d = desc()
    c = ctypes.addressof(d)

    def write(cache=c, k=P, v=P, dtype=BF16, strides=(256, 128, 256, 128), slots=P, tokens=3):
        return lib.b200_kv_cache_write(cache, k, v, dtype, *strides, slots, tokens, None)

    assert "null pointer" in err(write(cache=None))
    assert "bf16 or f16" in err(write(dtype=F32), _lib.ERR_UNSUPPORTED)
    assert "own type" in err(write(dtype=F16))
    assert "token count" in err(write(tokens=-1))
    assert "2^31 - 1 vectors" in err(write(tokens=1 << 31))
    assert "slots" in err(write(slots=None))
    assert "slots" in err(write(slots=ctypes.c_void_p(4100)))
    assert "null pointer" in err(write(k=None))
    assert "k: every vector" in err(write(strides=(257, 128, 256, 128)))
    assert "v: every vector" in err(write(v=ctypes.c_void_p(4098)))
    assert "negative strides" in err(write(strides=(256, 128, -256, 128)))
    assert write(tokens=0, k=None, v=None, slots=None) == 0
    read = lib.b200_kv_cache_read
    assert "overlap" in err(read(c, P, 3, P, P, BF16, 128, 128, None))
    assert "overlap" in err(read(c, P, 3, P, P, BF16, 256, 0, None))
    assert "own type" in err(read(c, P, 3, P, P, F16, 256, 128, None))
    assert read(c, None, 0, None, None, BF16, 256, 128, None) == 0


def attention(cache, **kw):
    a = dict(q=P, dtype=BF16, q_tokens=3, q_heads=4, q_ts=512, q_hs=128, table=P, table_stride=2,
             table_width=2, kv_lens=P, q_starts=P, seqs=3, max_q_len=1, scale=0.1, causal=1,
             window=0, out=P, out_ts=512, out_hs=128, lse=None, ws=P, ws_bytes=1 << 40, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return _lib.load().b200_paged_attention(cache, *a.values())


@pytest.mark.parametrize("kw,text", [
    (dict(dtype=F32), "bf16 or f16"),
    (dict(dtype=F16), "own type"),
    (dict(q_heads=3), "cannot share"),
    (dict(q_heads=0), "cannot share"),
    (dict(q_heads=258), "at most 128"),
    (dict(seqs=-1), "count"),
    (dict(q_tokens=-1), "count"),
    (dict(q_tokens=1 << 31), "count"),
    (dict(max_q_len=-1), "count"),
    (dict(table_width=-1), "count"),
    (dict(window=-1), "window"),
    (dict(window=3, causal=0), "window"),
    (dict(scale=float("nan")), "finite"),
    (dict(scale=1e300), "finite"),
    (dict(q=None), "null pointer"),
    (dict(q_ts=513), "q: every vector"),
    (dict(out=ctypes.c_void_p(4104)), "out: every vector"),
    (dict(out_ts=0), "overlap"),
    (dict(out_hs=64), "overlap"),
    (dict(out_ts=256), "overlap"),
    (dict(kv_lens=None), "null pointer"),
    (dict(q_starts=None), "null pointer"),
    (dict(table=None), "null pointer"),
    (dict(lse=ctypes.c_void_p(4097)), "4-byte aligned"),
    (dict(table_stride=-2), "negative strides"),
    (dict(ws=None), "workspace"),
    (dict(ws=ctypes.c_void_p(4096 + 128)), "workspace"),
    (dict(ws_bytes=4096), "workspace"),
])
def test_attention_refusals(kw, text):
    d = desc()
    assert text in err(attention(ctypes.addressof(d), **kw))


def test_attention_over_nothing_is_no_error():
    d = desc()
    for kw in (dict(seqs=0), dict(q_tokens=0, q=None), dict(max_q_len=0, out=None)):
        assert attention(ctypes.addressof(d), **kw) == 0


def test_attention_workspace_sizes():
    lib = _lib.load()
    size = lib.b200_paged_attention_workspace_bytes
    assert size(96, 1, 1) == -1 and size(128, -1, 1) == -1 and size(128, 1, -1) == -1
    for dim in (64, 128, 256):  # a workspace for more tokens and sequences serves fewer
        assert 0 < size(dim, 1, 1) <= size(dim, 1, 64) <= size(dim, 8192, 64) <= size(dim, 8192, 9000)
