"""What a row sees and what it does not: pages freed before a window, and values of
very different sizes.

Tolerances: P and the output are rounded once each, so an output element is off
by at most (u_p + u_out + 2 s_err) sum p|v| (u, s_err as in
test_gpu_attention.py), with the sum of its own column. Below f16's normal range
P's step is absolute, 2^-24, so each token may add half of that: of an e4m3 cache
relative to the row's largest P * 2^e, which the kernel keeps at 1 to 2^8, times a
code of at most 448, where the largest code of a vector is above 224: together
below 2^-24 of sum p max|v| a token; of an f16 cache 2^-25 max|v|.
"""

from __future__ import annotations

import pytest
import torch

from oracle import attention as ref
from sglang_restomod_b200 import ops
from tests.test_gpu_attention import BF16, E4M3, F16, U, bounds, build

pytestmark = pytest.mark.gpu


def run(case, max_q, **kw):
    cache, q, table, kv_lens, starts = case[:5]
    return ops.paged_attention(q.cuda(), cache, table.cuda(), kv_lens.cuda(), starts.cuda(), max_q,
                               return_lse=True, **kw)


def column_bound(q, kc, vc, table, kv_lens, starts, scale, window, products, quantized, causal=True):
    """(bound of each output element, bound of lse) by the file's docstring."""
    def mean(values):
        return ref.paged_attention_ref(q, kc, values, table, kv_lens, starts, scale, causal, window)[0]

    a = abs(scale) * float(q.double().norm(dim=-1).max()) * \
        float(torch.nan_to_num(kc).norm(dim=-1).max())
    s_err = q.shape[-1] * 2.0 ** -22 * a + 2.0 ** -20
    tol = (U[products] + U[q.dtype] + 2 * s_err) * mean(vc.abs())
    if quantized and products == F16:
        peak = mean(vc.abs().amax(-1, keepdim=True).expand_as(vc))
        tol = tol + 2.0 ** -24 * peak * int(kv_lens.max())
    elif products == F16:
        tol = tol + 2.0 ** -25 * int(kv_lens.max()) * float(torch.nan_to_num(vc).abs().max())
    return tol, s_err + 2.0 ** -20 * a


def check_columns(case, max_q, *, window=0, scale=None, products, causal=True):
    """The bound of the file's docstring, element by element."""
    cache, q, table, kv_lens, starts, kc, vc = case
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    out, lse = run(case, max_q, window=window, scale=scale, causal=causal)
    assert ops.attention_status() == 0
    want, want_lse = ref.paged_attention_ref(q, kc, vc, table, kv_lens, starts, scale, causal, window)
    tol, lse_tol = column_bound(q, kc, vc, table, kv_lens, starts, scale, window, products,
                                cache.k_scale is not None, causal)
    assert ((out.cpu().double() - want).abs() <= tol).all()
    seen = torch.isfinite(want_lse)
    assert torch.equal(torch.isfinite(lse.cpu()), seen)
    assert ((lse.cpu().double() - want_lse)[seen].abs() <= lse_tol).all()


@pytest.mark.parametrize("store,q_dtype", [(BF16, BF16), (F16, F16), (E4M3, BF16)])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("page", [1, 8, 16, 24, 64])
@pytest.mark.parametrize("q_len", [1, 30])
def test_pages_before_the_window_may_be_gone(cuda_device, store, q_dtype, dim, page, q_len):
    window, kv = 53, 331
    case = build(dim + page, [q_len, 1], [kv, 77], 2, 4, dim, page, q_dtype, store)
    table = case[2]
    for s, n in ((0, kv - q_len), (1, 76)):
        table[s, :max(0, n - window + 1) // page] = -1
    want, want_lse = run(build(dim + page, [q_len, 1], [kv, 77], 2, 4, dim, page, q_dtype, store),
                         q_len, window=window)
    got, lse = run(case, q_len, window=window)
    assert ops.attention_status() == 0
    assert torch.equal(got, want) and torch.equal(lse, want_lse)


def rewrite(case, s, tokens, k=None, v=None):
    """Other keys and values for some tokens of sequence s; the float64 values follow."""
    cache, q, table, kv_lens, starts, kc, vc = case
    page = cache.page_size
    t = torch.as_tensor(tokens)
    slots = (table[s].long()[t // page] * page + t % page).cuda()
    old_k, old_v = ops.kv_cache_read(cache, slots, q.dtype)
    ops.kv_cache_write(cache, old_k if k is None else k.cuda(), old_v if v is None else v.cuda(), slots)
    if cache.k_scale is not None:
        kc = ref.kv_values_ref(cache.k.cpu(), cache.k_scale.cpu())
        vc = ref.kv_values_ref(cache.v.cpu(), cache.v_scale.cpu())
    else:
        kc, vc = cache.k.cpu().double(), cache.v.cpu().double()
    return cache, q, table, kv_lens, starts, kc, vc


@pytest.mark.parametrize("q_dtype", [BF16, F16])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("page", [1, 8, 16, 64])
@pytest.mark.parametrize("byte", [134, 254])
@pytest.mark.parametrize("q_len,groups", [(1, 8), (3, 4)])
def test_stale_scales_before_the_window(cuda_device, q_dtype, dim, page, byte, q_len, groups):
    """A token that no row sees does not touch what the others contribute,
    whatever its scale bytes hold."""
    window, kv = 53, 331
    case = build(dim + page, [q_len, 1], [kv, 20], 2, groups, dim, page, q_dtype, E4M3)
    cache, table = case[0], case[2]
    for t in range(kv - q_len - window + 1):
        at = (table[0, t // page].item(), t % page)
        cache.k_scale[at] = cache.v_scale[at] = byte
    check_columns(case, q_len, window=window, products=F16)


@pytest.mark.parametrize("q_dtype,store", [(BF16, E4M3), (F16, E4M3), (BF16, BF16)])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("page", [1, 16])
@pytest.mark.parametrize("q_len,groups,kv", [(1, 8, 200), (2, 8, 200), (1, 1, 9001)])
def test_large_value_of_no_weight(cuda_device, q_dtype, store, dim, page, q_len, groups, kv):
    """One value 2^25 times the others whose weight is e^-60 or so: the others
    keep their bits."""
    case = build(dim + page, [q_len], [kv], 1, groups, dim, page, q_dtype, store)
    cache, q = case[0], case[1]
    g = torch.Generator().manual_seed(5)
    q[:] = q.abs()  # so that one key is far from all queries
    case = rewrite(case, 0, range(kv), v=torch.randn(kv, 1, dim, generator=g).to(q_dtype) * 2.0 ** -14)
    far = torch.full((1, 1, dim), -80.0 / dim ** 0.5, dtype=q_dtype)
    # |q| has a mean of 0.8, so q . far * scale is about -0.8 dim 80 / dim = -64
    case = rewrite(case, 0, [5], k=far, v=torch.full((1, 1, dim), 2.0 ** 11, dtype=q_dtype))
    check_columns(case, q_len, products=F16 if store == E4M3 else q_dtype)


@pytest.mark.parametrize("q_dtype", [BF16, F16])
@pytest.mark.parametrize("page", [1, 16])
@pytest.mark.parametrize("q_len,groups", [(1, 8), (40, 4), (150, 4)])
@pytest.mark.parametrize("scale", [0.0, 1e-30, -1e-30, 0.09])
@pytest.mark.parametrize("size", [0.0, 2.0 ** -120])
def test_queries_of_no_size(cuda_device, q_dtype, page, q_len, groups, scale, size):
    """Rows of zeros and of tiny values, over an e4m3 cache: every score is about
    zero, so that each row is the mean of what it sees."""
    case = build(q_len, [q_len, 2], [q_len + 190, 2], 1, groups, 128, page, q_dtype, E4M3)
    case[1][::2] *= size
    check_columns(case, max(q_len, 2), scale=scale, products=F16)


@pytest.mark.parametrize("q_dtype,store", [(BF16, BF16), (F16, F16), (BF16, E4M3)])
@pytest.mark.parametrize("page", [1, 16])
@pytest.mark.parametrize("window", [0, 21])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("q_len,max_q,groups", [(4, 2, 4), (9, 1, 8), (90, 50, 4), (700, 300, 2)])
def test_more_new_tokens_than_the_call_takes(cuda_device, q_dtype, store, page, window, causal, q_len,
                                             max_q, groups):
    """The first max_q_len new tokens of a sequence see what they see in a call
    that takes all of them; the others are left as they were."""
    if window and not causal:
        return
    case = build(q_len, [q_len, 1, 3], [q_len + 100, 40, 3], 1, groups, 128, page, q_dtype, store)
    cache, q, table, kv_lens, starts, kc, vc = case
    out = torch.full(q.shape, 7.0, dtype=q_dtype, device="cuda")
    run(case, max_q, window=window, causal=causal, out=out)
    want, _ = ref.paged_attention_ref(q, kc, vc, table, kv_lens, starts, 128 ** -0.5, causal, window)
    tol, _ = bounds(q, kc, vc, 128 ** -0.5, q_dtype, q_dtype)
    for a, n in zip(starts.tolist(), (q_len, 1, 3)):
        took = min(n, max_q)
        assert (out[a:a + took].cpu().double() - want[a:a + took]).abs().max().item() <= tol
        assert (out[a + took:a + n] == 7.0).all()


@pytest.mark.parametrize("store", [BF16, E4M3])
@pytest.mark.parametrize("page", [1, 16])
@pytest.mark.parametrize("q_len,groups", [(4, 2), (40, 4), (300, 2)])
@pytest.mark.parametrize("window", [(1 << 31) - 1, 1 << 30, 160, 320])
def test_windows_beyond_the_table(cuda_device, store, page, q_len, groups, window):
    """A window wider than anything cached is no window, also where new tokens
    outnumber the cached ones and the first of them see nothing."""
    case = build(q_len, [q_len, 2], [q_len - 3, 9], 1, groups, 128, page, BF16, store)
    want, want_lse = run(case, q_len)
    got, lse = run(case, q_len, window=window)
    if window > q_len:
        assert torch.equal(got, want) and torch.equal(lse, want_lse)
    check_columns(case, q_len, window=window, products=F16 if store == E4M3 else BF16)


@pytest.mark.parametrize("q_len", [1, 150])
@pytest.mark.parametrize("store", [BF16, E4M3])
def test_scales_beyond_fp32(cuda_device, store, q_len):
    """The kernels take the scale in units of log2, where it must be finite too."""
    case = build(3, [q_len], [q_len + 5], 1, 4, 64, 16, BF16, store)
    with pytest.raises(RuntimeError, match="finite"):
        run(case, q_len, scale=3e38)
    case[1].zero_()
    check_columns(case, q_len, scale=2e38, products=F16 if store == E4M3 else BF16)


@pytest.mark.parametrize("page", [1, 16])
@pytest.mark.parametrize("q_len,groups", [(1, 4), (40, 4), (300, 2)])
@pytest.mark.parametrize("byte,known", [(103, True), (134, True), (0, True), (102, False), (1, False),
                                        (135, False), (254, False)])
@pytest.mark.parametrize("which", ["k", "v"])
def test_scale_bytes_and_their_range(cuda_device, page, q_len, groups, byte, known, which):
    """Bytes that no write makes: decode takes them as they are, a chunk reports them
    and stays finite."""
    case = build(q_len, [q_len], [q_len + 90], 1, groups, 64, page, BF16, E4M3)
    cache, table = case[0], case[2]
    at = (table[0, 30 // page].item(), 30 % page)
    (cache.k_scale if which == "k" else cache.v_scale)[at] = byte
    case = (*case[:5], ref.kv_values_ref(cache.k.cpu(), cache.k_scale.cpu()),
            ref.kv_values_ref(cache.v.cpu(), cache.v_scale.cpu()))
    out, lse = run(case, q_len)
    status = ops.attention_status()
    if q_len == 1 and (which == "v" or byte < 200):  # (k at 2^127: scores beyond fp32)
        assert status == 0
    elif q_len > 1:
        assert status == (0 if known else 32)
        assert torch.isfinite(out).all() and torch.isfinite(lse).all()
    if known and (which == "v" or byte < 130):
        check_columns(case, q_len, products=F16)


@pytest.mark.parametrize("q_dtype,store", [(BF16, BF16), (F16, F16), (BF16, E4M3), (F16, E4M3)])
@pytest.mark.parametrize("dim,groups,page", [(64, 8, 16), (128, 8, 64), (256, 4, 16), (128, 3, 1),
                                             (128, 16, 24)])
@pytest.mark.parametrize("q_len,kv,window", [(1, 20011, 0), (1, 20011, 15000), (2, 9001, 0),
                                             (40, 9001, 0), (40, 9001, 5000), (150, 12007, 0)])
def test_every_part_of_a_long_context(cuda_device, q_dtype, store, dim, groups, page, q_len, kv,
                                      window):
    """Column d holds a one for the tokens of the d-th of head_dim equal pieces of the
    context, so the output tells the weight of each piece: one that a part, a tile or
    a merge drops is missing whole."""
    case = build(dim + kv, [q_len], [kv], 1, groups, dim, page, q_dtype, store)
    v = torch.zeros(kv, 1, dim, dtype=q_dtype)
    t = torch.arange(kv)
    v[t, 0, t * dim // kv] = 1.0
    case = rewrite(case, 0, range(kv), v=v)
    # (e4m3 chunks and decode multiply in f16, the others in q's type)
    check_columns(case, q_len, window=window, products=F16 if store == E4M3 else q_dtype)


@pytest.mark.parametrize("store", [BF16, E4M3])
@pytest.mark.parametrize("q_len", [1, 40])
def test_every_part_of_many_sequences(cuda_device, store, q_len):
    lens = [q_len + (37 * i) % 900 for i in range(60)]
    case = build(61, [q_len] * 60, lens, 2, 4, 64, 16, BF16, store)
    check_columns(case, q_len, products=F16 if store == E4M3 else BF16)
