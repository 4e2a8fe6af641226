"""GPU parity of the norm, the key/value cache and paged attention with 64-bit
references (oracle/attention.py).

Tolerances come from the roundings each operator makes, u = 2^-8 for bf16 and
2^-11 for f16 (half a unit in the last place of 8 and 11 significant bits),
2^-4 for e4m3 normals:

* norm: one rounding of the output, plus fp32 arithmetic over a row (the sum of
  n squares in any order is within n 2^-24; sqrt halves it): below 2^-12 for
  the widths here, so u + 2^-12 relative.
* cache: codes and scale bytes are exact (scaling by a power of two is).
* attention: P is rounded once (to the products' 16-bit type), the output once:
  |error| <= (u_p + u_out) max|v|, plus fp32 products: s is off by at most
  D 2^-22 A with A = scale max|q| max|k| (norms), which moves weights by that
  factor; lse is off by the same.
"""

from __future__ import annotations

import math

import pytest
import torch

import oracle
from oracle import attention as ref
from sglang_restomod_b200 import kv_cache, ops

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
BF16, F16, E4M3 = torch.bfloat16, torch.float16, torch.float8_e4m3fn


def gen(seed):
    return torch.Generator().manual_seed(seed)


# --------------------------------------------------------------------- norm
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("rows,hidden", [(1, 8), (3, 128), (5, 264), (17, 1000), (9, 1032), (2, 7168),
                                         (301, 2048), (3, 16384), (2, 20488), (1, 32768)])
def test_add_rms_norm(cuda_device, dtype, rows, hidden):
    g = gen(rows * hidden)
    x = torch.randn(rows, hidden, generator=g).to(dtype)
    r = (3 * torch.randn(rows, hidden, generator=g)).to(dtype)
    w = (0.2 * torch.randn(hidden, generator=g)).to(torch.float32)
    for residual, bias, wt in ((None, 1.0, torch.float32), (r, 0.0, dtype), (r, 1.0, BF16)):
        y, h = ops.add_rms_norm(x.cuda(), w.to(wt).cuda(), 1e-5, weight_bias=bias,
                                residual=None if residual is None else residual.cuda())
        want_y, want_h = ref.add_rms_norm_ref(x, w.to(wt), 1e-5, residual, bias)
        tol = U[dtype] + 2.0 ** -12
        # f16's subnormal step bounds what is below its normal range
        assert ((y.cpu().double() - want_y).abs() <= tol * want_y.abs() + 2.0 ** -24).all()
        if residual is None:
            assert h is None
        else:
            # the fp32 sum of two 16-bit values, rounded once
            assert torch.equal(h.cpu(), (x.float() + r.float()).to(dtype))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("rows,hidden", [(1, 128), (7, 384), (33, 1152), (5, 7168), (2, 16512)])
def test_add_rms_norm_fp8(cuda_device, dtype, rows, hidden):
    g = gen(rows + hidden)
    x = torch.randn(rows, hidden, generator=g).to(dtype)
    r = torch.randn(rows, hidden, generator=g).to(dtype)
    x[0, :128], r[0, :128] = 0, 0  # a group of zeros takes the 1e-8 floor
    w = torch.randn(hidden, generator=g).to(dtype)
    both = torch.empty(rows, hidden, dtype=dtype, device="cuda")
    q, s, h = ops.add_rms_norm_fp8(x.cuda(), w.cuda(), 1e-6, residual=r.cuda(), out=both,
                                   scales_ld=rows + 3)
    want, _ = ref.add_rms_norm_ref(x, w, 1e-6, r)
    scale = (want.reshape(rows, -1, 128).abs().amax(-1) / 448).clamp_min(1e-8)
    got_s = s[:, :rows].T.cpu().double()
    assert ((got_s - scale).abs() <= 2.0 ** -12 * scale).all()
    # one e4m3 rounding of y / scale, which is itself within 2^-11: relative
    # 2^-4, or half the smallest step (2^-10) near zero
    got = q.cpu().double() * got_s.repeat_interleave(128, -1)
    bound = (2.0 ** -4 + 2.0 ** -10) * want.abs() + 2.0 ** -9 * scale.repeat_interleave(128, -1)
    assert ((got - want).abs() <= bound).all()
    plain, h2 = ops.add_rms_norm(x.cuda(), w.cuda(), 1e-6, residual=r.cuda())
    assert torch.equal(both, plain) and torch.equal(h, h2)


def test_norm_in_place_strides_and_streams(cuda_device):
    g = gen(0)
    wide = torch.randn(37, 3 * 512, generator=g).to(BF16).cuda()
    x, r = wide[:, :512], wide[:, 512:1024]
    w = torch.ones(512, dtype=BF16, device="cuda")
    want_y, want_h = ops.add_rms_norm(x.contiguous(), w, residual=r.contiguous())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y, h = ops.add_rms_norm(x, w, residual=r, out=x, residual_out=r)
    torch.cuda.current_stream().wait_stream(side)
    assert y.data_ptr() == x.data_ptr() and h.data_ptr() == r.data_ptr()
    assert torch.equal(x, want_y) and torch.equal(r, want_h)
    # one row of x for all rows of the residual
    one = torch.randn(1, 512, generator=g).to(BF16).cuda()
    y, h = ops.add_rms_norm(one.expand(37, 512), w, residual=want_h)
    y2, h2 = ops.add_rms_norm(one.repeat(37, 1), w, residual=want_h)
    assert torch.equal(y, y2) and torch.equal(h, h2)


def test_norm_not_finite(cuda_device):
    x = torch.randn(3, 256, generator=gen(1)).to(BF16)
    x[1, 5] = math.nan
    w = torch.ones(256, dtype=BF16)
    y, _ = ops.add_rms_norm(x.cuda(), w.cuda())
    q, s, _ = ops.add_rms_norm_fp8(x.cuda(), w.cuda())
    assert torch.isnan(y[1]).all() and torch.isfinite(y[0]).all() and torch.isfinite(y[2]).all()
    assert torch.isnan(s[:, 1]).all() and torch.isfinite(s[:, 0]).all()
    assert torch.isnan(q[1].float()).all() and torch.isfinite(q[2].float()).all()


def test_norm_feeds_the_w8a8_linear(cuda_device):
    """norm -> quantized linear equals norm -> quantize -> linear but for the
    norm's 16-bit rounding, which the fused form leaves out."""
    from sglang_restomod_b200 import synth

    m, k, n = 45, 512, 384
    wq, ws = synth.fp8_bank(1, n, k, cuda_device, seed=2)
    x = synth.activations(m, k, cuda_device, seed=3)
    w = torch.ones(k, dtype=BF16, device="cuda")
    q, s, _ = ops.add_rms_norm_fp8(x, w, scales_ld=ops.w8a8_scales_ld(m))
    got = ops.w8a8_linear_quantized(q, s, wq[0], ws[0])
    dense = oracle.dequant_block_fp8(wq[0].cpu(), ws[0].cpu()).double()
    qx = q.cpu().double() * s[:, :m].T.cpu().double().repeat_interleave(128, -1)
    want = qx @ dense.T
    # exact products, fp32 sums of 512 terms, one bf16 rounding
    bound = 2.0 ** -8 * want.abs() + 2.0 ** -13 * (qx.abs() @ dense.abs().T)
    assert ((got.cpu().double() - want).abs() <= bound).all()
    assert ops.workspace_status() == 0


# -------------------------------------------------------------------- cache
def make_cache(pages, page, heads, dim, dtype, token_major=False):
    """A cache full of NaN: what an operator must not read shows."""
    shape = (pages, page, heads, dim) if token_major else (pages, heads, page, dim)
    raw = torch.uint8 if dtype == E4M3 else dtype
    fill = 0x7f if dtype == E4M3 else math.nan

    def view(t):
        return t if token_major else t.transpose(1, 2)

    kv = [view(torch.full(shape, fill, dtype=raw, device="cuda").view(dtype)) for _ in range(2)]
    sc = [view(torch.full(shape[:3], 255, dtype=torch.uint8, device="cuda"))
          if dtype == E4M3 else None for _ in range(2)]
    return kv_cache.PagedKVCache(*kv, *sc)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("store", ["same", E4M3])
@pytest.mark.parametrize("tokens,heads,dim,page,token_major",
                         [(1, 1, 64, 1, False), (37, 3, 128, 16, False), (130, 2, 256, 24, True),
                          (65, 5, 64, 8, True), (515, 8, 128, 64, False)])
def test_cache_round_trip(cuda_device, dtype, store, tokens, heads, dim, page, token_major):
    g = gen(tokens)
    store = dtype if store == "same" else store
    pages = -(-tokens // page) + 2
    cache = make_cache(pages, page, heads, dim, store, token_major)
    fused = torch.randn(tokens, 2 * heads, dim, generator=g) * 4
    fused[0, 0] = 0                      # a vector of zeros
    fused[-1, heads] *= 1e-6             # a small one
    fused[tokens // 2, 0, 3] = 448.0     # on a scale's edge
    if dtype == BF16:
        fused[tokens // 2, heads, 1] = 1e6  # saturates at 57344
    fused = fused.to(dtype)
    slots = torch.randperm(pages * page, generator=g)[:tokens]
    skip = tokens // 3 if tokens > 2 else -1
    if skip >= 0:
        slots[skip] = -1
    before = cache.k.view(torch.uint8).clone() if store == E4M3 else cache.k.clone()
    k, v = fused[:, :heads], fused[:, heads:]
    dev = fused.cuda()
    ops.kv_cache_write(cache, dev[:, :heads], dev[:, heads:], slots.cuda())
    at = [i for i in range(tokens) if i != skip]
    page_of, off = slots[at] // page, slots[at] % page
    for x, data, scale in ((k, cache.k, cache.k_scale), (v, cache.v, cache.v_scale)):
        if store == E4M3:
            codes, e = ref.kv_quantize_ref(x[at])
            assert torch.equal(scale.cpu()[page_of, off], e)
            got = data.view(torch.uint8).cpu()[page_of, off]
            assert torch.equal(got, codes.view(torch.uint8))
        else:
            assert torch.equal(data.cpu()[page_of, off], x[at])
    # slots that were not written keep their bytes
    free = torch.ones(pages * page, dtype=torch.bool)
    free[slots[at]] = False
    left = torch.nonzero(free).flatten()
    now = (cache.k.view(torch.uint8) if store == E4M3 else cache.k).cpu()[left // page, left % page]
    was = before.cpu()[left // page, left % page]
    if store == E4M3:
        assert torch.equal(now, was)
    else:
        assert torch.isnan(now.float()).all()
    rk, rv = ops.kv_cache_read(cache, slots.cuda(), dtype)
    for x, got in ((k, rk), (v, rv)):
        want = x[at].double()
        if store == E4M3:
            want = ref.kv_values_ref(*ref.kv_quantize_ref(x[at]))
        assert torch.equal(got.cpu()[at].double(), want.to(dtype).double())
        if skip >= 0:
            assert (got[skip] == 0).all()


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_cache_not_finite(cuda_device, dtype):
    cache = make_cache(2, 16, 1, 128, E4M3)
    k = torch.randn(4, 1, 128, generator=gen(3)).to(dtype)
    k[1, 0, 7], k[2, 0, 0] = math.inf, math.nan
    slots = torch.arange(4, device="cuda")
    ops.kv_cache_write(cache, k.cuda(), k.cuda(), slots)
    got, _ = ops.kv_cache_read(cache, slots, dtype)
    assert torch.isnan(got[1:3]).all() and torch.isfinite(got[[0, 3]].float()).all()


def test_cache_slots_outside(cuda_device):
    cache = make_cache(3, 8, 2, 64, BF16)
    k = torch.randn(5, 2, 64, generator=gen(4)).to(BF16).cuda()
    slots = torch.tensor([-7, 24, 23, 1 << 40, 0], device="cuda")
    ops.kv_cache_write(cache, k, k, slots)
    got, _ = ops.kv_cache_read(cache, slots)
    assert torch.equal(got[[2, 4]], k[[2, 4]]) and (got[[0, 1, 3]] == 0).all()


# ---------------------------------------------------------------- attention
def build(seed, q_lens, kv_lens, heads, groups, dim, page, q_dtype, store, *, token_major=False,
          k_scale=1.0):
    """A filled cache on shuffled pages (NaN wherever nothing was written), q,
    and the float64 values the cache stands for."""
    g = gen(seed)
    need = [-(-n // page) for n in kv_lens]
    pages = sum(need) + 1
    cache = make_cache(pages, page, heads, dim, store, token_major)
    order = torch.randperm(pages, generator=g)
    width = max(1, max(need))
    table = torch.full((len(kv_lens), width + 1), 1 << 29, dtype=torch.int32)  # a wider row, poisoned
    at = 0
    slots = []
    for s, n in enumerate(need):
        table[s, :n] = order[at:at + n].int()
        t = torch.arange(kv_lens[s])
        slots.append(table[s].long()[t // page] * page + t % page)
        at += n
    slots = torch.cat(slots) if slots else torch.empty(0, dtype=torch.int64)
    total = int(slots.shape[0])
    kv = torch.randn(total, 2 * heads, dim, generator=g)
    kv[:, :heads] *= k_scale
    kv = kv.to(q_dtype)
    dev = kv.cuda()
    if total:
        ops.kv_cache_write(cache, dev[:, :heads], dev[:, heads:], slots.cuda())
    q = torch.randn(sum(q_lens), heads * groups, dim, generator=g).to(q_dtype)
    starts = torch.tensor([0] + q_lens).cumsum(0).int()
    if store == E4M3:
        kc = ref.kv_values_ref(cache.k.cpu(), cache.k_scale.cpu())
        vc = ref.kv_values_ref(cache.v.cpu(), cache.v_scale.cpu())
    else:
        kc, vc = cache.k.cpu().double(), cache.v.cpu().double()
    return cache, q, table, torch.tensor(kv_lens, dtype=torch.int32), starts, kc, vc


def bounds(q, kc, vc, scale, p_dtype, out_dtype):
    finite = torch.nan_to_num
    a = scale * float(q.double().norm(dim=-1).max()) * float(finite(kc).norm(dim=-1).max())
    s_err = q.shape[-1] * 2.0 ** -22 * a + 2.0 ** -20
    top = float(finite(vc).abs().max())
    return (U[p_dtype] + U[out_dtype] + 2 * s_err) * top, s_err + 2.0 ** -20 * a


def check(case, *, causal=True, window=0, scale=None, max_q=None, products=None):
    cache, q, table, kv_lens, starts, kc, vc = case
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    max_q = int((starts[1:] - starts[:-1]).max()) if max_q is None else max_q
    out, lse = ops.paged_attention(q.cuda(), cache, table.cuda(), kv_lens.cuda(), starts.cuda(),
                                   max_q, scale=scale, causal=causal, window=window, return_lse=True)
    want, want_lse = ref.paged_attention_ref(q, kc, vc, table, kv_lens, starts, scale, causal, window)
    rows = max_q * (q.shape[1] // cache.kv_heads)
    p_dtype = products or (q.dtype if cache.k_scale is None else F16 if rows <= 16 else q.dtype)
    tol, lse_tol = bounds(q, kc, vc, scale, p_dtype, q.dtype)
    assert ops.attention_status() == 0
    assert torch.equal(torch.isinf(lse.cpu()), torch.isinf(want_lse))
    seen = torch.isfinite(want_lse)
    assert (lse.cpu().double() - want_lse)[seen].abs().max().item() <= lse_tol if seen.any() else True
    assert (out.cpu().double() - want).abs().max().item() <= tol
    assert (out.cpu()[~seen] == 0).all()
    return out


TYPES = [(BF16, BF16), (F16, F16), (BF16, E4M3), (F16, E4M3)]
LENS = [1, 15, 16, 17, 0, 63, 64, 65, 130, 1000]


@pytest.mark.parametrize("q_dtype,store", TYPES)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("heads,groups,page", [(2, 8, 16), (1, 3, 1), (3, 1, 24), (2, 16, 64)])
def test_decode(cuda_device, q_dtype, store, dim, heads, groups, page):
    check(build(dim + page, [1] * len(LENS), LENS, heads, groups, dim, page, q_dtype, store,
                token_major=page == 24))


@pytest.mark.parametrize("q_dtype,store", TYPES)
@pytest.mark.parametrize("q_lens,kv_lens,groups", [
    ([3, 1, 0, 4, 2], [200, 1, 77, 4, 0], 4),   # new tokens of several lengths, one sequence idle
    ([5, 5], [5, 300], 3),                      # a prompt from its first token
])
def test_decode_of_a_few_tokens(cuda_device, q_dtype, store, q_lens, kv_lens, groups):
    case = build(7, q_lens, kv_lens, 2, groups, 128, 16, q_dtype, store)
    check(case)
    check(case, causal=False)


@pytest.mark.parametrize("q_dtype,store", TYPES)
@pytest.mark.parametrize("window", [1, 16, 100, 5000])
def test_decode_window(cuda_device, q_dtype, store, window):
    check(build(window, [1, 2, 1], [700, 333, 50], 2, 4, 64, 16, q_dtype, store), window=window)


@pytest.mark.parametrize("store", [BF16, E4M3])
def test_decode_long_and_many(cuda_device, store):
    # one long sequence over the whole GPU, and more sequences than threads
    check(build(1, [1], [20011], 1, 8, 128, 16, BF16, store))
    check(build(2, [1] * 300, [(37 * i) % 90 for i in range(300)], 1, 2, 64, 16, BF16, store))


@pytest.mark.parametrize("store", [BF16, E4M3])
def test_decode_large_scores(cuda_device, store):
    """Scores in the hundreds: maxima far apart from tile to tile."""
    check(build(3, [1, 1], [900, 64], 2, 8, 128, 16, BF16, store, k_scale=30.0), scale=1.0)


def test_decode_same_result_every_time(cuda_device):
    case = build(4, [1] * 5, [3000, 10, 777, 2048, 1], 2, 8, 128, 16, BF16, E4M3)
    first = check(case)
    for _ in range(5):
        assert torch.equal(check(case), first)


def test_decode_scales_far_apart(cuda_device):
    """Values whose scales differ by 2^20 within a tile, growing and shrinking."""
    case = build(5, [1], [200], 1, 4, 128, 16, BF16, BF16)
    cache, q, table, kv_lens, starts, kc, vc = case
    g = gen(6)
    kv = torch.randn(200, 2, 128, generator=g)
    kv[:, 1] *= torch.pow(2.0, torch.randint(-12, 8, (200, 1), generator=g).float())
    kv = kv.to(BF16)
    t = torch.arange(200)
    slots = table[0].long()[t // 16] * 16 + t % 16
    quant = make_cache(cache.num_pages, 16, 1, 128, E4M3)
    ops.kv_cache_write(quant, kv[:, :1].cuda(), kv[:, 1:].cuda(), slots.cuda())
    kc = ref.kv_values_ref(quant.k.cpu(), quant.k_scale.cpu())
    vc = ref.kv_values_ref(quant.v.cpu(), quant.v_scale.cpu())
    check((quant, q, table, kv_lens, starts, kc, vc))


@pytest.mark.parametrize("store", [BF16, E4M3])
def test_decode_bad_pages_and_lengths(cuda_device, store):
    """A page number outside the cache reads as zeros and is reported; lengths
    beyond the page table are cut to it."""
    case = list(build(8, [1, 1], [40, 33], 1, 2, 64, 16, BF16, store))
    cache, q, table, kv_lens, starts, kc, vc = case
    bad = table.clone()
    bad[1, 1] = cache.num_pages + 5
    out = ops.paged_attention(q.cuda(), cache, bad.cuda(), kv_lens.cuda(), starts.cuda(), 1)
    assert ops.attention_status() == 16
    assert ops.attention_status() == 0
    want, _ = ref.paged_attention_ref(q, kc, vc, table, kv_lens, starts, 64 ** -0.5)
    assert (out.cpu().double() - want)[0].abs().max() < 0.1 and torch.isfinite(out).all()
    long = kv_lens.clone()
    long[0] = 1 << 30
    out = ops.paged_attention(q.cuda(), cache, table[:, :2].contiguous().cuda(), long.cuda(),
                              starts.cuda(), 1)
    want, _ = ref.paged_attention_ref(q, kc, vc, table, torch.tensor([32, 32]), starts, 64 ** -0.5)
    tol, _ = bounds(q, kc, vc, 0.125, BF16, BF16)
    assert (out.cpu().double() - want).abs().max().item() <= tol


def test_decode_strided_q_and_out(cuda_device):
    case = build(9, [1, 1, 1], [70, 20, 300], 2, 4, 128, 16, F16, F16)
    cache, q, table, kv_lens, starts, kc, vc = case
    want = check(case)
    wide = torch.zeros(3, 8, 3, 128, dtype=F16, device="cuda")
    wide[:, :, 1] = q.cuda()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.paged_attention(wide[:, :, 1], cache, table.cuda(), kv_lens.cuda(), starts.cuda(), 1,
                            out=wide[:, :, 2])
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(wide[:, :, 2], want)
    assert (wide[:, :, 0] == 0).all()


def test_decode_not_finite(cuda_device):
    """A NaN that a row sees makes that row NaN, and only rows of its head."""
    case = build(10, [1, 1], [100, 100], 2, 2, 64, 16, BF16, E4M3)
    cache, q, table, kv_lens, starts, kc, vc = case
    p = table[0, 3].item()
    cache.v_scale[p, 5, 1] = 255
    out, lse = ops.paged_attention(q.cuda(), cache, table.cuda(), kv_lens.cuda(), starts.cuda(), 1,
                                   return_lse=True)
    assert torch.isnan(out[0, 2:]).all() and torch.isfinite(out[0, :2].float()).all()
    assert torch.isfinite(out[1].float()).all() and torch.isfinite(lse).all()
    cache.k_scale[p, 5, 0] = 255
    out, lse = ops.paged_attention(q.cuda(), cache, table.cuda(), kv_lens.cuda(), starts.cuda(), 1,
                                   return_lse=True)
    assert torch.isnan(out[0, :2]).all() and torch.isnan(lse[0, :2]).all()
    assert torch.isfinite(out[1].float()).all()


def test_attention_graph_replay_sees_new_lengths(cuda_device):
    case = build(11, [1, 1], [500, 40], 2, 8, 128, 16, BF16, E4M3)
    cache, q, table, kv_lens, starts, kc, vc = case
    dq, dt, dl, ds = q.cuda(), table.cuda(), kv_lens.cuda(), starts.cuda()
    ops.paged_attention(dq, cache, dt, dl, ds, 1)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.paged_attention(dq, cache, dt, dl, ds, 1)
    tol, _ = bounds(q, kc, vc, 128 ** -0.5, F16, BF16)
    for lens in ([500, 40], [3, 40], [129, 0]):
        dl.copy_(torch.tensor(lens, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        want, _ = ref.paged_attention_ref(q, kc, vc, table, torch.tensor(lens), starts, 128 ** -0.5)
        assert (out.cpu().double() - want).abs().max().item() <= tol


# ------------------------------------------------- chunks of many new tokens
CHUNKS = [
    ([1], [1]), ([129], [129]), ([7, 130, 1, 64], [7, 400, 90, 1000]), ([33, 2], [33, 0]),
    ([256, 0, 300], [256, 5, 811]),
]


@pytest.mark.parametrize("q_dtype,store", TYPES)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("q_lens,kv_lens", CHUNKS)
def test_chunk(cuda_device, q_dtype, store, dim, q_lens, kv_lens):
    case = build(dim, q_lens, kv_lens, 2, 3, dim, 16, q_dtype, store)
    # a bound above the longest chunk also takes short calls through this path
    check(case, max_q=max(max(q_lens), 6), products=q_dtype)


@pytest.mark.parametrize("q_dtype,store", [(BF16, BF16), (F16, E4M3)])
@pytest.mark.parametrize("heads,groups,page", [(1, 1, 1), (2, 8, 24), (1, 17, 64), (1, 128, 128)])
def test_chunk_heads_and_pages(cuda_device, q_dtype, store, heads, groups, page):
    check(build(page, [70, 20], [300, 20], heads, groups, 128, page, q_dtype, store,
                token_major=page == 24), products=q_dtype, max_q=70)


@pytest.mark.parametrize("q_dtype,store", TYPES)
@pytest.mark.parametrize("window", [1, 100, 129, 4096])
def test_chunk_window(cuda_device, q_dtype, store, window):
    check(build(window, [200, 31], [900, 50], 1, 4, 128, 16, q_dtype, store), window=window,
          products=q_dtype)


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_chunk_not_causal(cuda_device, dim):
    check(build(20 + dim, [140, 3], [140, 500], 2, 2, dim, 16, BF16, BF16), causal=False,
          products=BF16)


@pytest.mark.parametrize("dim,store", [(64, F16), (128, BF16), (128, E4M3), (256, BF16)])
def test_chunk_long_context(cuda_device, dim, store):
    """Few rows on a long context: the keys of one tile of rows are split over
    many blocks."""
    check(build(30, [40], [9001], 1, 4, dim, 64, F16 if store == F16 else BF16, store),
          products=F16 if store == F16 else BF16)


def test_chunk_many_sequences(cuda_device):
    n = 300
    q_lens = [(7 * i) % 23 for i in range(n)]
    kv = [q + (13 * i) % 60 for i, q in enumerate(q_lens)]
    check(build(31, q_lens, kv, 1, 2, 64, 16, BF16, BF16), products=BF16)


@pytest.mark.parametrize("dim,store", [(128, BF16), (128, E4M3), (256, BF16)])
def test_chunk_large_scores(cuda_device, dim, store):
    check(build(32, [150], [700], 1, 2, dim, 16, BF16, store, k_scale=30.0), scale=1.0,
          products=BF16)


def test_chunk_same_result_every_time(cuda_device):
    case = build(33, [300, 20, 1], [3000, 20, 777], 2, 4, 128, 16, BF16, BF16)
    first = check(case, products=BF16)
    for _ in range(5):
        assert torch.equal(check(case, products=BF16), first)


@pytest.mark.parametrize("store", [BF16, E4M3])
def test_chunk_bad_page(cuda_device, store):
    cache, q, table, kv_lens, starts, kc, vc = build(34, [40, 20], [40, 50], 1, 2, 64, 16, BF16, store)
    bad = table.clone()
    bad[0, 1] = -3
    out = ops.paged_attention(q.cuda(), cache, bad.cuda(), kv_lens.cuda(), starts.cuda(), 40)
    assert ops.attention_status() == 16
    want, _ = ref.paged_attention_ref(q, kc, vc, table, kv_lens, starts, 64 ** -0.5)
    tol, _ = bounds(q, kc, vc, 0.125, BF16, BF16)
    assert (out.cpu().double() - want)[40:].abs().max().item() <= tol
    assert torch.isfinite(out).all()


@pytest.mark.parametrize("store", [BF16, E4M3])
def test_chunk_strides_stream_and_graph(cuda_device, store):
    cache, q, table, kv_lens, starts, kc, vc = build(35, [50, 9], [200, 9], 2, 4, 128, 16, BF16, store)
    wide = torch.zeros(59, 8, 3, 128, dtype=BF16, device="cuda")
    wide[:, :, 1] = q.cuda()
    dt, dl, ds = table.cuda(), kv_lens.cuda(), starts.cuda()
    tol, _ = bounds(q, kc, vc, 128 ** -0.5, BF16, BF16)

    def call():
        ops.paged_attention(wide[:, :, 1], cache, dt, dl, ds, 50, out=wide[:, :, 2])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for lens in ([200, 9], [50, 9], [60, 0]):
        dl.copy_(torch.tensor(lens, dtype=torch.int32))
        wide[:, :, 2] = -1
        graph.replay()
        torch.cuda.synchronize()
        want, _ = ref.paged_attention_ref(q, kc, vc, table, torch.tensor(lens), starts, 128 ** -0.5)
        assert (wide[:, :, 2].cpu().double() - want).abs().max().item() <= tol
    assert (wide[:, :, 0] == 0).all()


# ----------------------------------------------------------------- refusals
def test_refusals(cuda_device):
    x = torch.zeros(4, 256, dtype=BF16, device="cuda")
    w = torch.ones(256, dtype=BF16, device="cuda")
    with pytest.raises(RuntimeError, match="multiple of 8"):
        ops.add_rms_norm(x[:, :12].contiguous(), w[:12].contiguous())
    with pytest.raises(RuntimeError, match="128-wide"):
        ops.add_rms_norm_fp8(x[:, :200].contiguous(), w[:200].contiguous())
    with pytest.raises(RuntimeError, match="scales_ld"):
        ops.add_rms_norm_fp8(x, w, scales_ld=3)
    with pytest.raises(RuntimeError, match="16-byte aligned"):
        ops.add_rms_norm(torch.zeros(4 * 256 + 1, dtype=BF16, device="cuda")[1:].view(4, 256), w)
    with pytest.raises(TypeError, match="bf16 or f16"):
        ops.add_rms_norm(x.float(), w)
    with pytest.raises(ValueError, match="weight"):
        ops.add_rms_norm(x, w[:128])
    with pytest.raises(ValueError, match="residual"):
        ops.add_rms_norm(x, w, residual=x[:3])
    with pytest.raises(ValueError, match="CUDA"):
        ops.add_rms_norm(x.cpu(), w.cpu())
    with pytest.raises(RuntimeError, match="rounded up to 128"):
        ops.w8a8_linear_quantized(torch.zeros(4, 256, device="cuda").to(E4M3),
                                  torch.zeros(2, 4, device="cuda"),
                                  torch.zeros(128, 256, device="cuda").to(E4M3),
                                  torch.zeros(1, 2, device="cuda"))
    with pytest.raises(TypeError, match="float8"):
        kv_cache.PagedKVCache.empty(2, 16, 1, 64, "cuda", torch.float32)
    ok = kv_cache.PagedKVCache.empty(2, 16, 2, 64, "cuda", BF16)
    with pytest.raises(ValueError, match="scales"):
        kv_cache.PagedKVCache(ok.k.to(E4M3), ok.v.to(E4M3))
    with pytest.raises(ValueError, match="alike"):
        kv_cache.PagedKVCache(ok.k, ok.v[:1])
    k = torch.zeros(3, 2, 64, dtype=BF16, device="cuda")
    slots = torch.zeros(3, dtype=torch.int64, device="cuda")
    with pytest.raises(RuntimeError, match="own type"):
        ops.kv_cache_write(ok, k.half(), k.half(), slots)
    with pytest.raises(ValueError, match="slots"):
        ops.kv_cache_write(ok, k, k, slots.int())
    with pytest.raises(ValueError, match="slots"):
        ops.kv_cache_write(ok, k, k, slots[:2])
    with pytest.raises(ValueError, match="k must be"):
        ops.kv_cache_write(ok, k[:, :1], k, slots)
    odd = kv_cache.PagedKVCache(*(torch.zeros(2, 16, 2, 96, dtype=BF16, device="cuda") for _ in "kv"))
    with pytest.raises(RuntimeError, match="head_dim"):
        ops.kv_cache_read(odd, slots)
    q = torch.zeros(3, 4, 64, dtype=BF16, device="cuda")
    i32 = dict(dtype=torch.int32, device="cuda")
    table, lens, starts = torch.zeros(3, 1, **i32), torch.ones(3, **i32), torch.arange(4, **i32)
    with pytest.raises(RuntimeError, match="share"):
        ops.paged_attention(q[:, :3], ok, table, lens, starts, 1)
    with pytest.raises(RuntimeError, match="window"):
        ops.paged_attention(q, ok, table, lens, starts, 1, causal=False, window=4)
    with pytest.raises(RuntimeError, match="own type"):
        ops.paged_attention(q.half(), ok, table, lens, starts, 1)
    with pytest.raises(RuntimeError, match="finite"):
        ops.paged_attention(q, ok, table, lens, starts, 1, scale=math.inf)
    with pytest.raises(RuntimeError, match="workspace"):
        ops.paged_attention(q, ok, table, lens, starts, 1,
                            workspace=torch.zeros(512, dtype=torch.uint8, device="cuda"))
    with pytest.raises(ValueError, match="int32"):
        ops.paged_attention(q, ok, table.long(), lens, starts, 1)
    with pytest.raises(ValueError, match="sequences"):
        ops.paged_attention(q, ok, table, lens, starts[:3], 1)
    # nothing to do is no error
    assert ops.paged_attention(q[:0], ok, table, lens, torch.zeros(4, **i32), 1).shape == (0, 4, 64)
    assert ops.add_rms_norm(x[:0], w)[0].shape == (0, 256)
    ops.kv_cache_write(ok, k[:0], k[:0], slots[:0])
