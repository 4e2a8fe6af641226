"""The 8-bit integer linear against whole-number sums in 64 bits.

The codes must be equal: the definition's two divisions are fp32. An output is
the exact sum brought to fp32 (2^-24), two products (2^-24 each) and the output's
own rounding: at most 3 * 2^-24 + eps / 2 of the value, eps / 2 = 2^-8 (bf16) or
2^-11 (f16), and half of f16's smallest step, 2^-25."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import int8 as oracle
from sglang_restomod_b200 import ops

pytestmark = pytest.mark.gpu


def inputs(m, n, k, dtype, seed=0, low=-127):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(m, k, generator=g, device="cuda")
    x *= torch.exp(torch.randn(k, generator=g, device="cuda"))
    w = torch.randint(low, 128, (n, k), generator=g, device="cuda", dtype=torch.int8)
    ws = torch.rand(n, generator=g, device="cuda") * 1e-3 + 1e-5
    return x.to(dtype), w, ws


def check(y, q, s, w, ws):
    want = torch.from_numpy(oracle.linear(q.cpu().numpy(), s.cpu().numpy(), w.cpu().numpy(),
                                          ws.cpu().numpy()))
    half = 2.0 ** -8 if y.dtype == torch.bfloat16 else 2.0 ** -11
    off = (y.double().cpu() - want).abs()
    bound = want.abs() * (half + 3 * 2.0 ** -24) * (1 + 2.0 ** -8) + 2.0 ** -25
    assert bool((off <= bound).all()), (off / bound).max()


SIZES = [(1, 1, 16), (1, 128, 128), (1, 5120, 25600), (2, 7, 16400), (3, 130, 144), (16, 129, 256),
         (17, 1000, 2064), (33, 300, 4112), (64, 64, 640), (65, 1021, 1008), (77, 7164, 2048),
         (127, 384, 4096), (128, 256, 16), (129, 2000, 512), (200, 515, 7168), (256, 640, 640),
         (257, 1153, 1040), (513, 4099, 272), (1000, 1000, 1008), (2300, 3071, 400)]


@pytest.mark.parametrize("m,n,k", SIZES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
def test_linear(cuda_device, m, n, k, dtype):
    x, w, ws = inputs(m, n, k, dtype, seed=m + n + k, low=-128)
    q, s = ops.int8_act_quant(x)
    want_q, want_s = oracle.quantize(x.float().cpu().numpy())
    assert np.array_equal(q.cpu().numpy(), want_q)
    assert np.array_equal(s.cpu().numpy(), want_s)
    y = ops.int8_linear(x, w, ws)
    assert y.dtype == dtype and y.shape == (m, n)
    check(y, q, s, w, ws)
    other = torch.float16 if dtype == torch.bfloat16 else torch.bfloat16
    z = ops.int8_linear_quantized(q, s, w, ws, out_dtype=dtype)
    assert torch.equal(y, z)  # the same sums, whatever the cut
    check(ops.int8_linear(x, w, ws, out_dtype=other), q, s, w, ws)
    assert ops.attention_status() == 0


def test_largest_sums(cuda_device):
    """131072 products of -128 and 127: the sum is the nearest that int32 comes to its end."""
    k = 131072
    q = torch.full((5, k), 127, dtype=torch.int8, device="cuda")
    w = torch.full((130, k), -128, dtype=torch.int8, device="cuda")
    s = torch.tensor([1.0, 2.0 ** -20, 0.0, 3.0, 1e-30], device="cuda")
    ws = torch.full((130,), 2.0 ** -24, device="cuda")
    check(ops.int8_linear_quantized(q, s, w, ws), q, s, w, ws)


@pytest.mark.parametrize("m,k", [(1, 8192), (5, 64), (9, 4096), (300, 4112), (1, 40000), (2, 131072)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
def test_rows_out_of_the_ordinary(cuda_device, m, k, dtype):
    """Zeros, one value, the smallest and largest magnitudes, halves between codes,
    infinities and NaN."""
    x = torch.zeros(m, k, dtype=torch.float64)
    g = torch.Generator().manual_seed(k)
    lo, hi = (2.0 ** -133, 3e38) if dtype == torch.bfloat16 else (2.0 ** -24, 65504.0)
    rows = [lambda r: r.zero_(), lambda r: r.fill_(lo), lambda r: r.fill_(-hi),
            lambda r: r.copy_(torch.randint(-254, 255, (k,), generator=g) / 2.0),
            lambda r: r.copy_(torch.randn(k, generator=g, dtype=torch.float64) * lo * 4),
            lambda r: r.copy_(torch.randn(k, generator=g)).__setitem__(k - 1, float("inf")),
            lambda r: r.copy_(torch.randn(k, generator=g)).__setitem__(k // 2, float("nan")),
            lambda r: r.fill_(1.0).__setitem__(0, 127.0)]
    for i in range(m):
        rows[(i + (m == 1) * 3) % len(rows)](x[i])
    x = x.to(dtype).cuda()
    q, s = ops.int8_act_quant(x)
    want_q, want_s = oracle.quantize(x.float().cpu().numpy())
    assert np.array_equal(q.cpu().numpy(), want_q)
    assert np.array_equal(s.cpu().numpy(), want_s, equal_nan=True)
    w = torch.ones(3, k, dtype=torch.int8, device="cuda")
    y = ops.int8_linear(x, w, torch.ones(3, device="cuda"), out_dtype=torch.bfloat16)
    assert torch.equal(y.isnan().all(1).cpu(), torch.from_numpy(np.isnan(want_s)))
    assert torch.equal(y.isnan().any(1).cpu(), torch.from_numpy(np.isnan(want_s)))


def test_no_tokens_and_three_dimensions(cuda_device):
    x, w, ws = inputs(6, 40, 96, torch.bfloat16)
    assert ops.int8_linear(x[:0], w, ws).shape == (0, 40)
    assert ops.int8_act_quant(x[:0])[0].shape == (0, 96)
    y = ops.int8_linear(x.view(2, 3, 96), w, ws)
    assert y.shape == (2, 3, 40) and torch.equal(y.view(6, 40), ops.int8_linear(x, w, ws))


@pytest.mark.parametrize("m", [1, 40, 700])
def test_captured_and_on_two_streams(cuda_device, m):
    """A graph's replays see new activations and weights; two streams do not meet."""
    x, w, ws = inputs(m, 1100, 2064, torch.bfloat16)
    x2, w2, ws2 = inputs(m, 1100, 2064, torch.bfloat16, seed=1)
    want, want2 = ops.int8_linear(x, w, ws), ops.int8_linear(x2, w2, ws2)
    out = torch.empty_like(want)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        ops.int8_linear(x, w, ws, out=out)
    graph.replay()
    assert torch.equal(out, want)
    for a, b in ((x, x2), (w, w2), (ws, ws2)):
        a.copy_(b)  # ordered before the replay, which reads the weight early
    graph.replay()
    assert torch.equal(out, want2)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for i in range(8):
        with torch.cuda.stream(streams[i & 1]):
            got.append(ops.int8_linear(x2, w2, ws2))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want2) for g in got)


def test_more_than_two_to_the_31_elements(cuda_device):
    """Offsets of outputs and weights past 2^31."""
    m, n, k = 70000, 31000, 16
    x, w, ws = inputs(m, n, k, torch.bfloat16)
    y = ops.int8_linear(x, w, ws)
    q, s = ops.int8_act_quant(x)
    for rows in (slice(0, 3), slice(34000, 34002), slice(m - 2, m)):
        check(y[rows], q[rows], s[rows], w, ws)
