"""The norm's e4m3 codes are fp8_act_quant's: the fp32 quotient y / scale, rounded
once, also for quotients on the border between two codes.

Rows of ones have mean(h^2) = 1 and eps = 0, so y is the fp32 weight itself and the
codes can be told bit by bit from the formula in fp32."""

from __future__ import annotations

import pytest
import torch

from sglang_restomod_b200 import ops

pytestmark = pytest.mark.gpu

BF16, F16, E4M3 = torch.bfloat16, torch.float16, torch.float8_e4m3fn


def want(y):
    """(codes, scales) of fp32 columns by groups of 128, in fp32 with IEEE division."""
    groups = y.view(-1, 128)
    scale = (groups.abs().amax(-1) / 448.0).clamp_min(1e-8)
    q = (groups / scale[:, None]).clamp(-448.0, 448.0).to(E4M3)
    return q.view(-1), scale


def borders(g):
    """Numbers next to the borders between codes, times a scale of each group."""
    codes = torch.arange(0x7f, dtype=torch.uint8).view(E4M3).float()
    mid = (codes[:-1] + codes[1:]) / 2  # exact: one more bit than a code has
    scale = torch.rand(256, 1, generator=g) * 2.0 ** torch.randint(-20, 20, (256, 1), generator=g)
    top = 448.0 * scale
    y = mid[torch.randint(0, mid.numel(), (256, 128), generator=g)] * scale
    # the group's largest value sets the scale; then neighbours of each product
    y = (y.view(torch.int32) + torch.randint(-2, 3, y.shape, generator=g)).view(torch.float32)
    y = torch.minimum(y, top)
    y[:, 5] = top[:, 0]
    return (y * torch.where(torch.rand(y.shape, generator=g) < 0.5, -1.0, 1.0)).flatten()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("hidden", [128, 512, 1024, 16384, 32768])
@pytest.mark.parametrize("kind", ["normal", "borders"])
def test_codes_are_the_quotients(cuda_device, dtype, hidden, kind):
    differ = 0
    for seed in range(20):
        g = torch.Generator().manual_seed(seed)
        w = torch.randn(32768, generator=g) if kind == "normal" else borders(g)
        for part in w.split(hidden)[:8]:
            x = torch.ones(3, hidden, dtype=dtype, device="cuda")
            q, s, _ = ops.add_rms_norm_fp8(x, part.cuda(), 0.0)
            codes, scale = want(part)
            assert torch.equal(s.cpu(), scale[:, None].expand(-1, 3))
            for row in q.cpu().view(torch.uint8):
                differ += int((row != codes.view(torch.uint8)).sum())
    assert differ == 0


def test_codes_agree_with_the_activation_quantizer(cuda_device):
    """A 16-bit y has the same codes from both."""
    x = torch.ones(5, 4096, dtype=BF16, device="cuda")
    w = torch.randn(4096, generator=torch.Generator().manual_seed(3)).to(BF16)
    q, s, _ = ops.add_rms_norm_fp8(x, w.cuda(), 0.0)
    q2, s2 = ops.fp8_act_quant(w.expand(5, 4096).contiguous().cuda())
    assert torch.equal(q.view(torch.uint8), q2.view(torch.uint8))
    assert torch.equal(s[:, :5], s2[:, :5])


@pytest.mark.parametrize("rows,hidden", [(1, 128), (700, 512), (3, 7168)])
def test_codes_of_infinities_nan_and_zeros(cuda_device, rows, hidden):
    """A group with an infinity has an infinite scale, zeros and NaN; one with a NaN is
    NaN; zeros keep their signs. (Rows of ones: y is the weight.)"""
    w = torch.randn(hidden, generator=torch.Generator().manual_seed(5))
    w[3], w[5], w[7] = float("inf"), 0.0, -0.0
    if hidden > 128:
        w[130], w[261], w[262] = float("nan"), 0.0, -0.0
    x = torch.ones(rows, hidden, dtype=BF16, device="cuda")
    q, s, _ = ops.add_rms_norm_fp8(x, w.cuda(), 0.0)
    groups = w.view(-1, 128)
    scale = torch.maximum(groups.abs().amax(-1) / 448.0, torch.tensor(1e-8))
    codes = (groups / scale[:, None]).clamp(-448.0, 448.0).to(E4M3).view(-1)
    assert torch.equal(torch.nan_to_num(s.cpu(), nan=-1.0), torch.nan_to_num(
        scale, nan=-1.0)[:, None].expand(-1, rows))
    for row in (q[0].cpu(), q[-1].cpu()):
        nan = torch.isnan(codes.float())
        assert torch.equal(torch.isnan(row.float()), nan)
        assert torch.equal(row.view(torch.uint8)[~nan], codes.view(torch.uint8)[~nan])


@pytest.mark.parametrize("hidden", [128, 1024, 4096])
def test_both_outputs_are_one_norm(cuda_device, hidden):
    g = torch.Generator().manual_seed(hidden)
    x, r = (torch.randn(37, hidden, generator=g).to(BF16).cuda() for _ in "xr")
    w = torch.randn(hidden, generator=g).cuda()
    y, h = ops.add_rms_norm(x, w, residual=r)
    both = torch.empty_like(x)
    q, s, h2 = ops.add_rms_norm_fp8(x, w, residual=r, out=both)
    q3, s3, _ = ops.add_rms_norm_fp8(x, w, residual=r)
    assert torch.equal(both, y) and torch.equal(h, h2)
    assert torch.equal(q.view(torch.uint8), q3.view(torch.uint8)) and torch.equal(s, s3)
