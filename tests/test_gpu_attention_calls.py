"""Norm, key/value cache and paged attention as calls: several threads, status
bits, workspaces."""

from __future__ import annotations

import threading

import pytest
import torch

from sglang_restomod_b200 import ops, synth
from tests.test_gpu_attention import BF16, E4M3, build

pytestmark = pytest.mark.gpu


def on_gpu(case, max_q, **kw):
    cache, q, table, kv_lens, starts = case[:5]
    args = (q.cuda(), cache, table.cuda(), kv_lens.cuda(), starts.cuda(), max_q)
    return lambda: ops.paged_attention(*args, **kw)


def in_fresh_thread(call):
    """The result of a thread's very first call."""
    got = []
    t = threading.Thread(target=lambda: got.append(call()))
    t.start()
    t.join(60)
    assert got, "the call raised"
    return got[0]


def test_first_call_of_a_thread(cuda_device):
    """A thread without a CUDA context of its own takes the same kernels: the same
    bits from decode, and no refusal from the linear."""
    decode = on_gpu(build(44, [1] * 5, [900, 3, 0, 77, 40], 2, 8, 128, 16, BF16, E4M3), 1)
    assert torch.equal(decode(), in_fresh_thread(decode))
    wq, ws = synth.fp8_bank(1, 256, 512, cuda_device, seed=2)
    q, s, _ = ops.add_rms_norm_fp8(synth.activations(45, 512, cuda_device, seed=3),
                                   torch.ones(512, dtype=BF16, device="cuda"),
                                   scales_ld=ops.w8a8_scales_ld(45))
    linear = lambda: ops.w8a8_linear_quantized(q, s, wq[0], ws[0])  # noqa: E731
    torch.cuda.synchronize()
    assert torch.equal(linear(), in_fresh_thread(linear))


def test_threads_on_one_stream(cuda_device):
    """Calls of several threads on one stream share its workspace; each call's
    launches stay together (chunk calls plan in one and attend in the next)."""
    calls = [on_gpu(build(41, [90, 3], [400, 700], 2, 4, 128, 16, BF16, BF16), 90),
             on_gpu(build(42, [20] * 9, [20 + 31 * i for i in range(9)], 1, 3, 64, 8, BF16, BF16), 20),
             on_gpu(build(43, [130], [130], 1, 2, 128, 1, BF16, E4M3), 130),
             on_gpu(build(44, [1] * 5, [900, 3, 0, 77, 40], 2, 8, 128, 16, BF16, E4M3), 1)]
    wants = [call() for call in calls]
    torch.cuda.synchronize()
    wrong, gate = [], threading.Barrier(len(calls))

    def work(call, want):
        gate.wait(20)
        got = [call() for _ in range(60)]
        torch.cuda.current_stream().synchronize()
        wrong.extend(not torch.equal(g, want) for g in got)

    threads = [threading.Thread(target=work, args=pair) for pair in zip(calls, wants)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    assert len(wrong) == 60 * len(calls) and not any(wrong)
    assert ops.attention_status() == 0
