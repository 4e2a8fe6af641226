"""Norm, key/value cache and paged attention as calls: several threads, status
bits, workspaces."""

from __future__ import annotations

import os
import subprocess
import sys
import threading
from pathlib import Path

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


@pytest.mark.parametrize("store", [BF16, E4M3])
@pytest.mark.parametrize("q_len", [1, 40])
@pytest.mark.parametrize("reserved", [False, True])
def test_errors_of_replayed_graphs_are_seen(cuda_device, store, q_len, reserved):
    cache, q, table, kv_lens, starts = build(45, [q_len, 1], [90, 33], 1, 4, 64, 16, BF16, store)[:5]
    args = (q.cuda(), cache, table.cuda(), kv_lens.cuda(), starts.cuda(), q_len)
    ops.paged_attention(*args)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    if reserved:
        with torch.cuda.stream(side):
            ops.reserve_attention_workspace(64, q.shape[0], 2)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = ops.paged_attention(*args)
    graph.replay()
    assert ops.attention_status() == 0
    want = out.clone()
    args[2][1, 0] = cache.num_pages + 7
    graph.replay()
    assert ops.attention_status(reset=False) == 16
    assert ops.attention_status() == 16
    assert ops.attention_status() == 0
    args[2][1, 0] = table[1, 0].item()
    graph.replay()
    assert ops.attention_status() == 0 and torch.equal(out, want)


def test_errors_outlive_their_workspace(cuda_device):
    cache, q, table, kv_lens, starts = build(46, [1, 1], [90, 33], 1, 4, 64, 16, BF16, BF16)[:5]
    ws = torch.zeros(ops.paged_attention_workspace_bytes(64, 2, 2), dtype=torch.uint8, device="cuda")
    bad = table.cuda()
    bad[0, 2] = -1
    ops.paged_attention(q.cuda(), cache, bad, kv_lens.cuda(), starts.cuda(), 1, workspace=ws)
    assert int(ws[:4].view(torch.int32)) == 16  # the call's own word has it too
    del ws
    assert ops.attention_status() == 16 and ops.attention_status() == 0


FIRST_CALL_IN_A_CAPTURE = """
import torch
from sglang_restomod_b200 import kv_cache, ops
x = torch.ones(3, 7168, dtype=torch.bfloat16, device="cuda")
w = torch.ones(7168, dtype=torch.bfloat16, device="cuda")
cache = kv_cache.PagedKVCache.empty(4, 16, 1, 64, "cuda", torch.bfloat16)
cache.k.zero_(), cache.v.zero_()
i32 = dict(dtype=torch.int32, device="cuda")
q = torch.ones(3, 4, 64, dtype=torch.bfloat16, device="cuda")
args = torch.zeros(3, 1, **i32), torch.ones(3, **i32), torch.arange(4, **i32), 1
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    y, _ = ops.add_rms_norm(x, w)
    o = ops.paged_attention(q, cache, *args)
graph.replay()
torch.cuda.synchronize()
assert (y == 1).all() and (o == 0).all() and ops.attention_status() == 0
"""


def test_first_call_of_a_process_in_a_capture(cuda_device):
    env = {**os.environ, "PYTHONPATH": str(Path(ops.__file__).resolve().parents[1])}
    done = subprocess.run([sys.executable, "-c", FIRST_CALL_IN_A_CAPTURE], env=env,
                          capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr


def test_workspaces_of_growing_batches(cuda_device):
    """What larger workspaces have replaced stays below the present one."""
    def kept():
        return sum(t.numel() for t in ops._ATTN_OUTGROWN)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        before = kept()
        sizes = {ops.reserve_attention_workspace(dim, 1 << n, 1 << max(0, n - 4)).numel()
                 for dim in (64, 256, 128) for n in range(19)}
        assert len(sizes) <= 3
        present = ops.reserve_attention_workspace(128, 1, 1)
        assert kept() - before < present.numel()
        assert present.numel() < 2 * ops.paged_attention_workspace_bytes(128, 1 << 18, 1 << 14)
    # a graph that holds an outgrown workspace still answers
    case = build(47, [60, 2], [200, 40], 1, 4, 128, 16, BF16, BF16)
    call = on_gpu(case, 60)
    want = call()
    torch.cuda.synchronize()
    other = torch.cuda.Stream()
    with torch.cuda.stream(other):
        ops.reserve_attention_workspace(128, 62, 2)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=other):
        out = call()
    with torch.cuda.stream(other):
        first = ops.reserve_attention_workspace(128, 62, 2)
        assert ops.reserve_attention_workspace(128, 1 << 18, 2).numel() >= 2 * first.numel()
        junk = torch.full((first.numel(),), 255, dtype=torch.uint8, device="cuda")
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want) and ops.attention_status() == 0 and junk.numel()


def test_quantized_linear_refuses_operands_that_do_not_fit(cuda_device):
    def zeros(*shape, dtype=torch.float32):
        return torch.zeros(*shape, device="cuda").to(dtype)

    q, s = zeros(4, 256, dtype=E4M3), zeros(2, 128)
    w, ws = zeros(384, 256, dtype=E4M3), zeros(3, 2)
    assert ops.w8a8_linear_quantized(q, s, w, ws).shape == (4, 384)
    for bad in (zeros(2, 2), zeros(3, 1), zeros(6)[:5]):
        with pytest.raises(ValueError, match="scales"):
            ops.w8a8_linear_quantized(q, s, w, bad)
    with pytest.raises(ValueError, match="weight must be"):
        ops.w8a8_linear_quantized(q, s, zeros(2, 384, 256, dtype=E4M3), ws)
    with pytest.raises(ValueError, match="scales"):
        ops.w8a8_linear_quantized(q, zeros(256), w, ws)
    with pytest.raises(ValueError, match="K differs"):
        ops.w8a8_linear_quantized(q, zeros(3, 128), w, ws)
