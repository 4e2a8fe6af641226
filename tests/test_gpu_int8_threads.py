"""The integer linear's entries from several threads, each on a stream of its own, from the
first call of each kernel on."""

from __future__ import annotations

import threading

import pytest
import torch

from sglang_restomod_b200 import ops, synth

pytestmark = pytest.mark.gpu


def test_both_entries_from_threads(cuda_device):
    """Sizes of every tile width, in other orders by thread."""
    sizes = [1, 20, 50, 100, 300]
    (w,), (ws,) = synth.int8_bank(1, 1000, 2048, cuda_device, 3)
    xs = [synth.activations(m, 2048, cuda_device, seed=m) for m in sizes]
    codes = [ops.int8_act_quant(x) for x in xs]
    torch.cuda.synchronize()
    got, gate = [], threading.Barrier(4)

    def work(n):
        stream = torch.cuda.Stream()
        gate.wait(20)
        with torch.cuda.stream(stream):
            for i in range(20):
                at = (i + n) % len(sizes)
                y = ops.int8_linear(xs[at], w, ws) if n % 2 else \
                    ops.int8_linear_quantized(*codes[at], w, ws)
                got.append((at, y))
        stream.synchronize()

    threads = [threading.Thread(target=work, args=(n,)) for n in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    assert len(got) == 80
    wants = [(q.double() @ w.double().T) * s.double()[:, None] * ws.double() for q, s in codes]
    for at, y in got:
        # the output's rounding, and two in fp32
        bound = wants[at].abs() * (2.0 ** -8 + 2.0 ** -22)
        assert bool(((y.double() - wants[at]).abs() <= bound).all())
        assert torch.equal(y, ops.int8_linear(xs[at], w, ws))
    assert ops.attention_status() == 0
