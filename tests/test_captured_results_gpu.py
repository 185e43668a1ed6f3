"""Calls that allocate their result, captured on a context whose stream is not torch's current one, after eager calls of
the same kind whose results have been dropped: torch's allocator must have nothing to ask the device during the capture."""
from __future__ import annotations

import pytest
import test_other_streams_gpu as other
import test_other_streams_fp32_gpu as fp32

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name", ["linear", "attention_window", "gemm_bias", "matmul_batched", "conv2d", "dqmm", "attention"])
@pytest.mark.parametrize("busy", [False, True])
def test_capture(name, busy):
    import torch

    from onnxsharp_b200.runtime import Context

    c = Context(0)
    call = other._calls(c)[name] if name in ("linear", "attention_window") else fp32._call(c, name)
    want = call()
    c.synchronize()
    want = want.clone()
    for _ in range(3):
        call()  # dropped at once
    kept = []
    if busy:  # work on torch's stream that the dropped results would be held back for
        torch.cuda._sleep(200_000_000)
        for _ in range(3):
            call()
    graph = c.capture(lambda: kept.append(call()))
    kept[-1].zero_()
    torch.cuda.synchronize()
    graph.launch()
    c.synchronize()
    assert bool((kept[-1] == want).all())
    graph.close()
    torch.cuda.synchronize()
    c.close()
