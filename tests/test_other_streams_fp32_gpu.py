"""The FP32 and integer entry points on a context whose stream is not torch's current one: as test_other_streams_gpu."""
from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu


def _call(c, name):
    import torch

    from onnxsharp_b200 import runtime as r

    rnd = lambda *s: torch.randn(s, device="cuda")  # noqa: E731
    if name == "gemm_bias":
        a, w = rnd(512, 256), r.GemmWeights(c, rnd(256, 1024), 256, 1024)
        call = lambda: r.gemm_bias(c, a, w)  # noqa: E731
    elif name == "matmul_batched":
        a, b = rnd(4, 256, 128), rnd(4, 128, 512)
        call = lambda: r.matmul_batched(c, a, b)  # noqa: E731
    elif name == "conv2d":
        x, w = rnd(2, 32, 80, 80), r.ConvWeights(c, rnd(64, 32, 3, 3), (64, 32, 3, 3))
        call = lambda: r.conv2d(c, x, w, pads=(1, 1, 1, 1))  # noqa: E731
    elif name == "dqmm":
        a = rnd(512, 256)
        w = r.DqmmWeights(c, torch.randint(-127, 128, (256, 1024), dtype=torch.int8, device="cuda"), 256, 1024)
        s = torch.full((1024,), 0.01, device="cuda")
        call = lambda: r.dqmm(c, a, w, s)  # noqa: E731
    else:
        q = rnd(16, 128, 256)
        call = lambda: r.attention(c, q, q, q, heads=4, scale=0.125)  # noqa: E731
    torch.cuda.synchronize()
    return call


@pytest.mark.parametrize("name", ["gemm_bias", "matmul_batched", "conv2d", "dqmm", "attention"])
def test_a_block_that_is_still_read(name):
    import torch

    from onnxsharp_b200.runtime import Context

    c = Context(0)
    call = _call(c, name)
    want = call()
    c.synchronize()
    want = want.clone()
    torch.cuda.synchronize()
    for _ in range(2):
        x = torch.full(want.shape, 3.0, dtype=want.dtype, device="cuda")
        torch.cuda._sleep(20_000_000)
        y = x.clone()
        del x
        got = call()
        c.synchronize()
        torch.cuda.synchronize()
        assert bool((y == 3.0).all()), "written before it was read"
        assert bool((got == want).all())
        del got, y
