"""linear() and attention_window() on a context whose stream is not torch's current one: the results that they allocate
must not lie in memory that kernels on torch's stream still read, nor go back to that stream too early."""
from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu


def _calls(c):
    import torch

    from onnxsharp_b200.runtime import LinearWeights, attention_window, linear

    a, w = torch.randn(512, 256, device="cuda").bfloat16(), torch.randn(256, 1024, device="cuda").bfloat16()
    q, k = torch.randn(64, 8, 16, 64, device="cuda").bfloat16(), torch.randn(64, 50, 4, 64, device="cuda").bfloat16()
    n = torch.full((64,), 50, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    weights = LinearWeights(c, w)
    return {"linear": lambda **kw: linear(c, a, weights, out_dtype=torch.float32, **kw),
            "attention_window": lambda **kw: attention_window(c, q, k, k, n, 0.1, **kw)}


@pytest.mark.parametrize("name", ["linear", "attention_window"])
def test_a_block_that_is_still_read(name):
    import torch

    from onnxsharp_b200.runtime import Context

    c = Context(0)  # its own stream
    call = _calls(c)[name]
    want = call()
    c.synchronize()
    want = want.clone()
    torch.cuda.synchronize()
    for _ in range(3):
        x = torch.full(want.shape, 3.0, dtype=want.dtype, device="cuda")
        torch.cuda._sleep(20_000_000)  # some 10 ms on torch's stream, before x is read
        y = x.clone()
        del x  # its block may be handed out at once: for torch's stream alone
        got = call()
        c.synchronize()
        torch.cuda.synchronize()
        assert bool((y == 3.0).all()), "written before it was read"
        assert bool((got == want).all())
        del got, y


@pytest.mark.parametrize("name", ["linear", "attention_window"])
def test_a_result_that_is_still_read(name):
    """Read on torch's stream after the context has been waited for, then dropped: the next result waits for its turn."""
    import torch

    from onnxsharp_b200.runtime import Context

    c = Context(0)
    call = _calls(c)[name]
    want = call()
    c.synchronize()
    want = want.clone()
    for _ in range(3):
        got = call()
        c.synchronize()
        got.add_(0)
        torch.cuda._sleep(20_000_000)
        kept = got.clone()
        del got
        other = [call().zero_() for _ in range(2)]
        c.synchronize()
        torch.cuda.synchronize()
        assert bool((kept == want).all())
        del other


def test_given_results_are_left_alone():
    import torch

    from onnxsharp_b200.runtime import Context

    c = Context(0)
    for name, call in _calls(c).items():
        want = call()
        c.synchronize()
        out = torch.empty_like(want)
        torch.cuda.synchronize()
        assert call(out=out) is out
        c.synchronize()
        assert bool((out == want).all()), name
