"""rmsnorm() of rows of many million elements, up to the most that an int counts. The bound does not grow with the
row: 16 squares a time in FP32 (17 * 2^-24), their sums in FP64, ten levels over the threads, else as in
test_rmsnorm_gpu."""
from __future__ import annotations

import pytest
import test_rmsnorm_gpu as norm

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,cols", [("f32", 2**24 + 3), ("f32", 2**27 + 5), ("bf16", 2**27 + 1), ("f16", 2**26)])
def test_equal_elements(ctx, dtype, cols, monkeypatch):
    """Sums of one size lose the most: every addition rounds the same way."""
    import torch

    from onnxsharp_b200 import ops

    x = torch.full((1, cols), 0.1, dtype=norm._dt(dtype), device="cuda")
    y = torch.empty_like(x)
    rel = norm._rel(1024)
    monkeypatch.setattr(norm, "_rel", lambda n: rel)
    q, s = torch.empty(x.shape, dtype=torch.int8, device="cuda"), torch.empty(1, device="cuda")
    ops.rmsnorm_quant(ctx, x, None, 1e-6, q, s, y=y)
    ctx.synchronize()
    norm._check(x, None, None, 1e-6, "s8", y, None, q, s)


def test_the_longest_row(ctx):
    """2^31 - 1 elements: the index steps past what an int holds."""
    import torch

    from onnxsharp_b200 import ops

    cols = 2**31 - 1
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    some = (torch.randn(2**16 - 1, generator=g, device="cuda") * 0.5).bfloat16()
    x = torch.empty((1, cols), dtype=torch.bfloat16, device="cuda")
    whole = cols // some.numel()
    x[0, : whole * some.numel()].view(whole, -1)[:] = some
    x[0, whole * some.numel() :] = some[: cols - whole * some.numel()]
    x[0, -1] = 3.0
    squares = whole * some.double().pow(2).sum() + x[0, whole * some.numel() :].double().pow(2).sum()
    rstd = 1 / (squares / cols + 1e-6).sqrt()
    guard = torch.full((cols + 64,), 7.0, dtype=torch.bfloat16, device="cuda")
    ops.rmsnorm(ctx, x, None, 1e-6, guard[:cols].view(1, cols))
    ctx.synchronize()
    assert bool((guard[cols:] == 7.0).all())
    rel = norm._rel(1024) + 2.0**-8
    for at in (0, cols // 2, 2**31 - 2048, cols - 1000):
        got, ref = guard[at : min(at + 1000, cols)].double(), x[0, at : at + 1000].double() * rstd
        assert bool(((got - ref).abs() <= ref.abs() * rel + 1e-38).all())
