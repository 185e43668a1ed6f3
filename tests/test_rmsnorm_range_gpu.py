"""rmsnorm() at the ends of FP32's range: rows of finite elements whose squares, also scaled down, add up to more than
FP32 holds. Tolerances as in test_rmsnorm_gpu; rstd is a subnormal number there (22 bits at 2^-128): 2^-22 more."""
from __future__ import annotations

import pytest
import test_rmsnorm_gpu as norm

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("kind", ["", "s8", "e4m3"])
@pytest.mark.parametrize("cols", [1, 40, 500, 512, 1000, 4096, 16384, 16385, 40000])
@pytest.mark.parametrize("size", [2.0**62, 2.0**100, 2.0**126, 3.38e38])
def test_large_rows(ctx, dtype, kind, cols, size, monkeypatch):
    import torch

    from onnxsharp_b200 import ops

    g = torch.Generator(device="cuda")
    g.manual_seed(cols)
    x = (torch.rand((5, cols), generator=g, device="cuda") * 2 - 1) * size
    x[1] = size
    x[2] = torch.where(torch.arange(cols, device="cuda") % 7 == 0, size, 1e-3)
    x[3] *= 2.0**-20
    x = x.to(norm._dt(dtype))
    assert bool(x.isfinite().all())
    y = torch.empty_like(x)
    rel = norm._rel
    monkeypatch.setattr(norm, "_rel", lambda n: rel(n) + 2.0**-22)
    if kind:
        q, s = torch.empty(x.shape, dtype=norm._dt(kind), device="cuda"), torch.empty(5, device="cuda")
        ops.rmsnorm_quant(ctx, x, None, 1e-6, q, s, y=y)
        ctx.synchronize()
        norm._check(x, None, None, 1e-6, kind, y, None, q, s)
    else:
        ops.rmsnorm(ctx, x, None, 1e-6, y)
        ctx.synchronize()
        norm._check(x, None, None, 1e-6, "", y)


@pytest.mark.parametrize("cols", [64, 2000, 20000])
def test_a_large_eps_counts_beside_large_rows(ctx, cols):
    import torch

    from onnxsharp_b200 import ops

    x = torch.full((2, cols), 2.0**63, device="cuda")
    x[1] = 2.0**66
    y = torch.empty_like(x)
    ops.rmsnorm(ctx, x, None, 2.0**125, y)
    ctx.synchronize()
    norm._check(x, None, None, 2.0**125, "", y)


@pytest.mark.parametrize("cols", [1, 3, 64, 20000])
def test_the_largest_eps(ctx, cols):
    """Squares and eps each fit FP32, their sum does not."""
    import torch

    from onnxsharp_b200 import ops

    x = torch.full((1, cols), 1.8e19, device="cuda")
    if cols > 3:
        x[0, 1:] = 1e17
    y = torch.empty_like(x)
    ops.rmsnorm(ctx, x, None, 3e38, y)
    ctx.synchronize()
    norm._check(x, None, None, 3e38, "", y)
