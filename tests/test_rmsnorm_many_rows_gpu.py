"""rmsnorm() of many narrow rows: a warp a row with 16 elements a thread, which few rows are not given, and its
neighbours by width and count. Checks and tolerances as in test_rmsnorm_gpu."""
from __future__ import annotations

import pytest
import test_rmsnorm_gpu as norm

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize(
    "dtype,rows,cols",
    [
        ("f32", 4096, 512), ("f32", 6001, 500), ("f32", 2371, 512), ("f32", 9002, 136), ("f32", 80003, 4),
        ("bf16", 6001, 512), ("bf16", 9001, 264), ("f16", 6001, 512), ("f16", 9001, 264), ("bf16", 40003, 8),
        # several warps a row of 16 elements a thread
        ("f32", 3001, 1000), ("bf16", 5003, 1024), ("f16", 2001, 5120),
    ],
)
@pytest.mark.parametrize("kind", ["", "s8", "e4m3"])
@pytest.mark.parametrize("residual", ["", "kept", "dropped"])
def test_rows(ctx, dtype, rows, cols, kind, residual):
    import torch

    from onnxsharp_b200 import ops

    x, res, gamma = norm._inputs(rows, cols, dtype, bool(residual))
    x[rows // 2] = 0.0
    if residual:
        res[rows // 2] = 0.0
    h = torch.empty((rows, cols), dtype=x.dtype, device="cuda") if residual == "kept" else None
    y = torch.empty((rows + 1, cols), dtype=x.dtype, device="cuda")
    y[-1] = 7.0
    q = s = None
    if kind:
        q = torch.empty((rows + 1, cols), dtype=torch.uint8, device="cuda").view(norm._dt(kind))
        q.view(torch.uint8)[-1] = 11
        s = torch.full((rows + 1,), 13.0, device="cuda")
        ops.rmsnorm_quant(ctx, x, gamma, 1e-6, q[:-1], s[:-1], residual=res, sum_out=h, y=y[:-1])
    else:
        ops.rmsnorm(ctx, x, gamma, 1e-6, y[:-1], residual=res, sum_out=h)
    ctx.synchronize()
    norm._check(x, res, gamma, 1e-6, kind, y[:-1], h, q[:-1] if kind else None, s[:-1] if kind else None)
    assert bool((y[-1] == 7.0).all())
    if kind:
        assert bool((q.view(torch.uint8)[-1] == 11).all()) and s[-1].item() == 13.0
        # without y beside them
        q2, s2 = torch.empty_like(q[:-1]), torch.empty_like(s[:-1])
        ops.rmsnorm_quant(ctx, x, gamma, 1e-6, q2, s2, residual=res, sum_out=h)
        ctx.synchronize()
        assert bool((q2.view(torch.uint8) == q[:-1].view(torch.uint8)).all()) and bool((s2 == s[:-1]).all())
