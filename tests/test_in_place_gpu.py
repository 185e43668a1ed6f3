"""rmsnorm() and linear() with the outputs that the header allows in an input's place, for every kernel that takes them.
Checks and tolerances as in test_rmsnorm_gpu and test_linear_gpu."""
from __future__ import annotations

import pytest
import test_linear_gpu as lin
import test_linear_plans_gpu as plans
import test_rmsnorm_gpu as norm

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,cols", [(4, 95), (5000, 512), (4, 512), (700, 4096), (3, 9001), (2, 20000)])
@pytest.mark.parametrize("sum_in,y_in", [("x", "residual"), ("residual", "x"), ("", "residual"), ("", "x"), ("own", "x"),
                                         ("own", "residual"), ("x", ""), ("residual", "")])
@pytest.mark.parametrize("kind", ["", "e4m3"])
def test_norm(ctx, dtype, rows, cols, sum_in, y_in, kind):
    import torch

    from onnxsharp_b200 import ops

    x, res, gamma = norm._inputs(rows, cols, dtype, True)
    x0, res0 = x.clone(), res.clone()
    place = {"x": x, "residual": res, "own": torch.empty_like(x), "": None}
    h, y = place[sum_in], place[y_in]
    if y is None:
        y = torch.empty_like(x)
    q = s = None
    if kind:
        q, s = torch.empty((rows, cols), dtype=norm._dt(kind), device="cuda"), torch.empty(rows, device="cuda")
        ops.rmsnorm_quant(ctx, x, gamma, 1e-6, q, s, residual=res, sum_out=h, y=y)
    else:
        ops.rmsnorm(ctx, x, gamma, 1e-6, y, residual=res, sum_out=h)
    ctx.synchronize()
    norm._check(x0, res0, gamma, 1e-6, kind, y, h, q, s)
    if "x" not in (sum_in, y_in):
        assert bool((x == x0).all())
    if "residual" not in (sum_in, y_in):
        assert bool((res == res0).all())


@pytest.mark.parametrize("kind,out", [("bf16", "bf16"), ("s8", "f32"), ("e4m3", "f16")])
@pytest.mark.parametrize("m,k,n,wide,narrow", plans.PLANS)
def test_product(ctx, kind, out, m, k, n, wide, narrow):
    c = lin.Case(ctx, kind, m, k, n, out=out, residual=True, act="relu")
    y = c.residual.clone()
    c.run(out=y, residual=y)
    ctx.synchronize()
    c.check(y)
