"""rmsnorm() and rmsnorm_quant() against the formula in float64.

h is compared bit for bit (one FP32 addition, one rounding). y: the sum of squares adds at most (16 + 10) * 2^-24
relative (16 elements a thread, ten levels of the tree; a row read by one thread more often: cols / 1024), half of it
through the root, then the quotient, the root's approximation (2^-22) and two products; half a step of y's type. The
codes are functions of exact products: they have to be equal, borders included. A scale: what y has and the quotient."""
from __future__ import annotations

import math

import pytest

pytestmark = pytest.mark.gpu
TOP = {"s8": 127.0, "e4m3": 448.0}


def _dt(name):
    import torch

    return {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16, "e4m3": torch.float8_e4m3fn,
            "s8": torch.int8}[name]


def _codes64(t, kind):
    """Codes of t [rows, cols] (float64, exact products) from the definition: nearest, ties to the even code."""
    import torch

    peak = t.abs().amax(dim=1, keepdim=True)
    r = t * TOP[kind] / torch.where(peak > 0, peak, torch.ones_like(peak))
    if kind == "s8":
        return r.round().to(torch.int8), peak[:, 0]
    grid = torch.arange(127, device=t.device, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    mid = (grid[1:] + grid[:-1]) / 2
    lo, hi = torch.bucketize(r.abs(), mid), torch.bucketize(r.abs(), mid, right=True)
    mag = grid[torch.where(lo % 2 == 0, lo, hi)]
    return torch.where(r < 0, -mag, mag).to(torch.float8_e4m3fn), peak[:, 0]


def _rel(cols):
    return (math.ceil(cols / 1024) + 16 + 10) * 2.0**-25 + 2.0**-22 + 4 * 2.0**-24


def _reference(x, res, gamma, eps):
    h = x if res is None else (x.float() + res.float()).to(x.dtype)
    v = h.double()
    rstd = 1 / (v.pow(2).mean(dim=1, keepdim=True) + eps).sqrt()
    t = v * (gamma.double() if gamma is not None else 1.0)
    return h, t, rstd


def _check(x, res, gamma, eps, kind, y=None, h=None, q=None, scales=None):
    import torch

    rh, t, rstd = _reference(x, res, gamma, eps)
    rel = _rel(x.shape[1])
    if h is not None:
        assert bool((h == rh).all())
    if y is not None:
        ref = t * rstd
        half = torch.finfo(x.dtype).eps / 2
        tol = ref.abs() * (rel + half * 1.001) + torch.finfo(x.dtype).smallest_normal * half
        assert bool(((y.double() - ref).abs() <= tol).all()), ((y.double() - ref).abs() / tol).max().item()
    if q is not None:
        code, peak = _codes64(t, kind)
        assert bool((q.double() == code.double()).all()), (q.double() != code.double()).sum().item()
        s = torch.where(peak > 0, peak * rstd[:, 0] / TOP[kind], torch.ones_like(peak))
        assert bool(((scales.double() - s).abs() <= s * (rel + 2.0**-23)).all())


def _inputs(rows, cols, dtype, residual, pad=0, seed=0, shift=0):
    import torch

    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 7919 + rows * 31 + cols)

    def rows_of():
        buf = torch.full((rows * (cols + pad) + shift,), math.nan, dtype=_dt(dtype), device="cuda")
        v = buf[shift:].view(rows, cols + pad)[:, :cols]
        v.copy_(torch.randn((rows, cols), generator=g, device="cuda") * torch.rand(cols, generator=g, device="cuda") * 3)
        return v

    gamma = (1 + 0.3 * torch.randn(cols, generator=g, device="cuda")).to(_dt(dtype))
    return rows_of(), rows_of() if residual else None, gamma


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("kind", ["", "s8", "e4m3"])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 4096), (3, 7), (5, 64), (33, 512), (9, 513), (130, 1001), (7, 4096),
                                       (3, 5120), (2, 16384), (2, 16385), (3, 20000)])
@pytest.mark.parametrize("residual", [False, True])
def test_sizes(ctx, dtype, kind, rows, cols, residual):
    import torch

    from onnxsharp_b200 import ops

    x, res, gamma = _inputs(rows, cols, dtype, residual)
    h = torch.empty((rows, cols), dtype=x.dtype, device="cuda") if residual else None
    y = torch.empty((rows, cols), dtype=x.dtype, device="cuda")
    if kind:
        q, s = torch.empty((rows, cols), dtype=_dt(kind), device="cuda"), torch.empty(rows, device="cuda")
        ops.rmsnorm_quant(ctx, x, gamma, 1e-6, q, s, residual=res, sum_out=h, y=y)
        ctx.synchronize()
        _check(x, res, gamma, 1e-6, kind, y, h, q, s)
    else:
        ops.rmsnorm(ctx, x, gamma, 1e-6, y, residual=res, sum_out=h)
        ctx.synchronize()
        _check(x, res, gamma, 1e-6, kind, y, h)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("pad,shift", [(8, 0), (8, 3), (1, 0), (5, 16)])
@pytest.mark.parametrize("cols", [256, 300, 2048])
def test_pitches_and_alignment(ctx, dtype, pad, shift, cols):
    import torch

    from onnxsharp_b200 import ops

    rows = 11
    x, res, gamma = _inputs(rows, cols, dtype, True, pad, shift=shift)
    wide = torch.full((rows + 2, cols + 24), 5.0, dtype=x.dtype, device="cuda")
    y = wide[1:-1, 16:-8]
    qw = torch.full((rows + 2, cols + 24), 3, dtype=torch.int8, device="cuda")
    q, s = qw[1:-1, 16:-8], torch.empty(rows, device="cuda")
    ops.rmsnorm_quant(ctx, x, gamma, 1e-5, q, s, residual=res, y=y)
    ctx.synchronize()
    _check(x, res, gamma, 1e-5, "s8", y, None, q, s)
    wide[1:-1, 16:-8] = 5.0
    qw[1:-1, 16:-8] = 3
    assert bool((wide == 5.0).all()) and bool((qw == 3).all())


@pytest.mark.parametrize("cols", [96, 3000, 18000])
@pytest.mark.parametrize("into", ["residual", "x"])
def test_the_stream_in_place(ctx, cols, into):
    import torch

    from onnxsharp_b200 import ops

    x, res, gamma = _inputs(4, cols, "bf16", True)
    x0, r0 = x.clone(), res.clone()
    q, s = torch.empty((4, cols), dtype=torch.int8, device="cuda"), torch.empty(4, device="cuda")
    ops.rmsnorm_quant(ctx, x, gamma, 1e-6, q, s, residual=res, sum_out=res if into == "residual" else x)
    ctx.synchronize()
    _check(x0, r0, gamma, 1e-6, "s8", None, res if into == "residual" else x, q, s)
    x, _, gamma = _inputs(4, cols, "f16", False)
    x0 = x.clone()
    ops.rmsnorm(ctx, x, gamma, 1e-6, x)
    ctx.synchronize()
    _check(x0, None, gamma, 1e-6, "", x)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("kind", ["s8", "e4m3"])
@pytest.mark.parametrize("cols", [254, 2032, 17000])
def test_codes_on_borders(ctx, dtype, kind, cols):
    """Rows whose ratios lie exactly on the middle between two codes: to the even one."""
    import torch

    from onnxsharp_b200 import ops

    top = TOP[kind]
    if kind == "s8":
        v = (torch.arange(cols, device="cuda") % 254 - 127).double() + 0.5  # -126.5 .. 126.5
        v = torch.where(v.abs() > 126.5, torch.full_like(v, top), v)
    else:
        grid = torch.arange(127, device="cuda", dtype=torch.uint8).view(torch.float8_e4m3fn).double()
        v = ((grid[1:] + grid[:-1]) / 2)[torch.arange(cols, device="cuda") % 126]
    v[0] = top
    x = torch.stack([v, -v, v * 0.25, v * 2.0**40 if dtype == "f32" else v]).to(_dt(dtype))
    q, s = torch.empty(x.shape, dtype=_dt(kind), device="cuda"), torch.empty(4, device="cuda")
    ops.rmsnorm_quant(ctx, x, None, 1e-6, q, s)
    ctx.synchronize()
    _check(x, None, None, 1e-6, kind, None, None, q, s)
    # the same with weights that make the products inexact in FP32
    gamma = (1 + torch.rand(cols, device="cuda")).to(x.dtype)
    ops.rmsnorm_quant(ctx, x, gamma, 1e-6, q, s)
    ctx.synchronize()
    _check(x, None, gamma, 1e-6, kind, None, None, q, s)


def test_many_codes(ctx):
    """16 million codes: what FP32 cannot decide is decided."""
    import torch

    from onnxsharp_b200 import ops

    for dtype, kind in (("f32", "s8"), ("bf16", "s8"), ("f16", "e4m3"), ("f32", "e4m3")):
        x, _, gamma = _inputs(4096, 1024, dtype, False, seed=3)
        q, s = torch.empty(x.shape, dtype=_dt(kind), device="cuda"), torch.empty(4096, device="cuda")
        ops.rmsnorm_quant(ctx, x, gamma, 1e-6, q, s)
        ctx.synchronize()
        _check(x, None, gamma, 1e-6, kind, None, None, q, s)


@pytest.mark.parametrize("cols", [40, 4000, 18000])
def test_rows_without_a_usable_maximum(ctx, cols):
    import torch

    from onnxsharp_b200 import ops

    x = torch.randn(6, cols, device="cuda")
    x[0] = 0.0
    x[1] = 1e-30
    x[2, 5] = math.nan
    x[3, 6] = math.inf
    x[4] = x[4] * 1e30  # squares overflow, the row does not
    gamma = torch.ones(cols, device="cuda")
    q, s, y = torch.full((6, cols), 9, dtype=torch.int8, device="cuda"), torch.empty(6, device="cuda"), torch.empty_like(x)
    ops.rmsnorm_quant(ctx, x, gamma, 1e-6, q, s, y=y)
    ctx.synchronize()
    assert not bool(q[:4].any()) and s[:2].tolist() == [1.0, 1.0] and bool(s[2:4].isnan().all())
    assert not bool(y[0].any()) and bool(y[2].isnan().all())
    assert bool(y[3, 6].isnan()) and not bool(y[3, 7:].any())
    _check(x[4:], None, gamma, 1e-6, "s8", y[4:], None, q[4:], s[4:])


def test_no_rows_and_leading_dimensions(ctx):
    import torch

    from onnxsharp_b200 import ops

    before = ctx.launch_count()
    e = torch.empty((0, 64), device="cuda")
    ops.rmsnorm(ctx, e, torch.ones(64, device="cuda"), 1e-6, torch.empty_like(e))
    assert ctx.launch_count() == before
    x, _, gamma = _inputs(30, 96, "bf16", False)
    y = torch.empty((2, 3, 5, 96), dtype=torch.bfloat16, device="cuda")
    ops.rmsnorm(ctx, x.view(2, 3, 5, 96), gamma, 1e-6, y)
    ctx.synchronize()
    _check(x, None, gamma, 1e-6, "", y.view(30, 96))


def test_captured_and_replayed(ctx):
    import torch

    from onnxsharp_b200 import ops
    from onnxsharp_b200.runtime import Context

    stream = torch.cuda.Stream()
    c = Context(0, stream.cuda_stream)
    x, res, gamma = _inputs(64, 1024, "bf16", True)
    q, s, h = torch.empty((64, 1024), dtype=torch.int8, device="cuda"), torch.empty(64, device="cuda"), torch.empty_like(x)
    torch.cuda.synchronize()
    g = c.capture(lambda: ops.rmsnorm_quant(c, x, gamma, 1e-6, q, s, residual=res, sum_out=h))
    x.mul_(2)
    torch.cuda.synchronize()
    g.launch()
    c.synchronize()
    _check(x, res, gamma, 1e-6, "s8", None, h, q, s)
    g.close()
    c.close()


def test_refusals(ctx):
    import torch

    from onnxsharp_b200 import OscError, ops

    x, res, gamma = _inputs(4, 64, "bf16", True)
    y = torch.empty_like(x)
    q, s = torch.empty((4, 64), dtype=torch.int8, device="cuda"), torch.empty(4, device="cuda")
    with pytest.raises(OscError, match="eps"):
        ops.rmsnorm(ctx, x, gamma, 0.0, y)
    with pytest.raises(OscError, match="eps"):
        ops.rmsnorm(ctx, x, gamma, math.nan, y)
    with pytest.raises(OscError, match="without a residual"):
        ops.rmsnorm(ctx, x, gamma, 1e-6, y, sum_out=res)
    with pytest.raises(OscError, match="code type"):
        ops.rmsnorm_quant(ctx, x, gamma, 1e-6, y, s)
    with pytest.raises(OscError, match="come together"):
        ops.rmsnorm_quant(ctx, x, gamma, 1e-6, q, None)
    with pytest.raises(TypeError, match="y is"):
        ops.rmsnorm(ctx, x, gamma, 1e-6, torch.empty((4, 64), device="cuda"))
    with pytest.raises(ValueError, match="expected"):
        ops.rmsnorm(ctx, x, gamma, 1e-6, y[:3])
    with pytest.raises(ValueError, match="gamma"):
        ops.rmsnorm(ctx, x, gamma[:63], 1e-6, y)
    with pytest.raises(ValueError, match="pitch"):
        ops.rmsnorm(ctx, x.t(), gamma, 1e-6, y.t())
    with pytest.raises(ValueError, match="cpu"):
        ops.rmsnorm(ctx, x.cpu(), gamma, 1e-6, y)
    with pytest.raises(TypeError, match="float64"):
        d = torch.zeros((4, 64), dtype=torch.float64, device="cuda")
        ops.rmsnorm(ctx, d, d[0], 1e-6, d)
