"""linear(): bf16, fp16, e4m3 and s8 products with scales, bias, activation and residual in the epilogue, against the
same formula in float64.

Tolerances count roundings. An FP32 sum on the tensor cores is off by at most one unit of the largest partial sum's
24th bit for each MMA step (32 bytes of K), and the partial sums stay below S = sum |a w|: STEP = 2^-22 * S a step (one
bit for the alignment of the products, one for the sum). S32 sums are exact. The epilogue rounds the sum, the scales'
product, their product with the sum, the bias' and the residual's addition (2^-24 each), the activations come from
instructions good to 4e-6, every activation's slope is below 1.2, and the output is off by half a step of its type."""
from __future__ import annotations

import math

import pytest

pytestmark = pytest.mark.gpu

KINDS = ["bf16", "f16", "e4m3", "s8"]
ACTS = {"none": 0, "silu": 1, "relu": 2, "sigmoid": 3, "gelu": 4, "gelu_tanh": 5}


def _dt(name):
    import torch

    return {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16, "e4m3": torch.float8_e4m3fn,
            "s8": torch.int8}[name]


def _operand(g, shape, kind):
    import torch

    v = torch.randn(shape, generator=g, device="cuda")
    if kind == "s8":
        return (v * 40).round().clamp(-128, 127).to(torch.int8)
    if kind == "e4m3":
        return (v * 100).clamp(-448, 448).to(torch.float8_e4m3fn)
    return v.to(_dt(kind))


def _act64(v, act):
    import torch

    if act == "silu":
        return v * torch.sigmoid(v)
    if act == "relu":
        return v.clamp(min=0)
    if act == "sigmoid":
        return torch.sigmoid(v)
    if act == "gelu":
        return 0.5 * v * torch.erfc(-v / math.sqrt(2))
    if act == "gelu_tanh":
        return 0.5 * v * (1 + torch.tanh(math.sqrt(2 / math.pi) * (v + 0.044715 * v**3)))
    return v


class Case:
    def __init__(self, ctx, kind, m, k, n, out="", layout=0, act="none", bias=False, residual=False, scales=None, pad=0,
                 shift=0, seed=0):
        import torch

        from onnxsharp_b200.runtime import LinearWeights

        g = torch.Generator(device="cuda")
        g.manual_seed(1000 + seed)
        coded = kind in ("s8", "e4m3")
        scales = coded if scales is None else scales
        self.ctx, self.kind, self.m, self.k, self.n, self.act = ctx, kind, m, k, n, act
        self.out_type = _dt(out or ("bf16" if coded else kind))
        a, w = _operand(g, (m, k), kind), _operand(g, (k, n), kind)
        unit = {"s8": 40.0, "e4m3": 100.0}.get(kind, 1.0)
        rand = lambda *s: torch.rand(s, generator=g, device="cuda")  # noqa: E731
        self.a_scale = (0.5 + rand(m)) / unit if scales else None
        self.w_scale = (0.5 + rand(n)) / (unit * math.sqrt(k)) if scales else None
        self.bias = torch.randn(n, generator=g, device="cuda") if bias else None
        self.residual = torch.randn((m, n), generator=g, device="cuda").to(self.out_type) if residual else None
        # the rows inside a wider buffer whose other bytes are not numbers
        buf = torch.full((m * (k + pad) + shift + 64,), 127, dtype=torch.uint8 if coded else torch.int16, device="cuda")
        self.a = buf.view(_dt(kind))[shift : shift + m * (k + pad)].view(m, k + pad)[:, :k]
        self.a.copy_(a)
        self.w = LinearWeights(ctx, w.t().contiguous() if layout else w, layout=layout)
        x, y = a.double(), w.double()
        v = x @ y
        size = x.abs() @ y.abs()
        steps = math.ceil(k * a.element_size() / 32) + 1
        err = torch.zeros_like(v) if kind == "s8" else steps * 2.0**-22 * size
        if scales:
            s = self.a_scale.double()[:, None] * self.w_scale.double()
            v, err = v * s, err * s
        err = err + 2.0**-22 * v.abs()
        if bias:
            v = v + self.bias.double()
            err = err + 2.0**-24 * v.abs()
        err = 1.2 * err + (0 if act in ("none", "relu") else 4e-6 * (1 + v.abs()))
        v = _act64(v, act)
        if residual:
            v = v + self.residual.double()
        half = torch.finfo(self.out_type).eps / 2
        tiny = torch.finfo(self.out_type).smallest_normal * half
        self.ref, self.tol = v, err + half * (v.abs() + err) * 1.0001 + 2.0**-23 * v.abs() + tiny

    def run(self, out=None, **kw):
        from onnxsharp_b200.runtime import linear

        return linear(self.ctx, self.a, self.w, bias=self.bias, act=ACTS[self.act],
                      residual=kw.pop("residual", self.residual), a_scale=self.a_scale, w_scale=self.w_scale, out=out,
                      out_dtype=None if out is not None else self.out_type, **kw)

    def check(self, got):
        import torch

        assert got.dtype == self.out_type
        far = ((got.double() - self.ref).abs() / self.tol).max().item() if got.numel() else 0.0
        assert torch.isfinite(got).all()
        assert far <= 1.0, f"{far:.3f} of the tolerance"


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("m,k,n", [(1, 1, 1), (1, 64, 128), (2, 7, 5), (3, 129, 127), (16, 256, 384), (17, 1000, 129),
                                   (33, 96, 1), (128, 512, 128), (129, 200, 257), (300, 1001, 400), (5, 4096, 640)])
def test_sizes(ctx, kind, m, k, n):
    c = Case(ctx, kind, m, k, n, seed=m + k + n)
    got = c.run()
    ctx.synchronize()
    c.check(got)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("m,k,n", [(1500, 2048, 1100), (2048, 512, 2048), (4100, 1024, 4000), (700, 192, 9000)])
def test_many_tokens(ctx, kind, m, k, n):
    """Several tiles a CTA: the ring and both accumulators wrap, ragged last tiles on both sides."""
    c = Case(ctx, kind, m, k, n, bias=True, residual=True, seed=m)
    got = c.run()
    ctx.synchronize()
    c.check(got)


@pytest.mark.parametrize("act", list(ACTS))
@pytest.mark.parametrize("out", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("m", [9, 200])
def test_epilogue(ctx, act, out, m):
    c = Case(ctx, "s8", m, 320, 200, out=out, act=act, bias=True, residual=True, seed=m)
    got = c.run()
    ctx.synchronize()
    c.check(got)


@pytest.mark.parametrize("kind,out", [("bf16", "f32"), ("bf16", "f16"), ("f16", "f32"), ("e4m3", "f32"), ("e4m3", "f16")])
@pytest.mark.parametrize("m,k", [(4, 8192), (500, 2048)])
def test_other_outputs(ctx, kind, out, m, k):
    c = Case(ctx, kind, m, k, 300, out=out, layout=1, bias=True)
    got = c.run()
    ctx.synchronize()
    c.check(got)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("layout", [0, 1])
@pytest.mark.parametrize("pad,shift", [(1, 0), (0, 1), (3, 5), (16, 0), (48, 16)])
@pytest.mark.parametrize("m,k,n", [(1, 333, 250), (40, 333, 250), (1000, 640, 700)])
def test_pitches_and_alignment(ctx, kind, layout, pad, shift, m, k, n):
    c = Case(ctx, kind, m, k, n, layout=layout, pad=pad, shift=shift, act="silu", residual=True)
    import torch

    wide = torch.full((m + 2, n + 5), 7.0, dtype=c.out_type, device="cuda")
    out = wide[1 : m + 1, 2 : n + 2]
    c.run(out=out)
    ctx.synchronize()
    c.check(out)
    rest = wide.clone()
    rest[1 : m + 1, 2 : n + 2] = 7.0
    assert bool((rest == 7.0).all()), "written outside of y"


@pytest.mark.parametrize("m", [1, 64, 700])
def test_residual_in_place(ctx, m):
    c = Case(ctx, "bf16", m, 512, 384, bias=True, residual=True)
    y = c.residual.clone()
    c.run(out=y, residual=y)
    ctx.synchronize()
    c.check(y)


def test_scales_are_optional(ctx):
    import torch

    from onnxsharp_b200.runtime import linear

    c = Case(ctx, "s8", 20, 64, 40, scales=False, out="f32")
    got = linear(ctx, c.a, c.w)
    ctx.synchronize()
    assert got.dtype == torch.float32 and bool((got.double() == c.ref).all())  # integers below 2^24
    one = torch.tensor([0.5], device="cuda")
    got = linear(ctx, c.a, c.w, w_scale=one)
    ctx.synchronize()
    assert bool((got.double() == c.ref * 0.5).all())
    row = torch.arange(20, device="cuda", dtype=torch.float32)
    got = linear(ctx, c.a, c.w, a_scale=row)
    ctx.synchronize()
    assert bool((got.double() == c.ref * row.double()[:, None]).all())


def test_extreme_s8_sums_are_exact(ctx):
    import torch

    from onnxsharp_b200.runtime import LinearWeights, linear

    k = 131071
    a = torch.full((2, k), -128, dtype=torch.int8, device="cuda")
    w = LinearWeights(ctx, torch.full((k, 3), -128, dtype=torch.int8, device="cuda"))
    got = linear(ctx, a, w, w_scale=torch.tensor([2.0**-14], device="cuda"))
    ctx.synchronize()
    assert bool((got == 131071.0).all())


@pytest.mark.parametrize("m", [3, 300])
def test_a_bad_row_stays_its_own(ctx, m):
    """NaN or infinity in one row of a, or in its scale, reaches that row of y alone."""
    import torch

    from onnxsharp_b200.runtime import linear

    c = Case(ctx, "bf16", m, 256, 130)
    c.a[1, 3] = math.nan
    got = c.run()
    ctx.synchronize()
    assert bool(got[1].isnan().all()) and bool(got[[i for i in range(m) if i != 1]].isfinite().all())
    c = Case(ctx, "s8", m, 256, 130)
    c.a_scale[2] = math.nan
    got = linear(ctx, c.a, c.w, a_scale=c.a_scale, w_scale=c.w_scale)
    ctx.synchronize()
    assert bool(got[2].isnan().all()) and bool(got[[i for i in range(m) if i != 2]].isfinite().all())


def test_no_rows(ctx):
    import torch

    c = Case(ctx, "f16", 1, 32, 16)
    before = ctx.launch_count()
    from onnxsharp_b200.runtime import linear

    assert linear(ctx, torch.empty((0, 32), dtype=torch.float16, device="cuda"), c.w).shape == (0, 16)
    assert ctx.launch_count() == before


@pytest.mark.parametrize("m,k", [(1, 4096), (48, 4096), (900, 640)])
def test_same_bits_every_time(ctx, m, k):
    c = Case(ctx, "bf16", m, k, 512, bias=True)
    first = c.run()
    again = [c.run() for _ in range(5)]
    ctx.synchronize()
    assert all(bool((first.view(dtype=_dt("f16")).view(-1) == x.view(dtype=_dt("f16")).view(-1)).all()) or
               bool((first == x).all()) for x in again)


@pytest.mark.parametrize("k", [2048, 2001])
def test_two_graphs_on_two_streams(ctx, k):
    """Captured once, replayed on new inputs, two graphs of two contexts at the same time (k 2001: with the copy of
    rows that TMA cannot take, a temporary of each graph)."""
    import torch

    from onnxsharp_b200.runtime import Context

    streams = [torch.cuda.Stream() for _ in range(2)]
    ctxs = [Context(0, s.cuda_stream) for s in streams]
    cases, outs, graphs = [], [], []
    for i, x in enumerate(ctxs):
        c = Case(x, "bf16", 20 + 300 * i, k, 512, bias=True, residual=True, seed=i)
        torch.cuda.synchronize()
        y = torch.zeros((c.m, c.n), dtype=c.out_type, device="cuda")
        torch.cuda.synchronize()
        graphs.append(x.capture(lambda c=c, y=y: c.run(out=y)))
        cases.append(c)
        outs.append(y)
    for _ in range(3):
        for y in outs:
            y.zero_()
        torch.cuda.synchronize()
        for _ in range(10):
            for g in graphs:
                g.launch()
        for x in ctxs:
            x.synchronize()
        for c, y in zip(cases, outs):
            c.check(y)
    for g in graphs:
        g.close()
    for x in ctxs:
        x.close()


def test_failing_allocation_is_reported(ctx, monkeypatch):
    from onnxsharp_b200 import OscError

    c = Case(ctx, "bf16", 5, 33, 16)
    monkeypatch.setenv("OSC_FAULT", "alloc")
    with pytest.raises(OscError, match="injected"):
        c.run()
    monkeypatch.delenv("OSC_FAULT")
    got = c.run()
    ctx.synchronize()
    c.check(got)


def test_host_weights(ctx):
    import torch

    from onnxsharp_b200.runtime import LinearWeights, linear

    w = torch.randn(96, 40).to(torch.bfloat16)
    a = torch.randn(7, 96, device="cuda").to(torch.bfloat16)
    x, y = linear(ctx, a, LinearWeights(ctx, w)), linear(ctx, a, LinearWeights(ctx, w.cuda()))
    ctx.synchronize()
    assert bool((x == y).all())


def test_refusals(ctx):
    import torch

    from onnxsharp_b200 import OscError
    from onnxsharp_b200.runtime import LinearWeights, linear

    c = Case(ctx, "bf16", 4, 64, 32)
    f32 = torch.zeros(4, device="cuda")
    with pytest.raises(OscError, match="scales belong"):
        linear(ctx, c.a, c.w, a_scale=f32)
    with pytest.raises(OscError, match="activation"):
        linear(ctx, c.a, c.w, act=16)
    with pytest.raises(ValueError, match="expected"):
        linear(ctx, c.a[:, :63], c.w)
    with pytest.raises(ValueError, match="dense"):
        linear(ctx, torch.zeros((64, 4), dtype=torch.bfloat16, device="cuda").t(), c.w)
    with pytest.raises(ValueError, match="cpu"):
        linear(ctx, c.a.cpu(), c.w)
    with pytest.raises(TypeError, match="weights are"):
        linear(ctx, c.a.to(torch.float16), c.w)
    with pytest.raises(TypeError, match="residual"):
        linear(ctx, c.a, c.w, residual=torch.zeros((4, 32), device="cuda"), out_dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="bias"):
        linear(ctx, c.a, c.w, bias=torch.zeros(31, device="cuda"))
    with pytest.raises(OscError, match="output dtype"):
        linear(ctx, c.a, c.w, out_dtype=torch.int8)
    with pytest.raises(OscError, match="overflows"):
        LinearWeights(ctx, torch.zeros((131072, 1), dtype=torch.int8, device="cuda"))
    with pytest.raises(OscError, match="not f16"):
        LinearWeights(ctx, torch.zeros((4, 4), device="cuda"))
