"""linear()'s activations relative to their own value, where they are small beside their argument too.

The product is one exact factor (k = 1, w = 1), so the pre-activation v is known. Relative errors, u = 2^-24:
  gelu       the formula's own sensitivity: an argument z = |v| / sqrt 2 off by 1.5 u relative moves erfc(z) by at most
             z (z + sqrt(z^2 + 2)) <= v^2 + 1 times that; beside it an erfc good to 4 ulp (8 u) and two products
  silu, sigmoid  ex2.approx 4 u and its argument's 1.5 u |v|, the sum u, rcp.approx 2 u, a product
  gelu_tanh  the argument a = 2 sqrt(2/pi) (v + 0.044715 v^3) takes six roundings and two constants (7 u |a|), then
             the sigmoid's own
and half a step of the output's type."""
from __future__ import annotations

import math

import pytest
import test_linear_gpu as lin

pytestmark = pytest.mark.gpu


def _relative(v, act):
    a = v.abs()
    if act == "gelu":
        return 1.5 * (v * v + 1) + 8 + 2
    if act in ("silu", "sigmoid"):
        return 4 + 1.5 * a + 1 + 2 + 1
    if act == "gelu_tanh":
        z = 1.5957691216057308 * (a + 0.044715 * a**3)
        return 7 * z + 4 + 1.5 * z + 1 + 2 + 1
    return 0 * a


def _exact(v, act):
    import torch

    if act == "gelu_tanh":  # (1 + tanh cancels in 64 bits too)
        return v * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (v + 0.044715 * v**3))
    return lin._act64(v, act)


@pytest.mark.parametrize("act", list(lin.ACTS))
@pytest.mark.parametrize("kind", ["bf16", "s8"])
@pytest.mark.parametrize("out", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n", [40, 8192])
def test_small_values(ctx, act, kind, out, n):
    import torch

    from onnxsharp_b200.runtime import LinearWeights, linear

    if kind == "s8":  # -8 .. 8 by a row scale of 1/16
        a = torch.arange(-128, 128, device="cuda")[:, None].to(torch.int8)
        v, scale = a.double() / 16, torch.full((256,), 1 / 16, device="cuda")
    else:
        a = torch.linspace(-8, 8, 1777, device="cuda")[:, None].bfloat16()
        v, scale = a.double(), None
    w = LinearWeights(ctx, torch.ones((1, n), dtype=a.dtype, device="cuda"))
    got = linear(ctx, a, w, act=lin.ACTS[act], a_scale=scale, out_dtype=lin._dt(out))
    ctx.synchronize()
    ref, eps = _exact(v, act), torch.finfo(lin._dt(out))
    rel = _relative(v, act) * 2.0**-24 * 1.01
    tol = ref.abs() * (rel + eps.eps / 2 * (1 + rel)) + eps.smallest_normal * eps.eps / 2
    far = ((got.double() - ref).abs() / tol.clamp(min=1e-300)).max().item()
    assert far <= 1.0, f"{far:.2f} of the tolerance"
