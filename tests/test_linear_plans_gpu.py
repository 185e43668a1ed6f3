"""linear() through every kernel that its cost rule picks: single CTAs and pairs of k_linear_tiles, k_linear_split alone
and over clusters of four and eight, small and large token tiles, each operand type, ragged columns (an odd number of
128-column blocks leaves a pair's second CTA without one). The profile says which plan a call took; should the rule
change, the sizes here have to be chosen again. Checks and tolerances as in test_linear_gpu."""
from __future__ import annotations

import pytest
import test_linear_gpu as lin

pytestmark = pytest.mark.gpu

# m, k, n, plan in 16 bits, in 8 bits
PLANS = [
    (129, 200, 129, "split 1 16", "split 1 16"),
    (2050, 200, 9000, "tiles single 208", "split 1 112"),
    (9, 4100, 9000, "split 4 16", "tiles single 16"),
    (129, 4100, 900, "split 8 48", "split 4 16"),
    (129, 8192, 3000, "split 4 48", "split 4 48"),
    (50, 4100, 100, "split 8 16", "split 8 16"),
    (333, 4100, 129, "split 8 32", "split 8 32"),
    (200, 8192, 2000, "split 8 112", "split 8 112"),
    (333, 1001, 777, "tiles single 16", "tiles single 16"),
    (70, 1001, 9000, "tiles single 48", "tiles single 48"),
    (257, 200, 9000, "tiles single 144", "tiles single 144"),
    (1500, 200, 3000, "tiles single 256", "tiles single 256"),
    (2050, 8192, 900, "tiles pair 128", "tiles pair 128"),
    (257, 8192, 9000, "tiles pair 160", "tiles pair 160"),
    (300, 2048, 9000, "tiles pair 160", "tiles single 160"),
    (700, 2048, 9000, "tiles pair 192", "tiles pair 192"),
    (2050, 2048, 9000, "tiles pair 224", "tiles pair 224"),
    (2050, 4100, 4000, "tiles pair 256", "tiles pair 256"),
]


def _run(ctx, c, plan):
    ctx.profile_reset()
    ctx.profile(True)
    try:
        recorded = c.run()
        took = ctx.profile_read(f"k_linear_{plan}")[1]
    finally:
        ctx.profile(False)
        ctx.profile_reset()
    assert took == 1, f"not by {plan}"
    got = c.run()
    ctx.synchronize()
    c.check(got)
    assert bool((got == recorded).all())


@pytest.mark.parametrize("kind", lin.KINDS)
@pytest.mark.parametrize("m,k,n,wide,narrow", PLANS)
def test_plans(ctx, kind, m, k, n, wide, narrow):
    c = lin.Case(ctx, kind, m, k, n, bias=True, residual=True, act="silu", seed=m + n)
    _run(ctx, c, wide if kind in ("bf16", "f16") else narrow)


@pytest.mark.parametrize("kind", ["bf16", "s8"])
@pytest.mark.parametrize("act", list(lin.ACTS))
@pytest.mark.parametrize("out", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("m,k,n,wide,narrow", [p for p in PLANS if p[:2] in ((129, 4100), (333, 1001), (257, 8192), (70, 1001))])
def test_epilogues(ctx, kind, act, out, m, k, n, wide, narrow):
    c = lin.Case(ctx, kind, m, k, n, out=out, bias=True, residual=True, act=act)
    _run(ctx, c, wide if kind == "bf16" else narrow)


@pytest.mark.parametrize("kind,k", [("s8", 8192), ("e4m3", 8192), ("bf16", 4100)])
@pytest.mark.parametrize("m,n,plan", [(2050, 4000, "tiles pair 256"), (200, 2000, "split 8 112")])
def test_a_hundred_calls_agree(ctx, kind, k, m, n, plan):
    c = lin.Case(ctx, kind, m, k if plan.startswith("tiles") else 8192, n, bias=True, residual=True)
    _run(ctx, c, plan)
    first = c.run()
    for i in range(100):
        assert bool((c.run() == first).all()), i
