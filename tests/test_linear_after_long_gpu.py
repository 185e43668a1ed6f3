"""linear() queued behind a kernel that runs longer than the limit of a kernel's internal waits (about 1.5 s): it starts
early, beside that kernel, and has to hold its own waits until that kernel is done."""
from __future__ import annotations

import pytest
import test_linear_gpu as lin

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m,k,n,name", [(8, 512, 640, "k_linear_tiles"), (50, 4100, 100, "k_linear_split")])
def test_behind_two_seconds(ctx, m, k, n, name):
    import torch

    from onnxsharp_b200 import ops

    c = lin.Case(ctx, "bf16", m, k, n, bias=True, residual=True)
    y = torch.zeros((m, n), dtype=torch.bfloat16, device="cuda")
    x = torch.ones((1, 2**31 - 1), dtype=torch.bfloat16, device="cuda")
    out = torch.empty_like(x)
    torch.cuda.synchronize()
    begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    begin.record()
    ops.rmsnorm(ctx, x, None, 1e-6, out)  # one CTA: the others' SMs are free for the product
    c.run(out=y)
    end.record()
    ctx.synchronize()
    assert begin.elapsed_time(end) > 1600
    c.check(y)
    ctx.profile(True)  # (which kernel it was: profiling keeps launches apart)
    ctx.profile_reset()
    c.run(out=y)
    assert ctx.profile_read(name)[1] == 1
    ctx.profile(False)
    ctx.profile_reset()
