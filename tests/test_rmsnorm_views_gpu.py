"""rmsnorm() on views with dimensions of length one: the last token of every sequence, in and out of wider buffers."""
from __future__ import annotations

import pytest
import test_rmsnorm_gpu as norm

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("cols", [64, 95])
def test_last_tokens(ctx, dtype, cols):
    import torch

    from onnxsharp_b200 import ops

    x, res, gamma = norm._inputs(5 * 7, cols, dtype, True, pad=9)
    x, res = (torch.as_strided(t, (5, 7, cols), (7 * (cols + 9), cols + 9, 1))[:, -1:] for t in (x, res))
    wide = torch.full((5, 3, cols), 5.0, dtype=x.dtype, device="cuda")
    y, q, s = wide[:, 1:2], torch.empty((5, 1, cols), dtype=torch.int8, device="cuda"), torch.empty(5, device="cuda")
    ops.rmsnorm_quant(ctx, x, gamma, 1e-6, q, s, residual=res, y=y)
    ctx.synchronize()
    norm._check(x[:, 0], res[:, 0], gamma, 1e-6, "s8", y[:, 0], None, q[:, 0], s)
    assert bool((wide[:, ::2] == 5.0).all())
    with pytest.raises(ValueError, match="pitch"):  # rows 0, 1, 3, 4, ..
        ops.rmsnorm(ctx, wide[:, None, :2], gamma, 1e-6, torch.empty((5, 1, 2, cols), dtype=x.dtype, device="cuda"))
