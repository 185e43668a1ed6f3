"""attention_window() where a query or a visible key is not a number: the rows that see it, and no others, are NaN,
whichever kernel the token count picks. Tolerances of the other rows as in test_attention_window_gpu."""
from __future__ import annotations

import math

import pytest
import test_attention_window_gpu as win

pytestmark = pytest.mark.gpu

B, S, H, HK, WINDOW, SINKS = 2, 500, 8, 2, 100, 3


def _rows_that_see(T, length, j, start=None):
    first = length - T if start is None else start
    return [t for t in range(T) if 0 <= first + t < length and j <= first + t and (first + t - j < WINDOW or j < SINKS)]


@pytest.mark.parametrize("dtype,D", [("bf16", 64), ("bf16", 128), ("f16", 64)])
@pytest.mark.parametrize("T", [1, 4, 17, 60, 300])
@pytest.mark.parametrize("what", ["query nan", "query inf", "key nan", "key inf", "sink nan"])
def test_what_is_not_a_number_reaches_its_rows(ctx, dtype, D, T, what):
    import torch

    from onnxsharp_b200.runtime import attention_window

    q, k, v = win._inputs(B, T, S, H, HK, D, dtype, seed=5)
    q = q.abs()  # (an infinite key then gives every row that sees it a score of +inf)
    lengths = torch.tensor([S, S // 2], dtype=torch.int32, device="cuda")
    ref, tol = win._reference(q, k, v, lengths, None, D**-0.5, WINDOW, SINKS)
    nan = torch.zeros((B, T, H), dtype=torch.bool, device="cuda")
    if what.startswith("query"):
        t, h = T // 2, 5
        q[0, t, h, 7] = math.nan if what == "query nan" else math.inf
        if what == "query inf":
            k[0, :, h // (H // HK), 7] = k[0, :, h // (H // HK), 7].abs() + 0.5
            ref, tol = win._reference(q.nan_to_num(posinf=1.0), k, v, lengths, None, D**-0.5, WINDOW, SINKS)
        nan[0, t, h] = True
    else:
        j, hk = (1 if what == "sink nan" else S - 1 - T // 2 - 20), 1
        k[0, j, hk, 9] = math.inf if what == "key inf" else math.nan
        rows = _rows_that_see(T, S, j)
        assert rows and (T < 200 or what == "sink nan" or len(rows) < T)
        for t in rows:
            nan[0, t, hk * (H // HK) : (hk + 1) * (H // HK)] = True
    got = attention_window(ctx, q, k, v, lengths, D**-0.5, window=WINDOW, sinks=SINKS)
    ctx.synchronize()
    assert bool((got.isnan().all(-1) == nan).all()) and bool((got.isnan().any(-1) == nan).all())
    win._check(got[~nan], ref[~nan], tol[~nan])


@pytest.mark.parametrize("T", [3, 60, 300])
def test_padding_queries_hold_anything(ctx, T):
    """Rows outside 0 .. lengths - 1 are zeros, whatever q holds there."""
    import torch

    from onnxsharp_b200.runtime import attention_window

    q, k, v = win._inputs(3, T, S, H, HK, 64, "bf16")
    lengths = torch.tensor([T - T // 3, 0, S], dtype=torch.int32, device="cuda")
    starts = torch.tensor([0, 0, -(T // 2)], dtype=torch.int32, device="cuda")
    ref, tol = win._reference(q, k, v, lengths, starts, 0.125, WINDOW, SINKS)
    q[0, T - T // 3 :] = math.nan
    q[1] = math.inf
    q[2, : T // 2] = math.nan
    got = attention_window(ctx, q, k, v, lengths, 0.125, window=WINDOW, sinks=SINKS, starts=starts)
    ctx.synchronize()
    assert not bool(got[0, T - T // 3 :].any()) and not bool(got[1].any()) and not bool(got[2, : T // 2].any())
    win._check(got, ref, tol)
