"""attention_window() of a prompt's later chunks: more rows than k_window_rows takes over caches of many key tiles, with
forgotten tokens, sinks, ragged lengths and starts, and the same call from two graphs. Tolerances as in
test_attention_window_gpu."""
from __future__ import annotations

import pytest
import test_attention_window_gpu as win

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,D,H,HK", [("bf16", 128, 8, 2), ("f16", 64, 5, 1), ("bf16", 64, 16, 16)])
@pytest.mark.parametrize("T", [17, 33, 65, 130, 257])
@pytest.mark.parametrize("window,sinks", [(10**6, 0), (5000, 70), (700, 3)])
@pytest.mark.parametrize("lengths,starts", [([8192], None), ([6001, 300, 0], None), ([8000, 5000], [7800, 4000])])
def test_chunks(ctx, dtype, D, H, HK, T, window, sinks, lengths, starts):
    win._case(ctx, len(lengths), T, 8192, H, HK, D, dtype, window, sinks, lengths, starts, gone=True)


@pytest.mark.parametrize("T", [33, 200])
def test_chunks_in_two_graphs(T):
    import torch

    from onnxsharp_b200.runtime import Context, attention_window

    streams = [torch.cuda.Stream() for _ in range(2)]
    ctxs = [Context(0, s.cuda_stream) for s in streams]
    lengths = torch.tensor([6000, 900, 3500], dtype=torch.int32, device="cuda")
    cases = []
    for i in range(2):
        q, k, v = win._inputs(3, T, 6000, 8, 2, 128, "bf16", seed=i)
        cases.append((q, k, v, torch.empty_like(q)))
    torch.cuda.synchronize()
    run = lambda c, x: attention_window(c, x[0], x[1], x[2], lengths, 0.1, window=4000, sinks=5, out=x[3])  # noqa: E731
    graphs = [c.capture(lambda c=c, x=x: run(c, x)) for c, x in zip(ctxs, cases)]
    want = [x[3].clone() for x in cases]
    for x, w in zip(cases, want):
        win._check(w, *win._reference(x[0], x[1], x[2], lengths, None, 0.1, 4000, 5))
    for _ in range(5):
        for x in cases:
            x[3].fill_(7.0)
        torch.cuda.synchronize()
        for _ in range(3):
            for g in graphs:
                g.launch()
        for c in ctxs:
            c.synchronize()
        assert all(bool((x[3] == w).all()) for x, w in zip(cases, want))
    for g in graphs:
        g.close()
    for c in ctxs:
        c.close()
