"""attention_window() against the same formula in float64, for every kernel that it picks.

Tolerance, from the roundings: a score is an FP32 sum on the tensor cores of D products in D / 16 steps (a unit of the
24th bit of the largest partial sum each, 2^-22 S a step with S = scale sum |q k|), which moves a probability by at most
twice its error relative; exp2, the running maximum's factors and the division add 2^-19; probabilities are rounded to
the type (half a step), in FP16 not finer than 2^-25 against a sum of at least 1; the second product adds a unit a step
of 16 keys; the result is off by half a step of its type. All of it multiplies softmax @ |v|."""
from __future__ import annotations

import math

import pytest

pytestmark = pytest.mark.gpu


def _dt(name):
    import torch

    return {"bf16": torch.bfloat16, "f16": torch.float16}[name]


def _reference(q, k, v, lengths, starts, scale, window, sinks):
    import torch

    B, T, H, D = q.shape
    S, G = k.shape[1], H // k.shape[2]
    out, tol = torch.zeros(q.shape, dtype=torch.float64, device="cuda"), torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    eps = torch.finfo(q.dtype).eps
    for b in range(B):
        n = int(lengths[b])
        first = n - T if starts is None else int(starts[b])
        p = torch.arange(first, first + T, device="cuda")[:, None]
        j = torch.arange(n, device="cuda")[None]
        seen = (p >= 0) & (p < n) & (j <= p) & ((p - j < window) | (j < sinks))
        if n == 0:
            continue
        for h in range(H):
            qq, kk, vv = q[b, :, h].double(), k[b, :n, h // G].double(), v[b, :n, h // G].double()
            s = torch.where(seen, scale * (qq @ kk.T), -math.inf)
            ds = ((D / 16 + 1) * 2.0**-22 * scale * (qq.abs() @ kk.abs().T) * seen).amax(dim=1, keepdim=True)
            e = torch.where(seen, torch.exp(s - torch.where(seen.any(1, keepdim=True), s.amax(1, keepdim=True), 0.0)), 0.0)
            total = e.sum(1, keepdim=True)
            w = e / torch.where(total > 0, total, 1.0)
            y, a = w @ vv, w @ vv.abs()
            t = a * (2 * ds + eps / 2 + 2.0**-19 + (seen.sum(1, keepdim=True) / 16 + 1) * 2.0**-22) + eps / 2 * y.abs()
            if q.dtype == torch.float16:
                t = t + 2.0**-25 * (seen.double() @ vv.abs()) + 2.0**-25
            out[b, :, h], tol[b, :, h] = y, t
    return out, 1.05 * tol


def _inputs(B, T, S, H, HK, D, dtype, seed=0):
    import torch

    g = torch.Generator(device="cuda")
    g.manual_seed(seed + 17 * T + S)
    r = lambda *s: torch.randn(s, generator=g, device="cuda").to(_dt(dtype))  # noqa: E731
    return r(B, T, H, D) * 1.5, r(B, S, HK, D), r(B, S, HK, D)


def _check(got, ref, tol):
    import torch

    assert bool(torch.isfinite(got).all())
    bad = (got.double() - ref).abs() > tol
    assert not bool(bad.any()), ((got.double() - ref).abs() / tol.clamp(min=1e-30)).max().item()


def _hide(k, v, lengths):
    """What a cache holds behind a sequence: anything."""
    for b, n in enumerate(lengths.tolist()):
        k[b, n:], v[b, n:] = math.nan, math.inf


def _case(ctx, B, T, S, H, HK, D, dtype, window, sinks, lengths, starts=None, scale=None, seed=0, gone=False):
    import torch

    from onnxsharp_b200.runtime import attention_window

    q, k, v = _inputs(B, T, S, H, HK, D, dtype, seed)
    lengths = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    starts = None if starts is None else torch.tensor(starts, dtype=torch.int32, device="cuda")
    scale = scale or D**-0.5
    ref, tol = _reference(q, k, v, lengths, starts, scale, window, sinks)
    _hide(k, v, lengths)
    if gone:  # tokens that no row sees any more
        for b, n in enumerate(lengths.tolist()):
            lo = max(0, n - T if starts is None else int(starts[b])) - window + 1
            k[b, sinks : max(lo, sinks)], v[b, sinks : max(lo, sinks)] = math.nan, math.inf
    got = attention_window(ctx, q, k, v, lengths, scale, window=window, sinks=sinks, starts=starts)
    ctx.synchronize()
    _check(got, ref, tol)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("H,HK", [(8, 8), (8, 2), (12, 1), (10, 2)])
@pytest.mark.parametrize("S,lengths", [(1, [1, 1]), (63, [63, 1]), (130, [129, 64]), (1000, [1000, 517]), (5000, [4999, 128])])
@pytest.mark.parametrize("window,sinks", [(1, 0), (64, 0), (100, 5), (10**6, 0), (7, 300)])
def test_one_token(ctx, dtype, D, H, HK, S, lengths, window, sinks):
    _case(ctx, 2, 1, S, H, HK, D, dtype, window, sinks, lengths)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("H,HK", [(2, 2), (8, 2), (5, 1), (3, 1), (24, 2)])
@pytest.mark.parametrize("T", [2, 5, 33, 128, 300])
@pytest.mark.parametrize("window,sinks", [(1, 1), (50, 0), (129, 3), (10**6, 0), (20, 200)])
def test_prompts(ctx, dtype, D, H, HK, T, window, sinks):
    """The cache's newest T tokens; a sequence shorter than T has padding in front."""
    _case(ctx, 2, T, 700, H, HK, D, dtype, window, sinks, [700 - T // 3, max(1, T // 2)])


@pytest.mark.parametrize("T", [3, 40, 400])
@pytest.mark.parametrize("window,sinks", [(1000, 0), (60, 4)])
def test_starts(ctx, T, window, sinks):
    """Batches padded at the end, sequences without a token, starts in the middle and nowhere."""
    _case(ctx, 6, T, 500, 4, 2, 64, "bf16", window, sinks, [T, T // 2, 0, 500, 10, 10],
          [0, 0, 0, 77, 2**31 - 1, -(2**31)])


@pytest.mark.parametrize("T,G", [(1, 1), (16, 128), (1, 32), (2, 16), (4, 8), (1, 33), (64, 100)])
def test_groups(ctx, T, G):
    _case(ctx, 1, T, 300, 2 * G, 2, 64, "bf16", 90, 2, [280])


@pytest.mark.parametrize("dtype,D", [("bf16", 128), ("f16", 64)])
@pytest.mark.parametrize(
    "T,H,HK,S,lengths,starts",
    [
        (1, 8, 1, 9001, [9001], None),
        (1, 8, 2, 3001, [3001, 1, 0, 2999, 64, 65, 0], None),
        (8, 8, 2, 2500, [2500, 3, 1300], [2492, 0, 1000]),  # two row tiles, padded batches
        (3, 6, 6, 1999, [5, 1999, 1998, 0], [2, 1999, 1990, 0]),
        (1, 74, 37, 2100, [2100, 900], None),  # SMs that the heads do not divide
        (1, 2, 1, 20000, [17777], None),
        (2, 16, 1, 4100, [4100, 1, 3, 0, 0, 4097, 2, 1, 1, 1], None),
        (16, 8, 2, 4100, [4100, 9], [4080, 0]),  # four row tiles
        (11, 5, 1, 3000, [3000], None),
    ],
)
@pytest.mark.parametrize("window,sinks", [(10**6, 0), (1000, 0), (1500, 70), (900, 3)])
def test_cut_sequences(ctx, dtype, D, T, H, HK, S, lengths, starts, window, sinks):
    """Few groups with many keys: CTAs share them, whatever sequence their keys belong to."""
    _case(ctx, len(lengths), T, S, H, HK, D, dtype, window, sinks, lengths, starts, gone=True)


@pytest.mark.parametrize("T", [1, 4, 9, 40, 300])
@pytest.mark.parametrize("window,sinks", [(64, 0), (65, 5), (200, 129), (10, 1)])
def test_forgotten_tokens(ctx, T, window, sinks):
    """NaN and infinities between the sinks and the window of the first query."""
    _case(ctx, 2, T, 777, 8, 2, 64, "bf16", window, sinks, [777, 600], gone=True)
    _case(ctx, 3, T, 777, 4, 4, 128, "f16", window, sinks, [777, 700, 0], [400, 650, 0], gone=True)


@pytest.mark.parametrize("T", [1, 200])
def test_long_windows(ctx, T):
    """Several hundred key tiles, the maximum growing from tile to tile."""
    import torch

    from onnxsharp_b200.runtime import attention_window

    q, k, v = _inputs(1, T, 20000, 2, 1, 128, "bf16")
    k *= torch.linspace(0.1, 6.0, 20000, device="cuda")[None, :, None, None].to(k.dtype)
    lengths = torch.tensor([20000], dtype=torch.int32, device="cuda")
    ref, tol = _reference(q, k, v, lengths, None, 128**-0.5, 10**6, 0)
    got = attention_window(ctx, q, k, v, lengths, 128**-0.5)
    ctx.synchronize()
    _check(got, ref, tol)


@pytest.mark.parametrize("T", [1, 5, 150])
def test_views(ctx, T):
    """q, k and v as slices of one projection, a head-major cache, an output inside a wider buffer."""
    import torch

    from onnxsharp_b200.runtime import attention_window

    B, S, H, HK, D = 2, 333, 8, 2, 64
    g = torch.Generator(device="cuda")
    g.manual_seed(T)
    r = lambda *s: torch.randn(s, generator=g, device="cuda").to(torch.bfloat16)  # noqa: E731
    qkv = r(B, T, H + 2 * HK, D)
    kc, vc = r(B, HK, S, D).transpose(1, 2), r(B, S, HK + 1, D)[:, :, 1:]
    lengths = torch.tensor([333, 200], dtype=torch.int32, device="cuda")
    wide = torch.full((B, T, H + 2, D + 8), 9.0, dtype=torch.bfloat16, device="cuda")
    out = wide[:, :, 1:-1, 8:]
    ref, tol = _reference(qkv[:, :, :H], kc, vc, lengths, None, 0.2, 100, 4)
    attention_window(ctx, qkv[:, :, :H], kc, vc, lengths, 0.2, window=100, sinks=4, out=out)
    ctx.synchronize()
    _check(out, ref, tol)
    wide[:, :, 1:-1, 8:] = 9.0
    assert bool((wide == 9.0).all())


@pytest.mark.parametrize("T", [1, 100])
def test_same_bits_and_replay(ctx, T):
    """Captured once; the lengths on the device grow between replays."""
    import torch

    from onnxsharp_b200.runtime import Context, attention_window

    stream = torch.cuda.Stream()
    c = Context(0, stream.cuda_stream)
    q, k, v = _inputs(3, T, 2000, 8, 2, 128, "f16")
    lengths = torch.tensor([500, 700, 900], dtype=torch.int32, device="cuda")
    out = torch.empty_like(q)
    torch.cuda.synchronize()
    g = c.capture(lambda: attention_window(c, q, k, v, lengths, 0.1, window=600, sinks=2, out=out))
    for grow in (0, 1, 400, 1100):
        lengths.copy_(torch.tensor([500 + grow, 700 + grow, 900 + grow], dtype=torch.int32))
        torch.cuda.synchronize()
        g.launch()
        c.synchronize()
        first = out.clone()
        torch.cuda.synchronize()
        g.launch()
        c.synchronize()
        assert bool((out == first).all())
        _check(out, *_reference(q, k, v, lengths, None, 0.1, 600, 2))
    g.close()
    c.close()


def test_nothing_to_do(ctx):
    import torch

    from onnxsharp_b200.runtime import attention_window

    before = ctx.launch_count()
    for B, T in ((0, 4), (2, 0)):
        q, k, v = _inputs(B, T, 10, 2, 1, 64, "bf16")
        got = attention_window(ctx, q, k, v, torch.ones(B, dtype=torch.int32, device="cuda"), 1.0)
        assert got.shape == (B, T, 2, 64)
    assert ctx.launch_count() == before


def test_refusals(ctx):
    import torch

    from onnxsharp_b200 import OscError
    from onnxsharp_b200.runtime import attention_window

    q, k, v = _inputs(2, 3, 10, 4, 2, 64, "bf16")
    n = torch.tensor([10, 10], dtype=torch.int32, device="cuda")
    for kw, match in (({"window": 0}, "window"), ({"sinks": -1}, "sinks")):
        with pytest.raises(OscError, match=match):
            attention_window(ctx, q, k, v, n, 1.0, **kw)
    for scale in (0.0, -1.0, math.inf, math.nan):
        with pytest.raises(OscError, match="scale"):
            attention_window(ctx, q, k, v, n, scale)
    with pytest.raises(OscError, match="heads over"):
        attention_window(ctx, q[:, :, :3], k, v, n, 1.0)
    with pytest.raises(OscError, match="head size"):
        attention_window(ctx, q[..., :32], k[..., :32], v[..., :32], n, 1.0)
    with pytest.raises(OscError, match="16-byte"):
        attention_window(ctx, torch.zeros((2, 3, 4, 68), dtype=q.dtype, device="cuda")[..., :64], k, v, n, 1.0)
    with pytest.raises(OscError, match="16-byte"):
        attention_window(ctx, torch.zeros(2 * 3 * 4 * 64 + 1, dtype=q.dtype, device="cuda")[1:].view(2, 3, 4, 64), k, v, n, 1.0)
    with pytest.raises(OscError, match="dtype"):
        attention_window(ctx, q.float(), k.float(), v.float(), n, 1.0)
    with pytest.raises(TypeError, match="one tensor is"):
        attention_window(ctx, q, k.half(), v, n, 1.0)
    with pytest.raises(ValueError, match="lengths"):
        attention_window(ctx, q, k, v, n.long(), 1.0)
    with pytest.raises(ValueError, match="cpu"):
        attention_window(ctx, q.cpu(), k, v, n, 1.0)
    with pytest.raises(ValueError, match="dense"):
        attention_window(ctx, q.transpose(2, 3).contiguous().transpose(2, 3), k, v, n, 1.0)


def test_cut_sequences_in_two_graphs():
    """The parts of cut sequences belong to a call: two graphs of one context and an eager call on another stream."""
    import torch

    from onnxsharp_b200.runtime import Context, attention_window

    streams = [torch.cuda.Stream() for _ in range(2)]
    ctxs = [Context(0, s.cuda_stream) for s in streams]
    lengths = torch.tensor([6000, 100, 3500], dtype=torch.int32, device="cuda")
    cases = []
    for i in range(2):
        q, k, v = _inputs(3, 1, 6000, 8, 2, 128, "bf16", seed=i)
        cases.append((q, k, v, torch.empty_like(q)))
    torch.cuda.synchronize()
    run = lambda c, x: attention_window(c, x[0], x[1], x[2], lengths, 0.1, out=x[3])  # noqa: E731
    graphs = [ctxs[0].capture(lambda x=x: run(ctxs[0], x)) for x in cases]
    want = [x[3].clone() for x in cases]
    for x, w in zip(cases, want):
        _check(w, *_reference(x[0], x[1], x[2], lengths, None, 0.1, 10**6, 0))
    for _ in range(5):
        for x in cases:
            x[3].fill_(7.0)
        torch.cuda.synchronize()
        graphs[0].launch()
        run(ctxs[1], cases[1])
        ctxs[1].synchronize()
        graphs[1].launch()
        graphs[0].launch()
        ctxs[0].synchronize()
        assert all(bool((x[3] == w).all()) for x, w in zip(cases, want))
    for g in graphs:
        g.close()
    for c in ctxs:
        c.close()


@pytest.mark.parametrize("T,S", [(1, 40), (1, 3001), (60, 300)])
def test_shared_cache(ctx, T, S):
    """One cache behind several sequences, one key/value head behind several groups (strides of 0)."""
    import torch

    from onnxsharp_b200.runtime import attention_window

    q, k, v = _inputs(3, T, S, 8, 1, 64, "bf16")
    k, v = (t[:1].expand(3, S, 2, 64) for t in (k, v))
    lengths = torch.tensor([S, S - 1, S // 2], dtype=torch.int32, device="cuda")
    got = attention_window(ctx, q, k, v, lengths, 0.1, window=200, sinks=1)
    ctx.synchronize()
    _check(got, *_reference(q, k, v, lengths, None, 0.1, 200, 1))


def test_failing_allocation_is_reported(ctx, monkeypatch):
    import torch

    from onnxsharp_b200 import OscError
    from onnxsharp_b200.runtime import attention_window

    q, k, v = _inputs(1, 1, 6000, 8, 2, 128, "bf16")
    lengths = torch.tensor([6000], dtype=torch.int32, device="cuda")
    monkeypatch.setenv("OSC_FAULT", "alloc")
    with pytest.raises(OscError, match="injected"):
        attention_window(ctx, q, k, v, lengths, 0.1)
    monkeypatch.delenv("OSC_FAULT")
    got = attention_window(ctx, q, k, v, lengths, 0.1)
    ctx.synchronize()
    _check(got, *_reference(q, k, v, lengths, None, 0.1, 10**6, 0))


@pytest.mark.parametrize("T,H,HK,D,lengths", [(1, 74, 37, 128, [2100, 900]), (1, 8, 8, 64, [4000, 70, 3000]),
                                              (16, 8, 2, 128, [4100]), (200, 8, 2, 128, [4100, 300])])
def test_a_thousand_calls_agree(ctx, T, H, HK, D, lengths):
    """Rings that are refilled while slower warps still read show up as bits that change, in one call of a hundred."""
    import torch

    from onnxsharp_b200.runtime import attention_window

    q, k, v = _inputs(len(lengths), T, max(lengths), H, HK, D, "bf16")
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    outs = [torch.full_like(q, math.nan) for _ in range(2)]
    for i in range(1000):
        attention_window(ctx, q, k, v, n, 0.1, window=1500, sinks=70, out=outs[min(i, 1)])
        if i:
            assert bool((outs[0] == outs[1]).all()), i
            outs[1].fill_(math.nan)
    _check(outs[0], *_reference(q, k, v, n, None, 0.1, 1500, 70))
