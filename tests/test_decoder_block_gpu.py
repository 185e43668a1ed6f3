"""Norms, products and window attention as a decoder runs them: a prompt, then single tokens out of one captured graph.

Each call is checked against float64 on the inputs that it really had (the previous calls' results), with the
tolerances that test_rmsnorm_gpu, test_linear_gpu and test_attention_window_gpu derive for it alone."""
from __future__ import annotations

import math

import pytest
import test_attention_window_gpu as win
import test_rmsnorm_gpu as norm

pytestmark = pytest.mark.gpu

H, HK, D, WIDE, HIDDEN, CACHE, WINDOW, SINKS = 8, 2, 64, 512, 1408, 400, 150, 4


class Block:
    """h += attention(norm(h)); h += down(silu(up(norm(h)))): attention in bf16, the second half in `kind` codes."""

    def __init__(self, ctx, batch, kind, seed):
        import torch

        from onnxsharp_b200.runtime import LinearWeights

        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        r = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
        self.ctx, self.batch, self.kind = ctx, batch, kind
        self.g1, self.g2 = (1 + 0.1 * r(WIDE)).bfloat16(), (1 + 0.1 * r(WIDE)).bfloat16()
        self.w = {"qkv": (r(WIDE, (H + 2 * HK) * D) / math.sqrt(WIDE)).bfloat16(),
                  "o": (r(H * D, WIDE) / math.sqrt(H * D)).bfloat16(), "down": (r(HIDDEN, WIDE) / math.sqrt(HIDDEN)).bfloat16()}
        up = r(WIDE, HIDDEN) * 30
        self.w["up"] = up.round().clamp(-127, 127).to(torch.int8) if kind == "s8" else up.to(torch.float8_e4m3fn)
        self.up_scale = (0.5 + torch.rand(HIDDEN, generator=g, device="cuda")) / (30 * math.sqrt(WIDE))
        self.bias = r(WIDE)
        self.packed = {n: LinearWeights(ctx, w) for n, w in self.w.items()}
        self.k = torch.full((batch, CACHE, HK, D), math.nan, dtype=torch.bfloat16, device="cuda")
        self.v = torch.full_like(self.k, math.inf)

    def buffers(self, tokens):
        import torch

        n = self.batch * tokens
        e = lambda *s, t=torch.bfloat16: torch.empty(s, dtype=t, device="cuda")  # noqa: E731
        codes = torch.int8 if self.kind == "s8" else torch.float8_e4m3fn
        return {"n1": e(n, WIDE), "qkv": e(n, (H + 2 * HK) * D), "at": e(self.batch, tokens, H, D), "h1": e(n, WIDE),
                "q": e(n, WIDE, t=codes), "s": e(n, t=torch.float32), "up": e(n, HIDDEN), "h2": e(n, WIDE)}

    def run(self, h, b, lengths, slots):
        """slots: int64 [batch, tokens], the rows of the cache that the new tokens take; lengths count them."""
        from onnxsharp_b200 import ops
        from onnxsharp_b200.runtime import attention_window, linear

        c, w, tokens = self.ctx, self.packed, slots.shape[1]
        ops.rmsnorm(c, h, self.g1, 1e-6, b["n1"])
        linear(c, b["n1"], w["qkv"], out=b["qkv"])
        heads = b["qkv"].view(self.batch, tokens, H + 2 * HK, D)
        at = slots[:, :, None, None].expand(-1, -1, HK, D)
        self.k.scatter_(1, at, heads[:, :, H : H + HK])
        self.v.scatter_(1, at, heads[:, :, H + HK :])
        attention_window(c, heads[:, :, :H], self.k, self.v, lengths, D**-0.5, window=WINDOW, sinks=SINKS, out=b["at"])
        linear(c, b["at"].view(-1, H * D), w["o"], residual=h, out=b["h1"])
        ops.rmsnorm_quant(c, b["h1"], self.g2, 1e-6, b["q"], b["s"])
        linear(c, b["q"], w["up"], act=1, a_scale=b["s"], w_scale=self.up_scale, out=b["up"])
        linear(c, b["up"], w["down"], bias=self.bias, residual=b["h1"], out=b["h2"])

    def check(self, h, b, lengths, tokens):
        norm._check(h, None, self.g1, 1e-6, "", y=b["n1"])
        self._product(b["n1"], "qkv", b["qkv"])
        heads = b["qkv"].view(self.batch, tokens, H + 2 * HK, D)
        for row, n in enumerate(lengths.tolist()):
            assert bool((self.k[row, n - tokens : n] == heads[row, :, H : H + HK]).all())
            assert bool((self.v[row, n - tokens : n] == heads[row, :, H + HK :]).all())
        win._check(b["at"], *win._reference(heads[:, :, :H], self.k, self.v, lengths, None, D**-0.5, WINDOW, SINKS))
        self._product(b["at"].view(-1, H * D), "o", b["h1"], residual=h)
        norm._check(b["h1"], None, self.g2, 1e-6, self.kind, q=b["q"], scales=b["s"])
        self._product(b["q"], "up", b["up"], scale=(b["s"], self.up_scale), silu=True)
        self._product(b["up"], "down", b["h2"], bias=self.bias, residual=b["h1"])

    def _product(self, a, name, got, bias=None, residual=None, scale=None, silu=False):
        import torch

        x, w = a.double(), self.w[name].double()
        v, size = x @ w, x.abs() @ w.abs()
        err = 0 * v if a.dtype == torch.int8 else (math.ceil(x.shape[1] * a.element_size() / 32) + 1) * 2.0**-22 * size
        if scale is not None:
            s = scale[0].double()[:, None] * scale[1].double()
            v, err = v * s, err * s
        err = err + 2.0**-22 * v.abs()
        if bias is not None:
            v = v + bias.double()
            err = err + 2.0**-24 * v.abs()
        if silu:
            err = 1.2 * err + 4e-6 * (1 + v.abs())
            v = v * torch.sigmoid(v)
        if residual is not None:
            v = v + residual.double()
        tol = err + torch.finfo(got.dtype).eps / 2 * (v.abs() + err) * 1.0001 + 2.0**-23 * v.abs() + torch.finfo(got.dtype).tiny
        assert bool(torch.isfinite(got).all())
        assert bool(((got.double() - v).abs() <= tol).all()), ((got.double() - v).abs() / tol).max().item()


@pytest.mark.parametrize("kind", ["e4m3", "s8"])
@pytest.mark.parametrize("batch,prompt", [(1, 1), (3, 40), (2, 257)])
def test_prompt_then_tokens(kind, batch, prompt):
    import torch

    from onnxsharp_b200.runtime import Context

    stream = torch.cuda.Stream()
    c = Context(0, stream.cuda_stream)
    with torch.cuda.stream(stream):
        blocks = [Block(c, batch, kind, s) for s in (1, 2)]
        g = torch.Generator(device="cuda")
        g.manual_seed(prompt)
        lengths = torch.full((batch,), prompt, dtype=torch.int32, device="cuda")
        h = torch.randn((batch * prompt, WIDE), generator=g, device="cuda").bfloat16()
        slots = torch.arange(prompt, device="cuda").expand(batch, prompt)
        for block in blocks:
            b = block.buffers(prompt)
            block.run(h, b, lengths, slots)
            block.check(h, b, lengths, prompt)
            h = b["h2"]
        # a token at a time, all of it one graph that moves the lengths on by itself
        pos = torch.full((batch, 1), prompt - 1, device="cuda")
        x = h.view(batch, prompt, WIDE)[:, -1].contiguous()
        bufs = [block.buffers(1) for block in blocks]

        def step():
            lengths.add_(1)
            pos.add_(1)
            inp = x
            for block, b in zip(blocks, bufs):
                block.run(inp, b, lengths, pos)
                inp = b["h2"]

        graph = c.capture(step)  # (runs the step once before it is recorded)
        for _ in range(4):
            graph.launch()
            c.synchronize()
            inp = x
            for block, b in zip(blocks, bufs):
                block.check(inp, b, lengths, 1)
                inp = b["h2"]
            x.copy_(inp)
        assert lengths.tolist() == [prompt + 5] * batch
        graph.close()
    torch.cuda.synchronize()
    c.close()


def _far(shape, seed):
    """A large bf16 tensor, cheaply: random rows repeated."""
    import torch

    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    row = torch.randn((4099, shape[-1]), generator=g, device="cuda").bfloat16()
    return row[torch.arange(shape[0], device="cuda") % 4099]


def test_norm_rows_behind_two_to_the_31(ctx):
    import torch

    from onnxsharp_b200 import ops

    rows, cols = 530000, 4096
    x = _far((rows, cols), 1)
    q, s = torch.empty((rows, cols), dtype=torch.int8, device="cuda"), torch.empty(rows, device="cuda")
    ops.rmsnorm_quant(ctx, x, None, 1e-6, q, s)
    y = ops.rmsnorm(ctx, x, None, 1e-6, torch.empty_like(x))
    ctx.synchronize()
    for part in (slice(0, 8), slice(2**31 // cols - 4, 2**31 // cols + 4), slice(rows - 8, rows)):
        norm._check(x[part], None, None, 1e-6, "s8", y=y[part], q=q[part], scales=s[part])


def test_product_rows_behind_two_to_the_31(ctx):
    import torch

    from onnxsharp_b200.runtime import LinearWeights, linear

    m, k, n = 140001, 72, 16000
    a, res = _far((m, k), 2), torch.zeros((m, n), dtype=torch.bfloat16, device="cuda")
    w = _far((k, n), 3)
    spots = (slice(0, 8), slice(2**31 // n - 4, 2**31 // n + 4), slice(m - 8, m))
    for p in spots:
        res[p] = _far((8, n), 4)
    kept = [res[p].clone() for p in spots]
    linear(ctx, a, LinearWeights(ctx, w), residual=res, out=res)
    ctx.synchronize()
    for p, r in zip(spots, kept):
        v = a[p].double() @ w.double()
        err = (math.ceil(k * 2 / 32) + 1) * 2.0**-22 * (a[p].double().abs() @ w.double().abs()) + 2.0**-22 * v.abs()
        v = v + r.double()
        tol = err + 2.0**-8 * (v.abs() + err) * 1.0001 + 2.0**-23 * v.abs()
        assert bool(((res[p].double() - v).abs() <= tol).all())


@pytest.mark.parametrize("T", [1, 40])
def test_cache_rows_behind_two_to_the_31(ctx, T):
    import torch

    from onnxsharp_b200.runtime import attention_window

    S, heads, dim, near = 2**21 + 700, 8, 128, 6000
    cache = torch.zeros((1, S, heads, dim), dtype=torch.bfloat16, device="cuda")
    g = torch.Generator(device="cuda")
    g.manual_seed(5)
    n = S - 37
    cache[:, n - near : n] = torch.randn((1, near, heads, dim), generator=g, device="cuda").bfloat16()
    q = torch.randn((1, T, 16, dim), generator=g, device="cuda").bfloat16()
    lengths = torch.tensor([n], dtype=torch.int32, device="cuda")
    got = attention_window(ctx, q, cache, cache, lengths, dim**-0.5, window=4000)
    ctx.synchronize()
    part = cache[:, n - near : n]
    win._check(got, *win._reference(q, part, part, torch.tensor([near]), None, dim**-0.5, 4000, 0))
