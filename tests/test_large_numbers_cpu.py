"""Sizes and windows that do not fit the C ABI's ints: ctypes keeps their low 32 bits without a word, so the Python entry
points have to look. Meta tensors have shapes and strides but no memory; the library call is caught."""
from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch

from onnxsharp_b200 import ops, runtime

BIG = 2**32 + 4  # its low 32 bits are 4
CTX = SimpleNamespace(device=-1, handle=None)


@pytest.fixture
def calls(monkeypatch):
    made = []
    for module in (runtime, ops):
        monkeypatch.setattr(module, "call", lambda *a: made.append(a))
    return made


def _empty(*shape, dtype=torch.bfloat16):
    return torch.empty(shape, dtype=dtype, device="meta")


def test_norm(calls):
    x = _empty(2, BIG)
    with pytest.raises(ValueError, match="columns"):
        ops.rmsnorm(CTX, x, None, 1e-6, x)
    x = _empty(BIG, 8)  # rows are 64 bits
    ops.rmsnorm(CTX, x, None, 1e-6, x)
    assert calls[-1][7] == BIG


def _weights(k, n, dtype=torch.bfloat16):
    w = runtime.LinearWeights.__new__(runtime.LinearWeights)
    w.handle, w.k, w.n, w.dtype = None, k, n, dtype
    return w


def test_product(calls):
    with pytest.raises(ValueError, match="rows"):
        runtime.linear(CTX, _empty(BIG, 8), _weights(8, 16))
    runtime.linear(CTX, _empty(100, 8), _weights(8, 16))
    assert len(calls) == 1


@pytest.mark.parametrize("shape", [(BIG, 8), (8, BIG)])
@pytest.mark.parametrize("layout", [0, 1])
def test_weights(calls, shape, layout):
    with pytest.raises(ValueError, match="too large"):
        runtime.LinearWeights(SimpleNamespace(device=0, handle=None), _empty(*shape), layout=layout)
    assert not calls


@pytest.mark.parametrize("value,given", [(5, 5), (None, 2**31 - 1), (2**31 - 1, 2**31 - 1), (2**31, 2**31 - 1),
                                         (2**32 + 5, 2**31 - 1), (0, 0), (-3, -3), (-(2**32) + 5, -(2**31))])
def test_window(calls, value, given):
    q, n = _empty(2, 1, 8, 64), _empty(2, dtype=torch.int32)
    runtime.attention_window(CTX, q, _empty(2, 100, 2, 64), _empty(2, 100, 2, 64), n, 0.1, window=value)
    assert calls[-1][17] == given
    if value is not None:
        runtime.attention_window(CTX, q, _empty(2, 100, 2, 64), _empty(2, 100, 2, 64), n, 0.1, sinks=value)
        assert calls[-1][18] == given


@pytest.mark.parametrize("q,k", [((BIG, 1, 8, 64), (BIG, 9, 8, 64)), ((2, BIG, 8, 64), (2, 9, 8, 64)),
                                 ((2, 1, 8, 64), (2, BIG, 8, 64)), ((2, 1, BIG, 64), (2, 9, 4, 64)),
                                 ((2, 1, 8, 64), (2, 9, BIG, 64)), ((2, 1, 8, BIG), (2, 9, 8, BIG))])
def test_window_shapes(calls, q, k):
    with pytest.raises(ValueError, match="too large"):
        runtime.attention_window(CTX, _empty(*q), _empty(*k), _empty(*k), _empty(q[0], dtype=torch.int32), 0.1)
    assert not calls


def test_a_scale_too_large_for_powers_of_two():
    """scale * log2(e) has to be finite: against infinity a score of 0 would be NaN."""
    import ctypes as C

    from onnxsharp_b200 import _lib

    lib, at = _lib.load(), 1 << 20
    strides = (C.c_longlong * 3)(512, 512, 64)
    args = lambda scale: [C.create_string_buffer(1 << 12), _lib.BF16, at, strides, at, strides, at, strides, at, 0, 2, 1,  # noqa: E731
                          500, 8, 2, 64, 100, 4, scale, at, strides]
    assert lib.osc_attention_window(*args(3e38)) != 0
    assert "scale" in lib.osc_last_error().decode()
