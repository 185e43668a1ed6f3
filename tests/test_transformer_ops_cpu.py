"""What osc_rmsnorm, osc_linear and osc_attention_window refuse, on the host alone: every argument is checked before
the device is touched, so the context and the weights are zeroed buffers, and every address is made up."""
from __future__ import annotations

import ctypes as C

import pytest

F32, F16, BF16, S8, E4M3 = range(5)
AT = 1 << 20  # an aligned address that nothing may read
INT_MAX = 2**31 - 1


@pytest.fixture(scope="module")
def lib():
    from onnxsharp_b200 import _lib

    return _lib.load()


@pytest.fixture(scope="module")
def fake():
    return C.create_string_buffer(1 << 12)


def _refused(lib, code, word):
    assert code != 0
    assert word in lib.osc_last_error().decode(), lib.osc_last_error().decode()


NORM = dict(dtype=BF16, x=AT, x_ld=0, residual=0, res_ld=0, rows=4, cols=64, gamma=AT, eps=1e-6, sum=0, sum_ld=0, y=AT,
            y_ld=0, q_dtype=0, q=0, q_ld=0, scales=0)


@pytest.mark.parametrize(
    "change,word",
    [
        (dict(dtype=S8), "not f32, f16 or bf16"),
        (dict(dtype=77), "not f32, f16 or bf16"),
        (dict(rows=-1), "bad shape"),
        (dict(rows=2**31), "bad shape"),
        (dict(cols=0), "bad shape"),
        (dict(eps=0.0), "eps"),
        (dict(eps=-1.0), "eps"),
        (dict(eps=float("nan")), "eps"),
        (dict(eps=float("inf")), "eps"),
        (dict(y=0), "neither"),
        (dict(q=AT, scales=AT, q_dtype=BF16), "not s8 or e4m3"),
        (dict(q=AT, q_dtype=S8), "come together"),
        (dict(scales=AT), "come together"),
        (dict(sum=AT), "without a residual"),
        (dict(x_ld=63), "pitch"),
        (dict(x_ld=-64), "pitch"),
        (dict(y_ld=1), "pitch"),
        (dict(x=0), "null x"),
        (dict(x=AT + 1), "aligned"),
        (dict(residual=AT + 1), "aligned"),
        (dict(gamma=AT + 1), "aligned"),
        (dict(q=AT, q_dtype=S8, scales=AT + 2), "aligned"),
    ],
)
def test_norm_refuses(lib, fake, change, word):
    a = {**NORM, **change}
    _refused(lib, lib.osc_rmsnorm(fake, *a.values()), word)


def test_norm_without_rows_or_a_context(lib, fake):
    assert lib.osc_rmsnorm(fake, *{**NORM, "rows": 0, "x": 0, "y": 0}.values()) == 0
    _refused(lib, lib.osc_rmsnorm(None, *NORM.values()), "null context")


WIN = dict(dtype=BF16, q=AT, qs=(512, 512, 64), k=AT, ks=(64000, 128, 64), v=AT, vs=(64000, 128, 64), lengths=AT, starts=0,
           B=2, T=1, S=500, H=8, HK=2, D=64, window=100, sinks=4, scale=0.125, out=AT, os=(512, 512, 64))


def _win(a):
    return [(C.c_longlong * 3)(*v) if isinstance(v, tuple) else v for v in a.values()]


@pytest.mark.parametrize(
    "change,word",
    [
        (dict(dtype=F32), "not f16 or bf16"),
        (dict(B=-1), "bad shape"),
        (dict(T=-1), "bad shape"),
        (dict(S=0), "bad shape"),
        (dict(S=INT_MAX), "bad shape"),
        (dict(T=INT_MAX), "bad shape"),
        (dict(HK=0), "bad shape"),
        (dict(H=7), "7 heads over 2"),
        (dict(H=258), "258 heads over 2"),
        (dict(D=96), "head size 96"),
        (dict(window=0), "window 0"),
        (dict(sinks=-1), "sinks -1"),
        (dict(scale=0.0), "scale"),
        (dict(scale=float("nan")), "scale"),
        (dict(scale=float("inf")), "scale"),
        (dict(B=65536), "at most 65535"),
        (dict(qs=None), "null strides"),
        (dict(q=0), "null pointer"),
        (dict(lengths=0), "null pointer"),
        (dict(k=AT + 8), "16-byte"),
        (dict(ks=(64000, 127, 64)), "16-byte"),
        (dict(vs=(-64000, 128, 64)), "16-byte"),
        (dict(vs=(1 << 40, 128, 64)), "16-byte"),
        (dict(os=(512, 512, 60)), "16-byte"),
        (dict(lengths=AT + 2), "aligned"),
        (dict(starts=AT + 1), "aligned"),
    ],
)
def test_window_refuses(lib, fake, change, word):
    _refused(lib, lib.osc_attention_window(fake, *_win({**WIN, **change})), word)


def test_window_without_rows_or_a_context(lib, fake):
    for change in (dict(B=0), dict(T=0)):
        assert lib.osc_attention_window(fake, *_win({**WIN, **change, "q": 0, "out": 0})) == 0
    _refused(lib, lib.osc_attention_window(None, *_win(WIN)), "null context")


def _weights(dtype, k, n, device=0):
    """The head of osc_linear_weights: device, dtype, k, n."""
    return (C.c_int * 256)(device, dtype, k, n)


LIN = dict(a=AT, m=4, lda=0, w=None, a_scale=0, w_scale=0, n_scale=0, bias=0, act=0, residual=0, ldr=0, out=BF16, y=AT, ldy=0)


@pytest.mark.parametrize(
    "kind,change,word",
    [
        (BF16, dict(m=-1), "m = -1"),
        (BF16, dict(m=INT_MAX), "m = 2147483647"),
        (BF16, dict(out=S8), "not f32, f16 or bf16"),
        (BF16, dict(out=9), "not f32, f16 or bf16"),
        (BF16, dict(act=-1), "activation"),
        (BF16, dict(act=6), "activation"),
        (BF16, dict(a_scale=AT), "8-bit"),
        (F16, dict(w_scale=AT, n_scale=1), "8-bit"),
        (S8, dict(w_scale=AT, n_scale=2), "2 column scales"),
        (E4M3, dict(w_scale=AT, n_scale=0), "0 column scales"),
        (BF16, dict(lda=63), "pitch"),
        (BF16, dict(ldy=31), "pitch"),
        (BF16, dict(residual=AT, ldr=-1), "pitch"),
        (BF16, dict(a=0), "null pointer"),
        (BF16, dict(y=0), "null pointer"),
        (BF16, dict(a=AT + 1), "aligned"),
        (S8, dict(out=F32, y=AT + 2), "aligned"),
        (BF16, dict(residual=AT + 1), "aligned"),
        (S8, dict(a_scale=AT + 2), "aligned"),
        (BF16, dict(bias=AT + 2), "aligned"),
    ],
)
def test_product_refuses(lib, fake, kind, change, word):
    a = {**LIN, "w": _weights(kind, 64, 32), **change}
    _refused(lib, lib.osc_linear(fake, *a.values()), word)


def test_product_without_rows_weights_or_a_context(lib, fake):
    w = _weights(BF16, 64, 32)
    assert lib.osc_linear(fake, *{**LIN, "w": w, "m": 0, "a": 0, "y": 0}.values()) == 0
    _refused(lib, lib.osc_linear(fake, *LIN.values()), "null weights")
    _refused(lib, lib.osc_linear(None, *{**LIN, "w": w}.values()), "null context")
    _refused(lib, lib.osc_linear(fake, *{**LIN, "w": _weights(BF16, 64, 32, device=1)}.values()), "weights of device 1")
    assert lib.osc_linear_weights_free(None) == 0


@pytest.mark.parametrize(
    "dtype,w,k,n,layout,word",
    [
        (F32, AT, 64, 32, 0, "not f16"),
        (BF16, 0, 64, 32, 0, "bad W"),
        (BF16, AT, 0, 32, 0, "bad W"),
        (BF16, AT, 64, -1, 0, "bad W"),
        (BF16, AT, 64, 32, 2, "layout 2"),
        (S8, AT, 1 << 17, 1, 0, "overflows S32"),
        (BF16, AT, INT_MAX, 1, 0, "too large"),
        (BF16, AT, 64, INT_MAX, 1, "too large"),
        (BF16, AT, 64, 65532 * 32 + 1, 0, "too large"),
        (BF16, AT + 1, 64, 32, 0, "aligned"),
    ],
)
def test_prepack_refuses(lib, fake, dtype, w, k, n, layout, word):
    out = C.c_void_p(1)
    _refused(lib, lib.osc_linear_prepack(fake, dtype, w, k, n, layout, 0, C.byref(out)), word)
    assert out.value is None
    _refused(lib, lib.osc_linear_prepack(None, BF16, AT, 64, 32, 0, 0, C.byref(out)), "null context")
