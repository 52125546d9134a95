"""CPU tests of the refusals of the linear-layer and MXINT8 entries: every invalid call fails
before it touches the device."""
import ctypes as C

import pytest
import torch

import gemmkit_amd as gk
from gemmkit_amd import _lib

A, B, X, R, Z, S, O = (0x100000 * i for i in range(1, 8))


def ref(data, length, rows, cols, rs, cs):
    return _lib.MatRefC(data, length, rows, cols, rs, cs)


def mut(data, length, rows, cols, rs, cs):
    return _lib.MatMutC(data, length, rows, cols, rs, cs)


def mx(codes=Z, codes_len=320, scales=S, scales_len=160, rows=10, cols=6, ld=32, lds=16):
    return _lib.Mxint8C(codes, codes_len, scales, scales_len, rows, cols, ld, lds)


def bias(data=O, n=6, dim=1):
    return _lib.BiasC(data, n, dim)


def by(x):
    return None if x is None else C.byref(x)


OK_A, OK_B, OK_C = ref(A, 80, 10, 8, 8, 1), ref(B, 48, 8, 6, 6, 1), mut(X, 60, 10, 6, 6, 1)


def linear(a=OK_A, b=OK_B, c=OK_C, bias=None, wide=0, act=0, slope=0.0, res=None, z=None, zq=None,
           entry="gk_gemm_linear_bf16"):
    rc = getattr(_lib.lib(), entry)(None, 1.0, by(a), by(b), by(bias), wide, act, slope, by(res),
                                    by(z), by(zq), by(c), 1)
    return rc, _lib.last_error()


@pytest.mark.parametrize("change,code,text", [
    (dict(a=None), -4, "null"),
    (dict(c=None), -4, "null"),
    (dict(a=ref(A, 90, 10, 9, 9, 1)), -1, "A.cols (9) != B.rows (8)"),
    (dict(c=mut(X, 66, 11, 6, 6, 1)), -1, "A.rows (10) != C.rows (11)"),
    (dict(c=mut(X, 70, 10, 7, 7, 1)), -1, "B.cols (6) != C.cols (7)"),
    (dict(a=ref(A, 79, 10, 8, 8, 1)), -2, "A view of 10x8"),
    (dict(a=ref(A, 80, 10, 8, -8, 1)), -2, "A view has negative strides"),
    (dict(b=ref(B, 47, 8, 6, 6, 1)), -2, "B view of 8x6"),
    (dict(c=mut(X, 59, 10, 6, 6, 1)), -2, "C view of 10x6"),
    (dict(c=mut(X, 60, 10, 6, 1, 1)), -3, "C view aliases itself"),
    (dict(c=mut(A + 64, 60, 10, 6, 6, 1)), -3, "C aliases A"),
    (dict(c=mut(B + 64, 60, 10, 6, 6, 1)), -3, "C aliases B"),
    (dict(act=6), -4, "activation (6)"),
    (dict(act=-1), -4, "activation (-1)"),
    (dict(act=2, slope=float("inf")), -4, "slope must be finite"),
    (dict(bias=bias(dim=0)), -4, "must be 1 (PerCol)"),
    (dict(bias=bias(n=5)), -1, "bias length (5)"),
    (dict(bias=bias(data=None)), -4, "bias is null"),
    (dict(bias=bias(data=O + 2), wide=1), -4, "not aligned"),
    (dict(bias=bias(data=X + 8)), -3, "C aliases bias"),
    (dict(res=ref(R, 60, 9, 6, 6, 1)), -1, "the residual is 9x6, the output 10x6"),
    (dict(res=ref(R, 59, 10, 6, 6, 1)), -2, "the residual view of 10x6"),
    (dict(res=ref(X, 60, 10, 6, 1, 10)), -3, "C aliases the residual"),
    (dict(res=ref(X + 2, 60, 10, 6, 6, 1)), -3, "C aliases the residual"),
    (dict(z=mut(Z, 60, 10, 5, 6, 1)), -1, "Z is 10x5, the output 10x6"),
    (dict(z=mut(Z, 59, 10, 6, 6, 1)), -2, "Z view of 10x6"),
    (dict(z=mut(Z, 60, 10, 6, 0, 1)), -3, "Z view aliases itself"),
    (dict(z=mut(X + 4, 60, 10, 6, 6, 1)), -3, "Z aliases C"),
    (dict(z=mut(A, 60, 10, 6, 6, 1)), -3, "Z aliases A"),
    (dict(res=ref(R, 60, 10, 6, 6, 1), z=mut(R, 60, 10, 6, 6, 1)), -3, "Z aliases the residual"),
    (dict(res=ref(X, 60, 10, 6, 6, 1), z=mut(X, 60, 10, 6, 6, 1)), -3, "Z aliases the residual"),
    (dict(z=mut(Z, 60, 10, 6, 6, 1), zq=mx()), -4, "given twice"),
    (dict(zq=mx(rows=9)), -1, "Z is 9x6"),
    (dict(zq=mx(ld=16)), -2, "MXINT8 Z needs 16-byte aligned"),
    (dict(zq=mx(ld=40)), -2, "MXINT8 Z needs 16-byte aligned"),
    (dict(zq=mx(lds=8)), -2, "MXINT8 Z needs 16-byte aligned"),
    (dict(zq=mx(codes=Z + 8)), -2, "MXINT8 Z needs 16-byte aligned"),
    (dict(zq=mx(codes_len=319)), -2, "needs more bytes"),
    (dict(zq=mx(scales_len=159)), -2, "needs more bytes"),
    (dict(zq=mx(scales=Z + 16)), -3, "Z's scales aliases Z's codes"),
    (dict(zq=mx(codes=X)), -3, "Z's codes aliases C"),
    (dict(zq=mx(scales=B)), -3, "Z's scales aliases B"),
    (dict(a=ref(A, 2 ** 40, 2 ** 31, 8, 8, 1), c=mut(X + 2 ** 42, 2 ** 40, 2 ** 31, 6, 6, 1)), -6,
     "below 2^31"),
    (dict(a=ref(A, 2 ** 30, 10, 2 ** 22, 2 ** 22, 1), b=ref(B + 2 ** 44, 2 ** 30, 2 ** 22, 6, 6, 1),
          c=mut(X + 2 ** 42, 60, 10, 6, 6, 1)), -6, "4 MiB"),
])
def test_linear_refusals(change, code, text):
    for entry in ("gk_gemm_linear_bf16", "gk_gemm_linear_f32out"):
        if "residual" in text and "C aliases" in text and entry.endswith("f32out"):
            continue  # (written for bf16's element size)
        rc, msg = linear(entry=entry, **change)
        assert rc == code, msg
        assert text in msg


def dgrad(a=OK_A, b=OK_B, act=3, slope=0.0, z=None, zq=None, dbias=None, n=6, d=OK_C,
          entry="gk_gemm_linear_dgrad_bf16"):
    rc = getattr(_lib.lib(), entry)(None, 1.0, by(a), by(b), act, slope, by(z), by(zq), dbias, n,
                                    by(d), 1)
    return rc, _lib.last_error()


OK_Z = ref(Z, 60, 10, 6, 6, 1)
GRADS = [
    (dict(), -4, "needs its pre-activations"),
    (dict(act=0, z=OK_Z), -4, "pre-activations without an activation"),
    (dict(z=OK_Z, zq=mx()), -4, "given twice"),
    (dict(act=9, z=OK_Z), -4, "activation (9)"),
    (dict(act=2, slope=float("nan"), z=OK_Z), -4, "slope must be finite"),
    (dict(z=ref(Z, 60, 10, 5, 6, 1)), -1, "Z is 10x5"),
    (dict(z=ref(Z, 59, 10, 6, 6, 1)), -2, "Z view of 10x6"),
    (dict(z=ref(X, 60, 10, 6, 6, 1)), -3, "D aliases Z"),
    (dict(zq=mx(scales=X)), -3, "D aliases Z's scales"),
    (dict(zq=mx(cols=7)), -1, "Z is 10x7"),
    (dict(z=OK_Z, dbias=O, n=5), -1, "dbias length (5)"),
    (dict(z=OK_Z, dbias=O + 2), -4, "dbias is not aligned"),
    (dict(z=OK_Z, dbias=X + 16), -3, "dbias aliases D"),
    (dict(z=OK_Z, dbias=Z + 16), -3, "dbias aliases Z"),
    (dict(z=OK_Z, d=mut(X, 60, 10, 6, 3, 1)), -3, "D view aliases itself"),
    (dict(z=OK_Z, d=None), -4, "null"),
]


@pytest.mark.parametrize("change,code,text", GRADS + [
    (dict(z=OK_Z, dbias=A), -3, "dbias aliases A"),
    (dict(z=OK_Z, d=mut(B, 60, 10, 6, 6, 1)), -3, "D aliases B"),
    (dict(z=OK_Z, a=ref(A, 90, 10, 9, 9, 1)), -1, "A.cols (9) != B.rows (8)"),
    (dict(z=OK_Z, d=mut(X, 66, 11, 6, 6, 1)), -1, "A.rows (10) != D.rows (11)"),
])
def test_dgrad_refusals(change, code, text):
    rc, msg = dgrad(**change)
    assert rc == code, msg
    assert text in msg


def act_grad(g=ref(R, 60, 10, 6, 6, 1), act=3, slope=0.0, z=None, zq=None, dbias=None, n=6,
             d=OK_C, entry="gk_activation_grad_bf16"):
    rc = getattr(_lib.lib(), entry)(None, by(g), act, slope, by(z), by(zq), dbias, n, by(d))
    return rc, _lib.last_error()


@pytest.mark.parametrize("change,code,text", GRADS + [
    (dict(z=OK_Z, g=None), -4, "null"),
    (dict(z=OK_Z, g=ref(R, 60, 10, 5, 6, 1)), -1, "G is 10x5"),
    (dict(z=OK_Z, g=ref(R, 59, 10, 6, 6, 1)), -2, "G view of 10x6"),
    (dict(z=OK_Z, g=ref(X, 60, 10, 6, 1, 10)), -3, "D aliases G"),
    (dict(z=OK_Z, g=ref(X, 60, 10, 6, 6, 1), entry="gk_activation_grad_f32"), -3, "D aliases G"),
    (dict(z=OK_Z, g=ref(O, 60, 10, 6, 6, 1), dbias=O), -3, "dbias aliases G"),
])
def test_activation_grad_refusals(change, code, text):
    rc, msg = act_grad(**change)
    assert rc == code, msg
    assert text in msg


@pytest.mark.parametrize("change,code,text", [
    (dict(x=None), -4, "null"),
    (dict(q=None), -4, "null"),
    (dict(x=ref(A, 60, 10, 5, 6, 1)), -1, "MXINT8 output is 10x6, the matrix 10x5"),
    (dict(x=ref(A, 59, 10, 6, 6, 1)), -2, "X view of 10x6"),
    (dict(x=ref(Z, 60, 10, 6, 6, 1)), -3, "codes aliases X"),
    (dict(q=mx(scales=Z)), -3, "scales aliases codes"),
    (dict(q=mx(lds=24)), -2, "MXINT8 output needs"),
    (dict(q=mx(codes=None)), -2, "MXINT8 output needs"),
    (dict(q=mx(rows=2 ** 31, cols=2 ** 31)), -6, "below"),
])
def test_quantize_refusals(change, code, text):
    args = dict(x=ref(A, 60, 10, 6, 6, 1), q=mx())
    args.update(change)
    for entry in ("gk_quantize_mxint8_bf16", "gk_quantize_mxint8_f32"):
        assert getattr(_lib.lib(), entry)(by(args["x"]), by(args["q"])) == code
        assert text in _lib.last_error()


@pytest.mark.parametrize("change,code,text", [
    (dict(c=None), -4, "null"),
    (dict(act=7), -4, "activation (7)"),
    (dict(c=mut(X, 60, 10, 5, 6, 1)), -1, "MXINT8 input is 10x6, the matrix 10x5"),
    (dict(c=mut(X, 60, 10, 6, 0, 1)), -3, "C view aliases itself"),
    (dict(c=mut(S, 60, 10, 6, 6, 1)), -3, "C aliases scales"),
])
def test_dequantize_refusals(change, code, text):
    args = dict(c=OK_C, q=mx(), act=0)
    args.update(change)
    for entry in ("gk_dequantize_mxint8_bf16", "gk_dequantize_mxint8_f32"):
        rc = getattr(_lib.lib(), entry)(by(args["q"]), args["act"], 0.0, by(args["c"]))
        assert rc == code
        assert text in _lib.last_error()


@pytest.mark.parametrize("change,code,text", [
    (dict(a=None), -4, "null"),
    (dict(b=ref(B, 88, 11, 8, 8, 1)), -1, "A.rows (10) != B.rows (11)"),
    (dict(c=mut(X, 56, 7, 8, 8, 1)), -1, "A.cols (6) != C.rows (7)"),
    (dict(c=mut(X, 54, 6, 9, 9, 1)), -1, "B.cols (8) != C.cols (9)"),
    (dict(b=ref(B, 79, 10, 8, 8, 1)), -2, "B view of 10x8"),
    (dict(c=mut(B, 48, 6, 8, 8, 1)), -3, "C aliases B"),
    (dict(c=mut(Z, 48, 6, 8, 8, 1)), -3, "C aliases A"),
    (dict(act=-3), -4, "activation (-3)"),
    (dict(a=mx(cols=2 ** 22, ld=2 ** 22, codes_len=2 ** 30, lds=2 ** 17, scales_len=2 ** 30,
               scales=S + 2 ** 40),
          c=mut(X + 2 ** 50, 2 ** 30, 2 ** 22, 8, 8, 1)), -6, "4 MiB"),
])
def test_wgrad_refusals(change, code, text):
    args = dict(a=mx(), b=ref(B, 80, 10, 8, 8, 1), c=mut(X, 48, 6, 8, 8, 1), act=0)
    args.update(change)
    for entry in ("gk_gemm_wgrad_mxint8_bf16", "gk_gemm_wgrad_mxint8_f32"):
        rc = getattr(_lib.lib(), entry)(None, 1.0, by(args["a"]), args["act"], 0.0, by(args["b"]),
                                        0.0, by(args["c"]), 1)
        assert rc == code, _lib.last_error()
        assert text in _lib.last_error()


def test_smooth_activations_are_not_the_fused_entries():
    for act in (3, 4, 5):
        for name, one in (("gk_gemm_fused_f32", 1.0), ("gk_gemm_fused_bf16", 0x3F80)):
            zero = 0.0 if isinstance(one, float) else 0
            rc = getattr(_lib.lib(), name)(None, one, by(OK_A), by(OK_B), zero, by(OK_C), None, act,
                                           zero, 1)
            assert rc == -4 and f"activation ({act})" in _lib.last_error()


def test_python_types():
    t = torch.zeros(60, dtype=torch.float16)
    m = gk.MatMut(t, 10, 6, 6, 1)
    for call in (lambda: gk.gemm_linear(1.0, m, m, m), lambda: gk.quantize_mxint8(m),
                 lambda: gk.gemm_linear_dgrad(1.0, m, m, m), lambda: gk.activation_grad(m, m),
                 lambda: gk.gemm_wgrad_mxint8(1.0, None, m, 0.0, m),
                 lambda: gk.dequantize_mxint8(None, m)):
        with pytest.raises(TypeError):
            call()


@pytest.mark.parametrize("n", [0, 5, 7])
def test_python_dbias_length(n):
    """A dbias of any wrong length, one of no elements (whose pointer is null) among them."""
    t = torch.zeros(60, dtype=torch.bfloat16)
    d = gk.MatMut(t, 10, 6, 6, 1)
    dbias = torch.empty(n)
    for call in (lambda: gk.gemm_linear_dgrad(1.0, gk.MatRef(t, 10, 6, 6, 1), gk.MatRef(t, 6, 6, 6, 1), d,
                                              dbias=dbias),
                 lambda: gk.activation_grad(gk.MatRef(t, 10, 6, 6, 1), d, dbias=dbias)):
        with pytest.raises(gk.GemmkitError, match=rf"dbias length \({n}\) != the output's columns \(6\)") as e:
            call()
        assert e.value.code == -1
