"""CPU tests of the refusals of the grouped and MXFP4 entries: every invalid call fails
before it touches the device."""
import ctypes as C

import pytest
import torch

import gemmkit_amd as gk
from gemmkit_amd import _lib

A, B, X, O = 0x100000, 0x400000, 0x800000, 0xC00000


def ref(data, length, rows, cols, rs, cs):
    return _lib.MatRefC(data, length, rows, cols, rs, cs)


def mut(data, length, rows, cols, rs, cs):
    return _lib.MatMutC(data, length, rows, cols, rs, cs)


def grouped(a, b, c, offsets=O, groups=2, b_gs=64):
    rc = _lib.lib().gk_gemm_grouped_bf16(None, 1.0, C.byref(a), offsets, groups, C.byref(b), b_gs,
                                         0.0, C.byref(c), 1)
    return rc, _lib.last_error()


OK_A, OK_B, OK_C = ref(A, 80, 10, 8, 8, 1), ref(B, 128, 8, 8, 8, 1), mut(X, 80, 10, 8, 8, 1)


@pytest.mark.parametrize("change,code,text", [
    (dict(a=ref(A, 90, 10, 9, 9, 1)), -1, "A.cols (9) != B.rows (8)"),
    (dict(c=mut(X, 88, 11, 8, 8, 1)), -1, "A.rows (10) != C.rows (11)"),
    (dict(c=mut(X, 90, 10, 9, 9, 1)), -1, "B.cols (8) != C.cols (9)"),
    (dict(a=ref(A, 79, 10, 8, 8, 1)), -2, "A view of 10x8"),
    (dict(a=ref(A, 80, 10, 8, -8, 1)), -2, "A view has negative strides"),
    (dict(b=ref(B, 127, 8, 8, 8, 1)), -2, "B batched view"),
    (dict(b_gs=-64), -2, "B batch stride (-64) must be non-negative"),
    (dict(c=mut(X, 79, 10, 8, 8, 1)), -2, "C view of 10x8"),
    (dict(c=mut(X, 80, 10, 8, 1, 1)), -3, "C view aliases itself"),
    (dict(c=mut(A + 64, 80, 10, 8, 8, 1)), -3, "C aliases A or B"),
    (dict(c=mut(B + 64, 80, 10, 8, 8, 1)), -3, "C aliases A or B"),
    (dict(offsets=X + 8), -3, "C aliases the group offsets"),
    (dict(offsets=None), -4, "group offsets"),
    (dict(offsets=O + 2), -4, "group offsets"),
    (dict(a=ref(A, 2 ** 40, 2 ** 31, 8, 8, 1), c=mut(X + 2 ** 42, 2 ** 40, 2 ** 31, 8, 8, 1)), -6,
     "below 2^31"),
    (dict(a=ref(A, 2 ** 30, 10, 2 ** 22, 2 ** 22, 1), b=ref(B, 2 ** 30, 2 ** 22, 8, 8, 1),
          c=mut(X + 2 ** 42, 80, 10, 8, 8, 1)), -6, "4 MiB"),
])
def test_grouped_refusals(change, code, text):
    args = dict(a=OK_A, b=OK_B, c=OK_C)
    args.update(change)
    rc, msg = grouped(**args)
    assert rc == code, msg
    assert text in msg


def wgrad(a, b, c, offsets=O, groups=2, c_gs=64):
    rc = _lib.lib().gk_gemm_grouped_wgrad_bf16_f32out(None, 1.0, C.byref(a), offsets, groups,
                                                      C.byref(b), 0.0, C.byref(c), c_gs, 1)
    return rc, _lib.last_error()


W_A, W_B, W_C = ref(A, 80, 10, 8, 8, 1), ref(B, 80, 10, 8, 8, 1), mut(X, 128, 8, 8, 8, 1)


@pytest.mark.parametrize("change,code,text", [
    (dict(b=ref(B, 88, 11, 8, 8, 1)), -1, "A.rows (10) != B.rows (11)"),
    (dict(c=mut(X, 200, 9, 8, 8, 1)), -1, "A.cols (8) != C.rows (9)"),
    (dict(c=mut(X, 200, 8, 9, 9, 1), c_gs=72), -1, "B.cols (8) != C.cols (9)"),
    (dict(a=ref(A, 79, 10, 8, 8, 1)), -2, "A view of 10x8"),
    (dict(b=ref(B, 79, 10, 8, 8, 1)), -2, "B view of 10x8"),
    (dict(c=mut(X, 127, 8, 8, 8, 1)), -2, "C batched view"),
    (dict(c_gs=63), -3, "C group stride (63)"),
    (dict(c=mut(X, 128, 8, 8, 0, 1)), -3, "aliases itself"),
    (dict(c=mut(A, 128, 8, 8, 8, 1)), -3, "C aliases A or B"),
    (dict(offsets=X), -3, "C aliases the group offsets"),
    (dict(offsets=None), -4, "group offsets"),
    (dict(b=ref(B, 2 ** 30, 10, 2 ** 22, 2 ** 22, 1), c=mut(X + 2 ** 42, 2 ** 30, 8, 2 ** 22, 2 ** 22, 1),
          c_gs=2 ** 25), -6, "4 MiB"),
])
def test_wgrad_refusals(change, code, text):
    args = dict(a=W_A, b=W_B, c=W_C)
    args.update(change)
    rc, msg = wgrad(**args)
    assert rc == code, msg
    assert text in msg


def q(codes=A, codes_len=10 * 32, scales=B, scales_len=160, rows=10, cols=64, ld=32, lds=16):
    return _lib.Mxfp4C(codes, codes_len, scales, scales_len, rows, cols, ld, lds)


@pytest.mark.parametrize("mx,code,text", [
    (q(codes=A + 8), -2, "16-byte aligned"),
    (q(scales=B + 1), -2, "16-byte aligned"),
    (q(ld=16), -2, "at least 32 and 16"),
    (q(ld=40), -2, "multiples of 16"),
    (q(lds=8), -2, "at least 32 and 16"),
    (q(codes_len=319), -2, "more bytes of codes"),
    (q(scales_len=159), -2, "more bytes of codes"),
    (q(rows=2 ** 31), -6, "below 2^31"),
    (q(cols=2 ** 24, ld=2 ** 23, lds=2 ** 19, codes_len=2 ** 40, scales_len=2 ** 40), -6, "4 MiB"),
])
def test_mxfp4_refusals(mx, code, text):
    L = _lib.lib()
    x = ref(X, 640, 10, 64, 64, 1)
    rc = L.gk_quantize_mxfp4_f32(C.byref(x), C.byref(mx))
    assert rc == code and text in _lib.last_error()
    c = mut(X, 640, 10, 64, 64, 1)
    rc = L.gk_dequantize_mxfp4_bf16(C.byref(mx), C.byref(c))
    assert rc == code and text in _lib.last_error()
    good = q(codes=O, scales=O + 4096)
    c = mut(X, 100, 10, 10, 10, 1)
    for a, b in ((mx, good), (good, mx)):
        rc = L.gk_gemm_mxfp4_f32(None, 1.0, C.byref(a), C.byref(b), 0.0, C.byref(c), 1)
        assert rc == code and text in _lib.last_error()


def test_mxfp4_shapes_and_aliases():
    L = _lib.lib()
    good = q()
    for x, code, text in ((ref(X, 650, 10, 65, 65, 1), -1, "MXFP4 output is 10x64"),
                          (ref(X, 639, 10, 64, 64, 1), -2, "X view"),
                          (ref(A + 64, 640, 10, 64, 64, 1), -3, "overlap"),
                          (ref(X, 640, 10, 64, -64, 1), -2, "negative")):
        assert L.gk_quantize_mxfp4_f32(C.byref(x), C.byref(good)) == code
        assert text in _lib.last_error()
    x = ref(X, 640, 10, 64, 64, 1)
    over = q(scales=A + 16)
    assert L.gk_quantize_mxfp4_f32(C.byref(x), C.byref(over)) == -3
    for c, code, text in ((mut(X, 650, 10, 65, 65, 1), -1, "MXFP4 input is 10x64"),
                          (mut(X, 640, 10, 64, 1, 1), -3, "aliases itself"),
                          (mut(B, 640, 10, 64, 64, 1), -3, "aliases the MXFP4")):
        assert L.gk_dequantize_mxfp4_f32(C.byref(good), C.byref(c)) == code
        assert text in _lib.last_error()
    b = q(codes=O, scales=O + 4096)
    for a, bb, c, code, text in (
            (q(cols=32), b, mut(X, 100, 10, 10, 10, 1), -1, "A.cols (32) != B.cols (64)"),
            (good, b, mut(X, 110, 11, 10, 10, 1), -1, "A.rows (10) != C.rows (11)"),
            (good, b, mut(X, 110, 10, 11, 11, 1), -1, "B.rows (10) != C.cols (11)"),
            (good, b, mut(X, 99, 10, 10, 10, 1), -2, "C view"),
            (good, b, mut(X, 100, 10, 10, 0, 1), -3, "aliases itself"),
            (good, b, mut(A, 100, 10, 10, 10, 1), -3, "C aliases A or B")):
        rc = L.gk_gemm_mxfp4_bf16(None, 1.0, C.byref(a), C.byref(bb), 0.0, C.byref(c), 1)
        assert rc == code and text in _lib.last_error()
    c = mut(X, 100, 10, 5, 5, 1)
    for groups, off, code, text in ((2, None, -4, "group offsets"), (2, X, -3, "offsets"),
                                    (3, O, -1, "for each of 3 groups")):
        rc = L.gk_gemm_grouped_mxfp4_bf16(None, 1.0, C.byref(good), off, groups, C.byref(b), 0.0,
                                          C.byref(c), 1)
        assert rc == code and text in _lib.last_error()


def test_null_arguments():
    L = _lib.lib()
    a, c, m = OK_A, OK_C, q()
    assert L.gk_gemm_grouped_bf16(None, 1.0, None, O, 2, C.byref(a), 0, 0.0, C.byref(c), 1) == -4
    assert L.gk_gemm_grouped_wgrad_bf16(None, 1.0, C.byref(a), O, 2, None, 0.0, C.byref(c), 0, 1) == -4
    assert L.gk_quantize_mxfp4_bf16(None, C.byref(m)) == -4
    assert L.gk_quantize_mxfp4_bf16(C.byref(a), None) == -4
    assert L.gk_dequantize_mxfp4_f32(C.byref(m), None) == -4
    assert L.gk_gemm_mxfp4_f32(None, 1.0, None, C.byref(m), 0.0, C.byref(c), 1) == -4
    assert L.gk_gemm_grouped_mxfp4_f32(None, 1.0, C.byref(m), O, 1, C.byref(m), 0.0, None, 1) == -4


def test_python_refuses_host_tensors_and_wrong_types():
    if torch.cuda.is_available():
        pytest.skip("host without a device")
    x = torch.zeros(64, dtype=torch.bfloat16)
    with pytest.raises(gk.GemmkitError):
        gk.quantize_mxfp4(gk.MatRef.from_row_major(x, 1, 64))
    with pytest.raises(gk.GemmkitError):
        gk.gemm_grouped(1.0, gk.MatRef.from_row_major(x, 8, 8), torch.zeros(2, dtype=torch.int32),
                        gk.MatRef.from_row_major(x, 8, 8), 0, 0.0, gk.MatMut.from_row_major(x, 8, 8))
