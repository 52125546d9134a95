"""MXFP4 over the whole range of its scales: every scale byte with every code, blocks below the
normal range, products whose scales meet at either end; and matrices whose rows lie apart."""
import pytest
import torch

import gemmkit_amd as gk
from test_gpu_mxfp4 import mx, quantize_ref, random_mx, sample, unpack, values_of

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("out", [BF16, F32])
@pytest.mark.parametrize("how", ["row", "col", "odd"])
def test_every_scale_byte_and_code(dev, out, how):
    """Exact where f32 holds the value, subnormal ones among them; 2^128 and more is infinite."""
    byte = torch.arange(256, dtype=torch.uint8).view(256, 1)
    code = torch.arange(32, dtype=torch.uint8).remainder(16).repeat(256, 1)
    c_t, s_t, *_ = mx(code, byte, dev)
    buf = torch.full((256 * 40,), 7.0, dtype=out, device=dev)
    rs, cs = {"row": (32, 1), "col": (1, 256), "odd": (33, 1)}[how]
    gk.dequantize_mxfp4(gk.MatMxfp4(c_t, s_t, 256, 32), gk.MatMut(buf, 256, 32, rs, cs))
    got = torch.as_strided(buf.cpu(), (256, 32), (rs, cs)).float()
    want = values_of(code, byte).float()  # (f64 to f32: beyond its range infinite)
    assert torch.isnan(got[255]).all()
    assert torch.equal(got[:255], want[:255])


@pytest.mark.parametrize("dt", [BF16, F32])
@pytest.mark.parametrize("how", ["row", "col", "odd"])
def test_quantize_below_the_normal_range(dev, dt, how):
    """Blocks whose largest magnitude is subnormal, or near enough for the scale 2^-127."""
    rows = 24
    unit = 2.0 ** -133 if dt == BF16 else 2.0 ** -149
    x = torch.zeros(rows, 32, dtype=torch.float64)
    for r in range(rows):
        x[r] = torch.arange(32) * unit * 2.0 ** (r * (8 if dt == BF16 else 24) // rows)
        x[r, 1::2] *= -1
    x[1] = 2.0 ** -130 * torch.arange(32)
    x[2] = 2.0 ** -128 * torch.arange(32) / 4
    x = x.to(dt)
    if how == "col":
        t, rs, cs = x.t().contiguous().flatten().to(dev), 1, rows
    else:
        ld = 32 if how == "row" else 33
        t, rs, cs = torch.zeros(rows, ld, dtype=dt), ld, 1
        t[:, :32] = x
        t = t.flatten().to(dev)
    q = gk.quantize_mxfp4(gk.MatRef(t, rows, 32, rs, cs))
    code, byte = unpack(q)
    want_code, want_byte = quantize_ref(x)
    assert torch.equal(byte, want_byte)
    assert torch.equal(code, want_code)


@pytest.mark.parametrize("m", [8, 40, 300])
def test_products_over_the_range_of_scales(dev, m):
    """One block a row, so its products share one scale: sums of multiples of 1/4 below 2^11
    times a power of two, exact while they and their magnitudes' sum stay in f32's normal
    range; below it each of the 32 products and sums is off by at most a step of 2^-149."""
    n = 128
    ca, cb = random_mx(m, 32, 1), random_mx(n, 32, 2)
    ca[1][:, 0] = (torch.arange(m) * 254 // (m - 1)).to(torch.uint8)
    cb[1][:, 0] = (torch.arange(n) * 2).to(torch.uint8)
    c = torch.zeros(m, n, device=dev)
    a_c, a_s, *_ = mx(*ca, dev)
    b_c, b_s, *_ = mx(*cb, dev)
    gk.gemm_mxfp4(1.0, gk.MatMxfp4(a_c, a_s, m, 32), gk.MatMxfp4(b_c, b_s, n, 32), 0.0,
                  gk.MatMut.from_row_major(c, m, n))
    a, b = values_of(*ca), values_of(*cb)
    want, most = a @ b.t(), a.abs() @ b.abs().t()
    got = c.cpu().double()
    scale = ca[1].double() + cb[1].double().t() - 254  # the exponents of the least products
    normal = (scale - 2 >= -126) & (most < 2.0 ** 127)
    assert torch.equal(got[normal], want[normal])
    low = scale - 2 < -126
    assert ((got - want)[low].abs() <= 64 * 2.0 ** -149).all()


@pytest.mark.parametrize("dt", [BF16, F32])
@pytest.mark.parametrize("rows,k", [(1, 33), (7, 1000), (70, 520), (300, 96), (5, 4100)])
@pytest.mark.parametrize("how", ["row", "col", "odd", "one"])
def test_rows_of_codes_that_lie_apart(dev, dt, rows, k, how):
    """Quantization writes a row's blocks and its padded scales, nothing between the rows;
    "one": every row is the same memory."""
    nb = -(-k // 32)
    ld, lds = nb * 16 + 48, -(-nb // 16) * 16 + 32
    x = sample(rows, k, dt, 7)
    if how == "one":
        x = x[:1].expand(rows, k)
        t, rs, cs = x[0].contiguous().to(dev), 0, 1
    elif how == "col":
        t, rs, cs = x.t().contiguous().flatten().to(dev), 1, rows
    else:
        rs, cs = k + (how == "odd"), 1
        t = torch.zeros(rows, rs, dtype=dt)
        t[:, :k] = x
        t = t.flatten().to(dev)
    codes = torch.full((rows, ld), 0x5A, dtype=torch.uint8, device=dev)
    scales = torch.full((rows, lds), 0x5A, dtype=torch.uint8, device=dev)
    q = gk.MatMxfp4(codes, scales, rows, k, ld, lds)
    gk.quantize_mxfp4(gk.MatRef(t, rows, k, rs, cs), q)
    code, byte = unpack(q)
    want_code, want_byte = quantize_ref(x)
    assert torch.equal(code, want_code) and torch.equal(byte, want_byte)
    assert (codes[:, nb * 16:] == 0x5A).all() and (scales[:, -(-nb // 16) * 16:] == 0x5A).all()
    back = torch.zeros(rows, k, device=dev)
    gk.dequantize_mxfp4(q, gk.MatMut.from_row_major(back, rows, k))
    assert torch.equal(back.cpu().double(), values_of(want_code, want_byte)[:, :k])
