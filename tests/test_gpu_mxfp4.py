"""MXFP4 quantization and products against their definition in 64 bits.

Quantized codes and scales are compared exactly.  Products: e2m1 products and their scales
are exact in f32 while the scales' product stays in range, and K of them are added in f32,
each addition off by at most 2^-23 of the sum of the magnitudes; then the output's half
step (2^-8 relative in bf16, 2^-24 in f32) and two roundings for alpha and beta."""
import pytest
import torch

import gemmkit_amd as gk

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
HALF_STEP = {BF16: 2.0 ** -8, F32: 2.0 ** -24}
E2M1 = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)


def quantize_ref(x):
    """(codes, scale bytes) of a CPU matrix, element by element in f64."""
    rows, k = x.shape
    nb = -(-k // 32)
    pad = torch.zeros(rows, nb * 32, dtype=torch.float64)
    pad[:, :k] = x.double()
    v = pad.view(rows, nb, 32)
    top = v.abs().amax(2)
    bad = ~torch.isfinite(v).all(2)
    e = torch.frexp(torch.where(bad | (top == 0), torch.ones_like(top), top))[1] - 3
    e = e.clamp(min=-127)
    byte = torch.where(bad, torch.full_like(e, 255), torch.where(top == 0, torch.zeros_like(e), e + 127))
    m = v.abs() * torch.pow(2.0, -(byte.double() - 127)).unsqueeze(2)
    # the code whose value is nearest; between two, the even one
    d = (m.unsqueeze(3).clamp(max=6.0) - E2M1).abs()
    near = d.amin(3, keepdim=True)
    cand = d == near
    even = torch.tensor([1, 0, 1, 0, 1, 0, 1, 0])
    score = cand.int() * (2 + even)
    code = score.argmax(3) | torch.signbit(v).long() << 3
    code = torch.where(bad.unsqueeze(2), torch.zeros_like(code), code)
    return code.view(rows, nb * 32).to(torch.uint8), byte.to(torch.uint8)


def values_of(code, byte):
    rows, n32 = code.shape
    s = torch.pow(2.0, byte.double() - 127)
    s[byte == 255] = float("nan")
    v = E2M1[(code & 7).long()] * torch.where(code >= 8, -1.0, 1.0)
    return (v.view(rows, -1, 32) * s.unsqueeze(2)).view(rows, n32)


def packed(code):
    c = code.view(code.shape[0], -1, 2)
    return c[:, :, 0] | c[:, :, 1] << 4


def unpack(q):
    """(codes, scale bytes) of a MatMxfp4."""
    nb = -(-q.cols // 32)
    c = torch.as_strided(q.codes.cpu().flatten(), (q.rows, nb * 16), (q.ld, 1))
    s = torch.as_strided(q.scales.cpu().flatten(), (q.rows, nb), (q.lds, 1))
    return torch.stack((c & 15, c >> 4), 2).view(q.rows, nb * 32), s


def sample(rows, k, dt, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, k, generator=g)
    x *= torch.pow(2.0, torch.randint(-20, 20, (rows, -(-k // 32)), generator=g).float()
                   ).repeat_interleave(32, 1)[:, :k]
    if rows * k > 64:  # values on the midpoints, signed zeros, a block of zeros
        mids = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0, -0.25, -5.0, 6.0, -0.0, 4.0])
        n = min(13, k)
        x[0, :n] = mids[:n]
        if k >= 64:
            x[-1, 32:64] = 0.0
    return x.to(dt)


def as_view(x, how, dev, fill=float("nan")):
    rows, k = x.shape
    if how == "col":
        return x.t().contiguous().flatten().to(dev), 1, rows
    ld, off = (k + 3, 0) if how == "odd" else ((k + 40) // 8 * 8, 0) if how == "pad" else (k, 0)
    if how == "mis":
        ld, off = k, 1
    buf = torch.full((off + rows * ld + 1,), fill, dtype=x.dtype)
    buf[off:off + rows * ld].view(rows, ld)[:, :k] = x
    return buf.to(dev)[off:], ld, 1


@pytest.mark.parametrize("dt", [BF16, F32])
@pytest.mark.parametrize("rows,k", [(1, 1), (1, 32), (3, 31), (5, 33), (7, 512), (130, 1000),
                                    (2, 4096), (65, 520), (64, 96)])
@pytest.mark.parametrize("how", ["row", "pad", "odd", "mis", "col"])
def test_quantize_and_back(dev, dt, rows, k, how):
    x = sample(rows, k, dt, 3)
    t, rs, cs = as_view(x, how, dev)
    q = gk.MatMxfp4.empty(rows, k, dev)
    q.codes.fill_(0x5A)
    q.scales.fill_(0x5A)
    assert gk.quantize_mxfp4(gk.MatRef(t, rows, k, rs, cs), q) is q
    code, byte = unpack(q)
    want_code, want_byte = quantize_ref(x)
    assert torch.equal(byte, want_byte)
    assert torch.equal(code, want_code)
    for out in (BF16, F32):
        c, crs, ccs = as_view(torch.full((rows, k), float("nan"), dtype=out), how, dev, fill=7.0)
        before = c.clone()
        gk.dequantize_mxfp4(q, gk.MatMut(c, rows, k, crs, ccs))
        got = torch.as_strided(c.cpu(), (rows, k), (crs, ccs))
        assert torch.equal(got.double(), values_of(want_code, want_byte)[:, :k])
        mask = torch.ones(c.numel(), dtype=torch.bool)
        torch.as_strided(mask, (rows, k), (crs, ccs)).fill_(False)
        assert torch.equal(c.cpu()[mask], before.cpu()[mask])


@pytest.mark.parametrize("how", ["row", "col", "odd"])
@pytest.mark.parametrize("dt", [BF16, F32])
def test_quantize_extremes(dev, dt, how):
    tiny = torch.finfo(dt).smallest_normal
    sub = 2.0 ** -133 if dt == BF16 else 2.0 ** -149
    x = torch.zeros(10, 64, dtype=torch.float64)
    x[0, 3] = float("inf")
    x[1, 40] = float("nan")
    x[2, 0], x[2, 1] = torch.finfo(dt).max, -torch.finfo(dt).max
    x[3, 0], x[3, 33] = tiny, -tiny
    x[4, 0], x[4, 33] = sub, -3 * sub
    x[5, :32] = torch.linspace(-8, 8, 32)
    x[6, :] = -0.0
    x[7, 31], x[7, 32] = 2.0 ** -120, 2.0 ** 120
    x[8, 2] = float("-inf")
    x[8, 3] = float("nan")
    x[9, :32] = 2.0 ** -126 * torch.arange(32)
    x = x.to(dt)
    t, rs, cs = as_view(x, how, dev)
    q = gk.quantize_mxfp4(gk.MatRef(t, 10, 64, rs, cs))
    code, byte = unpack(q)
    want_code, want_byte = quantize_ref(x)
    assert torch.equal(byte, want_byte)
    assert torch.equal(code, want_code)
    for out in (BF16, F32):
        c = torch.zeros(640, dtype=out, device=dev)
        gk.dequantize_mxfp4(q, gk.MatMut.from_row_major(c, 10, 64))
        want = values_of(want_code, want_byte).to(out)
        got = c.cpu().view(10, 64)
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        assert torch.equal(got.nan_to_num(0.0), want.nan_to_num(0.0))


def mx(code, byte, dev, pad_codes=0, pad_scales=0, garbage=255):
    """A MatMxfp4 of CPU codes and scales; the scales' padding holds `garbage`."""
    rows, nb = byte.shape
    ld, lds = nb * 16 + pad_codes, -(-nb // 16) * 16 + pad_scales
    c = torch.full((rows, ld), 0x77, dtype=torch.uint8)
    c[:, :nb * 16] = packed(code)
    s = torch.full((rows, lds), garbage, dtype=torch.uint8)
    s[:, :nb] = byte
    return c.to(dev), s.to(dev), ld, lds


def random_mx(rows, k, seed):
    g = torch.Generator().manual_seed(seed)
    nb = -(-k // 32)
    code = torch.randint(0, 16, (rows, nb * 32), generator=g, dtype=torch.uint8)
    code[:, k:] = 0
    byte = torch.randint(115, 135, (rows, nb), generator=g, dtype=torch.uint8)
    return code, byte


def check(got, a, b, k, dt, alpha, beta, c0):
    want = alpha * (a @ b.t()) + (beta * c0.double() if beta else 0.0)
    tol = (k + 3) * 2.0 ** -23 * abs(alpha) * (a.abs() @ b.abs().t())
    tol = tol + 2.0 ** -23 * abs(beta) * c0.double().abs().nan_to_num(0.0)
    tol = tol + HALF_STEP[dt] * (want.abs() + tol) * 1.0001 + 1e-38
    err = (got.double() - want).abs()
    bad = ~(err <= tol)
    assert not bad.any(), (int(bad.sum()), float((err / tol).nan_to_num(1e9).max()))


@pytest.mark.parametrize("m", [1, 5, 16, 17, 64, 100, 300])
@pytest.mark.parametrize("n,k", [(1, 32), (40, 31), (64, 256), (136, 260), (130, 1000), (300, 544),
                                 (520, 2080)])
@pytest.mark.parametrize("out,c_lay,alpha,beta", [(BF16, "row", 1.0, 0.0), (F32, "col", 0.5, 1.0),
                                                  (F32, "odd", 1.0, 0.0), (BF16, "odd", -1.0, 0.5)])
def test_product(dev, m, n, k, out, c_lay, alpha, beta):
    ca, cb = random_mx(m, k, 1), random_mx(n, k, 2)
    g = torch.Generator().manual_seed(3)
    c0 = torch.randn(m, n, generator=g).to(out) if beta else torch.full((m, n), float("nan"), dtype=out)
    c, rs, cs = as_view(c0, c_lay, dev, fill=7.0)
    before = c.clone()
    a_c, a_s, ald, alds = mx(*ca, dev)
    b_c, b_s, bld, blds = mx(*cb, dev, pad_codes=32, pad_scales=16)
    gk.gemm_mxfp4(alpha, gk.MatMxfp4(a_c, a_s, m, k, ald, alds),
                  gk.MatMxfp4(b_c, b_s, n, k, bld, blds), beta, gk.MatMut(c, m, n, rs, cs))
    got = torch.as_strided(c.cpu(), (m, n), (rs, cs))
    check(got, values_of(*ca), values_of(*cb), k, out, alpha, beta, c0)
    mask = torch.ones(c.numel(), dtype=torch.bool)
    torch.as_strided(mask, (m, n), (rs, cs)).fill_(False)
    assert torch.equal(c.cpu()[mask], before.cpu()[mask])


def test_nan_scale_spoils_its_row_only(dev):
    m, n, k = 40, 50, 96
    ca, cb = random_mx(m, k, 1), random_mx(n, k, 2)
    ca[1][7, 1] = 255
    cb[1][9, 2] = 255
    c = torch.zeros(m, n, device=dev)
    a_c, a_s, *_ = mx(*ca, dev)
    b_c, b_s, *_ = mx(*cb, dev)
    gk.gemm_mxfp4(1.0, gk.MatMxfp4(a_c, a_s, m, k), gk.MatMxfp4(b_c, b_s, n, k), 0.0,
                  gk.MatMut.from_row_major(c, m, n))
    nan = torch.isnan(c.cpu())
    assert nan[7].all() and nan[:, 9].all()
    nan[7] = False
    nan[:, 9] = False
    assert not nan.any()


@pytest.mark.parametrize("sizes", [(1,), (0, 1, 3, 0, 17, 2), (65, 0, 40, 128, 1), (300, 257, 0, 600),
                                   tuple(i * 7 % 5 for i in range(70))])
@pytest.mark.parametrize("n,k", [(40, 31), (136, 260), (72, 1000)])
@pytest.mark.parametrize("out,c_lay,alpha,beta", [(BF16, "row", 1.0, 0.0), (F32, "col", 0.5, 1.0)])
def test_grouped_product(dev, sizes, n, k, out, c_lay, alpha, beta):
    start, groups = 2, len(sizes)
    offsets = [start]
    for s in sizes:
        offsets.append(offsets[-1] + s)
    rows = offsets[-1] + 3
    ca, cb = random_mx(rows, k, 1), random_mx(groups * n, k, 2)
    for r in (0, 1, rows - 1, rows - 2, rows - 3):
        ca[1][r] = 255  # rows of no group
    g = torch.Generator().manual_seed(3)
    c0 = torch.randn(rows, n, generator=g).to(out)
    c, rs, cs = as_view(c0, c_lay, dev, fill=7.0)
    before = c.clone()
    a_c, a_s, *_ = mx(*ca, dev)
    b_c, b_s, *_ = mx(*cb, dev)
    gk.gemm_grouped_mxfp4(alpha, gk.MatMxfp4(a_c, a_s, rows, k),
                          torch.tensor(offsets, dtype=torch.int32, device=dev),
                          gk.MatMxfp4(b_c, b_s, groups * n, k), beta,
                          gk.MatMut(c, rows, n, rs, cs))
    got = torch.as_strided(c.cpu(), (rows, n), (rs, cs))
    va, vb = values_of(*ca), values_of(*cb)
    mask = torch.ones(c.numel(), dtype=torch.bool)
    for i in range(groups):
        lo, hi = offsets[i], offsets[i + 1]
        if hi > lo:
            check(got[lo:hi], va[lo:hi], vb[i * n:(i + 1) * n], k, out, alpha, beta, c0[lo:hi])
            torch.as_strided(mask, (hi - lo, n), (rs, cs), lo * rs).fill_(False)
    assert torch.equal(c.cpu()[mask], before.cpu()[mask])


@pytest.mark.parametrize("sizes,n,k", [((1400, 300, 800), 2600, 160), ((130,) * 40, 1000, 288),
                                       ((40,) * 60, 700, 400), ((6,) * 100, 1100, 520),
                                       ((2,) * 70, 1500, 2080), ((3, 0, 1), 24, 8200),
                                       ((200,), 136, 4100), ((3000, 0, 2900, 100), 4000, 288)])
def test_grouped_tiles(dev, sizes, n, k):
    test_grouped_product(dev, sizes, n, k, F32, "row", 1.0, 0.0)


@pytest.mark.parametrize("m,n,k", [(4096, 4096, 288), (3000, 5000, 96), (300, 20000, 160),
                                   (30, 9000, 1100), (8, 14336, 800)])
def test_plain_tiles(dev, m, n, k):
    test_product(dev, m, n, k, BF16, "row", 1.0, 0.0)


def test_degenerate_products(dev):
    def product(m, n, k, alpha, beta):
        ca, cb = random_mx(max(m, 1), max(k, 1), 1), random_mx(max(n, 1), max(k, 1), 2)
        a_c, a_s, *_ = mx(*ca, dev)
        b_c, b_s, *_ = mx(*cb, dev)
        c = torch.full((max(m * n, 1),), 3.0, device=dev)
        gk.gemm_mxfp4(alpha, gk.MatMxfp4(a_c, a_s, m, k), gk.MatMxfp4(b_c, b_s, n, k), beta,
                      gk.MatMut.from_row_major(c, m, n))
        return c.cpu()

    assert (product(4, 6, 0, 1.0, 0.0) == 0).all()
    assert (product(4, 6, 0, 1.0, 0.5) == 1.5).all()
    assert (product(4, 6, 64, 0.0, 2.0) == 6.0).all()
    assert (product(0, 6, 64, 1.0, 0.0) == 3.0).all()
    assert (product(4, 0, 64, 1.0, 0.0) == 3.0).all()


@pytest.mark.parametrize("m,n,k", [(8, 9000, 2080), (16, 12288, 2300), (1, 14336, 2048), (5, 25000, 520),
                                   (16, 32768, 96), (9, 20000, 31)])
def test_short_products_of_many_columns(dev, m, n, k):
    """Up to 16 rows on one or two 64-column tiles per compute unit."""
    test_product(dev, m, n, k, F32, "row", 1.0, 0.0)


@pytest.mark.parametrize("sizes,n,k", [((2, 0, 5, 1), 3000, 2080), ((1, 2, 3), 6000, 2100),
                                       ((4,) * 12, 2560, 160), ((1,) * 9, 3333, 31)])
def test_short_groups_of_many_columns(dev, sizes, n, k):
    test_grouped_product(dev, sizes, n, k, BF16, "row", 1.0, 0.0)


def test_groups_of_several_rows_over_many_columns(dev):
    test_grouped_product(dev, (0, 20, 5, 11, 3, 9, 7, 9), 3900, 160, F32, "row", 1.0, 0.0)
