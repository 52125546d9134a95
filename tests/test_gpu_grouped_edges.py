"""Grouped products at the edges of what their documentation allows: rows of one element
with very many columns, group strides of any alignment, values below the normal range.
Tolerances as in test_gpu_grouped.py."""
import pytest
import torch

import gemmkit_amd as gk
from test_gpu_grouped import bounds_of, check, offs, rand

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


def offsets(sizes, dev):
    return torch.tensor(offs(*sizes), dtype=torch.int32, device=dev)


@pytest.mark.parametrize("k,n", [(1, 3_000_000), (1, 16_600_008), (1, 20_000_000), (1, 17_000_001),
                                 (2, 17_000_000), (3, 17_000_001)])
@pytest.mark.parametrize("groups", [1, 3])
def test_few_k_and_very_many_columns(dev, k, n, groups):
    """Sums of up to three exact products: two roundings at most in f32."""
    sizes = (2,) if groups == 1 else (2, 0, 1)
    rows = sum(sizes)
    g = torch.Generator(device="cuda").manual_seed(1)
    a = torch.randn(rows, k, generator=g, device=dev).to(BF16)
    b = torch.randn(groups, k, n, generator=g, device=dev).to(BF16)
    c = torch.full((rows, n), float("nan"), device=dev)
    gk.gemm_grouped(1.0, gk.MatRef.from_row_major(a, rows, k), offsets(sizes, dev),
                    gk.MatRef.from_row_major(b, k, n), k * n, 0.0,
                    gk.MatMut.from_row_major(c, rows, n))
    for z, (s, e) in enumerate(bounds_of(offs(*sizes), rows)):
        for r in range(s, e):
            terms = a[r].double()[:, None] * b[z].double()
            err = (c[r].double() - terms.sum(0)).abs()
            assert (err <= (k - 1) * 2.0 ** -23 * terms.abs().sum(0)).all(), r


def test_most_columns(dev):
    """One row, one k, the most columns that the entry takes in whole 16 bytes."""
    n = 2 ** 31 - 1024 - 8
    g = torch.Generator(device="cuda").manual_seed(2)
    a = torch.full((1, 1), -1.5, dtype=BF16, device=dev)
    b = torch.empty(n, dtype=BF16, device=dev).random_(-64, 64, generator=g)
    c = torch.full((n,), float("nan"), dtype=BF16, device=dev)
    gk.gemm_grouped(1.0, gk.MatRef.from_row_major(a, 1, 1), offsets((1,), dev),
                    gk.MatRef.from_row_major(b, 1, n), 0, 0.0, gk.MatMut.from_row_major(c, 1, n))
    for at in range(0, n, 1 << 28):
        assert torch.equal(c[at:at + (1 << 28)], b[at:at + (1 << 28)] * -1.5)


@pytest.mark.parametrize("layout", ["c", "r"])
@pytest.mark.parametrize("sizes,k,n", [((3, 0, 2), 64, 72), ((20, 33, 9), 200, 136), ((300, 0, 257), 520, 264),
                                       ((1, 2, 1), 1032, 4000)])
@pytest.mark.parametrize("more", [1, 4, 1000])
def test_group_strides_of_any_alignment(dev, sizes, k, n, layout, more):
    groups, rows = len(sizes), sum(sizes)
    a, b = rand(1, rows, k), rand(2, groups, k, n)
    step = k * n + more
    buf = torch.full((groups * step,), float("nan"), dtype=BF16)
    for g in range(groups):
        flat = b[g] if layout == "r" else b[g].t().contiguous()
        buf[g * step:g * step + k * n] = flat.flatten()
    c = torch.full((rows, n), float("nan"), device=dev)
    rs, cs = (n, 1) if layout == "r" else (1, k)
    gk.gemm_grouped(1.0, gk.MatRef.from_row_major(a.to(dev), rows, k), offsets(sizes, dev),
                    gk.MatRef(buf.to(dev), k, n, rs, cs), step, 0.0,
                    gk.MatMut.from_row_major(c, rows, n))
    for g, (s, e) in enumerate(bounds_of(offs(*sizes), rows)):
        if e > s:
            x, w = a[s:e].double(), b[g].double()
            check(c[s:e].cpu(), x @ w, x.abs() @ w.abs(), k, F32, 1.0, 0.0, torch.zeros(e - s, n).double())


def near(c, a, b, k):
    """f32 rows of an MXFP4 product of the values a and b against 64 bits."""
    a, b = a.double(), b.double()
    want = a @ b.t()
    tol = k * 2.0 ** -23 * (a.abs() @ b.abs().t()) + 2.0 ** -24 * want.abs()
    assert ((c.double() - want).abs() <= tol).all()


def mx_values(codes, scales, k):
    rows = codes.shape[0]
    v = torch.zeros(rows, k, device=codes.device)
    gk.dequantize_mxfp4(gk.MatMxfp4(codes, scales, rows, k), gk.MatMut.from_row_major(v, rows, k))
    return v


def test_mxfp4_rows_past_32_bits(dev):
    """Activations of more than 2^32 bytes: the last rows."""
    rows, k, n, last = 2_200_000, 4096, 72, 300
    g = torch.Generator(device="cuda").manual_seed(4)
    codes = torch.zeros(rows, k // 2, dtype=torch.uint8, device=dev)
    scales = torch.full((rows, k // 32), 120, dtype=torch.uint8, device=dev)
    codes[-last:] = torch.randint(0, 256, (last, k // 2), generator=g, device=dev, dtype=torch.uint8)
    wc = torch.randint(0, 256, (2 * n, k // 2), generator=g, device=dev, dtype=torch.uint8)
    ws = torch.randint(115, 130, (2 * n, k // 32), generator=g, device=dev, dtype=torch.uint8)
    c = torch.full((rows, n), float("nan"), device=dev)
    gk.gemm_grouped_mxfp4(1.0, gk.MatMxfp4(codes, scales, rows, k), offsets((rows - 100, 100), dev),
                          gk.MatMxfp4(wc, ws, 2 * n, k), 0.0, gk.MatMut.from_row_major(c, rows, n))
    av, wv = mx_values(codes[-last:], scales[-last:], k), mx_values(wc, ws, k)
    near(c[-last:-100], av[:-100], wv[:n], k)
    near(c[-100:], av[-100:], wv[n:], k)
    assert not c[:-last].any()


def test_mxfp4_weights_past_32_bits(dev):
    """Weights of more than 2^32 bytes: the last group's."""
    groups, k, n = 300, 4096, 8192
    g = torch.Generator(device="cuda").manual_seed(5)
    wc = torch.zeros(groups * n, k // 2, dtype=torch.uint8, device=dev)
    ws = torch.full((groups * n, k // 32), 120, dtype=torch.uint8, device=dev)
    wc[-n:] = torch.randint(0, 256, (n, k // 2), generator=g, device=dev, dtype=torch.uint8)
    for rows in (20, 700):  # all but one of the last group
        ac = torch.randint(0, 256, (rows, k // 2), generator=g, device=dev, dtype=torch.uint8)
        asc = torch.randint(115, 130, (rows, k // 32), generator=g, device=dev, dtype=torch.uint8)
        c = torch.full((rows, n), float("nan"), device=dev)
        gk.gemm_grouped_mxfp4(1.0, gk.MatMxfp4(ac, asc, rows, k),
                              offsets((1,) + (0,) * (groups - 2) + (rows - 1,), dev),
                              gk.MatMxfp4(wc, ws, groups * n, k), 0.0,
                              gk.MatMut.from_row_major(c, rows, n))
        near(c[1:], mx_values(ac, asc, k)[1:], mx_values(wc[-n:], ws[-n:], k), k)
        assert not c[:1].any()


@pytest.mark.parametrize("sizes", [(2, 1), (40, 30), (300, 200)])
def test_values_below_the_normal_range(dev, sizes):
    """Subnormal inputs count as what they are, and subnormal sums are kept."""
    k, n, rows, groups = 64, 72, sum(sizes), len(sizes)
    g = torch.Generator().manual_seed(3)

    def ints(*shape):
        return torch.randint(-3, 4, shape, generator=g).double()

    for ea, eb in ((-133, 20), (-133, 0), (-70, -70), (20, -133)):
        a, b = (ints(rows, k) * 2.0 ** ea).to(BF16), (ints(groups, k, n) * 2.0 ** eb).to(BF16)
        c = torch.full((rows, n), float("nan"), device=dev)
        gk.gemm_grouped(1.0, gk.MatRef.from_row_major(a.to(dev), rows, k), offsets(sizes, dev),
                        gk.MatRef.from_row_major(b.to(dev), k, n), k * n, 0.0,
                        gk.MatMut.from_row_major(c, rows, n))
        for z, (s, e) in enumerate(bounds_of(offs(*sizes), rows)):
            # whole numbers below 2^10 times a power of two of at least 2^-149: exact
            assert torch.equal(c[s:e].cpu().double(), a[s:e].double() @ b[z].double()), (ea, eb)


@pytest.mark.parametrize("sizes,k,n", [((3, 0, 2), 64, 72), ((40, 33, 9), 200, 136), ((300, 0, 257), 96, 264)])
@pytest.mark.parametrize("out", [BF16, F32])
@pytest.mark.parametrize("beta", [0.0, -0.5])
def test_output_of_any_strides(dev, sizes, k, n, out, beta):
    """C with neither stride 1: elements between stay as they are, for all three products."""
    rows, groups = sum(sizes), len(sizes)
    bounds = bounds_of(offs(*sizes), rows)
    a, b = rand(1, rows, k), rand(2, groups, k, n)
    for rs, cs in ((2 * n + 1, 2), (3, 3 * rows + 1)):
        buf0 = torch.randn((rows - 1) * rs + (n - 1) * cs + 1, generator=torch.Generator().manual_seed(3)).to(out)
        buf = buf0.to(dev)
        gk.gemm_grouped(1.0, gk.MatRef.from_row_major(a.to(dev), rows, k), offsets(sizes, dev),
                        gk.MatRef.from_row_major(b.to(dev), k, n), k * n, beta,
                        gk.MatMut(buf, rows, n, rs, cs))
        got, old = buf.cpu(), torch.as_strided(buf0, (rows, n), (rs, cs)).double()
        view = torch.as_strided(got, (rows, n), (rs, cs))
        for g, (s, e) in enumerate(bounds):
            if e > s:
                x, w = a[s:e].double(), b[g].double()
                check(view[s:e], x @ w + beta * old[s:e], x.abs() @ w.abs(), k, out, 1.0, beta, old[s:e])
        mask = torch.ones(buf0.numel(), dtype=torch.bool)
        torch.as_strided(mask, (rows, n), (rs, cs)).fill_(False)
        assert torch.equal(got[mask], buf0[mask])
    d = rand(4, rows, n)
    for rs, cs in ((2 * n + 1, 2), (3, 3 * k + 1)):
        step = (k - 1) * rs + (n - 1) * cs + 4
        buf0 = torch.randn(groups * step, generator=torch.Generator().manual_seed(5)).to(out)
        buf = buf0.to(dev)
        gk.gemm_grouped_wgrad(1.0, gk.MatRef.from_row_major(a.to(dev), rows, k), offsets(sizes, dev),
                              gk.MatRef.from_row_major(d.to(dev), rows, n), beta,
                              gk.MatMut(buf, k, n, rs, cs), step)
        got, mask = buf.cpu(), torch.ones(buf0.numel(), dtype=torch.bool)
        for g, (s, e) in enumerate(bounds):
            old = torch.as_strided(buf0, (k, n), (rs, cs), g * step).double()
            x, w = a[s:e].double().t(), d[s:e].double()
            check(torch.as_strided(got, (k, n), (rs, cs), g * step), x @ w + beta * old,
                  x.abs() @ w.abs(), e - s, out, 1.0, beta, old)
            torch.as_strided(mask, (k, n), (rs, cs), g * step).fill_(False)
        assert torch.equal(got[mask], buf0[mask])


@pytest.mark.parametrize("sizes", [(3, 0, 2), (40, 30), (300, 100)])
def test_operands_that_overlap_themselves(dev, sizes):
    """Broadcast and sliding rows, columns and group matrices."""
    rows, k, n, groups = sum(sizes), 72, 88, len(sizes)
    flat, w = rand(1, rows + k + 8), rand(2, groups, k + n + 8)
    for a_rs, a_cs in ((0, 1), (1, 1), (1, 0), (0, 0), (1, 2)):
        for b_rs, b_cs, b_gs in ((0, 1, 168), (1, 0, 168), (1, 1, 168), (1, 1, 3), (0, 0, 1)):
            if a_rs * (rows - 1) + a_cs * (k - 1) >= flat.numel():
                continue
            c = torch.full((rows, n), float("nan"), device=dev)
            gk.gemm_grouped(1.0, gk.MatRef(flat.to(dev), rows, k, a_rs, a_cs), offsets(sizes, dev),
                            gk.MatRef(w.to(dev), k, n, b_rs, b_cs), b_gs, 0.0,
                            gk.MatMut.from_row_major(c, rows, n))
            a = torch.as_strided(flat, (rows, k), (a_rs, a_cs)).double()
            for g, (s, e) in enumerate(bounds_of(offs(*sizes), rows)):
                if e > s:
                    b = torch.as_strided(w, (k, n), (b_rs, b_cs), g * b_gs).double()
                    check(c[s:e].cpu(), a[s:e] @ b, a[s:e].abs() @ b.abs(), k, F32, 1.0, 0.0,
                          torch.zeros(e - s, n).double())
        d = rand(3, rows + n + 8)
        c = torch.full((groups, k, n), float("nan"), device=dev)
        if a_rs * (rows - 1) + a_cs * (k - 1) < flat.numel():
            gk.gemm_grouped_wgrad(1.0, gk.MatRef(flat.to(dev), rows, k, a_rs, a_cs), offsets(sizes, dev),
                                  gk.MatRef(d.to(dev), rows, n, 1, 1), 0.0,
                                  gk.MatMut.from_row_major(c, k, n), k * n)
            dv = torch.as_strided(d, (rows, n), (1, 1)).double()
            for g, (s, e) in enumerate(bounds_of(offs(*sizes), rows)):
                x, y = a[s:e].t(), dv[s:e]
                check(c[g].cpu(), x @ y, x.abs() @ y.abs(), e - s, F32, 1.0, 0.0, torch.zeros(k, n).double())
