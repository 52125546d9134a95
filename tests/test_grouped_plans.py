"""Every kernel that products of ragged groups, their weight gradients and MXFP4 products
choose between: the plan of a product that reaches it (host-only), and that product against
64 bits.

Tolerance as in test_gpu_grouped.py: exact products (bf16; e2m1 with scales in range) added in
f32, each addition off by at most 2^-23 of the sum of the magnitudes, then half a step of the
output (2^-8 relative in bf16, 2^-24 in f32)."""
import pytest
import torch

import gemmkit_amd as gk

BF16, F32 = torch.bfloat16, torch.float32

# operator, rows, groups, k, n, operands of 16-byte alignment, plan
PRODUCTS = [
    ("grouped_c", 1451, 21, 104, 2952, True, "big 256x256"),
    ("grouped_c", 1798, 43, 103, 619, False, "reg 128x128 any"),
    ("grouped_c", 1107, 42, 103, 350, False, "reg 128x64 any"),
    ("grouped_c", 100, 48, 105, 301, False, "reg 32x64 any"),
    ("grouped_c", 5, 2, 100, 105, False, "regwave 16x32x4 any"),
    ("grouped_c", 5, 2, 404, 113, False, "regwave 16x32x8 any"),
    ("grouped_c", 3869, 76, 96, 264, True, "ring 128x128"),
    ("grouped_c", 351, 10, 1112, 6440, True, "ring 128x128 once"),
    ("grouped_c", 9498, 79, 96, 264, True, "ring 128x256"),
    ("grouped_c", 3, 2, 104, 96, True, "ring 16x64"),
    ("grouped_c", 9, 9, 272, 27544, True, "ring 16x64 once"),
    ("grouped_c", 862, 52, 96, 328, True, "ring 64x128"),
    ("grouped_c", 1051, 65, 664, 1576, True, "ring 64x128 once"),
    ("grouped_c", 1040, 4, 104, 104, True, "ring 64x64"),
    ("grouped_c", 1311, 68, 2344, 432, True, "ring 64x64 once"),
    ("grouped_c", 34, 2, 96, 96, True, "wave 16x32x4"),
    ("grouped_c", 15, 15, 2312, 1936, True, "wave 16x32x4 once"),
    ("grouped_c", 797, 27, 264, 104, True, "wave 32x64x4"),
    ("grouped_r", 1025, 15, 96, 4280, True, "big 256x256"),
    ("grouped_r", 675, 16, 112, 2022, False, "reg 128x128 any"),
    ("grouped_r", 4827, 4, 113, 134, False, "reg 128x64 any"),
    ("grouped_r", 39, 33, 109, 226, False, "reg 32x64 any"),
    ("grouped_r", 3, 2, 100, 108, False, "regwave 16x32x4 any"),
    ("grouped_r", 4, 2, 323, 115, False, "regwave 16x32x8 any"),
    ("grouped_r", 2297, 58, 112, 400, True, "ring 128x128"),
    ("grouped_r", 1273, 35, 2440, 816, True, "ring 128x128 once"),
    ("grouped_r", 885, 51, 136, 1264, True, "ring 128x256"),
    ("grouped_r", 31, 29, 104, 520, True, "ring 16x128"),
    ("grouped_r", 16, 16, 3616, 1168, True, "ring 16x128 once"),
    ("grouped_r", 4, 2, 96, 112, True, "ring 16x64"),
    ("grouped_r", 7, 7, 15392, 624, True, "ring 16x64 once"),
    ("grouped_r", 29, 6, 96, 4232, True, "ring 64x128"),
    ("grouped_r", 52, 49, 544, 2520, True, "ring 64x128 once"),
    ("grouped_r", 1015, 3, 96, 112, True, "ring 64x64"),
    ("grouped_r", 850, 53, 2952, 520, True, "ring 64x64 once"),
    ("grouped_r", 36, 2, 112, 104, True, "wave 16x32x4"),
    ("grouped_r", 4, 3, 23816, 944, True, "wave 16x32x4 once"),
    ("grouped_r", 827, 2, 264, 136, True, "wave 32x64x4"),
    ("mxfp4", 2290, 21, 104, 2941, True, "big 256x256"),
    ("mxfp4", 4096, 1, 4096, 4096, True, "big 256x256"),
    ("mxfp4", 6655, 53, 107, 135, True, "ring 128x128"),
    ("mxfp4", 1024, 1, 2048, 4096, True, "ring 128x128"),
    ("mxfp4", 852, 25, 9560, 1260, True, "ring 128x128 once"),
    ("mxfp4", 2607, 34, 101, 1025, True, "ring 128x256"),
    ("mxfp4", 41, 39, 112, 386, True, "ring 16x128"),
    ("mxfp4", 61, 58, 17885, 264, True, "ring 16x128 once"),
    ("mxfp4", 3, 1, 100, 110, True, "ring 16x64"),
    ("mxfp4", 21, 19, 2920, 4839, True, "ring 16x64 once"),
    ("mxfp4", 64, 32, 2048, 4096, True, "ring 16x64 once"),
    ("mxfp4", 33, 6, 104, 4115, True, "ring 64x128"),
    ("mxfp4", 238, 59, 3288, 1396, True, "ring 64x128 once"),
    ("mxfp4", 827, 4, 101, 132, True, "ring 64x64"),
    ("mxfp4", 201, 11, 19502, 1351, True, "ring 64x64 once"),
    ("mxfp4", 19, 1, 105, 101, True, "wave 16x32x4"),
    ("mxfp4", 4, 4, 37914, 1808, True, "wave 16x32x4 once"),
    ("mxfp4", 101, 65, 1898, 101, True, "wave 16x64x4"),
    ("mxfp4", 39, 36, 30717, 247, True, "wave 16x64x4 once"),
    ("mxfp4", 679, 1, 270, 164, True, "wave 32x64x4"),
    ("wgrad", 7064, 23, 2744, 136, True, "big 256x256"),
    ("wgrad", 11015, 2, 1160, 1304, True, "big 256x256 /4"),
    ("wgrad", 8395, 4, 129, 212, False, "reg 128x128 /16 any"),
    ("wgrad", 4, 32, 138, 333, False, "reg 128x128 any"),
    ("wgrad", 1078, 2, 103, 145, False, "reg 64x64 /4 any"),
    ("wgrad", 10, 2, 101, 101, False, "reg 64x64 any"),
    ("wgrad", 22, 40, 264, 144, True, "ring 128x128"),
    ("wgrad", 9665, 2, 200, 4296, True, "ring 128x128 /4"),
    ("wgrad", 5, 30, 136, 136, True, "ring 64x128"),
    ("wgrad", 11568, 2, 136, 2776, True, "ring 64x128 /4"),
    ("wgrad", 12, 2, 96, 96, True, "ring 64x64"),
    ("wgrad", 4919, 2, 104, 144, True, "ring 64x64 /16"),
    ("wgrad", 209, 2, 96, 96, True, "wave 32x64x4"),
    ("wgrad", 5926, 2, 112, 120, True, "wave 32x64x4 /16"),
]


@pytest.mark.parametrize("op,rows,groups,k,n,aligned,plan", PRODUCTS)
def test_plan(op, rows, groups, k, n, aligned, plan):
    for out in ("bf16", "f32"):
        assert gk.debug_plan_grouped(op, rows, groups, k, n, out, aligned) == plan


def test_every_plan_is_listed():
    """What products drawn over a wide range choose is in the list (row ranges of a weight
    gradient in any number)."""
    import random
    import re

    def kernel(plan):
        return re.sub(r"/\d+", "/", plan)

    listed = {(p[0], kernel(p[-1])) for p in PRODUCTS}
    rng = random.Random(1)

    def size(lo, hi):
        return round(lo * (hi / lo) ** rng.random())

    for _ in range(20000):
        op = rng.choice(("grouped_c", "grouped_r", "wgrad", "mxfp4"))
        rows, groups = size(1, 40000), rng.choice((1, size(1, 256)))
        k, n = size(1, 30000), size(1, 30000)
        if rng.random() < 0.5:
            k, n = -(-k // 8) * 8, -(-n // 8) * 8
        plan = gk.debug_plan_grouped(op, rows, groups, k, n, rng.choice(("bf16", "f32")))
        assert (op, kernel(plan)) in listed, (op, rows, groups, k, n, plan)


def test_plan_refusals():
    for rows, groups, k, n in ((0, 1, 1, 1), (1, 0, 1, 1), (1, 1, 0, 1), (1, 1, 1, 0), (2 ** 31, 1, 1, 1),
                             (1, 2 ** 30, 2 ** 30, 2 ** 30)):
        with pytest.raises(gk.GemmkitError):
            gk.debug_plan_grouped("mxfp4", rows, groups, k, n)


def uneven(rows, groups):
    """Bounds of groups that differ, an empty one among them where there are several."""
    w = [0 if g == 1 else 1 + g * 7 % 5 for g in range(groups)]
    sizes = [rows * v // sum(w) for v in w]
    sizes[0] += rows - sum(sizes)
    at, bounds = 0, []
    for s in sizes:
        bounds.append((at, at + s))
        at += s
    return bounds


def matrix(g, rows, cols, aligned):
    """(flat values, row stride) of a random matrix, rows of odd stride where not aligned."""
    ld = cols if aligned else cols + 1 + cols % 2
    return torch.randn(rows * ld, generator=g, device=g.device).to(BF16), ld


def rows_of(flat, ld, rows, cols, at=0):
    return torch.as_strided(flat, (rows, cols), (ld, 1), at)


def near(got, a, b, terms, out):
    a, b = a.double(), b.double()
    want = a @ b
    tol = terms * 2.0 ** -23 * (a.abs() @ b.abs())
    tol = tol + (2.0 ** -8 if out == BF16 else 2.0 ** -24) * (want.abs() + tol) * 1.0001
    assert ((got.double() - want).abs() <= tol).all()


def mx_values(q):
    v = torch.zeros(q.rows, q.cols, device=q.codes.device)
    gk.dequantize_mxfp4(q, gk.MatMut.from_row_major(v, q.rows, q.cols))
    return v


def mx_random(g, rows, k):
    blocks = -(-k // 32)
    codes = torch.randint(0, 256, (rows, 16 * blocks), generator=g, device=g.device, dtype=torch.uint8)
    scales = torch.randint(115, 135, (rows, -(-blocks // 16) * 16), generator=g, device=g.device,
                           dtype=torch.uint8)
    return gk.MatMxfp4(codes, scales, rows, k)


@pytest.mark.gpu
@pytest.mark.parametrize("op,rows,groups,k,n,aligned,plan", PRODUCTS)
@pytest.mark.parametrize("out", [BF16, F32])
def test_product(dev, op, rows, groups, k, n, aligned, plan, out):
    name = "bf16" if out == BF16 else "f32"
    assert gk.debug_plan_grouped(op, rows, groups, k, n, name, aligned) == plan
    g = torch.Generator(device=dev).manual_seed(1)
    bounds = uneven(rows, groups)
    off = torch.tensor([0] + [e for _, e in bounds], dtype=torch.int32, device=dev)
    if op == "wgrad":
        (a, lda), (b, ldb) = matrix(g, rows, k, aligned), matrix(g, rows, n, aligned)
        c = torch.full((groups, k, n), float("nan"), dtype=out, device=dev)
        gk.gemm_grouped_wgrad(1.0, gk.MatRef(a, rows, k, lda, 1), off, gk.MatRef(b, rows, n, ldb, 1),
                              0.0, gk.MatMut.from_row_major(c, k, n), k * n)
        a, b = rows_of(a, lda, rows, k), rows_of(b, ldb, rows, n)
        for z, (s, e) in enumerate(bounds):
            near(c[z], a[s:e].t().contiguous(), b[s:e], max(e - s, 1), out)
        return
    c = torch.full((rows, n), float("nan"), dtype=out, device=dev)
    view = gk.MatMut.from_row_major(c, rows, n)
    if op == "mxfp4":
        a, b = mx_random(g, rows, k), mx_random(g, groups * n, k)
        if groups == 1:
            gk.gemm_mxfp4(1.0, a, b, 0.0, view)
        else:
            gk.gemm_grouped_mxfp4(1.0, a, off, b, 0.0, view)
        av, bv = mx_values(a), mx_values(b)
        for z, (s, e) in enumerate(bounds):
            if e > s:
                near(c[s:e], av[s:e], bv[z * n:(z + 1) * n].t().contiguous(), k, out)
        return
    a, lda = matrix(g, rows, k, aligned)
    shape = (n, k) if op == "grouped_c" else (k, n)
    b, ldb = matrix(g, groups * shape[0], shape[1], aligned)
    gk.gemm_grouped(1.0, gk.MatRef(a, rows, k, lda, 1), off,
                    gk.MatRef(b, k, n, *((1, ldb) if op == "grouped_c" else (ldb, 1))),
                    shape[0] * ldb, 0.0, view)
    a = rows_of(a, lda, rows, k)
    for z, (s, e) in enumerate(bounds):
        if e > s:
            w = rows_of(b, ldb, *shape, z * shape[0] * ldb)
            near(c[s:e], a[s:e], w.t().contiguous() if op == "grouped_c" else w, k, out)
