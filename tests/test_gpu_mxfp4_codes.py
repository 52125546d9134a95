"""MXFP4 matrices whose arrays hold more than their columns: codes past the last column in a
row's last block, and whole blocks beyond.  A product is the product of what the matrices
dequantize to.

Compared as in test_gpu_mxfp4.py: K exact products added in f32, each addition
off by at most 2^-23 of the sum of the magnitudes, then the output's half step."""
import pytest
import torch

import gemmkit_amd as gk
from test_gpu_mxfp4 import check, mx, random_mx, values_of

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
NO_C = torch.zeros(())


def spoiled(rows, k, seed, more=0):
    """(codes, scales) of `more` blocks beyond k's own, no code past k zero."""
    code, byte = random_mx(rows, (-(-k // 32) + more) * 32, seed)
    code[:, k:] |= 1
    return code, byte


def only(code, byte, k):
    """The values of the first k columns."""
    nb = -(-k // 32)
    return values_of(code[:, :nb * 32], byte[:, :nb])[:, :k]


# m, n, k: every tile with one stage, an odd and an even number of them (a stage is 256
# codes), the tail in each half of the last stage, and the transposed output, which swaps the
# operands.
@pytest.mark.parametrize("m,n,k", [
    (1, 40, 31), (7, 64, 250), (16, 200, 2049), (16, 600, 2201), (5, 20000, 33), (16, 12288, 2300),
    (3, 9000, 2100), (8, 25000, 520), (64, 300, 1), (100, 130, 333), (64, 4096, 777), (130, 2000, 510),
    (700, 3000, 129), (1500, 2000, 1000), (2600, 2600, 95), (4096, 4096, 300), (3000, 4100, 1025),
])
@pytest.mark.parametrize("c_lay", ["row", "col"])
def test_codes_past_the_last_column_do_not_count(dev, m, n, k, c_lay):
    ca, cb = spoiled(m, k, 1, more=1), spoiled(n, k, 2, more=1)
    ca[1][:, -1] = 255  # scales of the blocks beyond
    a_c, a_s, ald, alds = mx(*ca, dev)
    b_c, b_s, bld, blds = mx(*cb, dev)
    c = torch.full((m * n,), float("nan"), device=dev)
    rs, cs = (n, 1) if c_lay == "row" else (1, m)
    gk.gemm_mxfp4(1.0, gk.MatMxfp4(a_c, a_s, m, k, ald, alds),
                  gk.MatMxfp4(b_c, b_s, n, k, bld, blds), 0.0, gk.MatMut(c, m, n, rs, cs))
    check(torch.as_strided(c, (m, n), (rs, cs)), only(*ca, k).to(dev), only(*cb, k).to(dev), k, F32,
          1.0, 0.0, NO_C)


@pytest.mark.parametrize("sizes,n,k", [
    ((3, 0, 1), 40, 31), ((2,) * 70, 300, 2049), ((4,) * 12, 2560, 167), ((6,) * 100, 1100, 333),
    ((40,) * 60, 700, 401), ((130,) * 40, 1000, 290), ((1400, 300, 800), 2600, 161),
    ((0, 20, 5, 11, 3, 9, 7, 9), 3900, 161),
])
def test_codes_past_the_last_column_of_groups(dev, sizes, n, k):
    rows, groups = sum(sizes), len(sizes)
    ca, cb = spoiled(rows, k, 1), spoiled(groups * n, k, 2)
    a_c, a_s, *_ = mx(*ca, dev)
    b_c, b_s, *_ = mx(*cb, dev)
    off = torch.tensor([0] + list(torch.tensor(sizes).cumsum(0)), dtype=torch.int32, device=dev)
    c = torch.full((rows, n), float("nan"), dtype=BF16, device=dev)
    gk.gemm_grouped_mxfp4(1.0, gk.MatMxfp4(a_c, a_s, rows, k), off,
                          gk.MatMxfp4(b_c, b_s, groups * n, k), 0.0,
                          gk.MatMut.from_row_major(c, rows, n))
    va, vb = only(*ca, k).to(dev), only(*cb, k).to(dev)
    at = 0
    for g, s in enumerate(sizes):
        if s:
            check(c[at:at + s], va[at:at + s], vb[g * n:(g + 1) * n], k, BF16, 1.0, 0.0, NO_C)
        at += s


def test_the_first_columns_of_a_quantized_matrix(dev):
    """A narrower MatMxfp4 on the arrays of a wider one: the product of what it
    dequantizes to."""
    g = torch.Generator().manual_seed(5)
    x, w = torch.randn(50, 300, generator=g).to(dev), torch.randn(70, 300, generator=g).to(dev)
    xq = gk.quantize_mxfp4(gk.MatRef.from_row_major(x, 50, 300))
    wq = gk.quantize_mxfp4(gk.MatRef.from_row_major(w, 70, 300))
    for k in (300, 299, 289, 288, 257, 45, 1):
        a = gk.MatMxfp4(xq.codes, xq.scales, 50, k, xq.ld, xq.lds)
        b = gk.MatMxfp4(wq.codes, wq.scales, 70, k, wq.ld, wq.lds)
        ad, bd = torch.zeros(50, k, device=dev), torch.zeros(70, k, device=dev)
        gk.dequantize_mxfp4(a, gk.MatMut.from_row_major(ad, 50, k))
        gk.dequantize_mxfp4(b, gk.MatMut.from_row_major(bd, 70, k))
        c = torch.zeros(50, 70, device=dev)
        gk.gemm_mxfp4(1.0, a, b, 0.0, gk.MatMut.from_row_major(c, 50, 70))
        check(c, ad.double(), bd.double(), k, F32, 1.0, 0.0, NO_C)
