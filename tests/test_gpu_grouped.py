"""Products of ragged groups (gemm_grouped) and their weight gradient
(gemm_grouped_wgrad) against the same sums in 64 bits.

Tolerance.  bf16 products are exact in f32 and the K of them are added in f32, each
addition off by at most 2^-23 of the partial sum (rounded or cut), which is at most the
sum of the magnitudes: |error| <= K * 2^-23 * (|A| |B|) before the output's own rounding, half a
step (2^-8 relative in bf16, 2^-24 in f32), with two more roundings for alpha and beta."""
import itertools

import pytest
import torch

import gemmkit_amd as gk

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
HALF_STEP = {BF16: 2.0 ** -8, F32: 2.0 ** -24}


def rand(seed, *shape, dt=BF16):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(*shape, generator=g).to(dt)


def bounds_of(offsets, rows):
    """The documented groups of any offsets."""
    top, s = 0, []
    for o in offsets:
        top = max(top, o)
        s.append(min(rows, top))
    return list(zip(s[:-1], s[1:]))


def check(got, want, mags, k, dt, alpha, beta, c0):
    """want: alpha * sums + beta * c0 in f64; mags: |alpha| (|A| |B|)."""
    tol = (k + 3) * 2.0 ** -23 * mags + (2.0 ** -23) * abs(beta) * c0.abs()
    tol = tol + HALF_STEP[dt] * (want.abs() + tol) * 1.0001 + 1e-38
    err = (got.double() - want).abs()
    bad = ~(err <= tol)
    assert not bad.any(), (int(bad.sum()), float((err / tol).nan_to_num(1e9).max()))


def same_bits(x, y):
    as_int = torch.int16 if x.dtype == BF16 else torch.int32
    return torch.equal(x.view(as_int), y.view(as_int))


def lay(x, how, fill=float("nan")):
    """The matrix x (rows x cols, CPU) in a larger buffer filled with `fill`: (flat
    buffer without its first `off` elements, rs, cs).  how: r row-major, r+ padded rows,
    ro rows of odd stride, c column-major, c+ padded columns, m row-major misaligned."""
    rows, cols = x.shape
    if how[0] == "c":
        buf, rs, cs = lay(x.t(), "r" + how[1:], fill)
        return buf, cs, rs
    ld = cols + {"r": 0, "r+": 24, "ro": 3, "m": 0, "rm": 0}[how]
    off = 3 if how in ("m", "rm") else 0
    buf = torch.full((off + max(rows, 1) * max(ld, 1),), fill, dtype=x.dtype)
    if x.numel():
        buf[off:off + rows * ld].view(rows, ld)[:, :cols] = x
    return (buf, off), ld, 1


def on(dev, laid):
    (buf, off), rs, cs = laid
    return buf.to(dev)[off:], rs, cs


def run_grouped(dev, offsets, rows, k, n, a_lay="r", b_lay="c", out=BF16, alpha=1.0, beta=0.0,
                c_lay="r", shared=False, seed=1, ws=None, values=None):
    groups = len(offsets) - 1
    a = rand(seed, rows, k)
    b = rand(seed + 1, 1 if shared else max(groups, 1), k, n)
    if values:
        values(a, b)
    c0 = rand(seed + 2, rows, n, dt=out)
    bounds = bounds_of(offsets, rows)
    covered = torch.zeros(rows, dtype=torch.bool)
    for s, e in bounds:
        covered[s:e] = True
    a_in = a.clone()
    a_in[~covered] = float("nan")  # rows of no group are not read into any sum
    if beta == 0.0:
        c_in = torch.full_like(c0, float("nan"))  # beta 0 never reads C
        c_in[~covered] = c0[~covered]
    else:
        c_in = c0.clone()
    at, ars, acs = on(dev, lay(a_in, a_lay))
    # the groups' matrices one after the other, each laid out alike
    parts = [lay(b[g], b_lay) for g in range(b.shape[0])]
    (p0, off), brs, bcs = parts[0]
    step = p0.numel() - off
    step += -step % 8  # group strides of whole 16 bytes
    bbuf = torch.full((off + step * len(parts),), float("nan"), dtype=BF16)
    for g, ((p, _), _, _) in enumerate(parts):
        bbuf[off + g * step:off + g * step + p.numel() - off] = p[off:]
    bt = bbuf.to(dev)[off:]
    ct, crs, ccs = on(dev, lay(c_in, c_lay, fill=7.0))
    cbuf0 = ct.clone()
    ot = torch.tensor(offsets, dtype=torch.int32, device=dev)
    gk.gemm_grouped(alpha, gk.MatRef(at, rows, k, ars, acs), ot, gk.MatRef(bt, k, n, brs, bcs),
                    0 if shared else step, beta, gk.MatMut(ct, rows, n, crs, ccs), ws=ws)
    torch.cuda.synchronize()
    got = torch.as_strided(ct.cpu(), (rows, n), (crs, ccs)) if rows and n else c0
    for g, (s, e) in enumerate(bounds):
        if e <= s or n == 0:
            continue
        bg = b[0 if shared else g].double()
        want = alpha * (a[s:e].double() @ bg) if alpha else torch.zeros(e - s, n).double()
        base = c0[s:e].double() if beta else torch.zeros(e - s, n).double()
        mags = abs(alpha) * (a[s:e].double().abs() @ bg.abs()) if alpha else torch.zeros(e - s, n).double()
        check(got[s:e], want + beta * base, mags, k, out, alpha, beta, base)
    # nothing else of C's buffer changed
    mask = torch.ones_like(cbuf0, dtype=torch.bool)
    if rows and n:
        rows_t = covered.nonzero().flatten().to(dev)
        idx = rows_t[:, None] * crs + torch.arange(n, device=dev)[None] * ccs
        mask[idx.flatten()] = False
    assert same_bits(ct[mask], cbuf0[mask])
    return got


def offs(*sizes, start=0):
    out = [start]
    for s in sizes:
        out.append(out[-1] + s)
    return out


SIZES = {
    "one_row": (1,),
    "few": (0, 1, 3, 0, 17, 2),
    "middle": (65, 0, 40, 128, 1),
    "large": (300, 257, 0, 600),
    "all_empty": (0, 0, 0),
    "many": tuple(i * 7 % 5 for i in range(70)),
    "many_large": tuple(130 if i % 3 else 0 for i in range(130)),
}


@pytest.mark.parametrize("layout", ["c", "r"])
@pytest.mark.parametrize("sizes", list(SIZES))
@pytest.mark.parametrize("out", [BF16, F32])
def test_sizes_and_layouts(dev, sizes, layout, out):
    o = offs(*SIZES[sizes])
    run_grouped(dev, o, o[-1] + 5, 200, 136, b_lay=layout, out=out)


@pytest.mark.parametrize("k", [1, 7, 8, 63, 64, 65, 128, 136, 1000])
@pytest.mark.parametrize("n", [1, 8, 63, 72, 264])
def test_every_k_and_n(dev, k, n):
    for layout, sizes in itertools.product(("c", "r"), ((2, 0, 5), (70, 30), (200, 0, 300))):
        run_grouped(dev, offs(*sizes), sum(sizes), k, n, b_lay=layout, out=F32)


@pytest.mark.parametrize("a_lay", ["r+", "ro", "c", "c+", "m"])
@pytest.mark.parametrize("b_lay", ["c+", "r+", "ro", "co", "rm", "c"])
def test_operand_layouts(dev, a_lay, b_lay):
    run_grouped(dev, offs(20, 0, 33, 9), 64, 96, 88, a_lay=a_lay, b_lay=b_lay)


@pytest.mark.parametrize("c_lay", ["r+", "ro", "c", "c+", "m"])
@pytest.mark.parametrize("beta", [0.0, 1.0, -0.5])
@pytest.mark.parametrize("out", [BF16, F32])
def test_output_layouts_alpha_beta(dev, c_lay, beta, out):
    for sizes in ((3, 0, 9), (150, 0, 290)):
        run_grouped(dev, offs(*sizes), sum(sizes) + 2, 72, 100, c_lay=c_lay, beta=beta,
                    alpha=-1.5, out=out)


@pytest.mark.parametrize("offsets", [[3, 10, 20, 20], [0, 30, 10, 25], [-5, 4, 2, 60],
                                     [50, 0, 0, 0], [0, 2 ** 31 - 1, -2 ** 31, 7], [40, 40, 40, 90],
                                     [0, 5]])
def test_any_offsets_give_disjoint_groups(dev, offsets):
    run_grouped(dev, offsets, 40, 64, 48)
    run_grouped(dev, offsets + [31] * 100, 40, 64, 48)


def test_degenerate_calls(dev):
    run_grouped(dev, [0], 4, 16, 16)                       # no groups
    run_grouped(dev, [0, 0], 0, 16, 16)                    # no rows
    run_grouped(dev, offs(3, 4), 7, 16, 0)                 # no columns
    run_grouped(dev, offs(3, 4), 8, 0, 16)                 # empty sums: zeros
    run_grouped(dev, offs(3, 4), 8, 0, 16, beta=0.5)
    # alpha 0 reads neither operand
    def nans(a, b):
        a.fill_(float("nan"))
        b.fill_(float("nan"))
    run_grouped(dev, offs(3, 4), 8, 64, 16, alpha=0.0, beta=2.0, values=nans)
    run_grouped(dev, offs(3, 300), 310, 64, 16, alpha=0.0, values=nans)


def test_shared_matrix(dev):
    run_grouped(dev, offs(20, 300, 1), 330, 80, 96, shared=True)


def test_infinities_stay_in_their_rows(dev):
    """A row with an infinity or a NaN spoils its own outputs only, also across the end
    of a group inside a tile."""
    rows, k, n = 60, 72, 80
    a, b = rand(1, rows, k), rand(2, 3, k, n).abs()
    a[19, 5] = float("inf")
    a[20, 6] = float("nan")
    o = [0, 20, 40, 60]
    c = torch.zeros(rows, n, device=dev)
    gk.gemm_grouped(1.0, gk.MatRef.from_row_major(a.to(dev), rows, k),
                    torch.tensor(o, dtype=torch.int32, device=dev),
                    gk.MatRef.from_row_major(b.to(dev), k, n), k * n, 0.0,
                    gk.MatMut.from_row_major(c, rows, n))
    c = c.cpu()
    assert torch.isinf(c[19]).all() and torch.isnan(c[20]).all()
    rest = torch.ones(rows, dtype=torch.bool)
    rest[19:21] = False
    assert torch.isfinite(c[rest]).all()


@pytest.mark.parametrize("sizes", [(1, 0, 3), (64, 65, 0, 1), (300, 0, 128, 700), (0, 0)])
@pytest.mark.parametrize("k,n", [(1, 1), (8, 16), (72, 136), (264, 300), (40, 520)])
@pytest.mark.parametrize("out,c_lay,alpha,beta", [(BF16, "r", 1.0, 0.0), (F32, "r", 0.5, 1.0),
                                                  (F32, "c", 1.0, 0.0), (BF16, "c+", -1.0, 0.5),
                                                  (F32, "ro", 1.0, 0.0)])
def test_wgrad(dev, sizes, k, n, out, c_lay, alpha, beta):
    run_wgrad(dev, offs(*sizes), sum(sizes) + 3, k, n, out, c_lay, alpha, beta)


@pytest.mark.parametrize("sizes,k,n", [((9000,), 40, 72), ((0, 4500), 130, 264), ((70, 6100, 0), 24, 520),
                                       ((4097, 4000), 264, 40)])
@pytest.mark.parametrize("out,c_lay,alpha,beta", [(F32, "r", 1.0, 0.0), (BF16, "c+", -0.5, 1.0)])
def test_wgrad_of_long_groups(dev, sizes, k, n, out, c_lay, alpha, beta):
    """Row ranges per group, their partial sums added afterwards."""
    run_wgrad(dev, offs(*sizes), sum(sizes) + 3, k, n, out, c_lay, alpha, beta)


@pytest.mark.parametrize("layout", ["c", "r"])
@pytest.mark.parametrize("k", [520, 1096, 4104])
@pytest.mark.parametrize("sizes", [(1,), (3, 0, 1), (16, 5), (70, 30), (200,), (7, 0, 90, 64)])
def test_long_k_on_few_tiles(dev, sizes, k, layout):
    for n in (24, 200):
        run_grouped(dev, offs(*sizes), sum(sizes) + 1, k, n, b_lay=layout, out=F32)


@pytest.mark.parametrize("layout", ["c", "r"])
@pytest.mark.parametrize("sizes,k,n", [((1400, 300, 800), 136, 2600), ((130,) * 40, 72, 1000),
                                       ((40,) * 60, 200, 700), ((6,) * 100, 264, 1100),
                                       ((2,) * 70, 1032, 1500), ((4096,), 72, 4096),
                                       ((3000, 0, 2900, 100), 136, 4000)])
def test_many_tiles(dev, sizes, k, n, layout):
    run_grouped(dev, offs(*sizes), sum(sizes) + 1, k, n, b_lay=layout)


@pytest.mark.parametrize("lays", ["ro co", "ro ro", "m rm", "r+ ro", "ro c+", "m c"])
@pytest.mark.parametrize("sizes", [(1, 0, 3), (16, 40, 0, 64), (200, 90), (7,) * 60, (130,) * 40])
@pytest.mark.parametrize("k,n", [(9, 15), (8, 8), (201, 137), (1031, 65), (66, 1101), (7, 40), (40, 7)])
def test_rows_of_any_alignment(dev, lays, sizes, k, n):
    a_lay, b_lay = lays.split()
    run_grouped(dev, offs(*sizes), sum(sizes) + 2, k, n, a_lay=a_lay, b_lay=b_lay, out=F32)


@pytest.mark.parametrize("lays", ["ro ro", "m r", "r ro"])
@pytest.mark.parametrize("sizes", [(1, 0, 3), (64, 65, 0, 1), (300, 0, 128, 700)])
@pytest.mark.parametrize("k,n", [(9, 15), (73, 137), (265, 301), (8, 9), (7, 9), (41, 521)])
def test_wgrad_rows_of_any_alignment(dev, lays, sizes, k, n):
    a_lay, b_lay = lays.split()
    run_wgrad(dev, offs(*sizes), sum(sizes) + 3, k, n, BF16, "ro", 1.0, 0.0, a_lay, b_lay)


@pytest.mark.parametrize("lays", ["r+ r", "r r+", "ro c", "m r", "c+ m"])
def test_wgrad_operand_layouts(dev, lays):
    a_lay, b_lay = lays.split()
    run_wgrad(dev, offs(30, 0, 70), 100, 48, 56, F32, "r", 1.0, 0.0, a_lay, b_lay)


@pytest.mark.parametrize("offsets", [[3, 10, 20, 20], [0, 30, 10, 25], [-5, 4, 2, 60], [50, 0, 0, 0]])
def test_wgrad_any_offsets(dev, offsets):
    run_wgrad(dev, offsets, 40, 64, 48, F32, "r", 1.0, 0.0)
    run_wgrad(dev, offsets + [31] * 100, 40, 64, 48, F32, "r", 1.0, 0.0)


def test_wgrad_degenerate(dev):
    run_wgrad(dev, [0, 0, 0], 0, 16, 24, F32, "r", 1.0, 0.0)
    run_wgrad(dev, [0, 0, 0], 0, 16, 24, BF16, "r", 1.0, 0.5)
    run_wgrad(dev, [0, 5, 9], 9, 16, 24, BF16, "r", 0.0, 0.5)
    run_wgrad(dev, [0], 9, 16, 24, BF16, "r", 1.0, 0.0)


def run_wgrad(dev, offsets, rows, k, n, out, c_lay, alpha, beta, a_lay="r", b_lay="r"):
    groups = len(offsets) - 1
    a, b = rand(5, rows, k), rand(6, rows, n)
    c0 = rand(7, max(groups, 1), k, n, dt=out)
    bounds = bounds_of(offsets, rows)
    covered = torch.zeros(rows, dtype=torch.bool)
    for s, e in bounds:
        covered[s:e] = True
    a_in, b_in = a.clone(), b.clone()
    a_in[~covered] = float("nan")
    b_in[~covered] = float("nan")
    at, ars, acs = on(dev, lay(a_in, a_lay))
    bt, brs, bcs = on(dev, lay(b_in, b_lay))
    parts = [lay(c0[g] if beta else torch.full_like(c0[g], float("nan")), c_lay, fill=7.0)
             for g in range(c0.shape[0])]
    (p0, off), crs, ccs = parts[0]
    step = p0.numel() - off + 5
    cbuf = torch.full((step * len(parts),), 7.0, dtype=out)
    for g, ((p, _), _, _) in enumerate(parts):
        cbuf[g * step:g * step + p.numel()] = p
    ct = cbuf.to(dev)
    ot = torch.tensor(offsets, dtype=torch.int32, device=dev)
    gk.gemm_grouped_wgrad(alpha, gk.MatRef(at, rows, k, ars, acs), ot,
                          gk.MatRef(bt, rows, n, brs, bcs), beta,
                          gk.MatMut(ct, k, n, crs, ccs), step)
    torch.cuda.synchronize()
    host = ct.cpu()
    mask = torch.ones_like(cbuf, dtype=torch.bool)
    for g, (s, e) in enumerate(bounds):
        view = torch.as_strided(host, (k, n), (crs, ccs), g * step)
        torch.as_strided(mask, (k, n), (crs, ccs), g * step).fill_(False)
        base = c0[g].double() if beta else torch.zeros(k, n).double()
        want, mags = torch.zeros(k, n).double(), torch.zeros(k, n).double()
        if alpha and e > s:
            want = alpha * (a[s:e].double().t() @ b[s:e].double())
            mags = abs(alpha) * (a[s:e].double().abs().t() @ b[s:e].double().abs())
        check(view, want + beta * base, mags, e - s, out, alpha, beta, base)
    assert same_bits(host[mask], cbuf[mask])


def uneven(rows, groups):
    """Group sizes that differ, an empty group among them where there are several."""
    w = [0 if g == 1 else 1 + g * 7 % 5 for g in range(groups)]
    sizes = [rows * v // sum(w) for v in w]
    sizes[0] += rows - sum(sizes)
    return sizes


# products that reach each tile for rows of any alignment, and the copies
@pytest.mark.parametrize("rows,groups,k,n,layout", [
    (459, 8, 9, 3101, "co"), (6419, 5, 9, 65, "co"), (5722, 3, 9, 9, "co"), (459, 8, 333, 301, "co"),
    (60, 8, 333, 301, "co"), (5, 3, 397, 9, "co"), (44, 7, 1397, 75, "co"), (404, 2, 11, 4345, "co"),
    (2254, 8, 9, 985, "ro"), (8467, 51, 9, 89, "ro"), (867, 5, 209, 189, "ro"), (33, 3, 69, 9, "ro"),
    (70, 3, 261, 77, "ro"), (23, 1, 3905, 9, "ro"), (4, 2, 517, 131, "ro"), (1500, 3, 129, 131, "ro"),
])
def test_tiles_for_any_alignment(dev, rows, groups, k, n, layout):
    run_grouped(dev, offs(*uneven(rows, groups)), rows + 3, k, n, a_lay="ro", b_lay=layout, out=F32)


# weight gradients that reach each tile, whole groups and ranges of them
@pytest.mark.parametrize("rows,groups,k,n", [
    (4, 35, 1288, 144), (6358, 1, 2088, 1688), (31, 32, 1032, 8), (7060, 1, 600, 1664), (9, 1, 8, 8),
    (4637, 2, 320, 8), (35, 54, 264, 8), (8172, 1, 136, 5600), (86, 1, 8, 16), (2142, 1, 16, 16),
    (9, 1, 9, 9), (635, 1, 9, 9), (9, 50, 69, 331), (8340, 4, 69, 327), (385, 2, 815, 2085),
    (6358, 1, 2087, 481), (8, 40, 1731, 259), (7060, 1, 597, 1657), (2215, 5, 623, 139),
    (8713, 1, 163, 211), (12, 44, 147, 631), (414, 1, 9, 9), (7833, 1, 9, 9), (3000, 2, 520, 1040),
    (900, 3, 520, 1040), (1200, 3, 521, 1041),
])
@pytest.mark.parametrize("out", [F32, BF16])
def test_wgrad_tiles(dev, rows, groups, k, n, out):
    lay = "ro" if k % 8 else "r"
    run_wgrad(dev, offs(*uneven(rows, groups)), rows + 3, k, n, out, "r", 1.0, 0.0, lay, lay)


@pytest.mark.parametrize("layout", ["c", "r"])
@pytest.mark.parametrize("sizes,k,n", [((2, 0, 5, 1), 520, 5000), ((1, 2, 3), 72, 9000),
                                       ((4,) * 12, 264, 2560), ((16,), 1032, 20000),
                                       ((1,) * 9, 8, 3336)])
def test_short_groups_of_many_columns(dev, sizes, k, n, layout):
    run_grouped(dev, offs(*sizes), sum(sizes) + 2, k, n, b_lay=layout)
