"""Linear layers' products, their gradients and 8-bit checkpoints against 64 bits.

Tolerances.  K products, exact in f32, are added in f32: each addition is off by at most 2^-23
of the sum of the magnitudes, S, so Z by (K + 2) 2^-23 S with bias and alpha.  An activation
carries that on with a slope of at most 1.13 and is off by 2^-20 max(|z|, 1) itself (as
documented), a derivative (whose own slope is at most 1.2) likewise.  A residual adds 2^-23 of
what it is added to, and the output's rounding half a step: 2^-8 (bf16) or 2^-24 of the value.
Column sums of M rows add up their terms' errors and M 2^-23 of the terms' magnitudes."""
import math

import pytest
import torch

import gemmkit_amd as gk

pytestmark = pytest.mark.gpu

BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
HALF = {BF16: 2.0 ** -8, F32: 2.0 ** -24}
E23, E20 = 2.0 ** -23, 2.0 ** -20
SLOPE = -0.3
ACTS = {"none": None, "relu": gk.Activation.Relu, "leaky": gk.Activation.LeakyRelu(SLOPE),
        "gelu": gk.Activation.Gelu, "tanh": gk.Activation.GeluTanh, "silu": gk.Activation.Silu}
C2 = math.sqrt(2 / math.pi)
SMOOTH = ("gelu", "tanh", "silu")


def act64(z, act):
    if act == "relu":
        return z.clamp(min=0)
    if act == "leaky":
        s = torch.tensor(SLOPE, dtype=F32).double().item()
        return z.clamp(min=0) + s * z.clamp(max=0)
    if act == "gelu":
        return z * torch.special.ndtr(z)
    if act == "tanh":
        return 0.5 * z * (1 + torch.tanh(C2 * (z + 0.044715 * z ** 3)))
    return z * torch.sigmoid(z) if act == "silu" else z


def slope64(z, act):
    if act == "none":
        return torch.ones_like(z)
    if act in ("relu", "leaky"):
        s = torch.tensor(SLOPE if act == "leaky" else 0.0, dtype=F32).double().to(z.device)
        return torch.where(z > 0, torch.ones_like(z), s)
    z = z.clone().requires_grad_()
    act64(z, act).sum().backward()
    return z.grad


def rnd(shape, dt, seed, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * std).to(dt)


def strides_of(rows, cols, how):
    """(rs, cs, length, offset) of a view."""
    if how == "row":
        return cols, 1, rows * cols, 0
    if how == "col":
        return 1, rows, rows * cols, 0
    if how == "pad":
        return cols + 8, 1, rows * (cols + 8), 0
    if how == "odd":
        return cols + 3, 1, rows * (cols + 3), 0
    if how == "mis":  # a base that is aligned to its element only
        return cols, 1, rows * cols, 1
    assert how == "gap"
    return 2 * cols + 1, 2, rows * (2 * cols + 1), 0


def placed(x, how, dev, fill=float("nan")):
    """x as a view of the layout, what lies between its elements filled; (buffer, rs, cs)."""
    rows, cols = x.shape
    rs, cs, n, off = strides_of(rows, cols, how)
    buf = torch.full((n + off,), fill, dtype=x.dtype)
    if rows * cols:
        torch.as_strided(buf, (rows, cols), (rs, cs), off).copy_(x)
    return buf.to(dev)[off:], rs, cs


def ref(x, how, dev):
    t, rs, cs = placed(x, how, dev)
    return gk.MatRef(t, x.shape[0], x.shape[1], rs, cs)


class Out:
    """An output view whose surroundings have to stay as they are."""

    def __init__(self, rows, cols, dt, how, dev, start=None):
        x = torch.full((rows, cols), float("nan"), dtype=dt) if start is None else start
        self.t, self.rs, self.cs = placed(x, how, dev, fill=7.0)
        self.shape = (rows, cols)
        self.view = gk.MatMut(self.t, rows, cols, self.rs, self.cs)

    def get(self):
        host = self.t.cpu()
        v = torch.as_strided(host, self.shape, (self.rs, self.cs), host.storage_offset())
        mask = torch.ones(host.numel(), dtype=torch.bool)
        torch.as_strided(mask, self.shape, (self.rs, self.cs)).fill_(False)
        assert (host[mask] == 7.0).all()
        return v.clone()


def values8(q):
    """(values, steps per element) of a MatMxint8."""
    nb = -(-q.cols // 32)
    c = torch.as_strided(q.codes.cpu().flatten(), (q.rows, nb * 32), (q.ld, 1)).double()
    s = torch.as_strided(q.scales.cpu().flatten(), (q.rows, nb), (q.lds, 1)).double()
    step = torch.pow(2.0, s - 133).repeat_interleave(32, 1)
    step[(s == 255).repeat_interleave(32, 1)] = float("nan")
    return (c * step)[:, :q.cols], step[:, :q.cols]


def quantize64(x):
    """(codes, scale bytes) by the definition."""
    rows, n = x.shape
    nb = -(-n // 32)
    v = torch.zeros(rows, nb * 32, dtype=F64)
    v[:, :n] = x.double()
    v = v.view(rows, nb, 32)
    bad = ~torch.isfinite(v).all(2)
    top = torch.where(bad.unsqueeze(2), torch.zeros_like(v), v).abs().amax(2)
    e = torch.where(top > 0, torch.frexp(top)[1] - 1, torch.full_like(top, -120).int()).clamp(min=-120)
    m = v / torch.pow(2.0, e.double() - 6).unsqueeze(2)
    code = torch.round(m).clamp(-127, 127)  # (half to even)
    code = torch.where(bad.unsqueeze(2), torch.zeros_like(code), code)
    byte = torch.where(bad, torch.full_like(e, 255), e + 127)
    return code.view(rows, nb * 32).to(torch.int8), byte.to(torch.uint8)


def mx_empty(rows, cols, dev, pad=0):
    nb = -(-cols // 32)
    ld, lds = nb * 32 + pad, -(-nb // 16) * 16 + pad
    codes = torch.full((max(rows * ld, 1),), 0x5A, dtype=torch.int8, device=dev)
    scales = torch.full((max(rows * lds, 1),), 0x5A, dtype=torch.uint8, device=dev)
    return gk.MatMxint8(codes, scales, rows, cols, ld, lds)


def mx_of(x, dev, pad=0):
    q = mx_empty(*x.shape, dev, pad)
    gk.quantize_mxint8(ref(x, "row", dev), q)
    return q


def close(got, want, tol, what):
    got = got.double()
    assert torch.isfinite(got).all(), what
    over = (got - want).abs() - tol
    assert (over <= 0).all(), f"{what}: off by {over.max().item()} more than its bound"


def product(a, b, alpha=1.0):
    """The product in 64 bits and the sums of its terms' magnitudes."""
    a, b = a.double(), b.double()
    return alpha * (a @ b), abs(alpha) * (a.abs() @ b.abs())


# ------------------------------------------------------------------ checkpoints

def sample(rows, k, dt, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, k, generator=g)
    x *= torch.pow(2.0, torch.randint(-30, 30, (rows, -(-k // 32)), generator=g).float()
                   ).repeat_interleave(32, 1)[:, :k]
    if rows * k > 64:
        # halves of a step under a largest magnitude of 64 steps, ties both ways, one that
        # rounds to 128 and stays at 127, signed zeros
        ties = torch.tensor([64.0, 0.5, 1.5, 2.5, -0.5, -1.5, 63.5, 62.5, -0.0, 0.25, -63.5])
        n = min(len(ties), k)
        x[0, :n] = ties[:n]
        if k >= 64:
            x[-1, 32:64] = 0.0
            x[0, 32:35] = torch.tensor([127.75, -127.5, 126.5])
            x[0, 35:64] = 1.0
    return x.to(dt)


@pytest.mark.parametrize("dt", [BF16, F32])
@pytest.mark.parametrize("rows,k", [(1, 1), (1, 32), (3, 31), (5, 33), (7, 512), (130, 1000),
                                    (2, 4096), (65, 520), (64, 96), (300, 4000)])
@pytest.mark.parametrize("how", ["row", "pad", "odd", "mis", "col", "gap"])
def test_quantize_and_back(dev, dt, rows, k, how):
    x = sample(rows, k, dt, 3)
    q = mx_empty(rows, k, dev, pad=16 if how == "pad" else 0)
    assert gk.quantize_mxint8(ref(x, how, dev), q) is q
    code, byte = quantize64(x)
    nb = -(-k // 32)
    got_c = torch.as_strided(q.codes.cpu(), (rows, nb * 32), (q.ld, 1))
    got_s = torch.as_strided(q.scales.cpu(), (rows, -(-nb // 16) * 16), (q.lds, 1))
    assert torch.equal(got_s[:, :nb], byte)
    assert (got_s[:, nb:] == 0).all()
    assert torch.equal(got_c, code)
    want = values8(q)[0]
    for out in (BF16, F32):
        c = Out(rows, k, out, how, dev)
        gk.dequantize_mxint8(q, c.view)
        assert torch.equal(c.get().double(), want)


@pytest.mark.parametrize("dt,rows", [(BF16, 4100), (F32, 2050)])
def test_large_matrices_as_their_halves(dev, dt, rows):
    """Matrices from 64 MiB on are read another way: the same bits as half of the rows at a time,
    with a last block that is not whole."""
    k = 8200
    x = torch.randn(rows, k, device=dev, generator=torch.Generator(dev).manual_seed(9)).to(dt)
    z = torch.randn(rows, k, device=dev, generator=torch.Generator(dev).manual_seed(10)).to(BF16)
    assert x.numel() * x.element_size() >= 64 << 20
    cuts = [(0, rows), (0, rows // 2), (rows // 2, rows)]
    codes, grads, sums = [], [], []
    for lo, hi in cuts:
        n = hi - lo
        xv = gk.MatRef(x[lo:hi], n, k, k, 1)
        q = mx_empty(n, k, dev)
        gk.quantize_mxint8(xv, q)
        codes.append((torch.as_strided(q.codes, (n, -(-k // 32) * 32), (q.ld, 1)),
                      torch.as_strided(q.scales, (n, -(-k // 32)), (q.lds, 1))))
        for act, zv in (("none", None), ("gelu", gk.MatRef(z[lo:hi], n, k, k, 1)), ("silu", q)):
            d, s = torch.empty(n, k, dtype=BF16, device=dev), torch.empty(k, device=dev)
            gk.activation_grad(xv, gk.MatMut(d, n, k, k, 1), act=ACTS[act], z=zv, dbias=s)
            grads.append(d)
            sums.append(s)
    for i in range(2):
        assert torch.equal(codes[0][i], torch.cat([codes[1][i], codes[2][i]]))
    for i in range(3):
        assert torch.equal(grads[i], torch.cat([grads[3 + i], grads[6 + i]]))
        # (two orders of one sum of `rows` terms, each off by rows half steps of the magnitudes' sum)
        bound = 2 * rows * E23 * (grads[i].double().abs().sum(0) * (1 + 2.0 ** -8) + 1e-30)
        assert ((sums[i].double() - sums[3 + i].double() - sums[6 + i].double()).abs() <= bound).all()


def test_quantize_extremes(dev):
    big, tiny, sub = 3.3895313892515355e38, 2.0 ** -126, 2.0 ** -133
    for dt in (BF16, F32):
        rows = [[big, -big], [tiny, 0.0], [sub, -sub], [2.0 ** -120, 2.0 ** -126], [2.0 ** -121, 0],
                [float("inf"), 1.0], [1.0, float("nan")], [float("-inf"), float("nan")], [0.0, -0.0],
                [2.0 ** -127, 3 * 2.0 ** -127]]
        x = torch.zeros(len(rows), 40)
        x[:, 3] = torch.tensor([r[0] for r in rows])
        x[:, 30] = torch.tensor([r[1] for r in rows])
        x[:, 35] = 5.0
        x = x.to(dt)
        for how in ("row", "col"):
            q = mx_empty(len(rows), 40, dev)
            gk.quantize_mxint8(ref(x, how, dev), q)
            code, byte = quantize64(x)
            assert torch.equal(q.scales.cpu().view(len(rows), -1)[:, :2], byte)
            assert torch.equal(q.codes.cpu().view(len(rows), -1), code)
            c = Out(len(rows), 40, F32, how, dev)
            gk.dequantize_mxint8(q, c.view)
            assert torch.equal(torch.nan_to_num(c.get().double(), nan=-1.0),
                               torch.nan_to_num(values8(q)[0], nan=-1.0))


def test_any_codes_and_scales(dev):
    """Every code under every scale byte, those that quantization never writes too."""
    q = mx_empty(256, 256, dev)
    codes = torch.arange(256).to(torch.uint8).view(torch.int8)
    q.codes.copy_(codes.repeat(256).to(dev))
    q.scales.view(256, 16)[:, :8] = torch.arange(256, dtype=torch.uint8, device=dev).unsqueeze(1)
    want = values8(q)[0].float().double()
    want[254, 128] = -float("inf")  # -128 * 2^121
    c = Out(256, 256, F32, "row", dev)
    gk.dequantize_mxint8(q, c.view)
    got = c.get().double()
    assert torch.isnan(got[255]).all() and torch.equal(got[:255], want[:255])


@pytest.mark.parametrize("act", [a for a in ACTS if a != "none"])
def test_dequantize_through_activation(dev, act):
    x = rnd((70, 333), F32, 5, std=3.0)
    q = mx_of(x, dev)
    z = values8(q)[0]
    for out in (BF16, F32):
        c = Out(70, 333, out, "odd", dev)
        gk.dequantize_mxint8(q, c.view, act=ACTS[act])
        want = act64(z, act)
        own = E20 * z.abs().clamp(min=1)
        close(c.get(), want, own + HALF[out] * (want.abs() + own), act)


def test_smooth_activations_far_out(dev):
    """Derivatives and activations where squares and exponentials overflow."""
    z = torch.tensor([[0.0, -0.0, 1e-30, -1e-30, 5.0, -5.0, 16.0, -16.0, 40.0, -40.0, 89.0, -89.0, 1e4,
                       -1e4, 1e18, -1e18, 3e19, -3e19, 1e30, -1e30, 3e38, -3e38, 1.0, -1.0]])
    zb = z.to(BF16)
    one = torch.ones_like(z)
    # limits: the derivative is 1 far right and 0 far left, the activation z and 0
    z64 = zb.double()
    for act in SMOOTH:
        near = z64.clamp(-60, 60)
        want = torch.where(z64.abs() > 60, (z64 > 0).double(), slope64(near, act))
        d = Out(1, z.shape[1], BF16, "row", dev)
        gk.activation_grad(ref(one, "row", dev), d.view, act=ACTS[act], z=ref(zb, "row", dev))
        close(d.get(), want, E20 * near.abs().clamp(min=1) + HALF[BF16] * want.abs(), act)
        nan = torch.full((1, 3), float("nan"), dtype=BF16)
        d = Out(1, 3, BF16, "row", dev)
        gk.activation_grad(ref(torch.ones(1, 3), "row", dev), d.view, act=ACTS[act],
                           z=ref(nan, "row", dev))
        assert torch.isnan(d.get()).all()


# ------------------------------------------------------------------ forward

def run_linear(dev, m, k, n, act="none", out=BF16, layout="c", bias=None, res=False, z=None,
               hows=("row", "row", "row"), alpha=1.0, in_place=False, seed=1, mx_pad=0, ws=None):
    a, w = rnd((m, k), BF16, seed), rnd((k, n), BF16, seed + 1, 1 / math.sqrt(max(k, 1)))
    av = ref(a, hows[0], dev)
    if layout == "c":
        t, rs, cs = placed(w.t().contiguous(), hows[1], dev)
        bv = gk.MatRef(t, k, n, cs, rs)
    else:
        bv = ref(w, hows[1], dev)
    p, s = product(a.to(dev), w.to(dev), alpha)
    p, s = p.cpu(), s.cpu()
    bt = None
    if bias is not None:
        bt = rnd((n,), bias, seed + 2)
        p, s = p + bt.double(), s + bt.double().abs()
    r = rnd((m, n), out, seed + 3) if res else None
    c = Out(m, n, out, hows[2], dev, start=r if in_place else None)
    rv = None if r is None else (c.view if in_place else ref(r, hows[2], dev))
    zo, zv = None, None
    if z == "mx":
        zv = mx_empty(m, n, dev, mx_pad)
    elif z:
        zo = Out(m, n, BF16, z, dev)
        zv = zo.view
    gk.gemm_linear(alpha, av, bv, c.view, bias=None if bt is None else gk.Bias.PerCol(bt.to(dev)),
                   act=ACTS[act], residual=rv, z=zv, ws=ws)
    dz = (k + 2) * E23 * s
    want = act64(p, act)
    tol = 1.13 * dz + (E20 * p.abs().clamp(min=1) if act in SMOOTH else E23 * p.abs())
    if r is not None:
        tol = tol + E23 * (want.abs() + r.double().abs())
        want = want + r.double()
    what = f"{m}x{k}x{n} {act} {out}"
    got = c.get()
    close(got, want, tol + HALF[out] * (want.abs() + tol), what)
    if zo is not None:
        close(zo.get(), p, dz + HALF[BF16] * (p.abs() + dz), what + " z")
    if z == "mx":
        v, step = values8(zv)
        top = torch.zeros(m, -(-n // 32) * 32, dtype=F64)
        top[:, :n] = (p.abs() + dz)
        top = top.view(m, -1, 32).amax(2).repeat_interleave(32, 1)[:, :n]
        assert (step <= torch.pow(2.0, torch.floor(torch.log2(top.clamp(min=2.0 ** -120))) - 6)).all()
        bound = torch.where(p.abs() + dz >= 127.5 * step, step, 0.5 * step)
        close(v, p, bound + dz, what + " z")
    return got, zv


SHAPES = [(1, 64, 32), (1, 1000, 1), (1, 7, 33), (3, 1, 5), (16, 4096, 256), (17, 130, 96), (40, 512, 200),
          (100, 1501, 333), (130, 264, 520), (257, 72, 260), (300, 1024, 1024), (513, 96, 1000)]


@pytest.mark.parametrize("m,k,n", SHAPES)
@pytest.mark.parametrize("layout", ["c", "r"])
@pytest.mark.parametrize("out", [BF16, F32])
def test_linear_shapes(dev, m, k, n, layout, out):
    run_linear(dev, m, k, n, "gelu", out, layout, bias=BF16, res=True, z="mx")
    run_linear(dev, m, k, n, "none", out, layout, z="row")


@pytest.mark.parametrize("act", list(ACTS))
@pytest.mark.parametrize("out", [BF16, F32])
@pytest.mark.parametrize("m", [5, 200])
def test_linear_activations(dev, act, out, m):
    run_linear(dev, m, 256, 160, act, out, bias=F32, res=True, z="row")
    run_linear(dev, m, 100, 75, act, out, "r", bias=BF16, z="mx")
    run_linear(dev, m, 100, 75, act, out, "r")


@pytest.mark.parametrize("hows", [("pad", "pad", "pad"), ("odd", "odd", "odd"), ("mis", "mis", "mis"),
                                  ("col", "col", "col"), ("gap", "gap", "gap"), ("row", "row", "col"),
                                  ("row", "odd", "gap"), ("col", "row", "odd")])
@pytest.mark.parametrize("out", [BF16, F32])
@pytest.mark.parametrize("m,k,n", [(9, 200, 72), (150, 130, 141)])
def test_linear_strides(dev, hows, out, m, k, n):
    run_linear(dev, m, k, n, "silu", out, "c", bias=BF16, res=True, z=hows[2], hows=hows)
    run_linear(dev, m, k, n, "tanh", out, "r", bias=F32, res=True, z="mx", hows=hows, mx_pad=16)
    run_linear(dev, m, k, n, "relu", out, "r", res=True, hows=hows, in_place=True, z="mx")


@pytest.mark.parametrize("m,k,n", [(4096, 320, 4096), (2500, 256, 3000), (8192, 128, 640),
                                   (1280, 512, 4000)])
@pytest.mark.parametrize("out", [BF16, F32])
def test_linear_many_tiles(dev, m, k, n, out):
    run_linear(dev, m, k, n, "gelu", out, "c", bias=BF16, res=True, z="mx")
    run_linear(dev, m, k, n, "silu", out, "r", bias=BF16, res=True, z="row", in_place=True)


def test_linear_broadcast_residual(dev):
    m, k, n = 70, 64, 96
    a, w, r = rnd((m, k), BF16, 1), rnd((k, n), BF16, 2), rnd((n,), BF16, 3)
    c = Out(m, n, BF16, "row", dev)
    gk.gemm_linear(1.0, ref(a, "row", dev), ref(w, "row", dev), c.view,
                   residual=gk.MatRef(r.to(dev), m, n, 0, 1))
    p, s = product(a, w)
    want = p + r.double()
    tol = (k + 2) * E23 * s + E23 * (p.abs() + r.double().abs())
    close(c.get(), want, tol + HALF[BF16] * (want.abs() + tol), "broadcast")


@pytest.mark.parametrize("alpha", [0.0, -2.5])
@pytest.mark.parametrize("k", [0, 48])
def test_linear_alpha_and_empty_k(dev, alpha, k):
    for m, n in ((1, 40), (70, 96), (600, 512)):
        run_linear(dev, m, k, n, "gelu", BF16, "c", bias=F32, res=True, z="mx", alpha=alpha)
    # alpha == 0 reads neither operand
    a = torch.full((33, 64), float("nan"), dtype=BF16)
    b = torch.full((64, 40), float("nan"), dtype=BF16)
    bias = rnd((40,), F32, 1)
    c = Out(33, 40, F32, "row", dev)
    gk.gemm_linear(0.0, ref(a, "row", dev), ref(b, "row", dev), c.view, bias=gk.Bias.PerCol(bias.to(dev)))
    assert torch.equal(c.get(), bias.expand(33, 40))


def test_linear_kept_z_is_the_unrounded_sum_rounded_once(dev):
    """The kept forms of Z are what rounding or quantizing the f32 Z gives."""
    for m, k, n in ((5, 300, 100), (200, 512, 333), (1024, 256, 1024)):
        z32, _ = run_linear(dev, m, k, n, "none", F32, bias=BF16)
        _, q = run_linear(dev, m, k, n, "none", F32, bias=BF16, z="mx")
        code, byte = quantize64(z32)
        nb = -(-n // 32)
        assert torch.equal(q.codes.cpu().view(m, nb * 32), code)
        assert torch.equal(q.scales.cpu().view(m, -1)[:, :nb], byte)


def test_linear_nan_and_infinity_stay_in_their_rows(dev):
    m, k, n = 60, 128, 130
    a, w = rnd((m, k), BF16, 1), rnd((k, n), BF16, 2, 0.1)
    a[7, 5], a[33, 1] = float("nan"), float("inf")
    for act in ("gelu", "silu"):
        c = Out(m, n, F32, "row", dev)
        q = mx_empty(m, n, dev)
        gk.gemm_linear(1.0, ref(a, "row", dev), ref(w, "row", dev), c.view, act=ACTS[act], z=q)
        got = c.get()
        keep = torch.ones(m, dtype=torch.bool)
        keep[[7, 33]] = False
        assert torch.isfinite(got[keep]).all() and torch.isnan(got[7]).all()
        s = q.scales.cpu().view(m, -1)[:, :5]
        assert (s[[7, 33]] == 255).all() and (s[keep] < 255).all()


@pytest.mark.parametrize("m,n", [(0, 8), (8, 0), (0, 0)])
def test_empty_outputs(dev, m, n):
    a, b = torch.ones(max(m * 4, 1), dtype=BF16, device=dev), torch.ones(max(4 * n, 1), dtype=BF16, device=dev)
    c = torch.full((max(m * n, 1),), 3.0, dtype=BF16, device=dev)
    d = torch.full((n,), 5.0, device=dev)
    gk.gemm_linear(1.0, gk.MatRef(a, m, 4, 4, 1), gk.MatRef(b, 4, n, n, 1), gk.MatMut(c, m, n, n, 1))
    gk.gemm_linear_dgrad(1.0, gk.MatRef(a, m, 4, 4, 1), gk.MatRef(b, 4, n, n, 1),
                         gk.MatMut(c, m, n, n, 1), dbias=d)
    assert (d == 0).all()
    d.fill_(5.0)
    gk.activation_grad(gk.MatRef(a, m, n, n, 1), gk.MatMut(c, m, n, n, 1), dbias=d)
    assert (d == 0).all() and (c == 3.0).all()
    q = gk.MatMxint8.empty(m, n, dev)
    gk.quantize_mxint8(gk.MatRef(a, m, n, n, 1), q)
    gk.dequantize_mxint8(q, gk.MatMut(c, m, n, n, 1))
    assert (c == 3.0).all()


# ------------------------------------------------------------------ gradients

def run_grad(dev, m, k, n, act="none", out=BF16, layout="r", z="row", dbias=True, alpha=1.0,
             hows=("row", "row", "row"), seed=11, product_first=True, gt=BF16, in_place=False, ws=None):
    """gemm_linear_dgrad, or activation_grad where the gradient is there already."""
    zx = rnd((m, n), F32, seed + 2, 2.0)
    zv, z64 = None, torch.zeros(m, n, dtype=F64)
    if act != "none":
        if z == "mx":
            zv = mx_of(zx, dev, 16)
            z64 = values8(zv)[0]
        else:
            zb = zx.to(BF16)
            zv, z64 = ref(zb, z, dev), zb.double()
    sums = torch.full((n,), float("nan"), device=dev) if dbias else None
    if product_first:
        a, w = rnd((m, k), BF16, seed), rnd((k, n), BF16, seed + 1, 1 / math.sqrt(max(k, 1)))
        if layout == "c":
            t, rs, cs = placed(w.t().contiguous(), hows[1], dev)
            bv = gk.MatRef(t, k, n, cs, rs)
        else:
            bv = ref(w, hows[1], dev)
        p, s = product(a.to(dev), w.to(dev), alpha)
        p, s = p.cpu(), s.cpu()
        dp = (k + 2) * E23 * s
        d = Out(m, n, out, hows[2], dev)
        gk.gemm_linear_dgrad(alpha, ref(a, hows[0], dev), bv, d.view, act=ACTS[act], z=zv,
                             dbias=sums, ws=ws)
    else:
        g = rnd((m, n), gt, seed)
        p, dp, out = g.double(), torch.zeros(m, n, dtype=F64), BF16
        d = Out(m, n, BF16, hows[2], dev, start=g if in_place else None)
        gv = d.view if in_place else ref(g, hows[0], dev)
        gk.activation_grad(gv, d.view, act=ACTS[act], z=zv, dbias=sums, ws=ws)
    slope = slope64(z64, act)
    want = p * slope
    tol = dp * slope.abs().clamp(min=1) + E23 * want.abs()
    if act in SMOOTH:
        tol = tol + (p.abs() + dp) * E20 * z64.abs().clamp(min=1)
    what = f"{m}x{k}x{n} {act} {out}"
    close(d.get(), want, tol + HALF[out] * (want.abs() + tol), what)
    if dbias:
        close(sums.cpu(), want.sum(0), tol.sum(0) + (m + 1) * E23 * (want.abs() + tol).sum(0),
              what + " dbias")
    return d, sums


@pytest.mark.parametrize("m,k,n", SHAPES)
@pytest.mark.parametrize("layout", ["c", "r"])
@pytest.mark.parametrize("out", [BF16, F32])
def test_dgrad_shapes(dev, m, k, n, layout, out):
    run_grad(dev, m, k, n, "gelu", out, layout, z="mx")
    run_grad(dev, m, k, n, "silu", out, layout, z="row")


@pytest.mark.parametrize("act", list(ACTS))
@pytest.mark.parametrize("out", [BF16, F32])
@pytest.mark.parametrize("m", [5, 200])
def test_dgrad_activations(dev, act, out, m):
    run_grad(dev, m, 256, 160, act, out, z="row")
    run_grad(dev, m, 100, 75, act, out, "c", z="mx")
    run_grad(dev, m, 100, 75, act, out, "c", dbias=False, alpha=-1.5)


@pytest.mark.parametrize("hows", [("pad", "pad", "pad"), ("odd", "odd", "odd"), ("mis", "mis", "mis"),
                                  ("col", "col", "col"), ("gap", "gap", "gap"), ("row", "odd", "gap")])
@pytest.mark.parametrize("m,k,n", [(9, 200, 72), (150, 130, 141)])
def test_dgrad_strides(dev, hows, m, k, n):
    for out in (BF16, F32):
        run_grad(dev, m, k, n, "silu", out, "c", z=hows[2], hows=hows)
        run_grad(dev, m, k, n, "tanh", out, "r", z="mx", hows=hows)


@pytest.mark.parametrize("m,k,n", [(4096, 320, 4096), (2500, 256, 3000), (8192, 128, 640),
                                   (1280, 512, 4000), (5000, 64, 70)])
@pytest.mark.parametrize("out", [BF16, F32])
def test_dgrad_many_tiles(dev, m, k, n, out):
    run_grad(dev, m, k, n, "gelu", out, "r", z="mx")
    run_grad(dev, m, k, n, "silu", out, "c", z="row")


@pytest.mark.parametrize("alpha,k", [(0.0, 64), (1.0, 0)])
def test_dgrad_of_nothing_is_zero(dev, alpha, k):
    for m, n in ((1, 40), (600, 512)):
        run_grad(dev, m, k, n, "gelu", BF16, z="mx", alpha=alpha)


@pytest.mark.parametrize("m,k,n", [(9, 64, 72), (130, 264, 520), (300, 1024, 1024), (2500, 256, 3000)])
@pytest.mark.parametrize("z", [None, "row", "mx"])
def test_dgrad_sums_of_infinite_columns(dev, m, k, n, z):
    """A column of B with an infinity: its sum is infinite, whatever the rows past the last one
    hold.  (Exact: every finite product is 2^-10, so that the sums are below 2^24 of them.)"""
    a = torch.ones((m, k), dtype=BF16)
    w = torch.full((k, n), 2.0 ** -10, dtype=BF16)
    w[k - 1, n - 1] = w[0, 5] = float("inf")
    zs = torch.ones((m, n), dtype=BF16)
    zv = None if z is None else mx_of(zs, dev) if z == "mx" else ref(zs, "row", dev)
    sums = torch.full((n,), float("nan"), device=dev)
    d = Out(m, n, BF16, "row", dev)
    gk.gemm_linear_dgrad(1.0, ref(a, "row", dev), ref(w, "row", dev), d.view,
                         act=ACTS["none" if z is None else "relu"], z=zv, dbias=sums)
    got = sums.cpu()
    want = torch.full((n,), m * k * 2.0 ** -10)
    want[n - 1] = want[5] = float("inf")
    assert torch.equal(got, want)


@pytest.mark.parametrize("m,n", [(1, 1), (1, 700), (3, 8), (700, 1), (333, 777), (1003, 520), (64, 5000),
                                 (5000, 40), (2048, 2048)])
@pytest.mark.parametrize("act", ["none", "gelu", "leaky"])
@pytest.mark.parametrize("gt", [BF16, F32])
def test_activation_grad(dev, m, n, act, gt):
    run_grad(dev, m, 0, n, act, z="row", product_first=False, gt=gt)
    run_grad(dev, m, 0, n, act, z="mx", product_first=False, gt=gt, dbias=m % 2 == 0)


@pytest.mark.parametrize("act", list(ACTS))
@pytest.mark.parametrize("how", ["row", "pad", "odd", "mis", "col", "gap"])
def test_activation_grad_strides(dev, act, how):
    run_grad(dev, 130, 0, 141, act, z=how, product_first=False, gt=F32, hows=(how, how, how))
    run_grad(dev, 130, 0, 141, act, z="mx", product_first=False, hows=(how, how, how), in_place=True)


@pytest.mark.parametrize("m", [64, 256, 257, 512, 513, 1023, 1024, 1025, 2048])
@pytest.mark.parametrize("n", [8, 72, 1000, 1001, 2080])
@pytest.mark.parametrize("z", ["row", "mx", "odd"])
def test_activation_grad_column_sums(dev, m, n, z):
    """Rows, widths and alignments on both sides of where the sums need no second launch."""
    run_grad(dev, m, 0, n, act="silu", z=z, product_first=False, gt=BF16 if m % 2 else F32)


def test_gradients_against_differences(dev):
    """d/dx and d/db of sum(G * act(X W + b)) against central differences in 64 bits."""
    m, k, n = 6, 40, 33
    x, w, b = rnd((m, k), BF16, 1), rnd((k, n), BF16, 2, 0.2), rnd((n,), F32, 3)
    g = rnd((m, n), BF16, 4)
    for act in SMOOTH:
        c, z = Out(m, n, F32, "row", dev), Out(m, n, BF16, "row", dev)
        gk.gemm_linear(1.0, ref(x, "row", dev), ref(w, "row", dev), c.view,
                       bias=gk.Bias.PerCol(b.to(dev)), act=ACTS[act], z=z.view)
        kept = z.get()
        d, db = Out(m, n, BF16, "row", dev), torch.zeros(n, device=dev)
        gk.activation_grad(ref(g, "row", dev), d.view, act=ACTS[act], z=ref(kept, "row", dev), dbias=db)
        h = 1e-4
        zk = kept.double()
        want = g.double() * (act64(zk + h, act) - act64(zk - h, act)) / (2 * h)
        # (differences: h^2 / 6 of a third derivative below 3, and rounding of 2^-52 / h)
        diff = g.double().abs() * (h * h + 1e-11)
        own = diff + g.double().abs() * E20 * zk.abs().clamp(min=1)
        close(d.get(), want, own + HALF[BF16] * (want.abs() + own), act)
        close(db.cpu(), want.sum(0), own.sum(0) + (m + 1) * E23 * want.abs().sum(0), act)
        dx = Out(m, k, F32, "row", dev)
        dz = d.get()
        gk.gemm_linear_dgrad(1.0, ref(dz, "row", dev), ref(w.t().contiguous(), "row", dev), dx.view)
        p, s = product(dz, w.t())
        close(dx.get(), p, (n + 2) * E23 * s + HALF[F32] * p.abs(), act)


# ------------------------------------------------------------------ weight gradient

@pytest.mark.parametrize("rows,k,n", [(1, 1, 1), (1, 33, 40), (3, 64, 7), (64, 32, 32), (65, 100, 200),
                                      (200, 256, 264), (333, 1000, 77), (1003, 1024, 704),
                                      (5000, 64, 64), (4096, 520, 300)])
@pytest.mark.parametrize("out", [BF16, F32])
@pytest.mark.parametrize("act", ["none", "gelu", "relu"])
def test_wgrad(dev, rows, k, n, out, act):
    q = mx_of(rnd((rows, k), F32, 1, 2.0), dev, 16)
    b = rnd((rows, n), BF16, 2)
    h = act64(values8(q)[0], act)
    dh = E20 * values8(q)[0].abs().clamp(min=1) if act in SMOOTH else torch.zeros_like(h)
    if act != "none":
        dh = dh + HALF[BF16] * (h.abs() + dh)
    for beta, how_b, how_c in ((0.0, "row", "row"), (0.5, "odd", "odd"), (1.0, "col", "col"),
                               (0.0, "mis", "pad")):
        c0 = rnd((k, n), out, 3)
        c = Out(k, n, out, how_c, dev, start=c0 if beta else None)
        gk.gemm_wgrad_mxint8(-1.25, q, ref(b, how_b, dev), beta, c.view, act=ACTS[act])
        p, s = product(h.t(), b, -1.25)
        want = p + (beta * c0.double() if beta else 0)
        tol = (rows + 2) * E23 * (s + (abs(beta) * c0.double().abs() if beta else 0))
        tol = tol + 1.25 * (dh.t() @ b.double().abs()) * (1 + rows * E23)
        close(c.get(), want, tol + HALF[out] * (want.abs() + tol), f"{rows}x{k}x{n} {act} {how_c}")


@pytest.mark.parametrize("rows", [1, 63, 64, 127, 128, 129, 256, 257])
@pytest.mark.parametrize("k,n", [(1, 8), (40, 72), (1025, 711), (2047, 1100), (64, 2048)])
@pytest.mark.parametrize("act", ["none", "leaky", "silu"])
def test_wgrad_of_few_rows(dev, rows, k, n, act):
    """Rows and tiles on both sides of where a checkpoint is decoded in the tiles; a block
    of NaN stays in its columns; what lies past the matrices' rows and columns is
    not read into them."""
    x = rnd((rows, k), F32, 5, 2.0)
    q = mx_of(x, dev, 16)
    if k % 32:
        torch.as_strided(q.codes, (rows, -(-k // 32) * 32), (q.ld, 1))[:, k:] = 55
    b = rnd((rows, n), BF16, 6)
    h = act64(values8(q)[0], act)
    dh = E20 * values8(q)[0].abs().clamp(min=1) if act in SMOOTH else torch.zeros_like(h)
    if act != "none":
        dh = dh + HALF[BF16] * (h.abs() + dh)
    p, s = product(h.t(), b)
    tol = (rows + 2) * E23 * s + (dh.t() @ b.double().abs()) * (1 + rows * E23)
    for how_b in ("row", "mis"):
        c = Out(k, n, F32, "row", dev)
        gk.gemm_wgrad_mxint8(1.0, q, ref(b, how_b, dev), 0.0, c.view, act=ACTS[act])
        close(c.get(), p, tol + HALF[F32] * (p.abs() + tol), f"{rows}x{k}x{n} {act} {how_b}")
    q.scales[(rows - 1) * q.lds] = 255
    c = Out(k, n, F32, "row", dev)
    gk.gemm_wgrad_mxint8(1.0, q, ref(b, "row", dev), 0.0, c.view, act=ACTS[act])
    got = c.get()
    bad = slice(0, min(k, 32))
    if act == "silu" or act == "none":
        assert torch.isnan(got[bad]).all()
    assert torch.isfinite(got[32:]).all()


def test_wgrad_of_no_rows_scales_c(dev):
    for rows, alpha in ((0, 1.0), (40, 0.0)):
        q = mx_empty(rows, 48, dev)
        b = torch.full((max(rows, 1) * 40,), float("nan"), dtype=BF16, device=dev)
        for beta in (0.0, 2.0):
            c0 = rnd((48, 40), F32, 3)
            c = Out(48, 40, F32, "row", dev, start=c0 if beta else None)
            gk.gemm_wgrad_mxint8(alpha, q, gk.MatRef(b, rows, 40, 40, 1), beta, c.view, act=ACTS["gelu"])
            assert torch.equal(c.get(), beta * c0)


def test_wgrad_of_nan_blocks(dev):
    x = rnd((100, 96), F32, 1)
    x[13, 40] = float("nan")
    q = mx_of(x, dev)
    c = Out(96, 50, F32, "row", dev)
    gk.gemm_wgrad_mxint8(1.0, q, ref(rnd((100, 50), BF16, 2), "row", dev), 0.0, c.view)
    got = c.get()
    assert torch.isnan(got[32:64]).all() and torch.isfinite(got[:32]).all() and torch.isfinite(got[64:]).all()


@pytest.mark.parametrize("m,n", [(512, 6143), (512, 6145), (96, 32767), (96, 32769), (512, 8192)])
@pytest.mark.parametrize("z", ["row", "mx"])
def test_activation_grad_column_sums_of_wide_rows(dev, m, n, z):
    """On both sides of 3 Mi elements, up to which rows without alignment are summed in one launch."""
    run_grad(dev, m, 0, n, act="silu", z=z, product_first=False)
