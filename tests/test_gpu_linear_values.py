"""Values of the linear layers' activations and derivatives where they are small, infinite or
NaN.  An activation's argument reaches it exactly as an f32 bias of a product without alpha, a
derivative's as a bfloat16 pre-activation under a gradient of 1."""
import pytest
import torch

import gemmkit_amd as gk

pytestmark = pytest.mark.gpu

BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
E20, E23 = 2.0 ** -20, 2.0 ** -23


def row(t):
    return gk.MatRef.from_row_major(t, *t.shape)


def out(t):
    return gk.MatMut.from_row_major(t, *t.shape)


def ones(dev, *shape, dt=BF16):
    return torch.ones(*shape, dtype=dt, device=dev)


def activated(z, act, dev):
    """act(z) of f32 values, in f32."""
    n = z.numel()
    c = torch.empty(1, n, device=dev)
    gk.gemm_linear(0.0, row(ones(dev, 1, 1)), row(ones(dev, 1, n)), out(c),
                   bias=gk.Bias.PerCol(z.to(dev)), act=act)
    return c.cpu().flatten()


def derivative(z, act, dev):
    """act'(z) of bfloat16 values, in f32."""
    n = z.numel()
    d = torch.empty(1, n, device=dev)
    gk.gemm_linear_dgrad(1.0, row(ones(dev, 1, 1)), row(ones(dev, 1, n)), out(d), act=act,
                         z=row(z.to(dev).view(1, n)))
    return d.cpu().flatten()


def bf16_between(lo, hi):
    """Every bfloat16 value of [lo, hi]."""
    v = torch.arange(-2 ** 15, 2 ** 15, dtype=torch.int32).to(torch.int16).view(BF16)
    return v[(v >= lo) & (v <= hi)]


def tail(z):
    """(P(-|z|), |z| p(z), how far either may be off, relative to itself) in 64 bits.

    An exponent of z^2 log2(e) / 2 that is rounded three times, by 2^-24 each, moves the exponential by
    z^2 / 2 * 3 * 2^-24, less than z^2 2^-23 of itself; the exponential, a reciprocal and the nine
    steps of a polynomial with positive sum, whose error the fit adds to by 2^-22, stay
    within 2^-20.  (P by erfc: as 1 + erf it would end at 2^-53.)"""
    a = z.double().abs()
    return torch.special.erfc(a * 0.5 ** 0.5) / 2, a * torch.exp(-a * a / 2) * 0.3989422804014327, E20 + a * a * E23


def test_gelu_keeps_the_tail(dev):
    """GELU of negative z is z P(z) to its own last bits, not only to those of 1: its sign is
    z's as far as f32 reaches."""
    g = torch.Generator().manual_seed(1)
    z = torch.cat([bf16_between(-13, 13).float(), torch.rand(20001, generator=g) * 26 - 13])
    got = activated(z, gk.Activation.Gelu, dev).double()
    p, _, rel = tail(z)
    z64 = z.double()
    want = torch.where(z64 < 0, z64 * p, z64 * (1 - p))
    tol = z64.abs() * p * rel + torch.where(z64 < 0, 0.0, E23 * z64) + 2.0 ** -126
    assert ((got - want).abs() <= tol).all(), ((got - want).abs() / tol).max()
    assert (got[(z < -0.01) & (z > -12.5)] < 0).all()


def test_gelu_derivative_keeps_the_tail(dev):
    z = bf16_between(-13, 13)
    got = derivative(z, gk.Activation.Gelu, dev).double()
    p, zp, rel = tail(z)
    want = torch.where(z < 0, p - zp, 1 - p + zp)
    tol = (p + zp) * rel + torch.where(z < 0, 0.0, 2 * E23) + 2.0 ** -126
    assert ((got - want).abs() <= tol).all(), ((got - want).abs() / tol).max()


def test_gelu_of_a_checkpoint_keeps_the_tail(dev):
    """The same through dequantization, in f32 and rounded once to bfloat16."""
    z = -torch.arange(32, 128).float().div(8).view(3, 32)  # -4 .. -15.9: codes of one scale each
    q = gk.quantize_mxint8(row(z.to(dev)))
    kept = torch.empty(3, 32, device=dev)
    gk.dequantize_mxint8(q, out(kept))
    assert torch.equal(kept.cpu(), z)
    p, _, rel = tail(z)
    want = z.double() * p
    for dt, half in ((F32, 0.0), (BF16, 2.0 ** -8)):
        c = torch.empty(3, 32, dtype=dt, device=dev)
        gk.dequantize_mxint8(q, out(c), act=gk.Activation.Gelu)
        tol = want.abs() * (rel + half * (1 + rel)) + 2.0 ** -126
        assert ((c.cpu().double() - want).abs() <= tol).all()


@pytest.mark.parametrize("act", ["Relu", "LeakyRelu", "Gelu", "GeluTanh", "Silu"])
def test_derivatives_at_infinity(dev, act):
    """Their limits: a pre-activation past bfloat16's range is kept as an infinity, and its column
    sum stays finite."""
    a = gk.Activation.LeakyRelu(-0.5) if act == "LeakyRelu" else getattr(gk.Activation, act)
    inf = float("inf")
    z = torch.tensor([inf, -inf, 1.0, inf, -inf], dtype=BF16)
    low = -0.5 if act == "LeakyRelu" else 0.0
    limits = torch.tensor([1.0, low])
    assert torch.equal(derivative(z, a, dev)[[0, 1]], limits)
    for rows in (1, 40, 700):
        zm = z.to(dev).repeat(rows, 1)
        d, sums = torch.empty(rows, 5, dtype=BF16, device=dev), torch.empty(5, device=dev)
        gk.activation_grad(row(ones(dev, rows, 5)), out(d), act=a, z=row(zm), dbias=sums)
        assert torch.equal(d.float().cpu()[:, [0, 1, 3, 4]], limits.repeat(rows, 2))
        assert torch.equal(sums.cpu()[[0, 1, 3, 4]], limits.repeat(2) * rows)
    big = torch.tensor([3.4e38], device=dev)  # rounds to an infinity in bfloat16
    zk, c = torch.empty(1, 1, dtype=BF16, device=dev), torch.empty(1, 1, device=dev)
    gk.gemm_linear(0.0, row(ones(dev, 1, 1)), row(ones(dev, 1, 1)), out(c), bias=gk.Bias.PerCol(big),
                   act=a, z=out(zk))
    assert torch.isinf(zk).all() and torch.isfinite(c).all()


def test_activations_at_infinity(dev):
    z = torch.tensor([float("inf"), -float("inf")])
    for act, low in ((gk.Activation.Relu, 0.0), (gk.Activation.LeakyRelu(0.25), -float("inf")),
                     (gk.Activation.Gelu, 0.0), (gk.Activation.GeluTanh, None),
                     (gk.Activation.Silu, None)):
        got = activated(z, act, dev)
        assert got[0] == float("inf")
        assert torch.isnan(got[1]) if low is None else got[1] == low


NAN_ACTS = [gk.Activation.Relu, gk.Activation.LeakyRelu(-0.3), gk.Activation.LeakyRelu(0.0),
            gk.Activation.Gelu, gk.Activation.GeluTanh, gk.Activation.Silu]


@pytest.mark.parametrize("act", NAN_ACTS)
def test_nan_stays_nan(dev, act):
    """Through every activation and derivative, from a value and from a checkpoint's block."""
    nan = float("nan")
    got = activated(torch.tensor([1.0, nan, -1.0, nan]), act, dev)
    assert torch.equal(torch.isnan(got), torch.tensor([False, True, False, True]))
    got = derivative(torch.tensor([1.0, nan, -1.0, nan], dtype=BF16), act, dev)
    assert torch.equal(torch.isnan(got), torch.tensor([False, True, False, True]))
    for rows in (70, 600):
        x = torch.randn(rows, 100, generator=torch.Generator().manual_seed(2))
        x[rows - 3, 40] = float("inf")
        q = gk.quantize_mxint8(row(x.to(dev)))
        bad = torch.zeros(rows, 100, dtype=torch.bool)
        bad[rows - 3, 32:64] = True
        c = torch.empty(rows, 100, device=dev)
        gk.dequantize_mxint8(q, out(c), act=act)
        assert torch.equal(torch.isnan(c.cpu()), bad)
        b = torch.randn(rows, 24, generator=torch.Generator().manual_seed(3)).to(BF16).to(dev)
        w = torch.empty(100, 24, device=dev)
        gk.gemm_wgrad_mxint8(1.0, q, row(b), 0.0, out(w), act=act)
        assert torch.equal(torch.isnan(w.cpu()), bad.any(0).unsqueeze(1).expand(100, 24))
        g = ones(dev, rows, 100)
        d, sums = torch.empty(rows, 100, dtype=BF16, device=dev), torch.empty(100, device=dev)
        gk.activation_grad(row(g), out(d), act=act, z=q, dbias=sums)
        assert torch.equal(torch.isnan(d.cpu()), bad) and torch.equal(torch.isnan(sums.cpu()), bad.any(0))
        a, k = ones(dev, rows, 8), ones(dev, 8, 100)
        gk.gemm_linear_dgrad(1.0, row(a), row(k), out(d), act=act, z=q, dbias=sums)
        assert torch.equal(torch.isnan(d.cpu()), bad) and torch.equal(torch.isnan(sums.cpu()), bad.any(0))


@pytest.mark.parametrize("act", [gk.Activation.Relu, gk.Activation.LeakyRelu(-0.3)])
def test_zeros_of_either_sign(dev, act):
    z = torch.tensor([0.0, -0.0])
    assert torch.equal(activated(z, act, dev), torch.zeros(2))
    assert torch.equal(derivative(z.to(BF16), act, dev), torch.full((2,), act.slope))
