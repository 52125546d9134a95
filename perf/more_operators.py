"""Training of linear layers: the cases whose time is looked after, their plain forms
and their 64-bit definitions.

  linear  Z = A B + bias, C = act(Z) + R, and Z kept for the backward pass, in
          bfloat16 or as an 8-bit checkpoint (MXINT8: int8 codes with one power of two
          per 32 columns).  "c": weights output-major, as a linear layer holds them;
          "r": input-major.
  dgrad   D = (A B) * act'(Z), the gradient at the pre-activation of the layer before,
          with its column sums (that layer's bias gradient) in float32.
  dz      D = G * act'(Z) and its column sums where G is there already.
  ckpt    a matrix to an 8-bit checkpoint and back to values.
  wgrad   dW = act(Z)^T D with Z an 8-bit checkpoint: the activations are computed
          again from it (without act: it holds the layer's input itself).
"""
import math
import random

import torch

own = False

BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
DTYPES = {"bf16": BF16, "f32": F32}
ACTS = ("none", "relu", "leaky", "gelu", "gelu_tanh", "silu")
SLOPE = 0.125  # of "leaky"
CUBIC = 0.044715  # of "gelu_tanh"


def listed():
    return [
        # Decoding one token through a gated layer's projection: the weights' read is the
        # whole cost.
        dict(name="linear_token", op="linear", m=1, k=4096, n=14336, layout="c", act="silu",
             bias="", residual=False, z="", out="bf16"),
        # An output projection at prefill: bias, and the residual stream added.
        dict(name="linear_prefill", op="linear", m=4096, k=4096, n=4096, layout="c", act="none",
             bias="bf16", residual=True, z="", out="bf16"),
        # A training step's up projection, its pre-activation kept in 8 bits (and decoded,
        # so that its values come back).
        dict(name="linear_train", op="linear", m=8192, k=4096, n=8192, layout="c", act="gelu",
             bias="bf16", residual=False, z="mx", out="bf16"),
        # Nothing aligned, an f32 residual stream, the pre-activation in bfloat16.
        dict(name="linear_odd", op="linear", m=1001, k=1501, n=777, layout="r", act="gelu_tanh",
             bias="f32", residual=True, z="bf16", out="f32"),
        # The down projection's input gradient in that training step, through the
        # activation to the up projection's pre-activation, with its bias gradient.
        dict(name="dgrad_train", op="dgrad", m=8192, k=4096, n=8192, layout="r", act="gelu",
             z="mx", dbias=True, out="bf16"),
        # The same for a small layer with sizes of no alignment.
        dict(name="dgrad_odd", op="dgrad", m=333, k=1000, n=1501, layout="c", act="silu", z="bf16",
             dbias=True, out="f32"),
        # A layer's own activation gradient and bias gradient.
        dict(name="dz_layer", op="dz", m=8192, n=8192, act="gelu", z="mx", g="bf16", dbias=True),
        # An f32 gradient of a small batch.
        dict(name="dz_odd", op="dz", m=1003, n=777, act="leaky", z="bf16", g="f32", dbias=True),
        # A small batch's activations whose rows are no whole number of blocks.
        dict(name="ckpt_odd", op="ckpt", m=333, n=1000, dtype="bf16"),
        # A training batch's activations.
        dict(name="ckpt_layer", op="ckpt", m=16384, n=4096, dtype="bf16"),
        # A layer's weight gradient from its checkpointed input, kept in f32.
        dict(name="wgrad_layer", op="wgrad", m=8192, k=4096, n=8192, act="none", out="f32"),
        # A small layer's, the activations computed again.
        dict(name="wgrad_act", op="wgrad", m=1003, k=1024, n=704, act="gelu", out="bf16"),
    ]


_MOST_FLOPS = 2 * 8192 * 4096 * 8192
_MOST_VALUES = 8192 * 8192  # of one matrix


def _size(rng, lo, hi):
    """A size in [lo, hi], spread over its logarithm; a third of them odd ones."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    step = rng.choice((1, 8, 64))
    return max(lo, min(hi, (v + step // 2) // step * step if v >= step else v))


def draw(rng):
    op = rng.choice(("linear", "linear", "dgrad", "dz", "ckpt", "wgrad"))
    while True:
        m, k, n = _size(rng, 1, 16384), _size(rng, 64, 14336), _size(rng, 64, 14336)
        if max(m * n, m * k, k * n) > _MOST_VALUES or m * k * n * 2 > _MOST_FLOPS:
            continue
        act = rng.choice(ACTS)
        kept = rng.choice(("bf16", "mx")) if act != "none" else ""
        wide = rng.choice(("bf16", "f32"))
        if op == "linear":
            return dict(op=op, m=m, k=k, n=n, layout=rng.choice("cr"), act=act,
                        bias=rng.choice(("", "bf16", "f32")), residual=rng.random() < 0.5,
                        z=rng.choice(("", kept)), out=wide)
        if op == "dgrad":
            return dict(op=op, m=m, k=k, n=n, layout=rng.choice("cr"), act=act, z=kept,
                        dbias=rng.random() < 0.7, out=wide)
        if op == "dz":
            if act != "none":
                return dict(op=op, m=m, n=n, act=act, z=kept, g=wide, dbias=rng.random() < 0.7)
        elif op == "ckpt":
            return dict(op=op, m=m, n=n, dtype=wide)
        else:
            # (activations are rounded to bfloat16 before the product, so the output that
            # goes with them is a bfloat16 one)
            return dict(op=op, m=m, k=k, n=n, act=act, out="bf16" if act != "none" else wide)


# ------------------------------------------------------------------ inputs

def _normal(g, *shape, std=1.0, dtype=BF16):
    return torch.randn(*shape, generator=g, device="cuda").mul_(std).to(dtype)


def _spread(g, rows, cols, dtype):
    """Activations: normal, one channel in 64 twelve times larger, a block of zeros."""
    x = torch.randn(rows, cols, generator=g, device="cuda")
    x[:, ::64] *= 12.0
    x[rows // 2, :32] = 0.0
    return x.to(dtype)


def _values(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op, m, n = case["op"], case["m"], case["n"]
    v = {}
    if op == "ckpt":
        return dict(x=_spread(g, m, n, DTYPES[case["dtype"]]))
    if op == "wgrad":
        v["q"] = _quantized(_spread(g, m, case["k"], F32))
        v["b"] = _normal(g, m, n, std=0.05)
        return v
    if op == "dz":
        v["g"] = _normal(g, m, n, std=0.05, dtype=DTYPES[case["g"]])
    else:
        k = case["k"]
        std = 1.0 if op == "linear" else 0.05
        v["a"] = _normal(g, m, k, std=std)
        shape = (n, k) if case["layout"] == "c" else (k, n)
        v["b"] = _normal(g, *shape, std=1.0 / math.sqrt(k))
    if op == "linear":
        if case["bias"]:
            v["bias"] = _normal(g, n, std=0.5, dtype=DTYPES[case["bias"]])
        if case["residual"]:
            v["r"] = _normal(g, m, n, dtype=DTYPES[case["out"]])
    elif case["z"] == "mx":
        v["z"] = _quantized(_spread(g, m, n, F32))
    elif case["z"]:
        v["z"] = _spread(g, m, n, BF16)
    return v


def prepare(case, seed):
    s = dict(case=case, **_values(case, seed))
    op, m, n = case["op"], case["m"], case["n"]
    empty = lambda *shape, dtype: torch.empty(*shape, dtype=dtype, device="cuda")
    if op == "ckpt":
        s["out"] = empty(m, n, dtype=DTYPES[case["dtype"]])
    elif op == "wgrad":
        s["out"] = empty(case["k"], n, dtype=DTYPES[case["out"]])
    elif op == "dz":
        s["out"] = empty(m, n, dtype=BF16)
    else:
        s["out"] = empty(m, n, dtype=DTYPES[case["out"]])
    if op == "linear" and case["z"]:
        s["kept"] = empty(m, n, dtype=BF16)
    if op == "ckpt" or op == "linear" and case["z"] == "mx":
        s["codes"] = empty(m, _blocks(n) * 32, dtype=torch.int8)
        s["scales"] = empty(m, (_blocks(n) + 15) // 16 * 16, dtype=torch.uint8)
    if case.get("dbias"):
        s["dbias"] = empty(n, dtype=F32)
    return s


# ------------------------------------------------------------------ plain form

def _blocks(n):
    return (n + 31) // 32


def _power(e):
    """2^e in 32 bits, exactly, for whole -126 <= e <= 127."""
    return ((e + 127) << 23).to(torch.int32).view(F32)


def _quantized(x):
    """(codes, scales) of a matrix: per 32 elements of a row e = floor(log2 of the
    largest magnitude), at least -120, codes the nearest whole multiple of 2^(e - 6),
    ties to even, at most 127 either way; the scale byte is e + 127.  Rows of codes are
    whole blocks, rows of scales whole 16 bytes."""
    rows, n = x.shape
    nb = _blocks(n)
    pad = torch.zeros(rows, nb * 32, dtype=F32, device=x.device)
    pad[:, :n] = x
    v = pad.view(rows, nb, 32)
    top = v.abs().amax(dim=2)
    e = torch.where(top == 0, -120, (torch.frexp(top)[1] - 1).clamp(min=-120))
    codes = (v * _power(6 - e).unsqueeze(2)).round_().clamp_(-127, 127).to(torch.int8)
    scales = torch.zeros(rows, (nb + 15) // 16 * 16, dtype=torch.uint8, device=x.device)
    scales[:, :nb] = (e + 127).to(torch.uint8)
    return codes.view(rows, nb * 32), scales


def _decoded(codes, scales, n):
    """The values of (codes, scales) in 32 bits."""
    rows, nb = codes.shape[0], _blocks(n)
    step = _power(scales[:, :nb].to(torch.int32) - 133)
    return (codes.view(rows, nb, 32).float() * step.unsqueeze(2)).view(rows, nb * 32)[:, :n]


def _act(z, act):
    if act == "relu":
        return torch.where(z > 0, z, 0.0)
    if act == "leaky":
        return torch.where(z > 0, z, SLOPE * z)
    if act == "gelu":
        return z * (0.5 * (1 + torch.erf(z * math.sqrt(0.5))))
    if act == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + CUBIC * z * z * z)))
    if act == "silu":
        return z / (1 + torch.exp(-z))
    return z


def _act_grad(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "leaky":
        return torch.where(z > 0, 1.0, SLOPE)
    if act == "gelu":
        density = torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * density
    if act == "gelu_tanh":
        c = math.sqrt(2 / math.pi)
        t = torch.tanh(c * (z + CUBIC * z * z * z))
        return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * CUBIC * z * z)
    s = 1 / (1 + torch.exp(-z))
    return s + z * s * (1 - s)


def _weights(s):
    b = s["b"].float()
    return b.t() if s["case"]["layout"] == "c" else b


def _kept(s):
    """The pre-activations in 32 bits."""
    return _decoded(*s["z"], s["case"]["n"]) if s["case"]["z"] == "mx" else s["z"].float()


def run(s):
    if own:
        return _run_own(s)
    case = s["case"]
    op = case["op"]
    if op == "ckpt":
        s["codes"], s["scales"] = _quantized(s["x"])
        return s["out"].copy_(_decoded(s["codes"], s["scales"], case["n"]))
    if op == "wgrad":
        h = _act(_decoded(*s["q"], case["k"]), case["act"])
        return s["out"].copy_(h.t() @ s["b"].float())
    if op == "linear":
        z = s["a"].float() @ _weights(s)
        if "bias" in s:
            z += s["bias"].float()
        c = _act(z, case["act"])
        if "r" in s:
            c = c + s["r"].float()
        s["out"].copy_(c)
        if not case["z"]:
            return s["out"]
        if case["z"] == "mx":
            s["codes"], s["scales"] = _quantized(z)
            z = _decoded(s["codes"], s["scales"], case["n"])
        return s["out"], s["kept"].copy_(z)
    d = s["g"].float() if op == "dz" else s["a"].float() @ _weights(s)
    if case["act"] != "none":
        d = d * _act_grad(_kept(s), case["act"])
    s["out"].copy_(d)
    if not case["dbias"]:
        return s["out"]
    return s["out"], s["dbias"].copy_(d.sum(dim=0, dtype=F64))


# ------------------------------------------------------------------ framework's calls

def _framework():
    import gemmkit_amd as gk

    gk.set_synchronous(False)
    return gk


def _run_own(s):
    gk = _framework()
    case, out = s["case"], s["out"]
    op, m, n, k = case["op"], case["m"], case["n"], case.get("k")
    act = {"none": lambda: None, "relu": lambda: gk.Activation.Relu,
           "leaky": lambda: gk.Activation.LeakyRelu(SLOPE), "gelu": lambda: gk.Activation.Gelu,
           "gelu_tanh": lambda: gk.Activation.GeluTanh,
           "silu": lambda: gk.Activation.Silu}[case.get("act", "none")]()
    if op == "ckpt":
        q = gk.MatMxint8(s["codes"], s["scales"], m, n)
        gk.quantize_mxint8(gk.MatRef.from_row_major(s["x"], m, n), q)
        gk.dequantize_mxint8(q, gk.MatMut.from_row_major(out, m, n))
        return out
    if op == "wgrad":
        gk.gemm_wgrad_mxint8(1.0, gk.MatMxint8(*s["q"], m, k),
                             gk.MatRef.from_row_major(s["b"], m, n), 0.0,
                             gk.MatMut.from_row_major(out, k, n), act=act)
        return out
    c = gk.MatMut.from_row_major(out, m, n)
    if op != "dz":
        a = gk.MatRef.from_row_major(s["a"], m, k)
        b = gk.MatRef(s["b"], k, n, 1, k) if case["layout"] == "c" else \
            gk.MatRef.from_row_major(s["b"], k, n)
    if op == "linear":
        bias = gk.Bias.PerCol(s["bias"]) if "bias" in s else None
        r = gk.MatRef.from_row_major(s["r"], m, n) if "r" in s else None
        z = None
        if case["z"] == "mx":
            z = gk.MatMxint8(s["codes"], s["scales"], m, n)
        elif case["z"]:
            z = gk.MatMut.from_row_major(s["kept"], m, n)
        gk.gemm_linear(1.0, a, b, c, bias=bias, act=act, residual=r, z=z)
        if z is None:
            return out
        if case["z"] == "mx":
            gk.dequantize_mxint8(z, gk.MatMut.from_row_major(s["kept"], m, n))
        return out, s["kept"]
    z = None
    if case["z"] == "mx":
        z = gk.MatMxint8(*s["z"], m, n)
    elif case["z"]:
        z = gk.MatRef.from_row_major(s["z"], m, n)
    if op == "dgrad":
        gk.gemm_linear_dgrad(1.0, a, b, c, act=act, z=z, dbias=s.get("dbias"))
    else:
        gk.activation_grad(gk.MatRef.from_row_major(s["g"], m, n), c, act=act, z=z,
                           dbias=s.get("dbias"))
    return (out, s["dbias"]) if case["dbias"] else out


# ------------------------------------------------------------------ work

def work(case):
    op, m, n = case["op"], case["m"], case["n"]
    size = {"bf16": 2, "f32": 4, "": 0}
    if op == "ckpt":
        return {"bytes": 2 * m * n * size[case["dtype"]], "flops": 4 * m * n}
    kept = lambda cols: m * _blocks(cols) * 33  # bytes of a checkpoint
    if op == "wgrad":
        k = case["k"]
        return {"bytes": kept(k) + 2 * m * n + k * n * size[case["out"]], "flops": 2 * m * k * n}
    z = kept(n) if case["z"] == "mx" else m * n * size[case["z"]]
    if op == "dz":
        return {"bytes": z + m * n * (size[case["g"]] + 2) + 4 * n * case["dbias"],
                "flops": 8 * m * n}
    k = case["k"]
    bytes_ = 2 * k * (m + n) + m * n * size[case["out"]]
    if op == "linear":
        # (an 8-bit checkpoint is written, and its values come back in bfloat16)
        bytes_ += n * size[case["bias"]] + m * n * (size[case["out"]] if case["residual"] else 0)
        bytes_ += m * n * 2 if case["z"] else 0
        bytes_ += z if case["z"] == "mx" else 0
    else:
        bytes_ += z + 4 * n * case["dbias"]
    return {"bytes": bytes_, "flops": 2 * m * k * n}


# ------------------------------------------------------------------ definition in 64 bits

def _power64(e):
    return ((e.long() + 1023) << 52).view(F64)


def _code64(x):
    """The value that every element of x stands for in a checkpoint."""
    rows, n = x.shape
    out = torch.empty(rows, n, dtype=F64, device=x.device)
    for lo in range(0, n, 32 * 64):
        part = x[:, lo:lo + 32 * 64].double()
        wide = -(-part.shape[1] // 32) * 32
        full = torch.nn.functional.pad(part, (0, wide - part.shape[1])).reshape(rows, -1, 32)
        top = full.abs().max(dim=2, keepdim=True).values.clamp(min=2.0 ** -120)
        step = _power64((top.view(torch.int64) >> 52) - 1023 - 6)
        code = full / step
        low = torch.floor(code)
        # up above the middle, and on it where the lower neighbour is odd
        up = (code - low > 0.5) | ((code - low == 0.5) & (low % 2 != 0))
        value = torch.minimum(torch.maximum(low + up, -127 * torch.ones_like(low)),
                              127 * torch.ones_like(low)) * step
        out[:, lo:lo + 32 * 64] = value.reshape(rows, wide)[:, :part.shape[1]]
    return out


def _kept64(v, cols):
    """The values of a checkpoint by its format: code / 64 times 2^(scale - 127)."""
    codes, scales = v
    power = _power64(scales.int() - 127).repeat_interleave(32, dim=1)[:, :codes.shape[1]]
    return (codes.double() / 64 * power)[:, :cols]


def _act64(z, act):
    if act == "relu":
        return z.clamp(min=0)
    if act == "leaky":
        return z.clamp(min=0) + SLOPE * z.clamp(max=0)
    if act == "gelu":
        return z * torch.special.ndtr(z)
    if act == "gelu_tanh":
        return z * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + CUBIC * z ** 3))
    return z * torch.sigmoid(z) if act == "silu" else z


def _slope64(z, act):
    if act == "relu":
        return torch.heaviside(z, torch.zeros_like(z))
    if act == "leaky":
        return SLOPE + (1 - SLOPE) * torch.heaviside(z, torch.zeros_like(z))
    if act == "gelu":
        return torch.special.ndtr(z) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if act == "gelu_tanh":
        inner = 2 * math.sqrt(2 / math.pi)
        p = torch.sigmoid(inner * (z + CUBIC * z ** 3))
        return p * (1 + z * (1 - p) * inner * (1 + 3 * CUBIC * z ** 2))
    if act == "silu":
        p = torch.sigmoid(z)
        return p * (1 + z * (1 - p))
    return torch.ones_like(z)


def exact(case, seed):
    v = _values(case, seed)
    op, n = case["op"], case["n"]
    if op == "ckpt":
        return _code64(v["x"])
    if op == "wgrad":
        return _act64(_kept64(v["q"], case["k"]), case["act"]).t() @ v["b"].double()
    if op == "dz":
        d = v["g"].double()
    else:
        b = v["b"].double()
        d = v["a"].double() @ (b.t() if case["layout"] == "c" else b)
    if op == "linear":
        if "bias" in v:
            d += v["bias"].double()
        c = _act64(d, case["act"])
        if "r" in v:
            c = c + v["r"].double()
        if not case["z"]:
            return c
        return c, (_code64(d) if case["z"] == "mx" else d)
    if case["act"] != "none":
        d = d * _slope64(_kept64(v["z"], n) if case["z"] == "mx" else v["z"].double(), case["act"])
    return (d, d.sum(dim=0)) if case["dbias"] else d
