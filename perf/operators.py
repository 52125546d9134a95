"""Products of routed expert layers and of 4-bit block-scaled layers: the cases
whose time is looked after, their plain forms and their 64-bit definitions.

  grouped   C[rows of group g] = A[rows of group g] B_g, ragged groups whose
            offsets lie on the device; "c": weights output-major, as a linear layer
            holds them (the forward product), "r": input-major (the same weights in
            the gradient of the layer's input).
  wgrad     dB_g = A[rows of group g]^T D[rows of group g]: the weights' gradient.
  quant     quantization to e2m1 codes with one e8m0 scale per 32 elements and back
            to values (calibration and quantization-aware training use the pair).
  mx        C = A B^T on such operands; "gmx": the same per group.
"""
import math
import random

import torch

own = False

BF16, F32 = torch.bfloat16, torch.float32
DTYPES = {"bf16": BF16, "f32": F32}
# magnitudes of the e2m1 codes 0..7
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def listed():
    return [
        # Decoding one token: eight of 64 experts see one row each; latency and
        # the chosen experts' weights are the whole cost.
        dict(name="grouped_token", op="grouped", rows=8, groups=64, k=2048, n=1024, layout="c",
             out="bf16", behind=0),
        # A prefill or training step through eight experts, tokens spread unevenly.
        dict(name="grouped_prefill", op="grouped", rows=16384, groups=8, k=4096, n=4096,
             layout="c", out="bf16", behind=0),
        # The gradient of the layer's input: the same output-major weights read as
        # an input-major matrix, with a padded batch behind the last group.
        dict(name="grouped_dgrad", op="grouped", rows=8192, groups=16, k=4096, n=2048, layout="r",
             out="bf16", behind=128),
        # Data-dependent sizes, nothing aligned, f32 sums kept.
        dict(name="grouped_odd", op="grouped", rows=1001, groups=5, k=1501, n=777, layout="r",
             out="f32", behind=0),
        # The weights' gradient of the prefill case's layer, kept in f32.
        dict(name="wgrad_layer", op="wgrad", rows=16384, groups=8, k=4096, n=4096, out="f32",
             behind=0),
        # Many small experts, few rows each, some of them none; a padded batch.
        dict(name="wgrad_small", op="wgrad", rows=1003, groups=32, k=1024, n=704, out="bf16",
             behind=21),
        # The activations of a small batch whose rows are no whole number of blocks.
        dict(name="quant_odd", op="quant", rows=333, k=1000, dtype="bf16"),
        # A layer's weight quantized from its f32 master copy.
        dict(name="quant_weight", op="quant", rows=14336, k=4096, dtype="f32"),
        # Eight sequences decoding through a 4-bit projection.
        dict(name="mx_decode", op="mx", m=8, k=4096, n=14336, out="bf16"),
        # A 4-bit linear layer at prefill.
        dict(name="mx_prefill", op="mx", m=4096, k=4096, n=4096, out="bf16"),
        # A decode batch through 32 4-bit experts, about two rows each.
        dict(name="gmx_decode", op="gmx", rows=64, groups=32, k=2048, n=4096, out="bf16",
             behind=0),
        # A prefill through eight 4-bit experts.
        dict(name="gmx_prefill", op="gmx", rows=16384, groups=8, k=4096, n=4096, out="bf16",
             behind=0),
    ]


_MOST_FLOPS = 2 * 16384 * 4096 * 4096
_MOST_BYTES = 6 << 30  # of all operands in memory, every group's weights among them


def _size(rng, lo, hi):
    """A size in [lo, hi], spread over its logarithm; a third of them odd ones."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    step = rng.choice((1, 8, 64))
    return max(lo, min(hi, (v + step // 2) // step * step if v >= step else v))


def draw(rng):
    op = rng.choice(("grouped", "grouped", "wgrad", "quant", "mx", "gmx"))
    while True:
        k, n = _size(rng, 128, 8192), _size(rng, 128, 8192)
        if op == "quant":
            case = dict(op=op, rows=_size(rng, 1, 16384), k=k, dtype=rng.choice(("bf16", "f32")))
            if case["rows"] * k <= 14336 * 4096:
                return case
            continue
        if op == "mx":
            case = dict(op=op, m=_size(rng, 1, 8192), k=k, n=n, out=rng.choice(("bf16", "f32")))
            if 2 * case["m"] * k * n <= 2 * 4096 ** 3:
                return case
            continue
        rows, groups = _size(rng, 1, 16384), _size(rng, 1, 128)
        case = dict(op=op, rows=rows, groups=groups, k=k, n=n, out=rng.choice(("bf16", "f32")),
                    behind=rng.choice((0, 0, rng.randint(1, 64))))
        if op == "grouped":
            case["layout"] = rng.choice(("c", "r"))
        held = groups * k * n * 4 + rows * (k + n) * 4
        if 2 * rows * k * n <= _MOST_FLOPS and held <= _MOST_BYTES:
            return case


# ------------------------------------------------------------------ inputs

def _group_sizes(case):
    """How many rows the groups get: every row picks its group with chances spread
    over about a factor of ten."""
    rng = random.Random(f"{case['rows']} {case['groups']} {case['k']} {case['n']}")
    chance = [math.exp(0.6 * rng.gauss(0, 1)) for _ in range(case["groups"])]
    sizes = [0] * case["groups"]
    for g in rng.choices(range(case["groups"]), chance, k=case["rows"]):
        sizes[g] += 1
    return sizes


def _bounds(case, seed):
    """(first row, row behind the last) of every group; the seed decides which
    group gets which size."""
    sizes = _group_sizes(case)
    random.Random(seed).shuffle(sizes)
    bounds, at = [], 0
    for s in sizes:
        bounds.append((at, at + s))
        at += s
    return bounds


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(g, *shape, std=1.0, dtype=BF16):
    return torch.randn(*shape, generator=g, device="cuda").mul_(std).to(dtype)


def _activations(g, rows, k, dtype):
    """Activations: normal, one channel in 64 twenty times larger, a block of zeros."""
    x = torch.randn(rows, k, generator=g, device="cuda")
    x[:, ::64] *= 20.0
    x[rows // 2, :32] = 0.0
    return x.to(dtype)


def _dims(case):
    if case["op"] in ("mx",):
        return case["m"], case["n"]
    return case["rows"] + case["behind"], case["groups"] * case["n"]


def _values(case, seed):
    g = _generator(seed)
    op, k = case["op"], case["k"]
    if op == "quant":
        return dict(x=_activations(g, case["rows"], k, DTYPES[case["dtype"]]))
    rows = _dims(case)[0]
    n = case["n"]
    if op == "wgrad":
        return dict(a=_normal(g, rows, k), b=_normal(g, rows, n))
    if op == "grouped":
        shape = (case["groups"], n, k) if case["layout"] == "c" else (case["groups"], k, n)
        return dict(a=_normal(g, rows, k), b=_normal(g, *shape, std=1.0 / math.sqrt(k)))
    a = _quantized(_activations(g, rows, k, F32))
    weight = [_quantized(_normal(g, n, k, std=1.0 / math.sqrt(k), dtype=F32))
              for _ in range(case.get("groups", 1))]
    return dict(a=a, b=tuple(torch.cat(part) for part in zip(*weight)))


def prepare(case, seed):
    s = dict(case=case, **_values(case, seed))
    op = case["op"]
    if op in ("grouped", "wgrad", "gmx"):
        s["bounds"] = _bounds(case, seed)
        ends = [0] + [e for _, e in s["bounds"]]
        s["offsets"] = torch.tensor(ends, dtype=torch.int32, device="cuda")
    if op == "quant":
        s["out"] = torch.zeros(case["rows"], case["k"], dtype=DTYPES[case["dtype"]], device="cuda")
    elif op == "wgrad":
        s["out"] = torch.zeros(case["groups"], case["k"], case["n"], dtype=DTYPES[case["out"]],
                               device="cuda")
    else:
        s["out"] = torch.zeros(_dims(case)[0], case["n"], dtype=DTYPES[case["out"]], device="cuda")
    if own:
        _prepare_own(s)
    return s


# ------------------------------------------------------------------ plain form

def _blocks(k):
    return (k + 31) // 32


def _quantized(x):
    """(codes, scales) of a float matrix: per 32 elements of a row e = floor(log2
    of the largest magnitude) - 2 and the nearest e2m1 value of x / 2^e, ties to the
    even code.  Two codes a byte, the lower nibble first; rows of scales padded to
    16 bytes."""
    rows, k = x.shape
    nb = _blocks(k)
    pad = torch.zeros(rows, nb * 32, dtype=F32, device=x.device)
    pad[:, :k] = x
    v = pad.view(rows, nb, 32)
    top = v.abs().amax(dim=2)
    e = torch.frexp(top.double())[1] - 3  # 2^(frexp - 1) <= top
    e = torch.where(top == 0, torch.full_like(e, -127), e.clamp(min=-127))
    m = torch.ldexp(v.abs().double(), -e.unsqueeze(2)).float()
    step = torch.where(m < 2, 0.5, torch.where(m < 4, 1.0, 2.0))
    m = (torch.round(m / step) * step).clamp_(max=6.0)
    code = torch.bucketize(m, torch.tensor(E2M1, device=x.device)).to(torch.uint8)
    code += torch.signbit(v).to(torch.uint8) * 8
    code = code.view(rows, nb * 16, 2)
    scales = torch.zeros(rows, (nb + 15) // 16 * 16, dtype=torch.uint8, device=x.device)
    scales[:, :nb] = (e + 127).to(torch.uint8)
    return code[:, :, 0] + code[:, :, 1] * 16, scales


def _decoded(codes, scales, k):
    """The values of (codes, scales) in 32 bits."""
    rows, nb = codes.shape[0], _blocks(k)
    code = torch.stack((codes & 15, codes >> 4), dim=2).view(rows, nb, 32).long()
    table = torch.tensor(E2M1 + tuple(-v for v in E2M1), device=codes.device)
    e = scales[:, :nb].to(torch.int32) - 127
    return torch.ldexp(table[code], e.unsqueeze(2)).view(rows, nb * 32)[:, :k]


def _weights(s, g):
    """The k x n matrix of group g in 32 bits."""
    b = s["b"][g].float()
    return b.t() if s["case"]["layout"] == "c" else b


def run(s):
    if own:
        return _run_own(s)
    case, out = s["case"], s["out"]
    op = case["op"]
    if op == "grouped":
        for g, (lo, hi) in enumerate(s["bounds"]):
            if hi > lo:
                out[lo:hi] = (s["a"][lo:hi].float() @ _weights(s, g)).to(out.dtype)
    elif op == "wgrad":
        for g, (lo, hi) in enumerate(s["bounds"]):
            out[g] = (s["a"][lo:hi].float().t() @ s["b"][lo:hi].float()).to(out.dtype)
    elif op == "quant":
        out.copy_(_decoded(*_quantized(s["x"]), case["k"]).to(out.dtype))
    elif op == "mx":
        out.copy_((_decoded(*s["a"], case["k"]) @ _decoded(*s["b"], case["k"]).t()).to(out.dtype))
    else:
        n, k = case["n"], case["k"]
        a = _decoded(*s["a"], k)
        for g, (lo, hi) in enumerate(s["bounds"]):
            if hi > lo:
                b = _decoded(*(part[g * n:(g + 1) * n] for part in s["b"]), k)
                out[lo:hi] = (a[lo:hi] @ b.t()).to(out.dtype)
    return out


# ------------------------------------------------------------------ framework's calls

def _prepare_own(s):
    import gemmkit_amd as gk

    gk.set_synchronous(False)
    case, out = s["case"], s["out"]
    op, k, n = case["op"], case["k"], case.get("n")
    rows = case["rows"] if op == "quant" else _dims(case)[0]
    if op == "quant":
        s["view"] = gk.MatRef.from_row_major(s["x"], rows, k)
        s["c"] = gk.MatMut.from_row_major(out, rows, k)
        s["q"] = gk.MatMxfp4.empty(rows, k, device="cuda")
        return
    s["c"] = (gk.MatMut.from_row_major(out, k, n) if op == "wgrad"
              else gk.MatMut.from_row_major(out, rows, n))
    if op in ("mx", "gmx"):
        s["va"] = gk.MatMxfp4(*s["a"], rows, k)
        s["vb"] = gk.MatMxfp4(*s["b"], s["b"][0].shape[0], k)
        return
    s["va"] = gk.MatRef.from_row_major(s["a"], rows, k)
    if op == "wgrad":
        s["vb"] = gk.MatRef.from_row_major(s["b"], rows, n)
    elif case["layout"] == "c":
        s["vb"] = gk.MatRef(s["b"], k, n, 1, k)
    else:
        s["vb"] = gk.MatRef.from_row_major(s["b"], k, n)


def _run_own(s):
    import gemmkit_amd as gk

    case = s["case"]
    op = case["op"]
    if op == "grouped":
        gk.gemm_grouped(1.0, s["va"], s["offsets"], s["vb"], case["k"] * case["n"], 0.0, s["c"])
    elif op == "wgrad":
        gk.gemm_grouped_wgrad(1.0, s["va"], s["offsets"], s["vb"], 0.0, s["c"],
                              case["k"] * case["n"])
    elif op == "quant":
        gk.quantize_mxfp4(s["view"], s["q"])
        gk.dequantize_mxfp4(s["q"], s["c"])
    elif op == "mx":
        gk.gemm_mxfp4(1.0, s["va"], s["vb"], 0.0, s["c"])
    else:
        gk.gemm_grouped_mxfp4(1.0, s["va"], s["offsets"], s["vb"], 0.0, s["c"])
    return s["out"]


# ------------------------------------------------------------------ work

def work(case):
    op, k = case["op"], case["k"]
    if op == "quant":
        size = 2 if case["dtype"] == "bf16" else 4
        return {"bytes": 2 * case["rows"] * k * size, "flops": 4 * case["rows"] * k}
    n, size = case["n"], 2 if case["out"] == "bf16" else 4
    held = _blocks(k) * 17  # bytes of a quantized row
    if op == "mx":
        m = case["m"]
        return {"bytes": (m + n) * held + m * n * size, "flops": 2 * m * n * k}
    rows, groups = case["rows"], case["groups"]
    busy = sum(1 for s in _group_sizes(case) if s)
    flops = 2 * rows * n * k
    offsets = 4 * (groups + 1)
    if op == "grouped":
        return {"bytes": 2 * rows * k + 2 * busy * k * n + rows * n * size + offsets, "flops": flops}
    if op == "wgrad":
        return {"bytes": 2 * rows * (k + n) + groups * k * n * size + offsets, "flops": flops}
    return {"bytes": (rows + busy * n) * held + rows * n * size + offsets, "flops": flops}


# ------------------------------------------------------------------ definition in 64 bits

def _decode64(codes, scales, k):
    """The values of (codes, scales) from the format's definition: sign, two bits of
    exponent with bias 1, one bit of mantissa, times 2^(scale - 127)."""
    nibbles = torch.empty(codes.shape[0], codes.shape[1] * 2, dtype=torch.uint8,
                          device=codes.device)
    nibbles[:, 0::2] = codes.bitwise_and(0x0F)
    nibbles[:, 1::2] = codes.bitwise_right_shift(4)
    nibbles = nibbles[:, :k]
    sign = 1.0 - 2.0 * (nibbles >= 8).double()
    exponent = (nibbles % 8 // 2).double()
    mantissa = (nibbles % 2).double()
    small = mantissa * 0.5
    value = torch.where(exponent == 0, small, (1 + mantissa / 2) * torch.pow(2.0, exponent - 1))
    block = torch.arange(k, device=codes.device) // 32
    return sign * value * torch.pow(2.0, scales.double()[:, block] - 127)


def _quantize64(x):
    """The value that every element is quantized to, by comparing with the midpoints
    of the format's values."""
    rows, k = x.shape
    out = torch.empty(rows, k, dtype=torch.float64, device=x.device)
    for lo in range(0, k, 32):
        part = x[:, lo:lo + 32].double()
        top = part.abs().max(dim=1, keepdim=True).values
        scale = torch.pow(2.0, torch.floor(torch.log2(top.clamp(min=2.0 ** -125))) - 2)
        m = part.abs() / scale
        value = torch.zeros_like(m)
        # above a midpoint, or on one whose upper neighbour has the even code
        for code in range(1, 8):
            mid = (E2M1[code - 1] + E2M1[code]) / 2
            over = m >= mid if code % 2 == 0 else m > mid
            value = torch.where(over, torch.full_like(m, E2M1[code]), value)
        out[:, lo:lo + 32] = torch.copysign(value * scale, part)
    return out


def exact(case, seed):
    v = _values(case, seed)
    op, k = case["op"], case["k"]
    if op == "quant":
        return _quantize64(v["x"])
    n = case["n"]
    if op == "mx":
        return _decode64(*v["a"], k) @ _decode64(*v["b"], k).t()
    bounds = _bounds(case, seed)
    if op == "wgrad":
        return torch.stack([v["a"][lo:hi].double().t() @ v["b"][lo:hi].double()
                            for lo, hi in bounds])
    out = torch.zeros(_dims(case)[0], n, dtype=torch.float64, device="cuda")
    for g, (lo, hi) in enumerate(bounds):
        if op == "grouped":
            b = v["b"][g].double()
            out[lo:hi] = v["a"][lo:hi].double() @ (b.t() if case["layout"] == "c" else b)
        else:
            b = _decode64(*(part[g * n:(g + 1) * n] for part in v["b"]), k)
            out[lo:hi] = _decode64(*(part[lo:hi] for part in v["a"]), k) @ b.t()
    return out
