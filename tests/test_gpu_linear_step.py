"""The linear-layer operators as a training step and a server use them: one after the other,
captured and replayed, on several streams and threads, and with matrices whose offsets pass 32
bits.  Tolerances as in test_gpu_linear.py: K exact products added in f32 are off by K 2^-23 of
their magnitudes' sum, an activation or its derivative by 2^-20 max(|z|, 1), bf16 by 2^-8."""
import threading

import pytest
import torch

import gemmkit_amd as gk

pytestmark = pytest.mark.gpu

BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
E23, E20, E8 = 2.0 ** -23, 2.0 ** -20, 2.0 ** -8


def rand(seed, *shape, dt=BF16, std=1.0, dev="cuda"):
    g = torch.Generator(device=dev).manual_seed(seed)
    return (torch.randn(*shape, generator=g, device=dev) * std).to(dt)


def row(t):
    return gk.MatRef.from_row_major(t, *t.shape)


def out(t):
    return gk.MatMut.from_row_major(t, *t.shape)


def transposed(w):
    """The k x n view of a weight stored output-major (n x k)."""
    n, k = w.shape
    return gk.MatRef(w, k, n, 1, k)


def values8(q):
    """The values of a MatMxint8 in 64 bits."""
    nb = -(-q.cols // 32)
    c = q.codes.view(q.rows, -1)[:, :nb * 32].double()
    s = q.scales.view(q.rows, -1)[:, :nb].double()
    return (c * torch.pow(2.0, s - 133).round(decimals=160).repeat_interleave(32, 1))[:, :q.cols]


def gelu64(z):
    return z * torch.special.ndtr(z)


def gelu_slope64(z):
    return torch.special.ndtr(z) + z * torch.exp(-z * z / 2) * 0.3989422804014327


def near(got, want, tol, what):
    over = ((got.double() - want).abs() - tol).max().item()
    assert over <= 0, f"{what}: {over} more than its bound"


class Layer:
    """x -> h = gelu(x w^T + b) -> y = h v^T + c + x, weights output-major."""

    def __init__(self, rows, width, hidden, ws=None):
        self.ws = ws
        self.x = rand(1, rows, width)
        self.w, self.b = rand(2, hidden, width, std=width ** -0.5), rand(3, hidden, dt=F32)
        self.v, self.c = rand(4, width, hidden, std=hidden ** -0.5), rand(5, width)
        self.dy = rand(6, rows, width, std=0.1)
        e = lambda *s, dt=BF16: torch.empty(*s, dtype=dt, device="cuda")
        self.h, self.y = e(rows, hidden), e(rows, width)
        self.zq, self.xq = gk.MatMxint8.empty(rows, hidden), gk.MatMxint8.empty(rows, width)
        self.dz, self.dx = e(rows, hidden), e(rows, width)
        self.dw, self.dv = e(hidden, width, dt=F32), e(width, hidden, dt=F32)
        self.db, self.dc = e(hidden, dt=F32), e(width, dt=F32)

    def forward(self):
        gk.gemm_linear(1.0, row(self.x), transposed(self.w), out(self.h), bias=gk.Bias.PerCol(self.b),
                       act=gk.Activation.Gelu, z=self.zq, ws=self.ws)
        gk.quantize_mxint8(row(self.x), self.xq)
        gk.gemm_linear(1.0, row(self.h), transposed(self.v), out(self.y), bias=gk.Bias.PerCol(self.c),
                       residual=row(self.x), ws=self.ws)

    def backward(self):
        rows, width = self.x.shape
        hidden = self.w.shape[0]
        gelu = gk.Activation.Gelu
        # dv (width x hidden) is the transposed hidden x width gradient
        gk.gemm_wgrad_mxint8(1.0, self.zq, row(self.dy), 0.0,
                             gk.MatMut(self.dv, hidden, width, 1, hidden), act=gelu, ws=self.ws)
        gk.gemm_linear_dgrad(1.0, row(self.dy), row(self.v), out(self.dz), act=gelu, z=self.zq,
                             dbias=self.db, ws=self.ws)
        same = torch.empty_like(self.dy)
        gk.activation_grad(row(self.dy), out(same), dbias=self.dc, ws=self.ws)
        gk.gemm_wgrad_mxint8(1.0, self.xq, row(self.dz), 0.0,
                             gk.MatMut(self.dw, width, hidden, 1, width), ws=self.ws)
        gk.gemm_linear(1.0, row(self.dz), row(self.w), out(self.dx), residual=row(self.dy), ws=self.ws)

    def results(self):
        # (scales past a row's blocks do not count, and gemm_linear leaves them)
        return [self.h, self.y, self.zq.codes, self.zq.scales[:, :-(-self.h.shape[1] // 32)], self.dz,
                self.dx, self.dw, self.dv, self.db, self.dc]


@pytest.mark.parametrize("rows,width,hidden", [(1, 64, 96), (70, 100, 260), (700, 256, 1024),
                                               (1003, 333, 777)])
def test_training_step(dev, rows, width, hidden):
    """Each result against 64 bits, from the values that the step itself kept."""
    s = Layer(rows, width, hidden)
    s.forward()
    s.backward()
    x, w, v, dy, h, dz = (t.double() for t in (s.x, s.w, s.v, s.dy, s.h, s.dz))
    z = x @ w.t() + s.b.double()
    dz_ = (width + 2) * E23 * (x.abs() @ w.t().abs() + s.b.double().abs())
    near(s.h, gelu64(z), 1.13 * dz_ + E20 * z.abs().clamp(min=1) + E8 * gelu64(z).abs() * 1.01, "h")
    y = h @ v.t() + s.c.double() + x
    dy_ = (hidden + 4) * E23 * (h.abs() @ v.t().abs() + s.c.double().abs() + x.abs())
    near(s.y, y, dy_ + E8 * (y.abs() + dy_), "y")
    zk, xk = values8(s.zq), values8(s.xq)
    # (a step is 2^-6 of its block's largest power of two: half of one, a whole one at the top)
    top = torch.nn.functional.pad(z.abs() + dz_, (0, -hidden % 32)).view(rows, -1, 32).amax(2)
    step = (torch.pow(2.0, torch.floor(torch.log2(top)) - 6) * 1.0001).repeat_interleave(32, 1)[:, :hidden]
    near(zk, z, step + dz_, "z")
    hk = gelu64(zk)
    dh = E20 * zk.abs().clamp(min=1) + E8 * hk.abs() * 1.01
    want = dy.t() @ hk
    near(s.dv, want, dy.t().abs() @ (dh + (rows + 2) * E23 * (hk.abs() + dh)) + 2 * E23 * want.abs(), "dv")
    p, slope = dy @ v, gelu_slope64(zk)
    dp = (width + 2) * E23 * (dy.abs() @ v.abs())
    own = dp * slope.abs().clamp(min=1) + (p.abs() + dp) * E20 * zk.abs().clamp(min=1) + E23 * (p * slope).abs()
    near(s.dz, p * slope, own + E8 * ((p * slope).abs() + own), "dz")
    near(s.db, (p * slope).sum(0), own.sum(0) + (rows + 1) * E23 * ((p * slope).abs() + own).sum(0), "db")
    near(s.dc, dy.sum(0), (rows + 1) * E23 * dy.abs().sum(0), "dc")
    want = dz.t() @ xk
    near(s.dw, want, (rows + 2) * E23 * (dz.t().abs() @ xk.abs()), "dw")
    want = dz @ w + dy
    bound = (hidden + 3) * E23 * (dz.abs() @ w.abs() + dy.abs())
    near(s.dx, want, bound + E8 * (want.abs() + bound), "dx")


def test_gradients_follow_the_loss(dev):
    """The step's gradients against central differences of the loss sum(dy * y) in 64 bits, over
    directions in each parameter: what separates them is the 8-bit checkpoints (a step of 2^-6
    of a block's largest power of two moves gelu' by at most 1.2 of half of it) and bf16."""
    rows, width, hidden = 64, 96, 160
    s = Layer(rows, width, hidden)
    s.forward()
    s.backward()

    def loss(x, w, b, v, c):
        h = gelu64(x @ w.t() + b)
        return (s.dy.double() * (h @ v.t() + c + x)).sum()
    at = [t.double() for t in (s.x, s.w, s.b, s.v, s.c)]
    grads = [s.dx, s.dw, s.db, s.dv, s.dc]
    z = at[0] @ at[1].t() + at[2]
    # the largest a kept z can be off by, relative to a hidden unit's slope (about 1)
    top = z.abs().view(rows, -1, 32).amax(2).max().item()
    off = 1.2 * 2.0 ** -7 * top + 3 * E8
    for i, g in enumerate(grads):
        for trial in range(3):
            d = rand(50 + 10 * i + trial, *at[i].shape, dt=F64)
            e = 1e-5
            up = [t + e * d if j == i else t for j, t in enumerate(at)]
            down = [t - e * d if j == i else t for j, t in enumerate(at)]
            want = (loss(*up) - loss(*down)) / (2 * e)
            got = (g.double() * d).sum()
            # (independent errors over the direction's terms)
            assert (got - want).abs() <= 4 * off * (g.double() * d).norm(), (i, got.item(), want.item())


def test_same_bits_every_time(dev):
    s = Layer(1003, 333, 777)
    s.forward()
    s.backward()
    first = [t.clone() for t in s.results()]
    for _ in range(3):
        for t in s.results():
            t.fill_(3)
        s.forward()
        s.backward()
        for a, b in zip(s.results(), first):
            assert torch.equal(a, b)


@pytest.mark.parametrize("rows,width,hidden", [(16, 256, 512), (333, 100, 260), (1003, 333, 777)])
def test_step_captured_and_replayed(dev, rows, width, hidden):
    """Replays with eager work and synchronizations between them, each against the eager bits."""
    ws = gk.Workspace.with_capacity(64 << 20)
    gk.set_synchronous(False)
    try:
        s = Layer(rows, width, hidden, ws)
        s.forward()
        s.backward()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            s.forward()
            s.backward()
        for i in range(4):
            s.x.copy_(rand(100 + i, rows, width))
            s.forward()
            s.backward()
            torch.cuda.synchronize()
            want = [t.clone() for t in s.results()]
            for t in s.results():
                t.fill_(1)
            graph.replay()
            torch.cuda.synchronize()
            for a, b in zip(s.results(), want):
                assert torch.equal(a, b), i
    finally:
        gk.set_synchronous(True)


def test_capture_needs_a_sized_workspace(dev):
    """Partial column sums, packed operands and decoded checkpoints under capture."""
    m, k, n = 2000, 64, 128
    a, b, d = rand(1, m, k), rand(2, k, n), torch.empty(m, n, dtype=BF16, device=dev)
    db = torch.empty(n, device=dev)
    q = gk.quantize_mxint8(row(a))
    c = torch.empty(k, n, device=dev)
    calls = [lambda ws: gk.gemm_linear_dgrad(1.0, row(a), row(b), out(d), dbias=db, ws=ws),
             lambda ws: gk.activation_grad(row(d), out(d), dbias=db, ws=ws),
             lambda ws: gk.gemm_wgrad_mxint8(1.0, q, row(d), 0.0, out(c), ws=ws),
             lambda ws: gk.gemm_linear(1.0, gk.MatRef(a, k, m, 1, k), gk.MatRef(d, m, n, n, 1),
                                       gk.MatMut(torch.empty(k, n, dtype=BF16, device=dev), k, n, n, 1),
                                       ws=ws)]
    gk.set_synchronous(False)
    try:
        for call in calls:
            call(None)
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with pytest.raises(gk.GemmkitError, match="HIP graph capture"):
                with torch.cuda.graph(graph):
                    call(gk.Workspace())
            torch.cuda.synchronize()
    finally:
        gk.set_synchronous(True)


def test_two_graphs_on_one_workspace(dev):
    """Graphs of different sizes that share a workspace, replayed in turn."""
    ws = gk.Workspace.with_capacity(64 << 20)
    gk.set_synchronous(False)
    try:
        steps, graphs, want = [], [], []
        for rows, width, hidden in ((300, 100, 260), (1003, 333, 777)):
            s = Layer(rows, width, hidden, ws)
            s.forward()
            s.backward()
            torch.cuda.synchronize()
            want.append([t.clone() for t in s.results()])
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                s.forward()
                s.backward()
            steps.append(s)
            graphs.append(g)
        for i in (0, 1, 1, 0, 1):
            for t in steps[i].results():
                t.fill_(1)
            graphs[i].replay()
            torch.cuda.synchronize()
            for a, b in zip(steps[i].results(), want[i]):
                assert torch.equal(a, b)
    finally:
        gk.set_synchronous(True)


def test_streams_share_the_default_workspace(dev):
    gk.set_synchronous(False)
    try:
        a, b = Layer(1003, 333, 777), Layer(700, 200, 520)
        want = []
        for s in (a, b):
            s.forward()
            s.backward()
            torch.cuda.synchronize()
            want.append([t.clone() for t in s.results()])
            for t in s.results():
                t.fill_(1)
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        for _ in range(5):
            for s, st in zip((a, b), streams):
                with torch.cuda.stream(st):
                    s.forward()
                    s.backward()
        torch.cuda.synchronize()
        for s, w in zip((a, b), want):
            for x, y in zip(s.results(), w):
                assert torch.equal(x, y)
    finally:
        gk.set_synchronous(True)


def test_threads(dev):
    steps = [Layer(300 + 50 * i, 130, 260) for i in range(3)]
    for s in steps:
        s.forward()
        s.backward()
    want = [[t.clone() for t in s.results()] for s in steps]
    failed = []

    def work(s, w):
        try:
            for _ in range(5):
                s.forward()
                s.backward()
                for x, y in zip(s.results(), w):
                    assert torch.equal(x, y)
        except BaseException as e:  # noqa: BLE001 -- reported by the test's own thread
            failed.append(e)
    threads = [threading.Thread(target=work, args=p) for p in zip(steps, want)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed[0]


def test_host_tensors_are_refused(dev):
    a, b, c = torch.zeros(4, 4, dtype=BF16), rand(1, 4, 4), rand(2, 4, 4)
    with pytest.raises(gk.GemmkitError):
        gk.gemm_linear(1.0, row(a), row(b), out(c))
    with pytest.raises(gk.GemmkitError):
        gk.activation_grad(row(b), out(a))
    with pytest.raises(gk.GemmkitError):
        gk.quantize_mxint8(row(a), gk.MatMxint8.empty(4, 4))
    with pytest.raises(TypeError):
        gk.gemm_linear(1.0, row(b), row(b), out(c), z=row(b))  # an output view is needed
    with pytest.raises(TypeError):
        gk.gemm_linear_dgrad(1.0, row(b), row(b), out(c), dbias=rand(3, 4))


def test_offsets_past_32_bits(dev):
    """Outputs, pre-activations and checkpoints of more than 2^32 elements."""
    m, k, n = 70016, 32, 65600
    x, w = rand(1, m, k), rand(2, k, n, std=k ** -0.5)
    c = torch.empty(m, n, dtype=BF16, device=dev)
    q = gk.MatMxint8.empty(m, n)
    gk.gemm_linear(1.0, row(x), row(w), out(c), act=gk.Activation.Gelu, z=q)
    rows = torch.tensor([0, 1, 32751, 65471, 65472, m - 129, m - 1], device=dev)
    z = x[rows].double() @ w.double()
    dz = (k + 2) * E23 * (x[rows].double().abs() @ w.double().abs())
    near(c[rows], gelu64(z), 1.13 * dz + E20 * z.abs().clamp(min=1) + 1.01 * E8 * gelu64(z).abs(), "c")
    kept = gk.MatMxint8(q.codes[rows].contiguous(), q.scales[rows].contiguous(), len(rows), n)
    zk = values8(kept)
    assert (zk - z).abs().max() <= 2.0 ** -6 * 2 * z.abs().max()
    # quantization of what c holds, and back
    gk.quantize_mxint8(row(c), q)
    part = gk.quantize_mxint8(row(c[rows].contiguous()))
    assert torch.equal(q.codes[rows], part.codes) and torch.equal(q.scales[rows], part.scales)
    gk.dequantize_mxint8(q, out(c))
    got = torch.empty(len(rows), n, dtype=BF16, device=dev)
    gk.dequantize_mxint8(part, out(got))
    assert torch.equal(c[rows], got)
    # the gradient through q, in place, and its column sums
    db = torch.empty(n, device=dev)
    d = c
    gk.gemm_linear_dgrad(1.0, row(x), row(w), out(d), act=gk.Activation.Gelu, z=q, dbias=db)
    slope = gelu_slope64(values8(part))
    bound = dz * slope.abs().clamp(min=1) + (z.abs() + dz) * 2 * E20 * 4
    near(d[rows], z * slope, bound + 1.01 * E8 * (z * slope).abs(), "d")
    cols = torch.tensor([0, 33, 32800, n - 1], device=dev)
    zc = x.double() @ w[:, cols].double()
    codes, scales = q.codes[:, cols].double(), q.scales[:, cols // 32].double()
    terms = zc * gelu_slope64(codes * torch.pow(2.0, scales - 133))
    near(db[cols], terms.sum(0), terms.abs().sum(0) * ((m + 2) * E23 + 4 * E20) + m * 4 * E20, "db")
    gk.activation_grad(row(d), out(d), act=gk.Activation.Relu, z=q)
    assert (d[rows].float()[values8(part) <= 0] == 0).all()
    # the weight gradient from q (decoded: 9 GB)
    b = rand(5, m, 8)
    g = torch.empty(n, 8, device=dev)
    gk.gemm_wgrad_mxint8(1.0, q, row(b), 0.0, out(g))
    want = (codes * torch.pow(2.0, scales - 133)).t() @ b.double()
    mags = (codes * torch.pow(2.0, scales - 133)).t().abs() @ b.double().abs()
    near(g[cols], want, (m + 2) * E23 * mags, "g")


def test_column_sums_of_more_than_2_28_columns(dev):
    """Their launch has more threads than 32 bits count: of no rows, and of two tiles' partial sums
    (whole numbers, exact)."""
    n, m, k = 2 ** 28 + 40, 129, 8
    db = torch.full((n,), float("nan"), device=dev)
    none = torch.empty(0, dtype=BF16, device=dev)
    gk.gemm_linear_dgrad(1.0, gk.MatRef(none, 0, 0, 0, 1), gk.MatRef(none, 0, n, n, 1),
                         gk.MatMut(none, 0, n, n, 1), dbias=db)
    assert not db.any()  # (a NaN counts as true)
    w = torch.randint(-8, 9, (n, k), dtype=torch.int8, device=dev).to(BF16)
    d = torch.empty(m, n, dtype=BF16, device=dev)
    gk.gemm_linear_dgrad(1.0, row(torch.ones(m, k, dtype=BF16, device=dev)), transposed(w), out(d), dbias=db)
    want = w.sum(1, dtype=F32)
    assert torch.equal(db, want * m)
    for r in (0, 64, 128):
        assert torch.equal(d[r], want.to(BF16))
