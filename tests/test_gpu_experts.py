"""The grouped and MXFP4 operators as a routed layer uses them: one after the other in a
training step and in a serving step, captured and replayed, on several streams and threads,
and with matrices whose offsets pass 32 bits."""
import threading

import pytest
import torch

import gemmkit_amd as gk

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


def rand(seed, *shape, dt=BF16, dev="cuda", std=1.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    return (torch.randn(*shape, generator=g, device=dev) * std).to(dt)


def offsets_of(sizes, dev="cuda"):
    return torch.tensor([0] + list(torch.tensor(sizes).cumsum(0)), dtype=torch.int32, device=dev)


def forward(x, off, w, out):
    """x (rows x k), w (groups x n x k) -> out (rows x n)."""
    groups, n, k = w.shape
    rows = x.shape[0]
    gk.gemm_grouped(1.0, gk.MatRef.from_row_major(x, rows, k), off, gk.MatRef(w, k, n, 1, k), n * k,
                    0.0, gk.MatMut.from_row_major(out, rows, n))
    return out


def backward(x, off, w, dy, dx, dw):
    groups, n, k = w.shape
    rows = x.shape[0]
    gk.gemm_grouped(1.0, gk.MatRef.from_row_major(dy, rows, n), off, gk.MatRef(w, n, k, k, 1), n * k,
                    0.0, gk.MatMut.from_row_major(dx, rows, k))
    # dw has w's layout: the k x n gradient with its strides swapped
    gk.gemm_grouped_wgrad(1.0, gk.MatRef.from_row_major(x, rows, k), off,
                          gk.MatRef.from_row_major(dy, rows, n), 0.0, gk.MatMut(dw, k, n, 1, k),
                          n * k)


SIZES = [[40, 0, 7, 130, 1], [300, 290, 0, 600], [3, 2, 0, 1]]


@pytest.mark.parametrize("sizes", SIZES)
@pytest.mark.parametrize("k,n", [(96, 136), (200, 72)])
def test_training_step(dev, sizes, k, n):
    """Output and gradients against autograd in 64 bits on the same (bf16) values.

    The output's gradient is an input of its own, so each result is one product: a sum of at
    most `terms` exact products, each addition off by 2^-23 of the sum of magnitudes, and
    bf16's half step of 2^-8."""
    rows, groups = sum(sizes), len(sizes)
    off = offsets_of(sizes)
    x, w = rand(1, rows, k), rand(2, groups, n, k, std=k ** -0.5)
    dy = rand(3, rows, n)
    y = forward(x, off, w, torch.zeros(rows, n, dtype=BF16, device=dev))
    dx = torch.zeros_like(x)
    dw = torch.full(w.shape, float("nan"), device=dev, dtype=F32)
    backward(x, off, w, dy, dx, dw)
    xr, wr = x.cpu().double().requires_grad_(), w.cpu().double().requires_grad_()
    parts, at = [], 0
    for g, s in enumerate(sizes):
        parts.append(xr[at:at + s] @ wr[g].t())
        at += s
    yr = torch.cat(parts)
    yr.backward(dy.cpu().double())

    def close(got, want, terms, mags, half):
        tol = terms * 2.0 ** -23 * mags + half * want.abs() * 1.001 + 1e-30
        assert ((got.cpu().double() - want).abs() <= tol + half * tol).all()

    xa, wa, da = xr.detach().abs(), wr.detach().abs(), dy.cpu().double().abs()
    at = 0
    for g, s in enumerate(sizes):
        r = slice(at, at + s)
        at += s
        close(y[r], yr.detach()[r], k, xa[r] @ wa[g].t(), 2.0 ** -8)
        close(dx[r], xr.grad[r], n, da[r] @ wa[g], 2.0 ** -8)
        close(dw[g], wr.grad[g], max(s, 1), da[r].t() @ xa[r], 2.0 ** -24)


def test_gradients_against_differences(dev):
    """d(sum(y * dy)) along a direction, by central differences in the weights and the input
    (f32 output; bf16 steps of exactly 2^-3 on values that hold them exactly)."""
    sizes, k, n = [20, 0, 45], 64, 48
    rows, groups, off = sum(sizes), 3, offsets_of(sizes)
    g = torch.Generator(device="cuda").manual_seed(4)

    def small_ints(*shape):  # multiples of 1/4 up to 2: products and sums are exact
        return (torch.randint(-8, 9, shape, generator=g, device=dev).float() / 4).to(BF16)

    x, w, dy = small_ints(rows, k), small_ints(groups, n, k), small_ints(rows, n)
    ux, uw = small_ints(rows, k), small_ints(groups, n, k)
    h = 0.125

    def loss(xv, wv):
        y = forward(xv, off, wv, torch.zeros(rows, n, device=dev))
        return (y.double() * dy.double()).sum()

    dx, dw = torch.zeros(rows, k, device=dev), torch.zeros(groups, n, k, device=dev)
    backward(x, off, w, dy, dx, dw)
    for ex, ew, got in ((ux, None, (dx.double() * ux.double()).sum()),
                        (None, uw, (dw.double() * uw.double()).sum())):
        xp, xm = (x.float() + h * ex.float(), x.float() - h * ex.float()) if ex is not None else (x, x)
        wp, wm = (w.float() + h * ew.float(), w.float() - h * ew.float()) if ew is not None else (w, w)
        for v in (xp, xm, wp, wm):
            assert torch.equal(v.to(BF16).float(), v.float())
        diff = (loss(xp.to(BF16), wp.to(BF16)) - loss(xm.to(BF16), wm.to(BF16))) / (2 * h)
        # the loss is linear in either; sums of multiples of 2^-7 below 2^16 are exact in f32
        assert float(diff) == float(got)


def mx_step(x, off, w_q, out, xq):
    rows, k = x.shape
    gk.quantize_mxfp4(gk.MatRef.from_row_major(x, rows, k), xq)
    gk.gemm_grouped_mxfp4(1.0, xq, off, w_q, 0.0, gk.MatMut.from_row_major(out, rows, out.shape[1]))
    return out


@pytest.mark.parametrize("sizes", SIZES)
def test_serving_step(dev, sizes):
    """Quantized activations through quantized experts, against the product of the
    dequantized matrices (exact products, f32 sums: k * 2^-23 of the magnitudes)."""
    rows, groups, k, n = sum(sizes), len(sizes), 200, 136
    off = offsets_of(sizes)
    x, w = rand(1, rows, k), rand(2, groups * n, k, dt=F32)
    w_q = gk.quantize_mxfp4(gk.MatRef.from_row_major(w, groups * n, k))
    xq = gk.MatMxfp4.empty(rows, k)
    y = mx_step(x, off, w_q, torch.zeros(rows, n, device=dev), xq)
    xd, wd = torch.zeros(rows, k, device=dev), torch.zeros(groups * n, k, device=dev)
    gk.dequantize_mxfp4(xq, gk.MatMut.from_row_major(xd, rows, k))
    gk.dequantize_mxfp4(w_q, gk.MatMut.from_row_major(wd, groups * n, k))
    xd, wd = xd.cpu().double(), wd.cpu().double()
    at = 0
    for g, s in enumerate(sizes):
        a, b = xd[at:at + s], wd[g * n:(g + 1) * n]
        err = (y[at:at + s].cpu().double() - a @ b.t()).abs()
        assert (err <= (k + 2) * 2.0 ** -23 * (a.abs() @ b.abs().t()) + 1e-30).all()
        at += s


def build_step(dev, ws, aligned=True):
    """(outputs, call) of a whole step; unaligned sizes and a long contraction take the
    workspace."""
    sizes = [150, 0, 33, 400] if aligned else [9000, 0, 33]
    k, n = (128, 264) if aligned else (77, 131)
    rows, groups, off = sum(sizes), len(sizes), offsets_of(sizes)
    x, w, dy = rand(1, rows, k), rand(2, groups, n, k), rand(3, rows, n)
    wq = gk.quantize_mxfp4(gk.MatRef.from_row_major(w.reshape(-1, k), groups * n, k))
    xq = gk.MatMxfp4.empty(rows, k)
    y, dx = torch.zeros(rows, n, dtype=BF16, device=dev), torch.zeros(rows, k, device=dev)
    dw, yq = torch.zeros(groups, n, k, device=dev), torch.zeros(rows, n, device=dev)
    xc = x.t().contiguous()  # column-major: packed

    def call():
        gk.gemm_grouped(1.0, gk.MatRef(xc, rows, k, 1, rows), off, gk.MatRef(w, k, n, 1, k), n * k,
                        0.0, gk.MatMut.from_row_major(y, rows, n), ws=ws)
        gk.gemm_grouped(1.0, gk.MatRef.from_row_major(dy, rows, n), off, gk.MatRef(w, n, k, k, 1),
                        n * k, 0.0, gk.MatMut.from_row_major(dx, rows, k), ws=ws)
        gk.gemm_grouped_wgrad(1.0, gk.MatRef.from_row_major(x, rows, k), off,
                              gk.MatRef.from_row_major(dy, rows, n), 0.0,
                              gk.MatMut(dw, k, n, 1, k), n * k, ws=ws)
        mx_step(x, off, wq, yq, xq)

    return (y, dx, dw, yq), call, (off, sizes)


def capture(call, side):
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            call()
    torch.cuda.current_stream().wait_stream(side)
    return graph


@pytest.mark.parametrize("aligned", [True, False])
def test_captured_step_follows_the_offsets(dev, aligned):
    """Replays equal the eager step bit for bit, with eager work between them, and follow
    offsets that change after the capture."""
    ws = gk.Workspace.with_capacity(64 << 20)
    outs, call, (off, sizes) = build_step(dev, ws, aligned)
    gk.set_synchronous(False)
    try:
        call()
        torch.cuda.synchronize()
        graph = capture(call, torch.cuda.Stream())
        for rep in range(4):
            bounds = [0] + list(torch.tensor(sizes[rep % len(sizes):] + sizes[:rep % len(sizes)]).cumsum(0))
            off.copy_(torch.tensor(bounds, dtype=torch.int32))
            for o in outs:
                o.zero_()
            call()
            want = [o.clone() for o in outs]
            for o in outs:
                o.fill_(7.0)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            for o, v in zip(outs, want):
                assert torch.equal(o, v), rep
    finally:
        gk.set_synchronous(True)


def test_graph_outlives_the_growth_of_its_workspace(dev):
    """A workspace that grows after a capture keeps what the graph was given."""
    ws = gk.Workspace.with_capacity(16 << 20)
    outs, call, _ = build_step(dev, ws, aligned=False)
    gk.set_synchronous(False)
    try:
        call()
        want = [o.clone() for o in outs]
        torch.cuda.synchronize()
        graph = capture(call, torch.cuda.Stream())
        before = ws.bytes()
        big = rand(9, 4096 * 4096)
        c = torch.zeros(1024 * 4096, dtype=BF16, device=dev)
        gk.gemm_grouped(1.0, gk.MatRef(big[:1024 * 4096], 1024, 4096, 1, 1024), offsets_of([1024]),
                        gk.MatRef(big, 4096, 4096, 1, 4096), 0, 0.0,
                        gk.MatMut.from_row_major(c, 1024, 4096), ws=ws)
        torch.cuda.synchronize()
        if ws.bytes() == before:
            gk.gemm_grouped(1.0, gk.MatRef(big, 4096, 4096, 1, 4096), offsets_of([4096]),
                            gk.MatRef(big, 4096, 1024, 1, 4096), 0, 0.0,
                            gk.MatMut.from_row_major(c, 4096, 1024), ws=ws)
            torch.cuda.synchronize()
        assert ws.bytes() > before
        for _ in range(3):
            for o in outs:
                o.fill_(7.0)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            for o, v in zip(outs, want):
                assert torch.equal(o, v)
    finally:
        gk.set_synchronous(True)


def test_two_streams_share_a_workspace(dev):
    ws = gk.Workspace.with_capacity(64 << 20)
    a, b = build_step(dev, ws, False), build_step(dev, ws, True)
    for _, call, _ in (a, b):
        call()
    want = [[o.clone() for o in outs] for outs, _, _ in (a, b)]
    gk.set_synchronous(False)
    try:
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        torch.cuda.synchronize()
        for _ in range(4):
            for s, (_, call, _) in zip(streams, (a, b)):
                with torch.cuda.stream(s):
                    call()
        torch.cuda.synchronize()
    finally:
        gk.set_synchronous(True)
    for (outs, _, _), w in zip((a, b), want):
        for o, v in zip(outs, w):
            assert torch.equal(o, v)


def test_threads(dev):
    """Steps of four threads at once, each on its own stream and default workspace."""
    steps = [build_step(dev, None, i % 2 == 0) for i in range(4)]
    for _, call, _ in steps:
        call()
    want = [[o.clone() for o in outs] for outs, _, _ in steps]
    torch.cuda.synchronize()
    errors = []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(5):
                    steps[i][1]()
            torch.cuda.synchronize()
        except Exception as e:  # noqa: BLE001 -- reported below
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    for (outs, _, _), w in zip(steps, want):
        for o, v in zip(outs, w):
            assert torch.equal(o, v)


def check_rows(got, a, b, k):
    """Rows of a bf16 product against 64 bits on the device."""
    a, b = a.double(), b.double()
    want = a @ b
    tol = k * 2.0 ** -23 * (a.abs() @ b.abs())
    assert ((got.double() - want).abs() <= tol + 2.0 ** -8 * (want.abs() + tol) * 1.001).all()


@pytest.mark.parametrize("layout", ["c", "r"])
def test_offsets_past_32_bits(dev, layout):
    """A and C of more than 2^31 elements, weights of more than 2^32 bytes."""
    rows, k, n = 1_100_000, 2048, 2000
    sizes = [rows - 900, 0, 899, 1]
    off = offsets_of(sizes)
    a = torch.zeros(rows, k, dtype=BF16, device=dev)
    a[-1000:] = rand(1, 1000, k)
    w = torch.zeros(4, 300 * 2 ** 20, dtype=BF16, device=dev)  # groups 600 MiB apart
    shape = (n, k) if layout == "c" else (k, n)
    for g in range(4):
        w[g, :n * k] = rand(2 + g, n * k, std=k ** -0.5)
    c = torch.zeros(rows, n, dtype=BF16, device=dev)
    view = gk.MatRef(w, k, n, 1, k) if layout == "c" else gk.MatRef(w, k, n, n, 1)
    gk.gemm_grouped(1.0, gk.MatRef.from_row_major(a, rows, k), off, view, w.shape[1], 0.0,
                    gk.MatMut.from_row_major(c, rows, n))
    mats = [m if layout == "r" else m.t() for m in (w[g, :n * k].view(shape) for g in range(4))]
    check_rows(c[-1000:-900], a[-1000:-900], mats[0], k)
    check_rows(c[-900:-1], a[-900:-1], mats[2], k)
    check_rows(c[-1:], a[-1:], mats[3], k)
    assert not c[:-1000].any()


def test_wgrad_offsets_past_32_bits(dev):
    rows, k, n = 1_100_000, 2048, 136
    sizes = [rows - 700, 200, 0, 500]
    a = torch.zeros(rows, k, dtype=BF16, device=dev)
    b = torch.zeros(rows, n, dtype=BF16, device=dev)
    a[-900:], b[-900:] = rand(1, 900, k), rand(2, 900, n)
    dw = torch.zeros(4, k, n, dtype=BF16, device=dev)
    gk.gemm_grouped_wgrad(1.0, gk.MatRef.from_row_major(a, rows, k), offsets_of(sizes),
                          gk.MatRef.from_row_major(b, rows, n), 0.0,
                          gk.MatMut.from_row_major(dw, k, n), k * n)
    check_rows(dw[0], a[-900:-700].t().contiguous(), b[-900:-700], 200)
    check_rows(dw[1], a[-700:-500].t().contiguous(), b[-700:-500], 200)
    assert not dw[2].any()
    check_rows(dw[3], a[-500:].t().contiguous(), b[-500:], 500)


def test_mxfp4_offsets_past_32_bits(dev):
    rows, k, n = 2_200_000, 4096, 64
    x = torch.zeros(rows, k, dtype=BF16, device=dev)
    x[-500:] = rand(1, 500, k)
    q = gk.quantize_mxfp4(gk.MatRef.from_row_major(x, rows, k))
    tail = gk.quantize_mxfp4(gk.MatRef.from_row_major(x[-500:], 500, k))
    assert torch.equal(q.codes[-500:], tail.codes) and torch.equal(q.scales[-500:], tail.scales)
    w = gk.quantize_mxfp4(gk.MatRef.from_row_major(rand(2, n, k), n, k))
    c, ct = torch.zeros(rows, n, device=dev), torch.zeros(500, n, device=dev)
    gk.gemm_grouped_mxfp4(1.0, q, offsets_of([rows]), w, 0.0, gk.MatMut.from_row_major(c, rows, n))
    gk.gemm_mxfp4(1.0, tail, w, 0.0, gk.MatMut.from_row_major(ct, 500, n))
    # (the tiles differ, and with them the order of the sums)
    assert torch.allclose(c[-500:], ct, rtol=0, atol=4096 * 2.0 ** -23 * float(c.abs().max()) * 64)
    back = torch.zeros(rows, k, dtype=BF16, device=dev)
    gk.dequantize_mxfp4(q, gk.MatMut.from_row_major(back, rows, k))
    want = torch.zeros(500, k, dtype=BF16, device=dev)
    gk.dequantize_mxfp4(tail, gk.MatMut.from_row_major(want, 500, k))
    assert torch.equal(back[-500:], want) and not back[:-500].any()


@pytest.mark.parametrize("aligned", [True, False])
def test_many_groups(dev, aligned):
    """More groups than a launch's z extent; without alignment the weights are copied in
    pieces (k below the 16 bytes that reading them as they are takes)."""
    groups, k, n = 70_000, 8 if aligned else 5, 8 if aligned else 6
    g = torch.Generator(device="cuda").manual_seed(5)
    sizes = torch.randint(0, 3, (groups,), generator=g, device=dev)
    off = torch.cat([torch.zeros(1, dtype=torch.int64, device=dev), sizes.cumsum(0)]).int()
    rows = int(off[-1])
    x, w, dy = rand(1, rows, k), rand(2, groups, n, k), rand(3, rows, n)
    y = forward(x, off, w, torch.zeros(rows, n, device=dev))
    of = torch.repeat_interleave(torch.arange(groups, device=dev), sizes)
    want = (w.double()[of] * x.double()[:, None, :]).sum(2)
    tol = 8 * 2.0 ** -23 * (w.double()[of].abs() * x.double()[:, None, :].abs()).sum(2)
    assert ((y.double() - want).abs() <= tol + 2.0 ** -24 * want.abs()).all()
    dx, dw = torch.zeros(rows, k, device=dev), torch.full((groups, n, k), 7.0, device=dev)
    backward(x, off, w, dy, dx, dw)
    outer = dy.double()[:, :, None] * x.double()[:, None, :]
    want = torch.zeros(groups, n, k, dtype=torch.float64, device=dev).index_add_(0, of, outer)
    tol = torch.zeros_like(want).index_add_(0, of, outer.abs()) * 2.0 ** -22
    assert ((dw.double() - want).abs() <= tol).all()


def test_one_mxfp4_matrix_in_several_products(dev):
    """A quantized matrix stays the caller's: its arrays may be replaced or grow, and both
    operands may be the same one."""
    x = rand(1, 96, 160)
    q = gk.quantize_mxfp4(gk.MatRef.from_row_major(x, 96, 160))
    xd = torch.zeros(96, 160, device=dev)
    gk.dequantize_mxfp4(q, gk.MatMut.from_row_major(xd, 96, 160))
    c = torch.zeros(96, 96, device=dev)
    gk.gemm_mxfp4(1.0, q, q, 0.0, gk.MatMut.from_row_major(c, 96, 96))
    want = xd.double() @ xd.double().t()
    tol = 160 * 2.0 ** -23 * (xd.double().abs() @ xd.double().abs().t())
    assert ((c.double() - want).abs() <= tol).all()
    codes, scales = q.codes, q.scales
    q.codes, q.scales = torch.zeros_like(codes), scales.clone()
    gk.gemm_mxfp4(1.0, q, q, 0.0, gk.MatMut.from_row_major(c, 96, 96))
    assert not c.any()
    q.codes = codes[:95]
    with pytest.raises(gk.GemmkitError):
        gk.gemm_mxfp4(1.0, q, q, 0.0, gk.MatMut.from_row_major(c, 96, 96))


def test_python_refusals(dev):
    x = rand(1, 8, 8)
    a, c = gk.MatRef.from_row_major(x, 8, 8), gk.MatMut.from_row_major(torch.zeros_like(x), 8, 8)
    good = offsets_of([8])
    for off, err in ((good.long(), TypeError), (good.view(1, 2), TypeError), (good[:0], TypeError),
                     (good.cpu(), gk.GemmkitError), (offsets_of([4, 4])[::2], TypeError),
                     ([0, 8], TypeError)):
        with pytest.raises(err):
            gk.gemm_grouped(1.0, a, off, a, 0, 0.0, c)
        with pytest.raises(err):
            gk.gemm_grouped_wgrad(1.0, a, off, a, 0.0, c, 64)
    f32 = gk.MatRef.from_row_major(x.float(), 8, 8)
    with pytest.raises(TypeError):
        gk.gemm_grouped(1.0, f32, good, a, 0, 0.0, c)
    half = gk.MatMut.from_row_major(x.half(), 8, 8)
    for call in (lambda: gk.gemm_grouped(1.0, a, good, a, 0, 0.0, half),
                 lambda: gk.gemm_grouped_wgrad(1.0, a, good, a, 0.0, half, 64),
                 lambda: gk.quantize_mxfp4(gk.MatRef.from_row_major(x.half(), 8, 8)),
                 lambda: gk.dequantize_mxfp4(gk.MatMxfp4.empty(8, 8), half)):
        with pytest.raises(TypeError):
            call()
    bad = gk.MatMxfp4(torch.zeros(8, 16, dtype=torch.int8, device=dev),
                      torch.zeros(8, 16, dtype=torch.uint8, device=dev), 8, 8)
    with pytest.raises(TypeError):
        gk.dequantize_mxfp4(bad, c)


def test_two_graphs_share_a_workspace(dev):
    """Replayed in turn, with eager work on the same workspace between them."""
    ws = gk.Workspace.with_capacity(64 << 20)
    steps = [build_step(dev, ws, False), build_step(dev, ws, True)]
    gk.set_synchronous(False)
    try:
        for _, call, _ in steps:
            call()
        torch.cuda.synchronize()
        want = [[o.clone() for o in outs] for outs, _, _ in steps]
        graphs = [capture(call, torch.cuda.Stream()) for _, call, _ in steps]
        for i in (0, 1, 1, 0, 1, 0):
            for o in steps[i][0]:
                o.fill_(7.0)
            steps[1 - i][1]()
            graphs[i].replay()
            steps[1 - i][1]()
            torch.cuda.synchronize()
            for o, v in zip(steps[i][0], want[i]):
                assert torch.equal(o, v)
    finally:
        gk.set_synchronous(True)


def test_a_capture_cannot_grow_its_workspace(dev):
    """Operands that have to be copied need a workspace of the size before the capture."""
    rows, k, n = 64, 40, 48
    a, w = rand(1, k, rows), rand(2, n, k)  # A column-major
    c, off = torch.zeros(rows, n, dtype=BF16, device=dev), offsets_of([30, 34])
    ws = gk.Workspace()

    def call():
        gk.gemm_grouped(1.0, gk.MatRef(a, rows, k, 1, rows), off, gk.MatRef(w, k, n, 1, k), 0, 0.0,
                        gk.MatMut.from_row_major(c, rows, n), ws=ws)

    gk.set_synchronous(False)
    try:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.stream(torch.cuda.Stream()):
            with torch.cuda.graph(graph):
                with pytest.raises(gk.GemmkitError, match="captur"):
                    call()
                c.fill_(3.0)
        call()
        torch.cuda.synchronize()
        want = c.clone()
        graph = capture(call, torch.cuda.Stream())
        for _ in range(3):
            c.fill_(7.0)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(c, want)
    finally:
        gk.set_synchronous(True)
    at = torch.cat([a.t()[:30].double() @ w.double().t(), a.t()[30:].double() @ w.double().t()])
    assert ((want.double() - at).abs() <= 2.0 ** -8 * at.abs() * 1.001 + 1e-4).all()


def test_tensors_of_another_device_are_refused(dev, monkeypatch):
    x = rand(1, 8, 32)
    a, c = gk.MatRef.from_row_major(x, 8, 32), gk.MatMut.from_row_major(torch.zeros(8, 8, device=dev), 8, 8)
    q, off = gk.quantize_mxfp4(a), offsets_of([8])
    w = gk.MatRef(rand(2, 8, 32), 32, 8, 1, 32)
    monkeypatch.setattr(gk, "_raw_stream", lambda device: 0)  # (there is no second device)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 1)
    for call in (lambda: gk.gemm_grouped(1.0, a, off, w, 0, 0.0, c),
                 lambda: gk.gemm_grouped_wgrad(1.0, a, off, a, 0.0, c, 0),
                 lambda: gk.quantize_mxfp4(a, q), lambda: gk.gemm_mxfp4(1.0, q, q, 0.0, c),
                 lambda: gk.gemm_grouped_mxfp4(1.0, q, off, q, 0.0, c)):
        with pytest.raises(gk.GemmkitError, match="current device"):
            call()
