"""GPU: odl_newton_schulz and odl_muon_step against the definition in 64 bits.

One step is held to a bound per element: with eps = 2^-18 for a product of 22-bit operands (see test_gpu_linear_ce.py) and
2^-36 of the largest entry for their grid,
  dA = eps |X||X|^T,  dS = |b| dA + |c| (2 |A| dA + eps |A||A|) + 2^-21 |S|,  dX' = dS |X| + eps |S||X|.
Five steps are held to what errors of that size do to the 64-bit iteration itself: the iteration is repeated with random
errors of relative size eps = 2^-20 (in the 2-norm over all elements, what such sums leave of the bound per element) put on A,
S and X in every step, and the kernel may be 4 times as far off as the furthest of four such runs.  PRECISION_TF32 keeps 11
bits per operand: eps = 2^-9 and 2^-11."""
import pytest
import torch

pytestmark = pytest.mark.gpu

A, B, C = 3.4445, -4.7750, 2.0315


@pytest.fixture(scope="module")
def ops():
    from origindl_b200 import capi, ops

    capi.init(0)
    yield ops
    capi.device_status()


def gradient(*shape, seed=0, rank=None, scale=1e-3):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rows, cols = shape[-2:]
    r = rank or max(1, min(rows, cols) // 8)
    lead = shape[:-2]
    strong = torch.randn(*lead, rows, r, device="cuda", generator=g) @ torch.randn(*lead, r, cols, device="cuda", generator=g)
    return (strong + 0.3 * torch.randn(*shape, device="cuda", generator=g)) * scale


def wide(x):
    return x.mT if x.shape[-2] > x.shape[-1] else x


def iterate(g, steps, eps=0.0, gen=None, floor=1e-7):
    x = wide(g.double())
    x = x / torch.linalg.matrix_norm(x, keepdim=True).clamp(min=floor)

    def off(v):
        if not eps:
            return v
        n = torch.randn(v.shape, device=v.device, dtype=v.dtype, generator=gen)
        return v + n * (eps * torch.linalg.matrix_norm(v, keepdim=True) / torch.linalg.matrix_norm(n, keepdim=True))

    x = off(x)
    for _ in range(steps):
        a = off(x @ x.mT)
        s = off(A * torch.eye(a.shape[-1], device=a.device, dtype=a.dtype) + B * a + C * (a @ a))
        x = off(s @ x)
    return x.mT if g.shape[-2] > g.shape[-1] else x


def bound(g, steps, precision):
    want = iterate(g, steps)
    gen = torch.Generator(device="cuda").manual_seed(99)
    eps = 2.0 ** -20 if precision == 0 else 2.0 ** -11
    far = max(torch.linalg.matrix_norm(iterate(g, steps, eps, gen) - want).max().item() for _ in range(4))
    return want, 4 * far


SHAPES = [(5, 5888), (16, 8192), (8192, 13), (17, 5120), (32, 8000), (6144, 40), (64, 6200), (2000, 31), (120, 1700), (16, 700), (700, 16), (64, 4096), (64, 4097), (4000, 60), (128, 1536), (128, 1537), (1500, 120), (65, 1000), (100, 2000), (8, 64), (1, 1), (1, 7), (9, 1), (2, 3), (31, 33), (64, 64), (65, 64), (63, 200), (128, 128), (129, 127), (100, 784), (784, 100),
          (256, 256), (257, 300), (300, 257), (513, 1000), (1000, 513), (1024, 384), (1100, 1100), (260, 2000)]


@pytest.mark.parametrize("rows,cols", SHAPES)
def test_one_step_per_element(ops, rows, cols):
    g = gradient(rows, cols, seed=rows + cols)
    got = wide(ops.newton_schulz(g, steps=1)).double()
    X = wide(g.double())
    X = X / torch.linalg.matrix_norm(X)
    eps, grid = 2.0 ** -18, 2.0 ** -36
    G = X @ X.mT
    S = A * torch.eye(G.shape[0], device="cuda", dtype=torch.float64) + B * G + C * (G @ G)
    dX = 2.0 ** -22 * X.abs() + grid
    dA = eps * (X.abs() @ X.abs().mT) + 2 * dX @ X.abs().mT + grid
    dS = abs(B) * dA + C * (2 * G.abs() @ dA + eps * G.abs() @ G.abs()) + 2.0 ** -21 * S.abs() + grid * 8
    tol = dS @ X.abs() + eps * (S.abs() @ X.abs()) + S.abs() @ dX
    err = (got - S @ X).abs()
    assert (err <= tol).all(), (err - tol).max().item()


@pytest.mark.parametrize("rows,cols", SHAPES)
def test_five_steps(ops, rows, cols):
    g = gradient(rows, cols, seed=rows * cols)
    want, far = bound(g, 5, 0)
    assert torch.linalg.matrix_norm(ops.newton_schulz(g).double() - want).item() <= far


@pytest.mark.parametrize("tile", [64, 128, 256])
@pytest.mark.parametrize("rows,cols", [(300, 520), (777, 260), (130, 130), (64, 600)])
def test_every_tile(ops, tile, rows, cols):
    from origindl_b200 import capi

    g = gradient(2, rows, cols, seed=tile)
    capi.call("odl_debug_set_tile_n", tile)
    try:
        got = ops.newton_schulz(g)
        plain = ops.newton_schulz(g, precision=ops.PRECISION_TF32)
    finally:
        capi.call("odl_debug_set_tile_n", 0)
    for i in range(2):
        want, far = bound(g[i], 5, 0)
        assert torch.linalg.matrix_norm(got[i].double() - want).item() <= far
        want, far = bound(g[i], 5, 1)
        assert torch.linalg.matrix_norm(plain[i].double() - want).item() <= far


@pytest.mark.parametrize("rows,cols", [(33, 70), (256, 512), (700, 300)])
def test_plain_tf32(ops, rows, cols):
    g = gradient(rows, cols, seed=1)
    want, far = bound(g, 5, 1)
    got = ops.newton_schulz(g, precision=ops.PRECISION_TF32)
    assert torch.linalg.matrix_norm(got.double() - want).item() <= far


@pytest.mark.parametrize("batch,rows,cols", [(40, 64, 512), (150, 9, 40), (300, 32, 130), (20, 500, 100), (3, 50, 70), (5, 130, 64), (2, 257, 513), (33, 16, 24), (4, 600, 300)])
def test_stack(ops, batch, rows, cols):
    g = gradient(batch, rows, cols, seed=batch)
    g[1] *= 1e-3   # each has its own norm
    got = ops.newton_schulz(g)
    for i in range(batch):
        want, far = bound(g[i], 5, 0)
        assert torch.linalg.matrix_norm(got[i].double() - want).item() <= far


def test_in_place_and_steps(ops):
    g = gradient(96, 160, seed=3)
    for steps in (0, 1, 2, 7):
        want = ops.newton_schulz(g, steps=steps)
        h = g.clone()
        assert ops.newton_schulz(h, steps=steps, out=h) is h
        assert torch.equal(h, want)
    X = g.double() / torch.linalg.matrix_norm(g.double())
    err = (ops.newton_schulz(g, steps=0).double() - X).abs()
    assert (err <= 2.0 ** -22 * X.abs() + 2.0 ** -38).all()


@pytest.mark.parametrize("scale", [1e-30, 1e-6, 1.0, 1e20, 1e37])
def test_any_size_of_gradient(ops, scale):
    """The norm is summed in 64 bits: nothing under- or overflows; below eps the matrix is divided by eps instead."""
    g = gradient(80, 120, seed=4, scale=1.0)
    g *= scale / g.abs().max()
    want, far = bound(g, 5, 0)
    assert torch.linalg.matrix_norm(ops.newton_schulz(g).double() - want).item() <= far + 1e-12


def test_zero_and_non_finite(ops):
    z = torch.zeros(40, 60, device="cuda")
    assert (ops.newton_schulz(z) == 0).all()
    g = gradient(3, 40, 60, seed=5)
    clean = ops.newton_schulz(g)
    g[1, 3, 4] = float("nan")
    got = ops.newton_schulz(g)
    assert torch.equal(got[0], clean[0]) and torch.equal(got[2], clean[2])
    assert not torch.isfinite(got[1]).any()


def test_one_strong_direction(ops):
    """Rank one and noise 1e-4 below it: the small directions are amplified 3.4445 times a step, and their errors too."""
    g = gradient(200, 320, seed=6, rank=1)
    g = g + 0 * g
    want, far = bound(g, 5, 0)
    assert torch.linalg.matrix_norm(ops.newton_schulz(g).double() - want).item() <= far


@pytest.mark.parametrize("rows,cols,layout", [(48, 100, "out_in"), (100, 48, "out_in"), (100, 48, "in_out"), (257, 130, "in_out"),
                                              (512, 512, "out_in"), (33, 1000, "in_out")])
@pytest.mark.parametrize("nesterov,decay,momentum", [(True, 0.1, 0.95), (False, 0.0, 0.9), (True, 0.0, 0.0)])
def test_muon_step(ops, rows, cols, layout, nesterov, decay, momentum):
    w_layout = ops.W_OUT_IN if layout == "out_in" else ops.W_IN_OUT
    lr, gs, hook = 0.03, 0.5, 1e-4
    p = torch.randn(rows, cols, device="cuda", generator=torch.Generator(device="cuda").manual_seed(7)) * 0.02
    g = gradient(rows, cols, seed=8)
    buf = gradient(rows, cols, seed=9) if momentum else None
    P, G, M = p.double(), g.double(), buf.double() if momentum else None
    G = G * gs + hook * P
    if momentum:
        M = momentum * M + G
        u = G + momentum * M if nesterov else M
    else:
        u = G
    want_u, far = bound(u.float(), 5, 0)
    fan = (rows, cols) if layout == "out_in" else (cols, rows)
    s = max(1.0, fan[0] / fan[1]) ** 0.5
    want = P * (1 - lr * decay) - lr * s * want_u
    small = torch.empty_like(p)
    ops.muon_step(p, g, buf, lr=lr, momentum=momentum, nesterov=nesterov, weight_decay=decay, hook_weight_decay=hook,
                  grad_scale=gs, w_layout=w_layout, p_small=small)
    # u itself is rounded to 32 bits (3 roundings) before the iteration sees it: within the injected errors' size
    assert torch.linalg.matrix_norm(p.double() - want).item() <= lr * s * far + 2.0 ** -23 * torch.linalg.matrix_norm(want).item()
    assert ((g.double() - G).abs() <= 2.0 ** -23 * (G.abs() + hook * P.abs())).all()
    if momentum:
        assert ((buf.double() - M).abs() <= 2.0 ** -22 * (M.abs() + G.abs())).all()
    assert torch.equal(small, ops.split_tf32(p))


def test_muon_stack_is_each_matrix_by_itself(ops):
    p, g, buf = (gradient(6, 90, 200, seed=s) for s in (1, 2, 3))
    q, h, m = p.clone(), g.clone(), buf.clone()
    ops.muon_step(p, g, buf)
    for i in range(6):
        a, b, c = (v[i].clone() for v in (q, h, m))
        ops.muon_step(a, b, c)
        torch.testing.assert_close(p[i], a, rtol=0, atol=2e-7)
        assert torch.equal(buf[i], c)
    assert torch.equal(g, h)   # nothing scaled it


def test_same_bits_again_and_on_other_streams(ops):
    a, c = gradient(300, 500, seed=1), gradient(2, 200, 100, seed=2)
    wa, wc = ops.newton_schulz(a), ops.newton_schulz(c)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    got = []
    for _ in range(4):
        with torch.cuda.stream(s1):
            ga = ops.newton_schulz(a)
        with torch.cuda.stream(s2):
            gc = ops.newton_schulz(c)
        got.append((ga, gc))
    torch.cuda.synchronize()
    for ga, gc in got:
        assert torch.equal(ga, wa) and torch.equal(gc, wc)


@pytest.mark.parametrize("shape", [(150, 260), (40, 300), (3, 100, 700), (2, 300, 140)])
def test_captured_and_replayed(ops, shape):
    p, g, buf = (gradient(*shape, seed=s) for s in (1, 2, 3))
    start = [v.clone() for v in (p, buf)]
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        ops.muon_step(p, g, buf)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            ops.muon_step(p, g, buf)
    p.copy_(start[0]), buf.copy_(start[1])
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    q, m = start
    for _ in range(3):
        ops.muon_step(q, g, m)
    assert torch.equal(p, q) and torch.equal(buf, m)


def test_unaligned_tensors(ops):
    off = lambda v: torch.empty(v.numel() + 1, device="cuda")[1:].view(v.shape).copy_(v)  # noqa: E731
    for rows, cols in ((64, 128), (200, 96), (256, 512)):
        p, g, buf = (gradient(rows, cols, seed=s) for s in (1, 2, 3))
        q, h, m = off(p), off(g), off(buf)
        ops.muon_step(p, g, buf)
        ops.muon_step(q, h, m)
        assert torch.equal(p, q) and torch.equal(buf, m)


def test_refusals(ops):
    g = gradient(8, 10)
    for bad in (lambda: ops.newton_schulz(g[0]), lambda: ops.newton_schulz(g, out=torch.empty(10, 8, device="cuda")),
                lambda: ops.newton_schulz(g.t()), lambda: ops.muon_step(g, g[:4].contiguous(), g.clone())):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        ops.newton_schulz(g.half())


def test_training_step_of_a_head_with_many_classes(ops):
    """The operators as they are used together: loss and gradients of the head, Muon on the hidden weight, SGD on the head.
    The parameters after three steps against the same three steps in 64 bits."""
    gen = torch.Generator(device="cuda").manual_seed(12)
    M, D, H, N = 192, 80, 136, 1111
    x = torch.randn(M, D, device="cuda", generator=gen)
    t = torch.randint(0, N, (M,), device="cuda", generator=gen)
    t[::7] = -100
    w1 = torch.randn(H, D, device="cuda", generator=gen) / D ** 0.5
    w2 = torch.randn(N, H, device="cuda", generator=gen) / H ** 0.5
    buf = torch.zeros_like(w1)
    W1, W2, BUF = w1.double(), w2.double(), buf.double()
    X = x.double()
    far = 0.0
    for _ in range(3):
        h = ops.linear_forward(x, w1, relu=True)
        loss, _, dh, dw2, _ = ops.linear_cross_entropy(h, w2, t)
        _, dw1, _ = ops.linear_backward(x, w1, dh, h, need_dx=False)
        ops.muon_step(w1, dw1, buf, lr=0.05)
        ops.sgd_step(w2, dw2, lr=0.1)
        W1g, W2g = W1.requires_grad_(), W2.requires_grad_()
        L = torch.nn.functional.cross_entropy(torch.relu(X @ W1g.t()) @ W2g.t(), t)
        G1, G2 = torch.autograd.grad(L, (W1g, W2g))
        assert abs(loss.item() - L.item()) <= 1e-4
        with torch.no_grad():
            BUF = 0.95 * BUF + G1
            u = G1 + 0.95 * BUF
            U, f = bound(u, 5, 0)
            far += f
            W1 = (W1 - 0.05 * max(1, H / D) ** 0.5 * U).detach()
            W2 = (W2 - 0.1 * G2).detach()
    # the gradient that enters the iteration is off by 1e-5 of its norm at most (two chained products of the bound above),
    # ten times the injected errors
    assert torch.linalg.matrix_norm(w1.double() - W1).item() <= 0.05 * 1.31 * 20 * far
    assert torch.linalg.matrix_norm(w2.double() - W2).item() <= 1e-4 * torch.linalg.matrix_norm(W2).item()
