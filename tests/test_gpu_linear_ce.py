"""GPU: odl_linear_cross_entropy against the definition in 64 bits.

Tolerances are bounds per element, from the arithmetic, with eps = 2^-18 for one matrix product of the 22-bit operands
(operand and dropped-term errors 2^-21, accumulation 12 * 2^-23 inside a chunk of 64 and K / 64 * 2^-24 over the chunks, for
K <= 4096: together below 2^-18 of the sum of the absolute products).  They are carried through the formulas:
  dz = eps |x||W|^T,  dlse = max_j dz + 2^-20 (1 + |lse|),  dP = P (dz + dlse + 2^-20) + 2^-38 (the grid of P),
  d(dx) = g (dP |W| + eps |P||W| + 2^-36 |P| max|W|),  and so on.
PRECISION_TF32 keeps 11 bits per operand: eps = 2^-9."""
import pytest
import torch

pytestmark = pytest.mark.gpu

EPS = {0: 2.0 ** -18, 1: 2.0 ** -9}
GRID = {0: 2.0 ** -38, 1: 2.0 ** -24}


@pytest.fixture(scope="module")
def ops():
    from origindl_b200 import capi, ops

    capi.init(0)
    yield ops
    capi.device_status()


def make(M, N, K, seed, in_out=False, bias=False, ignored=0.0, sharp=0.0, itype=torch.int64):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(M, K, device="cuda", generator=g)
    w = torch.randn(N, K, device="cuda", generator=g) * (0.7 / K ** 0.5)
    t = torch.randint(0, N, (M,), device="cuda", generator=g)
    if sharp:
        x += sharp * w[t]
    if ignored:
        t[torch.rand(M, device="cuda", generator=g) < ignored] = -100
    b = torch.randn(N, device="cuda", generator=g) * 0.1 if bias else None
    return x, (w.t().contiguous() if in_out else w), t.to(itype), b


def reference(x, w, t, b, in_out, grad_scale, precision):
    """Values and per-element bounds, all in 64 bits."""
    eps, grid = EPS[precision], GRID[precision]
    valid = t != -100
    x64 = torch.where(valid[:, None], x, torch.zeros_like(x)).double()
    w64 = (w.t() if in_out else w).double()
    b64 = torch.zeros(w64.shape[0], dtype=torch.float64, device=x.device) if b is None else b.double()
    z = x64 @ w64.t() + b64
    dz = eps * (x64.abs() @ w64.abs().t() + b64.abs().nan_to_num(posinf=0.0))
    lse = torch.logsumexp(z, 1)
    dlse = dz.max(1).values + 2.0 ** -20 * (1 + lse.abs())
    n = int(valid.sum())
    at = torch.where(valid, t, torch.zeros_like(t)).long()[:, None]
    rows = torch.where(valid, lse - z.gather(1, at)[:, 0], torch.zeros_like(lse))
    drows = torch.where(valid, dlse + dz.gather(1, at)[:, 0], torch.zeros_like(lse))
    loss, dloss = (rows.sum() / n, drows.sum() / n) if n else (rows.sum() * 0, drows.sum() * 0)
    soft = torch.exp(z - lse[:, None])
    P = soft.scatter_add(1, at, torch.full_like(at, -1, dtype=torch.float64)) * valid[:, None]
    dP = (soft * (dz + dlse[:, None] + 2.0 ** -20) + grid) * valid[:, None]
    g = grad_scale / n if n else 0.0
    E = dP + eps * P.abs()
    wide = lambda o, dim: 2.0 ** 2 * grid * o.abs().max()  # noqa: E731
    out = dict(loss=(loss, dloss + 1e-7 * loss.abs()), lse=(torch.where(valid, lse, 0 * lse), torch.where(valid, dlse, 0 * dlse)))
    out["dx"] = (g * (P @ w64), abs(g) * (E @ w64.abs() + P.abs().sum(1, keepdim=True) * wide(w64, 1)))
    dw, ddw = g * (P.t() @ x64), abs(g) * (E.t() @ x64.abs() + P.abs().sum(0)[:, None] * wide(x64, 0))
    out["dw"] = (dw.t(), ddw.t()) if in_out else (dw, ddw)
    out["db"] = (g * P.sum(0), abs(g) * (dP.sum(0) + P.abs().sum(0) * 2.0 ** -18))
    return out


def check(got, want, names):
    for name, value in zip(("loss", "lse", "dx", "dw", "db"), got):
        if name not in names:
            assert value is None or name in ("loss", "lse")
            continue
        ref, tol = want[name]
        err = (value.double() - ref).abs()
        assert torch.isfinite(value).all(), name
        worst = (err - tol).max().item()
        assert worst <= 0, f"{name}: over its bound by {worst:.3e} (largest error {err.max().item():.3e}, value {ref.abs().max().item():.3e})"


SIZES = [(1, 2, 1), (1, 1, 5), (1, 32000, 512), (2, 3, 7), (5, 129, 65), (16, 1000, 64), (31, 257, 100), (33, 4096, 128),
         (64, 130, 1001), (127, 511, 63), (128, 256, 64), (129, 255, 66), (200, 2049, 300), (255, 5000, 129), (257, 1000, 1000),
         (512, 10, 1000), (700, 10007, 96), (1025, 513, 257), (2100, 700, 72)]


@pytest.mark.parametrize("in_out", [False, True])
@pytest.mark.parametrize("M,N,K", SIZES)
def test_values_and_gradients(ops, M, N, K, in_out):
    x, w, t, b = make(M, N, K, seed=M + N + K, in_out=in_out, bias=True, ignored=0.3 if M > 4 else 0.0, sharp=4.0)
    layout = ops.W_IN_OUT if in_out else ops.W_OUT_IN
    got = ops.linear_cross_entropy(x, w, t, b=b, w_layout=layout, grad_scale=1.5)
    check(got, reference(x, w, t, b, in_out, 1.5, 0), ("loss", "lse", "dx", "dw", "db"))


@pytest.fixture
def chosen(ops):
    """Sets the overrides of include/odl_b200_test.h and puts them back."""
    from origindl_b200 import capi

    def set_(tile=0, splits=0, piece=0):
        capi.call("odl_debug_set_tile_n", tile)
        capi.call("odl_debug_set_split_k", splits)
        capi.call("odl_debug_set_loss_piece", piece)

    yield set_
    set_()


@pytest.mark.parametrize("in_out", [False, True])
@pytest.mark.parametrize("precision", [0, 1])
@pytest.mark.parametrize("tile,splits,piece", [(64, 1, 0), (128, 1, 256), (256, 1, 0), (256, 3, 256), (128, 2, 0), (64, 5, 256)])
def test_every_tile_and_split(ops, chosen, tile, splits, piece, precision, in_out):
    x, w, t, b = make(600, 1100, 200, seed=tile + splits, in_out=in_out, bias=True, ignored=0.3)
    chosen(tile, splits, piece)
    got = ops.linear_cross_entropy(x, w, t, b=b, w_layout=ops.W_IN_OUT if in_out else ops.W_OUT_IN, precision=precision)
    check(got, reference(x, w, t, b, in_out, 1.0, precision), ("loss", "lse", "dx", "dw", "db"))
    got = ops.linear_cross_entropy(x, w, t, b=b, need_dx=False, need_dw=False, need_db=False, precision=precision,
                                   w_layout=ops.W_IN_OUT if in_out else ops.W_OUT_IN)
    check(got, reference(x, w, t, b, in_out, 1.0, precision), ("loss", "lse"))


def test_pieces_with_few_rows_left(ops, chosen):
    """Most rows are ignored: later pieces are empty, the first is not full."""
    x, w, t, b = make(1300, 300, 100, seed=21, bias=True, ignored=0.97)
    chosen(256, 1, 256)
    check(ops.linear_cross_entropy(x, w, t, b=b), reference(x, w, t, b, False, 1.0, 0), ("loss", "lse", "dx", "dw", "db"))


@pytest.mark.parametrize("in_out", [False, True])
@pytest.mark.parametrize("precision", [0, 1])
@pytest.mark.parametrize("M,N,K", [(1, 4, 4), (1, 1, 1), (1, 7, 3), (2, 1001, 77), (3, 130, 999), (4, 50021, 65), (5, 999, 4001), (8, 5001, 130),
                                   (8, 40000, 64), (8, 300, 7000), (1, 20, 8), (1, 5000, 2048), (2, 128, 32), (9, 2500, 36), (15, 132, 100), (16, 4096, 64), (17, 33000, 96),
                                   (32, 1000, 260), (33, 7000, 128), (48, 19000, 64), (64, 300, 1000), (64, 40000, 68)])
def test_few_rows(ops, M, N, K, precision, in_out):
    """Up to 64 rows without gradients: read straight from the weights (aligned ones above 8 rows)."""
    x, w, t, b = make(M, N, K, seed=N, in_out=in_out, bias=True, ignored=0.3 if M > 4 else 0.0, sharp=3.0)
    got = ops.linear_cross_entropy(x, w, t, b=b, need_dx=False, need_dw=False, need_db=False, precision=precision,
                                   w_layout=ops.W_IN_OUT if in_out else ops.W_OUT_IN)
    check(got, reference(x, w, t, b, in_out, 1.0, precision), ("loss", "lse"))


def test_few_rows_garbage_masks_and_bad_labels(ops):
    from origindl_b200 import capi

    x, w, t, b = make(20, 3000, 64, seed=30, bias=True)
    t[::3] = -100
    x[::3] = float("nan")
    b[:2000] = float("-inf")
    t[t != -100] = 2500
    kw = dict(need_dx=False, need_dw=False, need_db=False)
    got = ops.linear_cross_entropy(x, w, t, b=b, **kw)
    want = reference(x, w[2000:].contiguous(), torch.where(t == -100, t, t - 2000), b[2000:].contiguous(), False, 1.0, 0)
    check(got, want, ("loss", "lse"))
    bad = t.clone()
    bad[1] = 3000
    t[1] = -100
    got = ops.linear_cross_entropy(x, w, bad, b=b, **kw)
    with pytest.raises(capi.OdlError, match="linear_cross_entropy"):
        capi.device_status()
    for u, v in zip(got[:2], ops.linear_cross_entropy(x, w, t, b=b, **kw)[:2]):
        assert torch.equal(u, v)
    t.fill_(-100)
    loss, lse = ops.linear_cross_entropy(x, w, t, b=b, **kw)[:2]
    assert loss == 0 and (lse == 0).all()


@pytest.mark.parametrize("M,N,K", [(1, 777, 130), (7, 50021, 64), (40, 3000, 515), (300, 1111, 192), (2000, 300, 64)])
@pytest.mark.parametrize("itype", [torch.int32, torch.int64])
def test_loss_alone(ops, M, N, K, itype):
    x, w, t, _ = make(M, N, K, seed=M, ignored=0.2 if M > 4 else 0.0, itype=itype)
    got = ops.linear_cross_entropy(x, w, t, need_dx=False, need_dw=False)
    check(got, reference(x, w, t, None, False, 1.0, 0), ("loss", "lse"))


@pytest.mark.parametrize("in_out", [False, True])
@pytest.mark.parametrize("M,N,K", [(3, 500, 64), (190, 1025, 130), (1030, 300, 520)])
def test_plain_tf32(ops, M, N, K, in_out):
    x, w, t, b = make(M, N, K, seed=5, in_out=in_out, bias=True, ignored=0.1 if M > 4 else 0.0)
    got = ops.linear_cross_entropy(x, w, t, b=b, w_layout=ops.W_IN_OUT if in_out else ops.W_OUT_IN,
                                   precision=ops.PRECISION_TF32)
    check(got, reference(x, w, t, b, in_out, 1.0, 1), ("loss", "lse", "dx", "dw", "db"))


@pytest.mark.parametrize("dx,dw,db", [(True, False, False), (False, True, False), (False, False, True), (True, False, True)])
def test_each_gradient_by_itself(ops, dx, dw, db):
    x, w, t, b = make(150, 400, 96, seed=9, bias=True, ignored=0.1)
    got = ops.linear_cross_entropy(x, w, t, b=b, need_dx=dx, need_dw=dw, need_db=db)
    names = ["loss", "lse"] + [n for n, f in (("dx", dx), ("dw", dw), ("db", db)) if f]
    check(got, reference(x, w, t, b, False, 1.0, 0), names)


@pytest.mark.parametrize("M", [1, 6, 300])
def test_no_row_left(ops, M):
    x, w, t, b = make(M, 100, 40, seed=2, bias=True)
    t.fill_(-100)
    x.fill_(float("nan"))
    loss, lse, dx, dw, db = ops.linear_cross_entropy(x, w, t, b=b)
    for v in (loss, lse, dx, dw, db):
        assert (v == 0).all()


@pytest.mark.parametrize("M", [8, 200, 520])
@pytest.mark.parametrize("garbage", [float("nan"), float("inf"), -3e38])
def test_what_ignored_rows_hold_reaches_nothing(ops, M, garbage):
    x, w, t, b = make(M, 333, 70, seed=3, bias=True)
    t[::3] = -100
    clean = ops.linear_cross_entropy(x, w, t, b=b)
    x[::3] = garbage
    for a, c in zip(ops.linear_cross_entropy(x, w, t, b=b), clean):
        assert torch.equal(a, c)


@pytest.mark.parametrize("low", [float("-inf"), torch.finfo(torch.float32).min])
@pytest.mark.parametrize("M,N", [(3, 50), (140, 1000)])
def test_classes_masked_by_the_bias(ops, low, M, N):
    x, w, t, b = make(M, N, 64, seed=4, bias=True)
    out = torch.arange(N, device="cuda") % 2 == 1
    out[:min(N - 2, 512)] = True   # whole tiles of classes that are out
    t.fill_(N - 1 if not out[N - 1] else N - 2)
    b[out] = low
    loss, lse, dx, dw, db = ops.linear_cross_entropy(x, w, t, b=b)
    keep = ~out
    t2 = (torch.cumsum(keep, 0) - 1)[t]
    want = reference(x, w[keep].contiguous(), t2, b[keep].contiguous(), False, 1.0, 0)
    check((loss, lse, dx), want, ("loss", "lse", "dx"))
    check((None, None, None, dw[keep], db[keep]), want, ("dw", "db"))
    assert (dw[out] == 0).all() and (db[out] == 0).all()


def test_rows_and_features_of_very_different_size(ops):
    """Scales per block: a block of rows 2^40 times another's keeps its precision."""
    x, w, t, _ = make(512, 640, 256, seed=6)
    x[128:256] *= 2.0 ** -20
    x[256:384] *= 2.0 ** -40
    w[:, 64:128] *= 2.0 ** 10
    x[:, 64:128] *= 2.0 ** -10
    got = ops.linear_cross_entropy(x, w, t, grad_scale=2.0 ** 30)
    want = reference(x, w, t, None, False, 2.0 ** 30, 0)
    check(got, want, ("loss", "lse", "dx", "dw"))


def test_label_out_of_range_is_reported_and_its_row_left_out(ops):
    from origindl_b200 import capi

    x, w, t, _ = make(150, 90, 32, seed=7)
    want_t = t.clone()
    t[3], t[100] = 90, -1
    want_t[3] = want_t[100] = -100
    got = ops.linear_cross_entropy(x, w, t)
    with pytest.raises(capi.OdlError, match="linear_cross_entropy"):
        capi.device_status()
    for a, c in zip(got, ops.linear_cross_entropy(x, w, want_t)):
        assert (a is None and c is None) or torch.equal(a, c)
    capi.device_status()


def test_another_ignore_index(ops):
    x, w, t, _ = make(64, 50, 32, seed=8)
    t[t == 7] = 8
    t[:10] = 7
    u = t.clone()
    u[:10] = -100
    for a, c in zip(ops.linear_cross_entropy(x, w, t, ignore_index=7), ops.linear_cross_entropy(x, w, u)):
        assert (a is None and c is None) or torch.equal(a, c)


@pytest.mark.parametrize("M,N,K", [(2, 40, 33), (140, 300, 65)])
def test_gradients_against_differences(ops, M, N, K):
    """Central differences of the 64-bit loss along random directions, and the call's gradients along the same."""
    x, w, t, b = make(M, N, K, seed=10, bias=True)
    _, _, dx, dw, db = ops.linear_cross_entropy(x, w, t, b=b)
    f = lambda x, w, b: torch.nn.functional.cross_entropy(x @ w.t() + b, t)  # noqa: E731
    gen = torch.Generator(device="cuda").manual_seed(1)
    X, W, B = x.double(), w.double(), b.double()
    for _ in range(3):
        vx, vw, vb = (torch.randn(v.shape, device="cuda", generator=gen, dtype=torch.float64) for v in (x, w, b))
        h = 1e-4
        num = (f(X + h * vx, W + h * vw, B + h * vb) - f(X - h * vx, W - h * vw, B - h * vb)) / (2 * h)
        parts = [(dx.double() * vx), (dw.double() * vw), (db.double() * vb)]
        ana = sum(p.sum() for p in parts)
        assert abs(num - ana) <= 1e-5 * sum(p.abs().sum() for p in parts) + 1e-6


def test_same_bits_again_and_on_other_streams(ops):
    a = make(700, 3001, 200, seed=11, bias=True, ignored=0.1)
    c = make(300, 5000, 100, seed=12, bias=True)
    run = lambda v: ops.linear_cross_entropy(v[0], v[1], v[2], b=v[3])  # noqa: E731
    wa, wc = run(a), run(c)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    got = []
    for _ in range(4):
        with torch.cuda.stream(s1):
            ga = run(a)
        with torch.cuda.stream(s2):
            gc = run(c)
        got.append((ga, gc))
    torch.cuda.synchronize()
    for ga, gc in got:
        for u, v in zip(ga + gc, wa + wc):
            assert torch.equal(u, v)


def test_captured_and_replayed(ops):
    from origindl_b200 import capi

    a = make(400, 2000, 128, seed=13, bias=True, ignored=0.2)
    other = make(400, 2000, 128, seed=14, bias=True, ignored=0.4)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        ops.linear_cross_entropy(a[0], a[1], a[2], b=a[3])
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            out = ops.linear_cross_entropy(a[0], a[1], a[2], b=a[3])
    for data in (other, a):
        keep = [v.clone() for v in data]
        for dst, src in zip(a, keep):
            dst.copy_(src)
        graph.replay()
        torch.cuda.synchronize()
        for u, v in zip(out, ops.linear_cross_entropy(a[0], a[1], a[2], b=a[3])):
            assert torch.equal(u, v)
    # a call that needs more scratch than the library holds is refused while it is being captured, and the capture goes on
    big = make(6000, 9001, 64, seed=15)
    if capi.lib().odl_scratch_bytes() < 6000 * 9001 * 4:
        with torch.cuda.stream(s):
            graph2 = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph2, stream=s):
                with pytest.raises(capi.OdlError, match="before the capture"):
                    ops.linear_cross_entropy(big[0], big[1], big[2])
    # the scratch block grows: the recorded one stays usable
    ops.linear_cross_entropy(big[0], big[1], big[2])
    graph.replay()
    torch.cuda.synchronize()
    for u, v in zip(out, ops.linear_cross_entropy(a[0], a[1], a[2], b=a[3])):
        assert torch.equal(u, v)


@pytest.mark.parametrize("M,N,K", [(3, 5000, 100), (40, 5000, 128), (200, 900, 64)])
def test_loss_alone_captured_and_on_another_stream(ops, M, N, K):
    x, w, t, b = make(M, N, K, seed=40, bias=True)
    run = lambda: ops.linear_cross_entropy(x, w, t, b=b, need_dx=False, need_dw=False, need_db=False)[:2]  # noqa: E731
    want = run()
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        again = run()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            out = run()
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    for a, c, d in zip(want, again, out):
        assert torch.equal(a, c) and torch.equal(a, d)


def test_unaligned_tensors(ops):
    """Every buffer starts 4 bytes off a 16-byte boundary."""
    off = lambda v: torch.empty(v.numel() + 1, device="cuda", dtype=v.dtype)[1:].view(v.shape).copy_(v)  # noqa: E731
    x, w, t, b = make(130, 517, 128, seed=16, bias=True)
    want = ops.linear_cross_entropy(x, w, t, b=b)
    for u, v in zip(ops.linear_cross_entropy(off(x), off(w), t, b=off(b)), want):
        assert torch.equal(u, v)


def test_refusals(ops):
    x, w, t, b = make(8, 9, 10, seed=17, bias=True)
    for bad in (lambda: ops.linear_cross_entropy(x[0], w, t), lambda: ops.linear_cross_entropy(x, w, t[:4]),
                lambda: ops.linear_cross_entropy(x, w[:, :5].contiguous(), t), lambda: ops.linear_cross_entropy(x, w, t, b=b[:3]),
                lambda: ops.linear_cross_entropy(x.t(), w, t), lambda: ops.linear_cross_entropy(x, w, t, w_layout=ops.W_IN_OUT)):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: ops.linear_cross_entropy(x.half(), w, t), lambda: ops.linear_cross_entropy(x, w, t.float())):
        with pytest.raises(TypeError):
            bad()
