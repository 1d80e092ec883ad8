"""The relation head (attention.linear) against its formula in 64 bits.

Error bounds.  With S = sum_k |x||w| of an output element:
 * fp32: each operand is hi + lo in two fp16 planes, off by 2^-22 of the value
   (2^-40 of its line's largest below that), and lo * lo is dropped: 3 * 2^-22 S;
   the sum takes 3 products per 16 of k, each addition off by at most 2^-23 S;
   the path for few rows adds k fp32 terms: k * 2^-24 S.  Both are below
   (4 * 2^-22 + (3 * ceil(k / 16) + 4) * 2^-23) S for the k used here, or
   (k + 4) * 2^-24 S: the larger of the two is taken.
 * 16-bit types: exact products, the same sums, one rounding of the result
   (half a step), and in a backward pass with an activation one rounding of dz.
"""
import itertools

import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
ACTS = ["none", "relu", "tanh", "silu", "gelu"]


@pytest.fixture(scope="module", autouse=True)
def _fault_free():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    from flashlog_b200 import ops
    yield
    assert not ops.gemm_fault()


def half(dt):
    return torch.finfo(dt).eps / 2


def sum_tol(k):
    return max(4 * 2.0 ** -22 + (3 * -(-k // 16) + 4) * 2.0 ** -23, (k + 4) * 2.0 ** -24)


def act64(z, act):
    return {"none": lambda t: t, "relu": torch.relu, "tanh": torch.tanh, "silu": torch.nn.functional.silu,
            "gelu": torch.nn.functional.gelu}[act](z)


def make(rows, k, n, dt, seed=0, res=False, bias=True, std=1.0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    x, w = (r(rows, k) * std).to(dt).cuda(), (r(n, k) * k ** -0.5).to(dt).cuda()
    return x, w, r(n).to(dt).cuda() if bias else None, r(rows, n).to(dt).cuda() if res else None


def forward64(x, w, b, res, act):
    z = x.double() @ w.double().T
    if b is not None:
        z = z + b.double()
    y = act64(z, act)
    return z, y if res is None else y + res.double()


def assert_forward(y, x, w, b, res, act):
    z, want = forward64(x, w, b, res, act)
    S = x.double().abs() @ w.double().abs().T
    if b is not None:
        S = S + b.double().abs()
    # slopes are at most 1.13; the functions and the final sum cost a few steps of fp32 each
    tol = 1.13 * sum_tol(x.shape[1]) * S + 8 * 2.0 ** -24 * (z.abs() + want.abs()) + half(y.dtype) * want.abs() + 1e-30
    if y.dtype == torch.float16:
        tol = tol + 2.0 ** -25  # subnormal results
    err = (y.double() - want).abs()
    assert y.dtype == x.dtype and y.shape == want.shape
    assert bool((err <= tol).all()), float((err / tol).max())


SHAPES = [(1, 1, 1), (1, 128, 475), (9, 128, 475), (16, 7, 29), (17, 65, 33), (64, 100, 130), (128, 64, 128),
          (257, 129, 255), (300, 1024, 1645), (1152, 128, 475), (513, 40, 2000)]


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_forward_shapes(shape, dt):
    from flashlog_b200 import attention
    x, w, b, res = make(*shape, DT[dt], res=True)
    assert_forward(attention.linear(x, w, b, res), x, w, b, res, "none")
    assert_forward(attention.linear(x, w), x, w, None, None, "none")


@pytest.mark.parametrize("dt,act", list(itertools.product(DT, ACTS)))
def test_forward_activations(dt, act):
    from flashlog_b200 import attention
    for rows, k, n in ((5, 33, 70), (200, 96, 300)):
        x, w, b, res = make(rows, k, n, DT[dt], seed=3, res=True, std=2.0)
        assert_forward(attention.linear(x, w, b, res, activation=act), x, w, b, res, act)


def backward64(x, w, b, res, act, gy):
    t = [None if v is None else v.double().requires_grad_() for v in (x, w, b, res)]
    z = t[0] @ t[1].T
    if b is not None:
        z = z + t[2]
    y = act64(z, act)
    if res is not None:
        y = y + t[3]
    got = torch.autograd.grad(y, [v for v in t if v is not None], gy.double())
    it = iter(got)
    z = z.detach()
    zz = z.clone().requires_grad_()
    slope = torch.autograd.grad(act64(zz, act).sum(), zz)[0]
    return [None if v is None else next(it) for v in t], z, slope


@pytest.mark.parametrize("dt,act", [(d, a) for d in DT for a in ACTS])
@pytest.mark.parametrize("shape", [(1, 5, 9), (13, 128, 475), (70, 33, 129), (300, 72, 520)], ids=str)
def test_backward(shape, dt, act):
    from flashlog_b200 import attention
    rows, k, n = shape
    x, w, b, res = make(rows, k, n, DT[dt], seed=5, res=True)
    gy = torch.randn(rows, n, generator=torch.Generator().manual_seed(9)).to(DT[dt]).cuda()
    leaves = [v.clone().requires_grad_() for v in (x, w, b, res)]
    y = attention.linear(*leaves, activation=act)
    dx, dw, db, dr = torch.autograd.grad(y, leaves, gy)
    (ex, ew, eb, er), z, slope = backward64(x, w, b, res, act, gy)
    # z is off by z_off, which moves the slope by at most 1.13 of it (every second derivative is below
    # 1.13); relu's slope is 0 or 1 for a z within z_off of its step
    S = x.double().abs() @ w.double().abs().T + b.double().abs()
    z_off = sum_tol(k) * S
    g = gy.double().abs()
    off = (1.13 * z_off + 16 * 2.0 ** -24) * g if act not in ("none", "relu") else torch.zeros_like(g)
    if act == "relu":
        off = torch.where(z.abs() <= z_off, g, off)
    if act != "none" and DT[dt] != torch.float32:
        off = off + half(DT[dt]) * (g * slope.abs()) + (2.0 ** -25 if dt == "fp16" else 0)
    d = g * slope.abs()
    sub = 2.0 ** -25 if dt == "fp16" else 1e-30
    for got, want, tol in (
            (dx, ex, off @ w.double().abs() + sum_tol(n) * (d @ w.double().abs())),
            (dw, ew, off.T @ x.double().abs() + sum_tol(rows) * (d.T @ x.double().abs())),
            (db, eb, off.sum(0) + (rows + 4) * 2.0 ** -24 * d.sum(0))):
        tol = tol + half(DT[dt]) * want.abs() + sub
        err = (got.double() - want).abs()
        assert got.dtype == DT[dt] and got.shape == want.shape
        assert bool((err <= tol).all()), float((err / tol).max())
    assert torch.equal(dr, gy)


# ---- what a caller may hand in ------------------------------------------------------------------
def test_strides_and_leading_dimensions():
    from flashlog_b200 import attention
    g = torch.Generator().manual_seed(21)
    r = lambda *s: torch.randn(*s, generator=g).cuda()  # noqa: E731
    for rows, k, n, dt in ((70, 48, 90, torch.float32), (300, 264, 520, torch.float32), (300, 264, 520, torch.bfloat16),
                           (5, 33, 70, torch.float16)):
        wide, tall = r(rows, k + 13).to(dt), r(k, n).to(dt)
        x, w = wide[:, 5:5 + k], tall.T  # a slice of wider rows (odd offset); a transposed weight
        res = r(n, rows).to(dt).T
        bias = r(2 * n).to(dt)[::2]
        y = attention.linear(x, w, bias, residual=res, activation="tanh")
        assert_forward(y, x, w, bias, res, "tanh")
        y3 = attention.linear(x.reshape(5, rows // 5, k), w, bias, residual=res.reshape(5, rows // 5, n), activation="tanh")
        assert torch.equal(y3.reshape(rows, n), y)
        one = attention.linear(x[0], w, bias)
        assert one.shape == (n,)
        assert_forward(one[None], x[:1], w, bias, None, "none")
        expanded = x[:1].expand(rows, k)
        assert_forward(attention.linear(expanded, w), expanded, w, None, None, "none")


def test_empty_rows():
    from flashlog_b200 import attention
    x, w, b, _ = make(4, 8, 16, torch.float32)
    e = x[:0].clone().requires_grad_()
    w.requires_grad_()
    b.requires_grad_()
    y = attention.linear(e, w, b)
    assert y.shape == (0, 16)
    gx, gw, gb = torch.autograd.grad(y.sum(), [e, w, b])
    assert gx.shape == (0, 8) and not gw.any() and not gb.any()


@pytest.mark.parametrize("rows", [7, 60, 700])
def test_lines_of_very_different_sizes(rows):
    """fp32 lines keep their own accuracy: rows and weight rows scaled by powers of two from 2^-90 to 2^90."""
    from flashlog_b200 import attention
    x, w, b, _ = make(rows, 300, 401, torch.float32, seed=8, bias=False)
    ex = torch.randint(-45, 46, (rows, 1), generator=torch.Generator().manual_seed(1)).cuda()
    ew = torch.randint(-45, 46, (401, 1), generator=torch.Generator().manual_seed(2)).cuda()
    xs, ws = torch.ldexp(x, 2 * ex), torch.ldexp(w, -2 * ew)
    y = attention.linear(xs, ws)
    want = xs.double() @ ws.double().T
    S = xs.double().abs() @ ws.double().abs().T
    tol = sum_tol(300) * S + half(torch.float32) * want.abs()
    # results that fp32 holds: partial sums are at most S, so a sum with S beyond fp32 may overflow on its way
    fits = (S < 3e38) & (S > 1e-30)
    assert bool(((y.double() - want).abs() <= tol)[fits].all())


def test_nonfinite_inputs_stay_in_their_rows():
    from flashlog_b200 import attention
    for rows, k, n in ((6, 40, 50), (300, 512, 700)):
        x, w, b, _ = make(rows, k, n, torch.float32, seed=12)
        clean = attention.linear(x, w, b)
        x[2, 3], x[4, 1] = float("nan"), float("inf")
        y = attention.linear(x, w, b)
        keep = [i for i in range(rows) if i not in (2, 4)]
        assert torch.equal(y[keep], clean[keep])
        assert bool(y[2].isnan().all()) and not bool(y[4].isfinite().any())


def test_other_stream_and_capture():
    """On a stream of the caller's, and captured with its gradients: the same bits."""
    from flashlog_b200 import attention
    for rows, k, n in ((9, 128, 475), (300, 256, 475)):
        x, w, b, _ = make(rows, k, n, torch.float32, seed=31)
        gy = torch.randn(rows, n, generator=torch.Generator().manual_seed(5)).cuda()

        def run(leaves):
            y = attention.linear(*leaves, activation="silu")
            return (y.detach(), *torch.autograd.grad(y, leaves, gy))

        first = run([t.clone().requires_grad_() for t in (x, w, b)])
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            leaves = [t.clone().requires_grad_() for t in (x, w, b)]
            second = run(leaves)
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                captured = run(leaves)
        torch.cuda.current_stream().wait_stream(s)
        for _ in range(2):
            g.replay()
        torch.cuda.synchronize()
        for a, c, d in zip(first, second, captured):
            assert torch.equal(a, c) and torch.equal(a, d)


def test_two_captured_graphs_do_not_share_memory():
    from flashlog_b200 import attention
    sets = [make(300, 200 + 8 * i, 333, torch.float32, seed=40 + i) for i in range(2)]
    want = [attention.linear(x, w, b) for x, w, b, _ in sets]
    graphs, outs = [], []
    s = torch.cuda.Stream()
    for x, w, b, _ in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            outs.append(attention.linear(x, w, b))
        graphs.append(g)
    for order in ((0, 1), (1, 0)):
        for i in order:
            graphs[i].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for o, w in zip(outs, want))


def test_gradient_against_differences():
    from flashlog_b200 import attention
    x, w, b, _ = make(6, 20, 15, torch.float32, seed=50)
    x.requires_grad_()
    gy = torch.randn(6, 15, generator=torch.Generator().manual_seed(3)).cuda()
    g, = torch.autograd.grad(attention.linear(x, w, b, activation="gelu"), [x], gy)
    d = torch.zeros_like(x)
    d[1, 2] = 2.0 ** -6
    with torch.no_grad():
        f = [(attention.linear(x + s * d, w, b, activation="gelu").double() * gy.double()).sum() for s in (1, -1)]
    # cubic term: h^2 / 6 of a third derivative below 2 per weight (sum |gy w^3| < 30 here); roundings 15 * 2^-24 / h
    assert abs(float((f[0] - f[1]) / 2.0 ** -5) - float(g[1, 2])) <= 30 * 2 * 2.0 ** -12 / 6 + 100 * 2.0 ** -24 * 2.0 ** 6


def test_only_wanted_gradients():
    from flashlog_b200 import attention
    for rows in (40, 700):
        x, w, b, res = make(rows, 300, 420, torch.float32, seed=60, res=True)
        gy = torch.randn(rows, 420, generator=torch.Generator().manual_seed(6)).cuda()
        full = [t.clone().requires_grad_() for t in (x, w, b, res)]
        all4 = torch.autograd.grad(attention.linear(*full, activation="relu"), full, gy)
        for k in range(4):
            leaves = [x, w, b, res]
            leaves[k] = leaves[k].clone().requires_grad_()
            got, = torch.autograd.grad(attention.linear(*leaves, activation="relu"), [leaves[k]], gy)
            assert torch.equal(got, all4[k])


def test_second_derivative_is_an_error():
    """Asking for a differentiable gradient is fine; differentiating it says so instead of giving zeros."""
    from flashlog_b200 import attention
    x, w, b, _ = make(5, 6, 7, torch.float32)
    x.requires_grad_()
    g, = torch.autograd.grad(attention.linear(x, w, b, activation="tanh").square().sum(), [x], create_graph=True)
    assert g.requires_grad
    with pytest.raises(RuntimeError, match="once"):
        torch.autograd.grad(g.sum(), [x])
    z = torch.randn(4, 9, device="cuda", requires_grad=True)
    g, = torch.autograd.grad(attention.relation_weights(z).square().sum(), [z], create_graph=True)
    with pytest.raises(RuntimeError, match="once"):
        torch.autograd.grad(g.sum(), [z])
