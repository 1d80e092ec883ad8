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
