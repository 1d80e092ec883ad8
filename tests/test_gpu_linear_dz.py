"""Gradients of 16-bit heads with an activation: dz = gy * act'(z) is kept beyond the operands' type.

Error bounds, element by element.  z is an fp32 sum of k terms, in at most k / 16 + 2 additions that truncate at 2^-23 of
the sum's terms; the slopes of the activations change by at most 1.2 per unit of z and are evaluated to 2^-20.  dz has two
planes: off by 2^-18 of it (bf16: 2^-9 of 2^-9) or less (fp16).  A product of length L adds with at most L / 8 + 4
truncations in its two accumulators.  The result is rounded once: half a step of its type, or of its smallest value.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

ROWS, K = 700, 320


def slope(z, act):
    if act == "relu":
        return (z > 0).double()
    if act == "tanh":
        return 1 - torch.tanh(z) ** 2
    if act == "silu":
        t = torch.sigmoid(z)
        return t * (1 + z * (1 - t))
    return 0.5 * (1 + torch.erf(z * 0.5 ** 0.5)) + z * torch.exp(-0.5 * z * z) * (2 * torch.pi) ** -0.5


def case(dt, n, scale, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(ROWS, K, generator=g).to(dt).cuda().requires_grad_()
    w = (torch.randn(n, K, generator=g) * K ** -0.5).to(dt).cuda().requires_grad_()
    b = (torch.randn(n, generator=g) * 0.1).to(dt).cuda().requires_grad_()
    gy = (torch.randn(ROWS, n, generator=g) * scale).to(dt).cuda()
    return x, w, b, gy


@pytest.mark.parametrize("act", ["relu", "tanh", "silu", "gelu"])
@pytest.mark.parametrize("n", [480, 481])
@pytest.mark.parametrize("dt,scale", [(torch.bfloat16, 1.0 / ROWS), (torch.bfloat16, 1e-20), (torch.float16, 1.0),
                                      (torch.float16, 1.0 / ROWS), (torch.float16, 2.0 ** -21)], ids=str)
def test_gradients_are_rounded_once(dt, scale, n, act):
    from flashlog_b200 import attention
    x, w, b, gy = case(dt, n, scale, n)
    dx, dw = torch.autograd.grad(attention.linear(x, w, b, activation=act), (x, w), gy)
    X, W, B, G = (t.detach().double() for t in (x, w, b, gy))
    z = X @ W.T + B
    dz = G * slope(z, act)
    off_z = (K / 16 + 2) * 2.0 ** -23 * (X.abs() @ W.abs().T + B.abs())
    off = G.abs() * (1.2 * off_z + 2.0 ** -20) + 2.0 ** -18 * dz.abs()
    if act == "relu":
        off = 2.0 ** -18 * dz.abs() + torch.where(z.abs() <= off_z, G.abs(), 0.0)
    if dt == torch.float16:
        off = off + 2.0 ** -35  # half of lo's smallest value, 2^-24 / 1024
    half, least = torch.finfo(dt).eps / 2, 2.0 ** -25 if dt == torch.float16 else 1e-38

    def close(got, want, terms, unsure, length):
        inner = unsure + (length / 8 + 4) * 2.0 ** -23 * terms
        bound = (1 + half) * inner + half * want.abs() + least
        err = (got.double() - want).abs()
        assert bool((err <= bound).all()), float((err / bound).max())

    close(dx, dz @ W, dz.abs() @ W.abs(), off @ W.abs(), n)
    close(dw, dz.T @ X, dz.abs().T @ X.abs(), off.T @ X.abs(), ROWS)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
def test_large_and_infinite_gradients(dt):
    """An infinity stays in its row of dx and its row of dweight; fp16 gradients up to the largest value do not overflow
    on the way (GELU's slope is up to 1.13)."""
    from flashlog_b200 import attention
    x, w, b, gy = case(dt, 481, 1.0, 5)
    big = torch.finfo(dt).max if dt == torch.float16 else 1e30
    with torch.no_grad():
        w.mul_(2.0 ** -6)
        b.fill_(1.4)  # where the slope is largest
        gy[3, 5] = float("inf")
        gy[7, 9] = big
        gy[8, 9] = float("nan")
    dx, dw = torch.autograd.grad(attention.linear(x, w, b, activation="gelu"), (x, w), gy)
    want = torch.sign(w[5].detach().double()) * float("inf")
    assert torch.equal(dx[3].double()[w[5] != 0], want[w[5] != 0])
    assert bool(dx[8].isnan().all()) and bool(dw[9].isnan().all())
    rows = torch.ones(ROWS, dtype=torch.bool)
    rows[[3, 8]] = False
    assert bool(dx[rows.cuda()].isfinite().all())
    lines = torch.ones(481, dtype=torch.bool)
    lines[[5, 9]] = False
    assert bool(dw[lines.cuda()].isfinite().all())
    z = x.detach().double()[7] @ w.detach().double().T + 1.4
    row = (gy[7].double() * slope(z, "gelu")) @ w.detach().double()
    assert float(((dx[7].double() - row).abs() / row.abs().max()).max()) <= torch.finfo(dt).eps
