"""Heads of very many rows and very few columns."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,k,n,dt", [(2_200_000, 8, 4, torch.float32), (3_000_001, 1, 25, torch.float32),
                                         (2_200_003, 8, 1, torch.float16), (2_097_121, 2, 3, torch.bfloat16),
                                         (20, 3, 2_200_001, torch.float32)], ids=str)
def test_many_rows(rows, k, n, dt):
    """More than 65535 tiles of 32 rows (and as many columns); every gradient."""
    from flashlog_b200 import attention
    g = torch.Generator(device="cuda").manual_seed(rows)
    draw = lambda *s: torch.randn(*s, generator=g, device="cuda").to(dt).requires_grad_()  # noqa: E731
    x, w, b, res = draw(rows, k), draw(n, k), draw(n), draw(rows, n)
    gy = torch.randn(rows, n, generator=g, device="cuda").to(dt)
    y = attention.linear(x, w, b, residual=res, activation="relu")
    got = torch.autograd.grad(y, (x, w, b, res), gy)
    X, W, B, R, G = (t.detach().double() for t in (x, w, b, res, gy))
    half, fp32 = torch.finfo(dt).eps / 2, 2.0 ** -24
    z = X @ W.T + B
    size = X.abs() @ W.abs().T + B.abs()  # a sum of k + 1 terms is off by at most (k + 1) roundings of this
    # the last size is not small: its product runs on two fp16 planes an operand.  Both are off by at most 2^-22 of their
    # value, and lo * lo, at most 2^-22 of the product, is left out: 3 * 2^-22 of each term, 12 roundings of fp32
    planes = 12 if dt == torch.float32 and rows * n * k > 96_000_000 else 0
    off = (k + 1 + planes) * fp32 * size
    tiny = 2.0 ** -24
    assert bool(((y.detach().double() - (z.clamp_min(0) + R)).abs() <=
                 (1 + half) * (off + fp32 * (size + R.abs())) + half * (z.clamp_min(0) + R).abs() + tiny).all())
    # where z is nearer to 0 than its error, the slope may be either
    sure = z.abs() > off
    dz = torch.where(z > 0, G, 0.0)
    loose = torch.where(sure, 0.0, G.abs())

    def close(got, want, terms, unsure, count):
        """Sums of count terms, added in parts: each part's and the parts' sums are off by at most their lengths."""
        bound = (1 + half) * ((count + planes) * fp32 * terms + unsure) + half * want.abs() + tiny
        return bool(((got.double() - want).abs() <= bound).all())

    chunk = lambda length: length / max(1, min(64, length // 64)) + 96  # noqa: E731
    assert close(got[0], dz @ W, dz.abs() @ W.abs(), loose @ W.abs(), chunk(n))
    assert close(got[1], dz.T @ X, dz.abs().T @ X.abs(), loose.T @ X.abs(), chunk(rows))
    assert close(got[2], dz.sum(0), dz.abs().sum(0), loose.sum(0), chunk(rows))
    assert torch.equal(got[3], gy)
