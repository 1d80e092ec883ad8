"""fp32 heads whose lines hold values of very different sizes: a huge feature that a weight of 0 leaves out must not cost
the small ones their bits.

Error bound, as for other heads: an operand's value is off by at most 2^-22 of it, or 2^-50 of its line's largest where
that is more (times the other operand's sum of magnitudes), lo * lo is dropped, and each of 3 additions per 16 terms and
of the chunks is off by at most 2^-23 of the terms' sum S: (4 * 2^-22 + (3 * ceil(k / 16) + 4) * 2^-23) S, and half a
step of the result.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu


def assert_close(got, a, b):
    """got = a b^T of fp32 matrices."""
    a, b = a.detach().double(), b.detach().double()
    want, terms = a @ b.T, a.abs() @ b.abs().T
    k = a.shape[1]
    bound = (4 * 2.0 ** -22 + (3 * -(-k // 16) + 4) * 2.0 ** -23) * terms + 2.0 ** -24 * want.abs()
    bound += 2.0 ** -50 * (a.abs().amax(1, keepdim=True) * b.abs().sum(1) + a.abs().sum(1, keepdim=True) * b.abs().amax(1))
    err = (got.detach().double() - want).abs()
    assert bool((err <= bound).all()), float((err / bound.clamp_min(1e-300)).max())


def draw(rows, k, seed):
    """Values of 0.5 to 2: none is small by chance."""
    g = torch.Generator().manual_seed(seed)
    return ((0.5 + 1.5 * torch.rand(rows, k, generator=g)) * torch.sign(torch.randn(rows, k, generator=g))).cuda()


@pytest.mark.parametrize("power", [16, 24, 32])
@pytest.mark.parametrize("rows,k,n", [(700, 300, 900), (2304, 1024, 1645)], ids=str)
def test_a_huge_feature_times_zero(rows, k, n, power):
    from flashlog_b200 import attention
    x, w, gy = draw(rows, k, 1), draw(n, k, 2), draw(rows, n, 3)
    x[:, 7] = 2.0 ** power
    w[:, 7] = 0.0
    gy[:, 11] = 2.0 ** power     # in dx, left out by a weight row of 0
    w[11] = 0.0
    gy[5] = gy[5] * 2.0 ** power  # in dweight, left out by a row of x that is 0
    x[5] = 0.0
    x.requires_grad_(), w.requires_grad_()
    y = attention.linear(x, w)
    assert_close(y, x, w)
    dx, dw = torch.autograd.grad(y, (x, w), gy)
    assert_close(dx, gy, w.detach().T.contiguous())
    assert_close(dw, gy.T.contiguous(), x.detach().T.contiguous())
