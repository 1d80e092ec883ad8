"""The temperature of the relation weights: w = 2^((u - max) log2 e / tau), whose factor is rounded once."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


# the forms of the kernel: short rows, rows that stay in registers, few long rows, two passes
@pytest.mark.parametrize("rows,n", [(50, 40), (50, 1000), (400, 5000), (1, 29649), (400, 40000)])
def test_weights_far_below_the_largest(rows, n):
    """Two finite logits, 0 and -d, whose difference is exact.  With X = d / tau the exponent is off by one half step
    (2^-24) of X for the factor and one for the product, the power by 2^-22, and the sum, its reciprocal and the last
    product by two half steps each at most."""
    from flashlog_b200 import attention
    worst = 0.0
    g = torch.Generator().manual_seed(n)
    for _ in range(40):
        tau = float(0.05 + 3.0 * torch.rand((), generator=g, dtype=torch.float64))
        d = torch.linspace(20.0, 80.0, rows, dtype=torch.float64) * tau
        z = torch.full((rows, n), -math.inf)
        z[:, 0] = 0.0
        z[:, n - 1] = -d.float()
        w = attention.relation_weights(z.cuda(), tau=tau)[:, n - 1].double().cpu()
        x = -z[:, n - 1].double() / tau
        want = torch.exp(-x) / (1 + torch.exp(-x))
        bound = 2 * 2.0 ** -24 * x + 2.0 ** -22 + 6 * 2.0 ** -24
        worst = max(worst, float(((w / want - 1).abs() / bound).max()))
    assert worst <= 1.0, worst
