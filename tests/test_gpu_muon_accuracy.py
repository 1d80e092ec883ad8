"""Newton-Schulz products on matrices whose singular values decay, as those of gradients do.

The reference is the polynomial of the singular values in 64 bits, the measure what the same steps in plain fp32 are
off by.  A stored matrix has two fp16 planes, 22 to 23 bits where fp32 has 24: off by at most 2^-23, two of fp32's
half steps of 2^-24.  A chunk of a product is at most 12 additions of the long form (24 of the nearly square one) to an
accumulator that the tensor cores truncate: each loses between 0 and 2^-23 of the sum so far, 2^-24 on average, and the
sum grows from 0 to its end, so one-sided sums lose 12 * 2^-24 / 2 of it, six half steps.  (Chunks are added with
rounding, and in the nearly square form nothing is squared, so that the doubled loss is not amplified.)  Plain fp32
rounds each stored value by up to one half step, so the result may be off by 2 + 6 = 8 times its error.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

C = (3.4445, -4.7750, 2.0315)


def steps_in(x, steps, dtype):
    x = x.to(dtype)
    for _ in range(steps):
        a = x @ x.mT
        x = C[0] * x + (C[1] * a + C[2] * (a @ a)) @ x
    return x


def spectrum(kind, m, n, seed):
    g = torch.Generator().manual_seed(seed)
    if kind == "rank 3":
        return torch.randn(m, 3, generator=g, dtype=torch.float64) @ torch.randn(3, n, generator=g, dtype=torch.float64) \
            + 1e-2 * torch.randn(m, n, generator=g, dtype=torch.float64)
    u, _ = torch.linalg.qr(torch.randn(m, m, generator=g, dtype=torch.float64))
    v, _ = torch.linalg.qr(torch.randn(n, m, generator=g, dtype=torch.float64))
    i = torch.arange(1, m + 1, dtype=torch.float64)
    s = {"1/i": 1 / i, "1/i^2": i ** -2, "exp": torch.exp(-10 * i / m)}[kind]
    return (u * s) @ v.mT


# long matrices, turned ones, and nearly square ones (the direct form)
@pytest.mark.parametrize("shape", [(128, 256), (128, 640), (256, 400), (640, 128), (130, 3000), (200, 210)], ids=str)
@pytest.mark.parametrize("kind", ["1/i", "1/i^2", "exp", "rank 3"])
@pytest.mark.parametrize("steps", [5, 7])
def test_decaying_spectra_are_as_close_as_in_fp32(shape, kind, steps):
    from flashlog_b200 import muon
    lo, hi = sorted(shape)
    u = spectrum(kind, lo, hi, seed=lo + hi).float()
    x = u.double() / (torch.linalg.matrix_norm(u.double()) + 1e-7)
    want = steps_in(x, steps, torch.float64)
    plain = steps_in(x, steps, torch.float32).double()
    u = (u.mT if shape[0] > shape[1] else u).cuda()
    got = muon.orthogonalize(u, steps=steps).double().cpu()
    got = got.mT if shape[0] > shape[1] else got
    scale = torch.linalg.matrix_norm(want)
    error, allowed = (torch.linalg.matrix_norm(t - want) / scale for t in (got, plain))
    print(f"{shape} {kind} {steps} steps: {float(error):.2e}, plain fp32 {float(allowed):.2e}")
    assert float(error) <= 8 * float(allowed)


@pytest.mark.parametrize("shape", [(128, 640), (200, 210), (20, 30)], ids=str)
def test_many_steps(shape):
    """As many steps as are allowed: small singular values grow by 1.5^64 at most, and end at 1."""
    from flashlog_b200 import muon
    u = spectrum("1/i", *shape, seed=7).float()
    w, _, v = torch.linalg.svd(u.double(), full_matrices=False)
    got = muon.orthogonalize(u.cuda(), steps=64, coefficients=(1.5, -0.5, 0.0)).double().cpu()
    # at 1 the polynomial's slope is 0: what is left are the last step's roundings, three products of matrices of
    # norm 1 in the spectral sense, each off by at most 4 * 2^-22 of its factors' Frobenius norms, sqrt(m) each
    assert float((got - w @ v).norm()) <= 3 * 4 * 2.0 ** -22 * shape[0]


@pytest.mark.parametrize("turned", [False, True])
def test_very_long_matrices(turned):
    """5 million rows of 8: near the steps in 64 bits, as other sizes are (white noise: nothing is amplified)."""
    from flashlog_b200 import muon
    g = torch.Generator(device="cuda").manual_seed(2)
    u = torch.randn(8, 5_000_000, generator=g, device="cuda")
    x = u.double() / (torch.linalg.matrix_norm(u.double()) + 1e-7)
    want = steps_in(x, 5, torch.float64)
    got = muon.orthogonalize(u.mT.contiguous()).mT if turned else muon.orthogonalize(u)
    assert float(torch.linalg.matrix_norm(got.double() - want) / torch.linalg.matrix_norm(want)) <= 2e-5
