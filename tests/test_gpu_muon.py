"""Newton-Schulz orthogonalisation and the Muon step against the polynomial of
the singular values in 64 bits.

Error bounds.  A relative perturbation d of the matrix in each of the 3 products
of a step is amplified by at most a = 3.4445 per later step in directions whose
singular values are still small (there p(s) = a s, so the signal grows as much)
and by p'(s), at most a, elsewhere.  Products on two fp16 planes are off by
4 * 2^-22 of |A||B| per element; in the Frobenius norm, with independent
roundings, by 4 * 2^-22 of the product's factors' norms.  The bound used is
|O - O64|_F <= 3 steps * 4 * 2^-22 * G + half a step of the dtype * |O|_F,
where G = sum over steps of a^(steps - k) |X_k|_F |P_k|_2 bounds how far a
relative error in step k moves the result, |P_k|_2 <= a.  The Gram form squares
singular values: an error of A relative to its norm |A|_2 = s1^2 moves a
singular value s of X by that over 2 s; for its matrices (white noise with a
few stronger directions, long/short ratio at least 1.5) the condition s1 / s is
computed and enters the bound.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
C = (3.4445, -4.7750, 2.0315)


@pytest.fixture(scope="module", autouse=True)
def _fault_free():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    from flashlog_b200 import ops
    yield
    assert not ops.gemm_fault()


def exact(u, steps=5, c=C, eps=1e-7):
    """The result in 64 bits and the error bound's factor per matrix."""
    u = u.double()
    turned = u.shape[-2] > u.shape[-1]
    x = u.mT if turned else u
    x = x / (torch.linalg.matrix_norm(x, keepdim=True) + eps)
    U, s, V = torch.linalg.svd(x, full_matrices=False)
    t, G = s, torch.zeros(s.shape[:-1], dtype=torch.float64, device=u.device)
    for k in range(steps):
        G = G + abs(c[0]) ** (steps - k) * t.norm(dim=-1)
        t = c[0] * t + c[1] * t ** 3 + c[2] * t ** 5
    o = (U * t[..., None, :]) @ V
    cond = s[..., 0] / s[..., -1].clamp_min(1e-300)
    return (o.mT if turned else o), G, cond


def assert_close(got, u, steps=5, c=C, eps=1e-7):
    want, G, cond = exact(u, steps, c, eps)
    lo, hi = sorted(u.shape[-2:])
    grow = torch.ones_like(cond)
    if hi >= 1.5 * lo and 1.5 * hi / lo + 2 * steps - 1.5 < steps * (1.5 * hi / lo + 0.5):
        grow = cond.clamp(1.0, 2.0 ** 20)
    dt = got.dtype
    tol = 3 * steps * 4 * 2.0 ** -22 * G * grow + torch.finfo(dt).eps / 2 * torch.linalg.matrix_norm(want)
    if dt == torch.float16:
        tol = tol + 2.0 ** -25 * math.sqrt(lo * hi)
    err = torch.linalg.matrix_norm(got.double() - want)
    assert got.shape == u.shape and bool((err <= tol).all()), float((err / tol).max())
    return float((err / torch.linalg.matrix_norm(want)).max())


def matrices(*shape, seed=0):
    g = torch.Generator().manual_seed(seed)
    m, n = shape[-2:]
    r = max(1, min(m, n) // 16)
    strong = torch.randn(*shape[:-1], r, generator=g) @ torch.randn(*shape[:-2], r, n, generator=g)
    return (torch.randn(*shape, generator=g) + strong * (0.5 / r ** 0.5)).cuda()


# one-block sizes, direct (nearly square) and Gram (long) forms, tiles that end inside 128 and 256
SHAPES = [(1, 1), (1, 9), (9, 1), (24, 25), (25, 24), (64, 64), (75, 74), (128, 129), (130, 127), (257, 260),
          (200, 500), (500, 200), (31, 2000), (2000, 31), (474, 475), (700, 720), (129, 1100)]


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_orthogonalize_shapes(shape, dt):
    from flashlog_b200 import muon
    u = matrices(2, *shape, seed=sum(shape)).to(DT[dt])
    rel = assert_close(muon.orthogonalize(u), u)
    # near the rounding of the result itself: each element's is at most half a step (eps / 2) of it, so their
    # Frobenius norm is at most eps / 2 of the result's (2^-8 for bf16, 2^-11 for fp16)
    assert rel <= 2e-5 + (torch.finfo(DT[dt]).eps / 2 if dt != "fp32" else 0.0)
