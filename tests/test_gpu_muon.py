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


def test_decaying_spectrum():
    """A strong low-rank part over noise, the case that single 16-bit planes lose (see the kernel's comment)."""
    from flashlog_b200 import muon
    g = torch.Generator().manual_seed(4)
    for m, n in ((200, 210), (128, 640)):
        u = torch.randn(m, 3, generator=g) @ torch.randn(3, n, generator=g) + 1e-3 * torch.randn(m, n, generator=g)
        u = u.cuda()
        got, (want, _, _) = muon.orthogonalize(u), exact(u)
        # what plain fp32 steps give is off by 5e-5 here; within ten times that
        assert float((got.double() - want).norm() / want.norm()) <= 5e-4


@pytest.mark.parametrize("shape", [(20, 30), (300, 310), (100, 900)], ids=str)
def test_zero_tiny_huge_and_nonfinite(shape):
    from flashlog_b200 import muon
    u = matrices(5, *shape, seed=9)
    u[0] = 0
    u[1] *= 1e25
    u[2] *= 1e-20
    u[3, 2, 3] = float("nan")
    o = muon.orthogonalize(u)
    assert not bool(o[0].any())
    assert bool(o[3].isnan().any()) and bool(o[[1, 2, 4]].isfinite().all())
    for k in (1, 2, 4):
        assert_close(o[k:k + 1], u[k:k + 1])


@pytest.mark.parametrize("steps,c", [(1, C), (2, C), (3, (1.5, -0.5, 0.0)), (8, C), (5, (2.0, -1.5, 0.5))])
@pytest.mark.parametrize("shape", [(30, 40), (200, 208), (100, 700)], ids=str)
def test_steps_and_coefficients(shape, steps, c):
    from flashlog_b200 import muon
    u = matrices(1, *shape, seed=steps)
    assert_close(muon.orthogonalize(u, steps=steps, coefficients=c), u, steps, c)


@pytest.mark.parametrize("shape", [(24, 25), (130, 140), (140, 900)], ids=str)
def test_strided_batches(shape):
    """Views of a table [m, T, N, n], transposed matrices, more batch dimensions than the kernels know."""
    from flashlog_b200 import muon
    m, n = shape
    table = matrices(m, 2, 3, n, seed=2)
    view = table.permute(1, 2, 0, 3)
    want = muon.orthogonalize(view.contiguous())
    assert torch.equal(muon.orthogonalize(view), want)
    torch.testing.assert_close(muon.orthogonalize(view.mT), want.mT, rtol=1e-4, atol=1e-4)
    odd = view[None].expand(2, -1, -1, -1, -1)
    assert torch.equal(muon.orthogonalize(odd), want[None].expand(2, -1, -1, -1, -1))
    assert muon.orthogonalize(view[:0]).shape == (0, 3, m, n)


def muon64(p, g, mo, lr, beta, nesterov, wd, scale):
    p, g, mo = p.double(), g.double(), mo.double()
    m2 = beta * mo + g
    o, _, _ = exact(g + beta * m2 if nesterov else m2)
    return p * (1 - lr * wd) - lr * scale * o, m2


@pytest.mark.parametrize("shape", [(24, 25), (300, 140), (200, 230), (90, 800)], ids=str)
@pytest.mark.parametrize("nesterov", [True, False])
def test_muon_update(shape, nesterov):
    from flashlog_b200 import muon
    m, n = shape
    p, g, mo = (matrices(2, m, n, seed=s) for s in (1, 2, 3))
    kw = dict(lr=0.1, beta=0.9, nesterov=nesterov, weight_decay=0.05)
    want_p, want_m = muon64(p, g, mo, 0.1, 0.9, nesterov, 0.05, max(1.0, m / n) ** 0.5)
    p0, m0 = p.clone(), mo.clone()
    p2, m2 = muon.muon_update(p, g, mo, **kw)
    assert torch.equal(p, p0) and torch.equal(mo, m0)
    # momentum: one rounding of each operation; parameter: three, and lr * scale of the orthogonalised update's 2e-5
    assert bool(((m2.double() - want_m).abs() <= 2 * 2.0 ** -24 * (0.9 * mo.double().abs() + g.double().abs())).all())
    tol = 4 * 2.0 ** -24 * p.double().abs().max() * math.sqrt(m * n) + 0.1 * max(1.0, m / n) ** 0.5 * 2e-5 * math.sqrt(min(m, n)) * 1.3
    assert float((p2.double() - want_p).flatten(1).norm(dim=1).max()) <= tol
    assert muon.muon_update_(p, g, mo, **kw) is p
    assert torch.equal(p, p2) and torch.equal(mo, m2)
    # strided tensors of different layouts, in place
    strided = [t.permute(1, 0, 2).contiguous().permute(1, 0, 2) for t in (p0, m0)]
    muon.muon_update_(strided[0], g.mT.contiguous().mT, strided[1], **kw)
    assert torch.equal(strided[0], p2) and torch.equal(strided[1], m2)


@pytest.mark.parametrize("shape", [(24, 25), (200, 230), (90, 800)], ids=str)
def test_closed_gate_changes_nothing(shape):
    from flashlog_b200 import muon
    p, g, mo = (matrices(2, *shape, seed=s) for s in (1, 2, 3))
    g[:] = float("nan")
    gate = torch.zeros(1, device="cuda")
    p2, m2 = muon.muon_update(p, g, mo, lr=0.1, weight_decay=0.1, gate=gate)
    assert torch.equal(p2, p) and torch.equal(m2, mo)
    gate.fill_(1.0)
    g = matrices(2, *shape, seed=7)
    a = muon.muon_update(p, g, mo, lr=0.1, weight_decay=0.1, gate=gate)
    b = muon.muon_update(p, g, mo, lr=0.1, weight_decay=0.1)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("shape", [(24, 25), (200, 230), (90, 800), (64, 4000)], ids=str)
def test_same_bits_on_other_streams_and_in_graphs(shape):
    """Repeated, on two streams at once, and replayed from two graphs: one result."""
    from flashlog_b200 import muon
    u = matrices(3, *shape, seed=5)
    want = muon.orthogonalize(u)
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(muon.orthogonalize(u))
    graphs = []
    for s in streams:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            outs.append(muon.orthogonalize(u))
        graphs.append(g)
    for s, g in zip(streams, graphs):
        with torch.cuda.stream(s):
            g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


def test_optimizer():
    from flashlog_b200 import attention, muon
    g = torch.Generator().manual_seed(6)
    w = torch.randn(70, 50, generator=g).cuda().requires_grad_()
    b = torch.randn(3, 20, 30, generator=g).cuda().requires_grad_()
    idle = torch.randn(5, 6, generator=g).cuda().requires_grad_()
    opt = muon.Muon([{"params": [w, idle]}, {"params": [b], "lr": 0.1}], lr=0.05, weight_decay=0.01)
    x = torch.randn(8, 50, generator=g).cuda()
    want = [w.detach().clone(), b.detach().clone()]
    mom = [torch.zeros_like(t) for t in want]
    for _ in range(3):
        opt.zero_grad()
        (attention.linear(x, w).square().sum() + (b ** 3).sum()).backward()
        for i, (t, lr) in enumerate(((w, 0.05), (b, 0.1))):
            muon.muon_update_(want[i], t.grad, mom[i], lr=lr, weight_decay=0.01)
        opt.step()
    assert torch.equal(w.detach(), want[0]) and torch.equal(b.detach(), want[1])
    assert idle not in opt.state or not opt.state[idle]


@pytest.mark.parametrize("shape", [(65, 129), (300, 520), (1025, 1600), (2, 700, 1100), (1200, 260), (1100, 4000)], ids=str)
def test_short_products_in_narrow_tiles(shape):
    """Few matrices of the Gram form: their short products and the last one are two launches."""
    from flashlog_b200 import muon
    u = matrices(*shape, seed=9)
    assert_close(muon.orthogonalize(u), u)
    assert_close(muon.orthogonalize(u, steps=1), u, steps=1)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = muon.orthogonalize(u)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, muon.orthogonalize(u))
