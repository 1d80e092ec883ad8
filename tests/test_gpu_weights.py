"""attention.relation_weights against its formula in 64 bits.

Error bounds.  A value u is off by at most 8 roundings of the largest |z|,
penalty or bias U; its exponent (top - u) / tau = A by as much over tau and two
more roundings; exp, the sum (at most 16 terms per thread, then 25 levels) and
the quotient add under 60 roundings: a weight is off by at most
rel = 2^-24 (16 U / tau + 4 A + 60) of itself.  A gradient w (g - dot) / tau is
off by rel (2 |g - dot| + 2 sum |w g|) w / tau and half a step of its dtype.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
NS = [1, 25, 32, 75, 128, 129, 475, 513, 1024, 1645, 2049, 4096, 4097, 8193, 29649, 65536]


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")


def plain64(z, tau=1.0, mask=None, states=None, bias=None, history=None, repetition=1.0, frequency=0.0, presence=0.0):
    """(u, slope, w) of 2-D inputs in 64 bits."""
    z = z.double()
    rows, n = z.shape
    u, slope = z, torch.ones_like(z)
    if history is not None:
        count = torch.zeros_like(z)
        for j in range(history.shape[1]):
            h = history[:, j]
            ok = (h >= 0) & (h < n)
            count[torch.arange(rows, device=z.device)[ok], h[ok]] += 1
        slope = torch.where(count > 0, torch.where(z > 0, 1 / repetition, repetition), 1.0)
        u = torch.where(count > 0, torch.where(z > 0, z / repetition, z * repetition), z)
        u = u - frequency * count - presence * (count > 0)
    if bias is not None:
        u = u + bias.double()
    if mask is not None:
        if states is None:
            allowed = mask.bool().expand(rows, n)
        else:
            inside = (states >= 0) & (states < mask.shape[0])
            allowed = mask.bool()[torch.where(inside, states, 0)] & inside[:, None]
        u = torch.where(allowed, u, -torch.inf)
    top = u.amax(1, keepdim=True)
    empty = top == -torch.inf
    w = torch.softmax(torch.where(empty, 0.0, u) / tau, 1)
    return u, slope, torch.where(empty, 0.0, w)


def relative(u, tau):
    fin = torch.isfinite(u)
    zero = torch.zeros_like(u)
    U = torch.where(fin, u.abs(), zero).amax(1, keepdim=True) + 4.0
    A = torch.where(fin, u.amax(1, keepdim=True) - u, zero).nan_to_num(posinf=0.0) / tau
    return 2.0 ** -24 * (16 * U / tau + 4 * A + 60)


def inputs(rows, n, dt, seed=0, states=7, hist=5, bias="shared"):
    g = torch.Generator().manual_seed(seed)
    z = (torch.randn(rows, n, generator=g) * 2).to(dt)
    kw = {}
    if states:
        m = torch.rand(states, n, generator=g) < 0.4
        m[0] = False
        kw["mask"] = m
        kw["states"] = torch.randint(-1, states + 1, (rows,), generator=g)
    if hist:
        kw["history"] = torch.randint(-1, n + 1, (rows, hist), generator=g)
        kw["history"][:, hist // 2:] = kw["history"][:, :1]  # repeated entries
    if bias:
        kw["bias"] = (torch.randn(*((n,) if bias == "shared" else (rows, n)), generator=g) * 0.5).to(dt)
    return z.cuda(), {k: v.cuda() for k, v in kw.items()}


RULES = dict(tau=0.8, repetition=1.3, frequency=0.2, presence=0.4)


def check(z, kw, rules, backward=True):
    from flashlog_b200 import attention
    lz = z.clone().requires_grad_()
    lb = kw["bias"].clone().requires_grad_() if "bias" in kw else None
    w = attention.relation_weights(lz, **{**kw, **({"bias": lb} if lb is not None else {})}, **rules)
    u, slope, want = plain64(z, **kw, **rules)
    tau = rules.get("tau", 1.0)
    rel = relative(u, tau)
    assert w.dtype == torch.float32
    assert torch.equal(w == 0, want < 2.0 ** -150) or bool((w[(w == 0) != (want < 2.0 ** -150)] < 1e-36).all())
    err = (w.double() - want).abs()
    assert bool((err <= rel * want + 1e-37).all()), float((err / (rel * want + 1e-37)).max())
    if not backward:
        return w
    g = torch.randn(z.shape, generator=torch.Generator().manual_seed(77)).cuda()
    got = torch.autograd.grad(w, [lz] + ([lb] if lb is not None else []), g)
    gd = g.double()
    dot = (gd * want).sum(1, keepdim=True)
    du = want * (gd - dot) / tau
    off = rel * want * (2 * (gd - dot).abs() + 2 * (gd * want).abs().sum(1, keepdim=True)) / tau
    step = torch.finfo(z.dtype).eps / 2
    sub = 2.0 ** -25 if z.dtype == torch.float16 else 2.0 ** -134  # half a subnormal step (bf16's and fp32's least)
    e = (got[0].double() - du * slope).abs()
    tol = off * slope * 1.01 + step * (du * slope).abs() + sub
    assert got[0].dtype == z.dtype and bool((e <= tol).all()), float((e / tol).max())
    if lb is not None:
        if lb.dim() == 1:
            want_b, off_b = du.sum(0), off.sum(0) + (z.shape[0] + 4) * 2.0 ** -24 * du.abs().sum(0)
        else:
            want_b, off_b = du, off
        e = (got[1].double() - want_b).abs()
        tol = off_b + step * want_b.abs() + sub
        assert got[1].dtype == z.dtype and bool((e <= tol).all()), float((e / tol).max())
    return w


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("n", NS)
def test_widths(n, dt):
    for rows in (1, 5, 70):
        z, kw = inputs(rows, n, DT[dt], seed=n)
        check(z, kw, RULES)


@pytest.mark.parametrize("n", [25, 475, 1645, 29649])
def test_parts_alone(n):
    z, kw = inputs(11, n, torch.float32, seed=4)
    check(z, {}, {})
    check(z, {"bias": kw["bias"]}, {"tau": 2.0})
    check(z, {"history": kw["history"]}, {"presence": 1.0})
    check(z, {"history": kw["history"]}, {"repetition": 0.7, "frequency": -0.1})
    check(z, {"mask": kw["mask"], "states": kw["states"]}, {})
    check(z, {"mask": kw["mask"][1].to(torch.uint8)}, {})
    z, kw = inputs(11, n, torch.bfloat16, seed=5, bias="full")
    check(z, kw, RULES)
    m = torch.rand(11, n, generator=torch.Generator().manual_seed(1)).cuda() < 0.2
    check(z, {"mask": m}, {})
