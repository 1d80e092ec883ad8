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


# ---- masks, infinities, odd inputs ----------------------------------------------------------------
@pytest.mark.parametrize("n", [25, 1645, 8193])
@pytest.mark.parametrize("rows", [6, 300])
def test_empty_rows_and_hidden_garbage(n, rows):
    """Rows whose mask leaves nothing are 0 with gradient 0; masked logits may hold NaN or infinities."""
    from flashlog_b200 import attention
    g = torch.Generator().manual_seed(n)
    z = torch.randn(rows, n, generator=g).cuda()
    mask = torch.rand(rows, n, generator=g).cuda() < 0.5
    mask[0] = False
    mask[1] = False
    mask[1, n // 2] = True  # one left: weight 1
    clean = attention.relation_weights(z, mask=mask)
    dirty = z.clone()
    dirty[~mask] = torch.tensor([float("nan"), float("inf"), -float("inf"), 3e38]).cuda()[
        torch.randint(0, 4, (int((~mask).sum()),), generator=g).cuda()]
    dirty.requires_grad_()
    w = attention.relation_weights(dirty, mask=mask)
    assert torch.equal(w, clean)
    assert not bool(w[0].any()) and float(w[1, n // 2].detach()) == 1.0
    gw = torch.randn(rows, n, generator=g).cuda()
    d, = torch.autograd.grad(w, [dirty], gw)
    assert bool(d.isfinite().all()) and not bool(d[~mask].any()) and not bool(d[0].any())


@pytest.mark.parametrize("n", [25, 475, 4097])
def test_lowest_values_and_infinities(n):
    from flashlog_b200 import attention
    low = torch.finfo(torch.float32).min
    z = torch.randn(5, n, generator=torch.Generator().manual_seed(2)).cuda()
    z[0] = low                      # all at the type's lowest: equal weights
    z[1] = -float("inf")            # nothing left
    z[2, 1:] = low                  # one above
    z[3, 0] = float("nan")
    z[4, 0] = float("inf")
    w = attention.relation_weights(z, tau=0.5)
    torch.testing.assert_close(w[0], torch.full((n,), 1.0 / n, device="cuda"), rtol=1e-5, atol=0)
    assert not bool(w[1].any())
    assert float(w[2, 0]) == 1.0 and not bool(w[2, 1:].any())
    assert bool(w[3].isnan().all()) and bool(w[4].isnan().any())
    # the additive form of a mask: the lowest value as a bias
    z = torch.randn(5, n, generator=torch.Generator().manual_seed(3)).cuda()
    bias = torch.where(torch.rand(n, generator=torch.Generator().manual_seed(4)).cuda() < 0.5, low, 0.0)
    bias[0] = 0.0
    a, b = attention.relation_weights(z, bias=bias), attention.relation_weights(z, mask=bias == 0)
    torch.testing.assert_close(a, b, rtol=1e-6, atol=0)
    for dt in (torch.float16, torch.bfloat16):
        zz = torch.full((2, n), torch.finfo(dt).min, dtype=dt, device="cuda")
        torch.testing.assert_close(attention.relation_weights(zz), torch.full((2, n), 1.0 / n, device="cuda"), rtol=1e-5, atol=0)


@pytest.mark.parametrize("n", [475, 29649])
def test_long_histories(n):
    """More entries than threads and than operators, every column used, the same one many times."""
    for rows in (3, 90):
        z, kw = inputs(rows, n, torch.float32, seed=6, states=0, hist=0, bias=None)
        g = torch.Generator().manual_seed(8)
        for hist in (700, 5000):
            h = torch.randint(-3, n + 3, (rows, hist), generator=g)
            h[0] = n - 1
            check(z, {"history": h.cuda()}, dict(repetition=1.1, frequency=0.001, presence=0.1))
    from flashlog_b200 import attention
    z = torch.zeros(2, n, device="cuda")
    h = torch.zeros(2, 65535, dtype=torch.int64, device="cuda")
    w = attention.relation_weights(z, history=h, frequency=2.0 ** -16)
    u = torch.zeros(n, dtype=torch.float64)
    u[0] = -65535 * 2.0 ** -16
    torch.testing.assert_close(w[1].double().cpu(), torch.softmax(u, 0), rtol=1e-5, atol=0)


def test_strides_leading_dimensions_and_shared_gradients():
    from flashlog_b200 import attention
    z, kw = inputs(24, 130, torch.float32, seed=9)
    plain = attention.relation_weights(z, **kw, **RULES)
    wide = torch.zeros(24, 200, device="cuda")
    wide[:, 7:137] = z
    table = torch.zeros(7, 131, dtype=torch.bool, device="cuda")
    table[:, 1:] = kw["mask"]
    hist = torch.zeros(24, 11, dtype=torch.int64, device="cuda")
    hist[:, ::2][:, :5] = kw["history"]
    odd = attention.relation_weights(wide[:, 7:137], mask=table[:, 1:], states=kw["states"], history=hist[:, ::2][:, :5],
                                     bias=kw["bias"], **RULES)
    assert torch.equal(odd, plain)
    lead = attention.relation_weights(z.view(2, 3, 4, 130), mask=kw["mask"], states=kw["states"].view(2, 3, 4),
                                      history=kw["history"].view(2, 3, 4, 5), bias=kw["bias"], **RULES)
    assert torch.equal(lead.view(24, 130), plain)
    lz = z.clone().requires_grad_()
    a, = torch.autograd.grad((attention.relation_weights(lz, **kw, **RULES) ** 2).sum(), [lz])
    w = attention.relation_weights(lz, **kw, **RULES)
    b, = torch.autograd.grad(w, [lz], 2 * w.detach())
    assert torch.equal(a, b)
    row = torch.randn(130, device="cuda")  # one gradient row for all rows, as a broadcast gives it
    c, = torch.autograd.grad(attention.relation_weights(lz, **kw, **RULES), [lz], row.expand(24, 130))
    d, = torch.autograd.grad(attention.relation_weights(lz, **kw, **RULES), [lz], row.expand(24, 130).contiguous())
    assert torch.equal(c, d)
    empty = attention.relation_weights(z[:0], bias=kw["bias"])
    assert empty.shape == (0, 130)


@pytest.mark.parametrize("rows,n", [(1, 29649), (40, 29649), (500, 1645), (60, 25)])
def test_same_bits_on_another_stream_and_in_a_graph(rows, n):
    from flashlog_b200 import attention
    z, kw = inputs(rows, n, torch.float32, seed=13)
    g = torch.randn(rows, n, generator=torch.Generator().manual_seed(1)).cuda()

    def run(lz, lb):
        w = attention.relation_weights(lz, **{**kw, "bias": lb}, **RULES)
        return (w.detach(), *torch.autograd.grad(w, [lz, lb], g))

    first = run(z.clone().requires_grad_(), kw["bias"].clone().requires_grad_())
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        lz, lb = z.clone().requires_grad_(), kw["bias"].clone().requires_grad_()
        second = run(lz, lb)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            third = run(lz, lb)
    torch.cuda.current_stream().wait_stream(s)
    graph.replay()
    graph.replay()
    torch.cuda.synchronize()
    for a, b, c in zip(first, second, third):
        assert torch.equal(a, b) and torch.equal(a, c)


def test_gradient_against_differences():
    from flashlog_b200 import attention
    z, kw = inputs(4, 60, torch.float32, seed=14)
    kw["states"][:] = 1
    g = torch.randn(4, 60, generator=torch.Generator().manual_seed(2)).cuda().double()
    lz = z.clone().requires_grad_()
    d, = torch.autograd.grad(attention.relation_weights(lz, **kw, **RULES), [lz], g.float())
    k = int(d[2].abs().argmax())
    h = 2.0 ** -7
    e = torch.zeros_like(z)
    e[2, k] = h
    with torch.no_grad():
        f = [(attention.relation_weights(z + s * e, **kw, **RULES).double() * g).sum() for s in (1, -1)]
    # the third derivative of a softmax is below 1 / tau^3 times the slope, penalties scale by at most 1.3
    assert abs(float((f[0] - f[1]) / (2 * h)) - float(d[2, k])) <= (1.3 / 0.8) ** 3 * 4 * h * h / 6 + 60 * 2.0 ** -23 * 4 / h


# ---- rows of thousands of columns, more of them than are in flight at once --------------------------
@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("rows,n", [(650, 4097), (600, 8186), (310, 16377), (310, 16378), (160, 24577), (150, 32761),
                                    (150, 32762)])
def test_long_rows(rows, n, dt):
    """Odd row starts (every position within 16 bytes), longer histories than a block has threads, states without
    a mask row, both kinds of bias."""
    z, kw = inputs(rows, n, DT[dt], seed=n, hist=7, bias="shared" if n % 2 else "full")
    check(z, kw, RULES, backward=False)
    wide = torch.zeros(rows, n + 3, dtype=z.dtype, device="cuda")
    wide[:, 1:n + 1] = z
    again = check(wide[:, 1:n + 1], {k: kw[k] for k in ("mask", "states")}, {"tau": 1.5}, backward=False)
    assert not bool(again[(kw["states"] < 0) | (kw["states"] >= 7)].any())
    few = z[:5].repeat(40, 1)[:100]  # few rows, long histories with many repetitions
    hist = torch.randint(-1, 40, (100, 1500), generator=torch.Generator().manual_seed(3)).cuda()
    check(few, {"history": hist}, {"frequency": 0.01, "repetition": 1.1}, backward=False)


def test_long_rows_in_a_graph_and_on_a_stream():
    from flashlog_b200 import attention
    z, kw = inputs(300, 29649, torch.float32, seed=8, bias=None)
    want = attention.relation_weights(z, **kw, **RULES)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        assert torch.equal(attention.relation_weights(z, **kw, **RULES), want)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            out = attention.relation_weights(z, **kw, **RULES)
    out.fill_(7.0)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)
