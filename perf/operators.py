"""The relation-attention operators: what is measured, in plain torch and through the framework.

Four operators learn and answer with the attention over relations that the hops propagate by:

* linear: y = act(x W^T + b) + residual, forward and backward (the head that turns a query's hidden
  state into a logit for each of the n = 2R + 1 relation operators, and the layers before it);
* weights: the repeat penalties, bias, grammar mask and softmax that turn logits into the hops' weights,
  forward and backward;
* ortho: Newton-Schulz orthogonalisation of (a batch of) matrices;
* muon: one whole momentum / orthogonalise / decay / update step of a parameter that is such a batch.

Sizes are those of the benchmark graphs: R = 12, 237, 37, 822, 14824 relations, hidden sizes 128, 256, 1024,
2 * batch queries (64 to 512) times 3 hops times 3 channels rows.
"""
import math

import torch

own = False

DEV = "cuda" if torch.cuda.is_available() else "cpu"
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
COEFFICIENTS = (3.4445, -4.7750, 2.0315)
STEPS = 5
EPS = 1e-7


def listed():
    return [
        # the hidden state of one query (3 hops x 3 channels) through the head of the 237-relation graph
        {"name": "head_one_query", "op": "linear", "back": False, "dtype": "fp32", "rows": 9, "k": 128, "n": 475, "act": "none", "bias": True, "res": False},
        # a training batch's logits on the 822-relation graph: 512 queries
        {"name": "head_822_relations", "op": "linear", "back": False, "dtype": "fp32", "rows": 4608, "k": 1024, "n": 1645, "act": "none", "bias": True, "res": False},
        # a residual hidden layer before that head, half types
        {"name": "hidden_layer_bf16", "op": "linear", "back": False, "dtype": "bf16", "rows": 4608, "k": 1024, "n": 1024, "act": "gelu", "bias": True, "res": True},
        # one training step of a head with its activation on the 237-relation graph, odd n
        {"name": "head_step_237_relations", "op": "linear", "back": True, "dtype": "fp32", "rows": 1152, "k": 128, "n": 475, "act": "silu", "bias": True, "res": False},
        # the largest: one training step of the head on the 14824-relation graph
        {"name": "head_step_14824_relations", "op": "linear", "back": True, "dtype": "bf16", "rows": 4608, "k": 1024, "n": 29649, "act": "none", "bias": True, "res": False},
        # one query's next operator on the largest graph (a single position)
        {"name": "weights_one_row", "op": "weights", "back": False, "dtype": "bf16", "rows": 1, "n": 29649, "states": 64, "history": 16, "bias": True},
        # a training batch's weights on the 822-relation graph, and their gradient
        {"name": "weights_step_822_relations", "op": "weights", "back": True, "dtype": "fp32", "rows": 4608, "n": 1645, "states": 1645, "history": 3, "bias": True},
        # the same on the largest graph, long histories
        {"name": "weights_14824_relations", "op": "weights", "back": False, "dtype": "fp32", "rows": 1536, "n": 29649, "states": 512, "history": 200, "bias": False},
        # the smallest table: 24 query relations x 25 operators, 9 hop-channel matrices
        {"name": "ortho_tables_12_relations", "op": "ortho", "dtype": "fp32", "batch": 9, "m": 24, "n": 25},
        # the update of the head's weight on the largest graph: a tall matrix in half type
        {"name": "ortho_head_14824_relations", "op": "ortho", "dtype": "bf16", "batch": 1, "m": 29649, "n": 1024},
        # the attention table of the 237-relation graph: a whole step
        {"name": "muon_table_237_relations", "op": "muon", "dtype": "fp32", "m": 474, "n": 475, "hops": 3, "channels": 3},
        # the attention table of the 822-relation graph: a whole step
        {"name": "muon_table_822_relations", "op": "muon", "dtype": "fp32", "m": 1644, "n": 1645, "hops": 3, "channels": 3},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["linear", "linear", "weights", "weights", "ortho", "muon"])
    dtype = rng.choice(["fp32", "fp32", "bf16", "fp16"])
    if op == "linear":
        rows, k, n = _log(rng, 1, 4608), _log(rng, 16, 1024), _log(rng, 25, 29649)
        return {"op": op, "back": rng.random() < 0.5, "dtype": dtype, "rows": rows, "k": k, "n": n,
                "act": rng.choice(["none", "none", "relu", "tanh", "silu", "gelu"]), "bias": rng.random() < 0.8,
                "res": rng.random() < 0.4}
    if op == "weights":
        return {"op": op, "back": rng.random() < 0.5, "dtype": dtype, "rows": _log(rng, 1, 1536), "n": _log(rng, 25, 29649),
                "states": rng.choice([0, 1, _log(rng, 2, 1645)]), "history": rng.choice([0, 1, _log(rng, 2, 256)]), "bias": rng.random() < 0.6}
    if op == "ortho":
        m, n = _log(rng, 8, 1645), _log(rng, 8, 4096)
        return {"op": op, "dtype": dtype, "batch": rng.randint(1, 9), "m": m, "n": n} if rng.random() < 0.5 else \
            {"op": op, "dtype": dtype, "batch": rng.randint(1, 3), "m": n, "n": m}
    m = _log(rng, 24, 1644)
    return {"op": op, "dtype": "fp32", "m": m, "n": rng.choice([m + 1, _log(rng, 16, 1645)]), "hops": rng.randint(1, 3), "channels": rng.randint(1, 3)}


def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    return g


def _normal(g, *shape, std=1.0):
    return torch.randn(*shape, generator=g, device=DEV) * std


def prepare(case, seed):
    g, op, dt = _gen(seed), case["op"], DTYPES[case["dtype"]]
    s = {"case": case}
    if op == "linear":
        rows, k, n = case["rows"], case["k"], case["n"]
        s["x"] = _normal(g, rows, k).to(dt)
        s["weight"] = _normal(g, n, k, std=k ** -0.5).to(dt)
        s["bias"] = _normal(g, n, std=0.1).to(dt) if case["bias"] else None
        s["residual"] = _normal(g, rows, n).to(dt) if case["res"] else None
        s["gy"] = _normal(g, rows, n, std=1.0 / rows).to(dt) if case["back"] else None
        if case["back"]:
            for name in ("x", "weight", "bias", "residual"):
                if s[name] is not None:
                    s[name].requires_grad_()
    elif op == "weights":
        rows, n, states, hist = case["rows"], case["n"], case["states"], case["history"]
        s["logits"] = _normal(g, rows, n, std=1.5).to(dt)
        s["bias"] = _normal(g, n, std=0.3).to(dt) if case["bias"] else None
        s["mask"] = s["states"] = s["history"] = None
        if states:
            # what may follow each state; the last of several states allows nothing
            s["mask"] = torch.rand(states, n, generator=g, device=DEV) < 0.3
            if states > 1:
                s["mask"][-1] = False
            s["states"] = torch.randint(0, states, (rows,), generator=g, device=DEV)
        if hist:
            # operators used so far, the frequent ones repeated, short histories padded with -1
            u = torch.rand(rows, hist, generator=g, device=DEV)
            h = (n * u * u * u).long().clamp_(max=n - 1)
            length = torch.randint(0, hist + 1, (rows, 1), generator=g, device=DEV)
            s["history"] = torch.where(torch.arange(hist, device=DEV) < length, h, torch.full_like(h, -1))
        s["gw"] = _normal(g, rows, n) if case["back"] else None
        if case["back"]:
            for name in ("logits", "bias"):
                if s[name] is not None:
                    s[name].requires_grad_()
    elif op == "ortho":
        s["update"] = _spectrum(g, case["batch"], case["m"], case["n"]).to(dt)
    else:
        # a table [query relations, hops, channels, operators]: its matrices are strided views
        m, n, T, N = case["m"], case["n"], case["hops"], case["channels"]
        view = lambda t: t.reshape(T, N, m, n).permute(2, 0, 1, 3).contiguous().permute(1, 2, 0, 3)  # noqa: E731
        s["param"] = view(_normal(g, T * N, m, n))
        s["grad"] = view(_spectrum(g, T * N, m, n) * 1e-3)
        s["momentum"] = view(_spectrum(g, T * N, m, n) * 1e-2)
    return s


def _spectrum(g, batch, m, n):
    """Matrices as gradients are: a few strong directions over noise."""
    r = max(1, min(m, n) // 16)
    strong = _normal(g, batch, m, r) @ _normal(g, batch, r, n)
    return _normal(g, batch, m, n) + strong * (0.5 / r ** 0.5)


LR, BETA, DECAY = 0.02, 0.95, 0.01
TAU, REPETITION, FREQUENCY, PRESENCE = 0.9, 1.2, 0.1, 0.2


def run(s):
    if own:
        return _run_own(s)
    with torch.no_grad():
        return _run_plain(s)


def _run_own(s):
    from flashlog_b200 import attention, muon
    c = s["case"]
    if c["op"] == "linear":
        y = attention.linear(s["x"], s["weight"], s["bias"], residual=s["residual"], activation=c["act"])
        if not c["back"]:
            return {"y": y}
        names = [k for k in ("x", "weight", "bias", "residual") if s[k] is not None]
        grads = torch.autograd.grad(y, [s[k] for k in names], s["gy"])
        return {"y": y.detach(), **{"d_" + k: v for k, v in zip(names, grads)}}
    if c["op"] == "weights":
        w = attention.relation_weights(s["logits"], tau=TAU, mask=s["mask"], states=s["states"], bias=s["bias"], history=s["history"],
                                       repetition=REPETITION, frequency=FREQUENCY, presence=PRESENCE)
        if not c["back"]:
            return {"w": w}
        names = [k for k in ("logits", "bias") if s[k] is not None]
        grads = torch.autograd.grad(w, [s[k] for k in names], s["gw"])
        return {"w": w.detach(), **{"d_" + k: v for k, v in zip(names, grads)}}
    if c["op"] == "ortho":
        return {"o": muon.orthogonalize(s["update"], steps=STEPS, coefficients=COEFFICIENTS, eps=EPS)}
    p, m = muon.muon_update(s["param"], s["grad"], s["momentum"], lr=LR, beta=BETA, nesterov=True, weight_decay=DECAY, steps=STEPS,
                            coefficients=COEFFICIENTS, eps=EPS)
    return {"param": p, "momentum": m}


# ---- the plain forms ----------------------------------------------------------------------------
def _act(z, name):
    if name == "relu":
        return torch.clamp_min(z, 0)
    if name == "tanh":
        return torch.tanh(z)
    if name == "silu":
        return z * torch.sigmoid(z)
    if name == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    return z


def _act_slope(z, name):
    if name == "relu":
        return (z > 0).to(z.dtype)
    if name == "tanh":
        return 1 - torch.tanh(z) ** 2
    if name == "silu":
        t = torch.sigmoid(z)
        return t * (1 + z * (1 - t))
    if name == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
    return None


def _newton_schulz(x):
    """In 32 bits; x [..., m, n]."""
    turned = x.shape[-2] > x.shape[-1]
    if turned:
        x = x.transpose(-1, -2)
    norm = (x.double() ** 2).sum(dim=(-2, -1), keepdim=True).sqrt().float()
    x = x / (norm + EPS)
    a, b, c = COEFFICIENTS
    for _ in range(STEPS):
        gram = x @ x.transpose(-1, -2)
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return x.transpose(-1, -2) if turned else x


def _run_plain(s):
    c = s["case"]
    if c["op"] == "linear":
        dt = s["x"].dtype
        x, w = s["x"].float(), s["weight"].float()
        z = x @ w.T
        if s["bias"] is not None:
            z = z + s["bias"].float()
        y = _act(z, c["act"])
        if s["residual"] is not None:
            y = y + s["residual"].float()
        if not c["back"]:
            return {"y": y.to(dt)}
        slope = _act_slope(z, c["act"])
        dz = s["gy"].float() if slope is None else s["gy"].float() * slope
        out = {"y": y.to(dt), "d_x": (dz @ w).to(dt), "d_weight": (dz.T @ x).to(dt)}
        if s["bias"] is not None:
            out["d_bias"] = dz.sum(0).to(dt)
        if s["residual"] is not None:
            out["d_residual"] = s["gy"]
        return out
    if c["op"] == "weights":
        z = s["logits"].float()
        n = z.shape[1]
        u, slope = z, None
        if s["history"] is not None:
            h = s["history"]
            inside = (h >= 0) & (h < n)
            count = torch.zeros(z.shape[0], n + 1, device=z.device)
            count.scatter_add_(1, torch.where(inside, h, torch.full_like(h, n)), torch.ones_like(h, dtype=torch.float32))
            count = count[:, :n]
            seen = count > 0
            slope = torch.where(seen, torch.where(z > 0, 1.0 / REPETITION, REPETITION), 1.0)
            u = torch.where(seen & (z > 0), z / REPETITION, torch.where(seen, z * REPETITION, z))
            u = u - FREQUENCY * count - PRESENCE * seen
        if s["bias"] is not None:
            u = u + s["bias"].float()
        if s["mask"] is not None:
            u = torch.where(s["mask"][s["states"]], u, -math.inf)
        top = u.amax(1, keepdim=True)
        some = top > -math.inf
        e = torch.exp((u - torch.where(some, top, 0.0)) / TAU)
        total = e.sum(1, keepdim=True)
        w = e / torch.where(some, total, 1.0)
        if not c["back"]:
            return {"w": w}
        g = s["gw"]
        du = w * (g - (g * w).sum(1, keepdim=True)) / TAU
        dt = s["logits"].dtype
        out = {"w": w, "d_logits": (du if slope is None else du * slope).to(dt)}
        if s["bias"] is not None:
            out["d_bias"] = du.sum(0).to(dt)
        return out
    if c["op"] == "ortho":
        return {"o": _newton_schulz(s["update"].float()).to(s["update"].dtype)}
    m2 = BETA * s["momentum"] + s["grad"]
    o = _newton_schulz(s["grad"] + BETA * m2)
    scale = math.sqrt(max(1.0, c["m"] / c["n"]))
    return {"param": s["param"] * (1 - LR * DECAY) - (LR * scale) * o, "momentum": m2}


def work(case):
    op, size = case["op"], 4 if case["dtype"] == "fp32" else 2
    if op == "linear":
        rows, k, n = case["rows"], case["k"], case["n"]
        b = rows * k + n * k + rows * n + (n if case["bias"] else 0) + (rows * n if case["res"] else 0)
        f = 2 * rows * k * n
        if case["back"]:  # gy read, dx, dw and db written (the residual's gradient is gy)
            b += rows * n + rows * k + n * k + (n if case["bias"] else 0)
            f *= 3
        return {"bytes": b * size, "flops": f}
    if op == "weights":
        rows, n = case["rows"], case["n"]
        b = rows * n * (size + 4) + (n * size if case["bias"] else 0) + min(rows, case["states"]) * n + (8 * rows if case["states"] else 0)
        b += 8 * rows * case["history"]
        f = 8 * rows * n
        if case["back"]:
            b += rows * n * (4 + size) + (n * size if case["bias"] else 0)
            f += 6 * rows * n
        return {"bytes": b, "flops": f}
    lo, hi = min(case["m"], case["n"]), max(case["m"], case["n"])
    batch = case["batch"] if op == "ortho" else case["hops"] * case["channels"]
    # a product with a symmetric result costs half
    f = batch * STEPS * (lo * lo * hi + lo ** 3 + 2 * lo * lo * hi)
    return {"bytes": batch * lo * hi * size * (2 if op == "ortho" else 5), "flops": f}


# ---- the definitions in 64 bits ------------------------------------------------------------------
def _exact_ortho(x):
    """Newton-Schulz maps each singular value by an odd polynomial: through the eigenvectors of the Gram matrix."""
    turned = x.shape[-2] > x.shape[-1]
    x = x.mT if turned else x
    x = x / (torch.linalg.matrix_norm(x, keepdim=True) + EPS)
    lam, v = torch.linalg.eigh(x @ x.mT)
    lam = lam.clamp_min(0)
    a, b, c = COEFFICIENTS
    factor = torch.ones_like(lam)
    for _ in range(STEPS):
        t = lam * factor * factor
        factor = factor * (a + b * t + c * t * t)
    o = (v * factor[..., None, :]) @ (v.mT @ x)
    return o.mT if turned else o


def exact(case, seed):
    s = prepare(case, seed)
    f64 = lambda t: None if t is None else t.detach().to(torch.float64)  # noqa: E731
    if case["op"] == "linear":
        names = [k for k in ("x", "weight", "bias", "residual") if s[k] is not None]
        v = {k: f64(s[k]).requires_grad_(case["back"]) for k in names}
        z = torch.nn.functional.linear(v["x"], v["weight"], v.get("bias"))
        fn = {"none": lambda t: t, "relu": torch.relu, "tanh": torch.tanh, "silu": torch.nn.functional.silu,
              "gelu": torch.nn.functional.gelu}[case["act"]]
        y = fn(z)
        if "residual" in v:
            y = y + v["residual"]
        if not case["back"]:
            return {"y": y}
        grads = torch.autograd.grad(y, [v[k] for k in names], f64(s["gy"]))
        return {"y": y.detach(), **{"d_" + k: t for k, t in zip(names, grads)}}
    if case["op"] == "weights":
        z = f64(s["logits"]).requires_grad_(case["back"])
        bias = None if s["bias"] is None else f64(s["bias"]).requires_grad_(case["back"])
        n = z.shape[1]
        u = z
        if s["history"] is not None:
            h = s["history"]
            rows = torch.arange(h.shape[0], device=h.device)[:, None].expand_as(h)
            keep = (h >= 0) & (h < n)
            count = torch.zeros(z.shape, dtype=torch.float64, device=z.device)
            count.index_put_((rows[keep], h[keep]), torch.ones((), dtype=torch.float64, device=z.device), accumulate=True)
            penalised = torch.where(z > 0, z / REPETITION, z * REPETITION)
            u = torch.where(count > 0, penalised, z) - FREQUENCY * count - PRESENCE * (count > 0)
        if bias is not None:
            u = u + bias
        if s["mask"] is None:
            w = torch.softmax(u / TAU, dim=1)
        else:
            allowed = s["mask"].index_select(0, s["states"])
            some = allowed.any(1, keepdim=True)
            w = torch.softmax((u / TAU).masked_fill(~(allowed | ~some), -math.inf), dim=1) * some
        if not case["back"]:
            return {"w": w}
        grads = torch.autograd.grad(w, [z] if bias is None else [z, bias], f64(s["gw"]))
        return {"w": w.detach(), **{"d_" + k: t for k, t in zip(("logits", "bias"), grads)}}
    if case["op"] == "ortho":
        return {"o": _exact_ortho(f64(s["update"]))}
    m2 = f64(s["momentum"]).mul(BETA).add(f64(s["grad"]))
    o = _exact_ortho(f64(s["grad"]).add(m2, alpha=BETA))
    scale = max(1.0, case["m"] / case["n"]) ** 0.5
    return {"param": f64(s["param"]).mul(1 - LR * DECAY).sub(o, alpha=LR * scale), "momentum": m2}
