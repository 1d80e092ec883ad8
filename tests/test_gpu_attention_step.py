"""The attention operators together, as a training step uses them: a head, rules
for the weights, three hops, the loss, their gradients and a Muon step -- the
static-buffer step against the autograd engine, eagerly and as a CUDA graph."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

Q, T, N, H = 16, 3, 3, 40


@pytest.fixture(scope="module")
def setup():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    from flashlog_b200 import ops
    from flashlog_b200.flashlog_kernel import build_csr_structure
    from flashlog_b200.synthetic import CONFIGS, generate_triples
    cfg = CONFIGS[1]
    train, _, _ = generate_triples(cfg)
    t = torch.from_numpy(train).cuda()
    csr = build_csr_structure(t[:, 0], t[:, 2], t[:, 1], cfg.entities)
    yield cfg, train, csr, ops.Graph.of(csr)
    assert not ops.gemm_fault()


def make(setup, with_head, seed=3, step=30):
    from flashlog_b200 import attention, rules
    from flashlog_b200.synthetic import training_queries
    cfg, train, csr, graph = setup
    R, n = cfg.relations, cfg.n
    ids, h, r, t = (torch.from_numpy(a).cuda() for a in training_queries(train, cfg, step=step))
    ids, h, r, t = ids[:8], h[:Q], r[:Q], t[:Q]
    g = torch.Generator().manual_seed(seed)
    table = torch.randn(2 * R, T, N, H if with_head else n, generator=g).cuda()
    head = (torch.randn(n, H, generator=g).cuda() * H ** -0.5, torch.randn(n, generator=g).cuda() * 0.1) if with_head else None
    # the first hop along an operator that leaves the head entity, the others free; the query's own relation penalised
    first = rules.first_operator_mask(h, csr, R)
    mask = torch.cat([first, torch.ones(1, n, dtype=torch.bool, device="cuda")])
    states = torch.full((T, Q), Q, dtype=torch.int64, device="cuda")
    states[0] = torch.arange(Q, device="cuda")
    op_rules = attention.OperatorRules(mask=mask, states=states, history=r[:, None].clone(), bias=torch.randn(n, generator=g).cuda() * 0.2,
                                       repetition=1.3, frequency=0.1, presence=0.5)
    return dict(ids=ids, h=h, r=r, t=t, table=table, head=head, rules=op_rules)


def engine_loss_and_grads(setup, p):
    from flashlog_b200 import engine
    cfg, train, csr, graph = setup
    mask = torch.ones(train.shape[0], dtype=torch.uint8, device="cuda")
    mask[p["ids"]] = 0
    table = p["table"].clone().requires_grad_()
    head = None if p["head"] is None else tuple(x.clone().requires_grad_() for x in p["head"])
    rp, ent, val = engine.drum_propagate(p["h"], table[p["r"]], graph, cfg.relations, c1=40, c2=16, mask_triple=mask,
                                         head=head, rules=p["rules"])
    loss = engine.readout_loss(rp, ent, val, p["t"], N)
    grads = torch.autograd.grad(loss, [table] + ([] if head is None else list(head)))
    return float(loss.detach()), grads


def make_step(setup, p, **kw):
    from flashlog_b200.step import DrumTrainStep
    cfg, _, _, graph = setup
    head = None if p["head"] is None else tuple(x.clone() for x in p["head"])
    step = DrumTrainStep(graph, cfg.relations, Q, T, N, 40, 16, p["table"].clone(), n_hide=8, head=head,
                         rules=p["rules"], **kw)
    step.load(p["h"], p["t"], p["r"], p["ids"])
    return step


def close(a, b, rel):
    """Frobenius distance relative to b's norm: sums over hops and rows, whose terms carry fp32 roundings."""
    a, b = a.double(), b.double()
    assert a.shape == b.shape and float((a - b).norm()) <= rel * float(b.norm()), float((a - b).norm() / b.norm())


@pytest.mark.parametrize("with_head", [False, True])
def test_step_matches_engine(setup, with_head):
    p = make(setup, with_head)
    loss, grads = engine_loss_and_grads(setup, p)
    step = make_step(setup, p, apply_update=False)
    got = float(step.run())
    step.check()
    assert got == pytest.approx(loss, rel=1e-5)
    close(step.grad, grads[0], 1e-5)
    if with_head:
        close(step.grad_head[0], grads[1], 1e-5)
        close(step.grad_head[1], grads[2], 1e-5)


def test_rules_shape_the_first_hop(setup):
    """No weight on operators that cannot leave the head, and less on the query's own relation than without rules."""
    p = make(setup, False)
    step = make_step(setup, p, apply_update=False)
    step.run()
    n = p["table"].shape[-1]
    w0 = step.w[0][:Q * N * n].view(Q, N, n)
    allowed = p["rules"].mask[:Q]
    assert bool((w0[~allowed[:, None].expand(-1, N, -1)] == 0).all())
    np.testing.assert_allclose(w0.sum(-1).cpu().numpy(), 1.0, rtol=1e-5)


@pytest.mark.parametrize("with_head", [False, True])
def test_muon_step_is_muon_of_the_gradient(setup, with_head):
    from flashlog_b200 import muon
    p = make(setup, with_head)
    lr, options = 0.03, dict(beta=0.9, weight_decay=0.01)
    plain = make_step(setup, p, apply_update=False)
    plain.run()
    step = make_step(setup, p, optimizer="muon", lr=lr, muon_options=options)
    step.run()
    step.check()
    view = lambda x: x.permute(1, 2, 0, 3)  # noqa: E731
    # contiguous copies: other strides than the step's views
    want, _ = muon.muon_update(view(p["table"]).contiguous(), view(plain.grad).contiguous(),
                               torch.zeros_like(view(p["table"]).contiguous()), lr=lr, **options)
    close(view(step.table), want, 1e-6)
    if with_head:
        w, _ = muon.muon_update(p["head"][0], plain.grad_head[0], torch.zeros_like(p["head"][0]), lr=lr, **options)
        close(step.head[0], w, 1e-6)
        close(step.head[1], p["head"][1] - lr * plain.grad_head[1], 1e-6)


def test_muon_step_replays_as_cuda_graph(setup):
    """Three steps on different batches, with the rules' tensors changed in place between replays."""
    batches = [make(setup, True, step=40 + k) for k in range(3)]
    eager = make_step(setup, batches[0], optimizer="muon", lr=0.02)
    graphed = make_step(setup, batches[0], optimizer="muon", lr=0.02)
    own = graphed.rules
    import dataclasses
    eager.rules = dataclasses.replace(own, mask=own.mask.clone(), states=own.states.clone(), history=own.history.clone())
    start = [x.clone() for x in (graphed.table, *graphed.head, graphed.momentum, graphed.momentum_head)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graphed.run()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        graphed.run()
    for x, y in zip((graphed.table, *graphed.head, graphed.momentum, graphed.momentum_head), start):
        x.copy_(y)
    for b in batches:
        for s in (eager, graphed):
            s.load(b["h"], b["t"], b["r"], b["ids"])
            s.rules.mask.copy_(b["rules"].mask)
            s.rules.history.copy_(b["rules"].history)
        want = float(eager.run())
        g.replay()
        torch.cuda.synchronize()
        assert float(graphed.loss) == pytest.approx(want, rel=1e-5)
    graphed.check()
    close(graphed.table, eager.table, 1e-5)
    close(graphed.head[0], eager.head[0], 1e-5)


def test_overflowed_step_leaves_everything_as_it_was(setup):
    """A forward that overflowed (here: the status word set by hand) changes neither table, head nor momentum."""
    p = make(setup, True)
    step = make_step(setup, p, optimizer="muon", lr=0.05)
    step.run()
    before = [x.clone() for x in (step.table, *step.head, step.momentum, step.momentum_head)]
    step.status.fill_(1)
    step.run()
    torch.cuda.synchronize()
    for a, b in zip((step.table, *step.head, step.momentum, step.momentum_head), before):
        assert torch.equal(a, b)
    with pytest.raises(RuntimeError):
        step.check()
    step.status.zero_()
    step.run()
    assert not torch.equal(step.table, before[0])


def test_engine_rules_gradient_of_bias(setup):
    """The engine differentiates the rules' bias: against a central difference of its own loss, in one operator."""
    from flashlog_b200 import engine
    import dataclasses
    cfg, train, csr, graph = setup
    p = make(setup, False)
    mask = torch.ones(train.shape[0], dtype=torch.uint8, device="cuda")
    mask[p["ids"]] = 0

    def loss_of(bias):
        r = dataclasses.replace(p["rules"], bias=bias)
        rp, ent, val = engine.drum_propagate(p["h"], p["table"][p["r"]], graph, cfg.relations, mask_triple=mask, rules=r)
        return engine.readout_loss(rp, ent, val, p["t"], N)

    bias = p["rules"].bias.clone().requires_grad_()
    g, = torch.autograd.grad(loss_of(bias), [bias])
    k = int(g.abs().argmax())
    d = torch.zeros_like(bias)
    d[k] = 1e-2
    with torch.no_grad():
        num = (float(loss_of(bias + d)) - float(loss_of(bias - d))) / 2e-2
    # the loss is a mean of Q logarithms, each off by a few 1e-6; the difference quotient's cubic term is of order
    # d^2 = 1e-4 of the slope
    assert abs(num - float(g[k])) <= 1e-3 * abs(float(g[k])) + 1e-3
