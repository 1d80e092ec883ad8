"""Training and propagation with a head and no rules: the hops' weights and their gradient come from the framework's own
kernels, as with rules."""
import pytest
import torch

from test_gpu_attention_step import close, engine_loss_and_grads, make, make_step, setup  # noqa: F401

pytestmark = pytest.mark.gpu


def torch_losses(p, setup):
    """Loss and gradients with the logits and their softmax by torch, through the engine without a head."""
    from flashlog_b200 import engine
    cfg, train, csr, graph = setup
    mask = torch.ones(train.shape[0], dtype=torch.uint8, device="cuda")
    mask[p["ids"]] = 0
    leaves = [t.clone().requires_grad_() for t in (p["table"], *p["head"])]
    logits = torch.nn.functional.linear(leaves[0][p["r"]], leaves[1], leaves[2])
    rp, ent, val = engine.drum_propagate(p["h"], logits, graph, cfg.relations, c1=40, c2=16, mask_triple=mask)
    loss = engine.readout_loss(rp, ent, val, p["t"], logits.shape[2])
    return float(loss.detach()), torch.autograd.grad(loss, leaves)


def test_head_without_rules_runs_on_the_own_kernels(setup, monkeypatch):  # noqa: F811
    p = make(setup, True)
    p["rules"] = None
    want, grads = torch_losses(p, setup)

    def no(*a, **k):
        raise AssertionError("a library softmax next to the head")
    for name in ("softmax", "_softmax_backward_data"):
        monkeypatch.setattr(torch, name, no)
    loss, engine_grads = engine_loss_and_grads(setup, p)
    assert loss == pytest.approx(want, rel=1e-5)
    step = make_step(setup, p, apply_update=False)
    assert float(step.run()) == pytest.approx(want, rel=1e-5)
    step.check()
    for got in (engine_grads, (step.grad, *step.grad_head)):
        for a, b in zip(got, grads):
            close(a, b, 1e-5)


def test_history_rows_follow_changes_in_place(setup):  # noqa: F811
    """Rules are read on every run; the backward sees the history that its forward saw."""
    p = make(setup, False)
    step = make_step(setup, p, apply_update=False)
    step.run()
    before = step.grad.clone()
    p["rules"].history.add_(1)
    step.load(p["h"], p["t"], p["r"], p["ids"])
    loss = float(step.run())
    want, grads = engine_loss_and_grads(setup, p)
    assert loss == pytest.approx(want, rel=1e-5) and not torch.equal(step.grad, before)
    close(step.grad, grads[0], 1e-5)
