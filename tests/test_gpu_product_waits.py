"""Newton-Schulz products that give up a wait: NaN in what was left, a fault word, and a context that goes on.

The waits are bounded; here the one for the product before gets a limit of 0, so that it runs out at its first look.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture
def no_patience():
    from flashlog_b200 import ops
    assert not ops.gemm_fault()
    ops.gemm_wait_limits(0.5, 0.0)
    yield
    ops.gemm_wait_limits()
    ops.gemm_fault()


# direct form (its last product takes X in), Gram form of one segment and of two, and many matrices
@pytest.mark.parametrize("shape,steps", [((300, 310), 5), ((300, 900), 3), ((900, 300), 5), ((9, 200, 210), 2)], ids=str)
def test_what_is_left_becomes_nan(no_patience, shape, steps):
    from flashlog_b200 import muon, ops
    g = torch.Generator().manual_seed(1)
    p, u = (torch.randn(*shape, generator=g).cuda() for _ in range(2))
    m = torch.zeros_like(p)
    before = p.clone()
    muon.muon_update_(p, u, m, lr=0.1, steps=steps)
    torch.cuda.synchronize()
    assert ops.gemm_fault() and not ops.gemm_fault()
    assert bool(p.isnan().all()) and torch.equal(m, u)
    ops.gemm_wait_limits()
    want, _ = muon.muon_update(before, u, torch.zeros_like(p), lr=0.1, steps=steps)
    assert bool(want.isfinite().all()) and not ops.gemm_fault()
    closed = torch.zeros(1).cuda()
    ops.gemm_wait_limits(0.5, 0.0)
    again = before.clone()
    muon.muon_update_(again, u, m, lr=0.1, steps=steps, gate=closed)  # a closed gate keeps what it kept
    assert torch.equal(again, before)


def test_orthogonalize_leaves_nothing_unwritten(no_patience):
    from flashlog_b200 import muon, ops
    for shape in ((300, 310), (300, 900), (500, 520)):
        o = muon.orthogonalize(torch.randn(*shape, device="cuda").to(torch.bfloat16))
        assert bool(o.isnan().all())
    assert ops.gemm_fault()


def test_step_check_raises(no_patience):
    from flashlog_b200 import muon
    from flashlog_b200.step import DrumTrainStep
    muon.orthogonalize(torch.randn(300, 310, device="cuda"))
    step = DrumTrainStep.__new__(DrumTrainStep)  # of a step, what its check looks at
    step.dev, step.head, step.optimizer = torch.device("cuda", torch.cuda.current_device()), None, "muon"
    step.status = torch.zeros(1, dtype=torch.int32, device="cuda")
    with pytest.raises(RuntimeError, match="wait of a matrix product"):
        step.check()
    step.check()


def test_limits_refuse():
    from flashlog_b200 import ops
    with pytest.raises((ValueError, RuntimeError)):
        ops.gemm_wait_limits(-1.0)
