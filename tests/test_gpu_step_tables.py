"""Steps on the first hops of a longer table: gradients only."""
import pytest
import torch

from test_gpu_attention_step import N, Q, T, make, setup  # noqa: F401

pytestmark = pytest.mark.gpu


def test_table_of_more_hops(setup):  # noqa: F811
    from flashlog_b200.step import DrumTrainStep
    p = make(setup, False)
    cfg, _, _, graph = setup
    longer = torch.cat([p["table"], torch.randn_like(p["table"][:, :1])], 1)
    got = []
    for table in (p["table"], longer):
        step = DrumTrainStep(graph, cfg.relations, Q, T, N, 40, 16, table.clone(), n_hide=8, apply_update=False)
        step.load(p["h"], p["t"], p["r"], p["ids"])
        got.append((float(step.run()), step.grad.clone()))
        step.check()
    assert got[0][0] == pytest.approx(got[1][0], rel=1e-6)
    torch.testing.assert_close(got[0][1], got[1][1], rtol=1e-5, atol=1e-8)
    for kw in (dict(apply_update=True), dict(apply_update=False, optimizer="muon")):
        with pytest.raises(ValueError, match="table must be"):
            DrumTrainStep(graph, cfg.relations, Q, T, N, 40, 16, longer.clone(), n_hide=8, **kw)
