"""Host-side parts of the attention operators' paths (CPU): the ranks' update, the first hop's mask."""
import os

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

from test_multigpu_host import _free_port


def _update_worker(rank, world, port, fails, out):
    os.environ["MASTER_ADDR"] = "127.0.0.1"
    os.environ["MASTER_PORT"] = str(port)
    dist.init_process_group("gloo", rank=rank, world_size=world)
    try:
        from flashlog_b200 import multigpu as MG
        T = 2
        grad_hop, table = torch.zeros(T, 4, 3), torch.ones(4, T, 3)
        grad_head = (torch.full((2,), float(rank + 1)), None)
        ok = torch.tensor([0.0 if fails and rank == 1 else 1.0])
        seen = []

        def part(hop):
            def run():
                if hop >= 0:
                    grad_hop[hop].fill_(float((rank + 1) * (hop + 1)))
            return run

        def update():
            seen.append((grad_hop[:, 0, 0].tolist(), grad_head[0].tolist(), float(ok)))

        MG.run_parts_with_overlapped_allreduce([part(1), part(0), part(-1)], grad_hop, grad_hop.permute(1, 0, 2), table,
                                               lr=0.5, update=update, extra_grads=grad_head, gate=ok)
        out.put((rank, seen, table.tolist()))
    finally:
        dist.destroy_process_group()


@pytest.mark.parametrize("fails", [False, True])
def test_update_sees_the_ranks_mean_once_and_one_gate(fails):
    ctx = mp.get_context("spawn")
    q, port = ctx.Queue(), _free_port()
    procs = [ctx.Process(target=_update_worker, args=(r, 2, port, fails, q)) for r in range(2)]
    for p in procs:
        p.start()
    res = sorted(q.get(timeout=120) for _ in range(2))
    for p in procs:
        p.join(timeout=60)
        assert p.exitcode == 0
    for _, seen, table in res:
        assert seen == [([1.5, 3.0], [1.5, 1.5], 0.0 if fails else 1.0)]
        assert table == torch.ones(4, 2, 3).tolist()  # the update's own business


@pytest.mark.parametrize("seed,entities,relations,keep", [(0, 9, 4, 0.4), (1, 1, 1, 1.0), (2, 30, 7, 0.05), (3, 6, 3, 0.0)])
def test_first_operator_mask_is_each_sources_own(seed, entities, relations, keep):
    """Groups (entity, relation) of both directions, some entities without any."""
    from flashlog_b200 import rules
    g = torch.Generator().manual_seed(seed)
    csr = [None] * 14
    for at in (8, 12):
        have = torch.rand(entities, relations, generator=g) < keep
        csr[at] = torch.cat([torch.zeros(1, dtype=torch.int64), have.sum(1).cumsum(0)]).int()
        csr[at + 1] = have.nonzero()[:, 1].int()
    sources = torch.cat([torch.arange(entities), torch.randint(0, entities, (5,), generator=g)])
    mask = rules.first_operator_mask(sources, csr, relations)
    assert mask.dtype == torch.bool and tuple(mask.shape) == (len(sources), 2 * relations + 1)
    for s, row in zip(sources, mask):
        assert torch.equal(row, rules.available_first_operators(s.view(1), csr, relations))
    assert rules.first_operator_mask(sources[:0], csr, relations).shape == (0, 2 * relations + 1)
