"""Pairs without an expert (the router's id -1) in the host-side dispatch plans: they go nowhere and add nothing, whatever the
experts return. torch products stand in for the CUDA entry points."""
import os

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

from tests.test_distributed_cpu import _free_port, _grouped_cpu
from tritonblas_b200 import distributed as tbd

E, H, F, T, K = 8, 16, 12, 14, 3


def _case(seed):
    g = torch.Generator().manual_seed(seed)
    w1, w2 = torch.randn(E, 2 * F, H, generator=g) * 0.2, torch.randn(E, H, F, generator=g) * 0.2
    x, wts = torch.randn(T, H, generator=g), torch.rand(T, K, generator=g)
    ids = torch.stack([torch.randperm(E - 1, generator=g)[:K] for _ in range(T)])     # nobody chooses the last expert
    ids[2] = -1                                 # a token without any expert
    ids[5, 1:] = -1
    ids[7, 0], ids[9, 2] = E, 1 << 40           # outside on the other side
    wts[(ids < 0) | (ids >= E)] = 0.0
    return w1, w2, x, ids, wts


def _reference(w1, w2, x, ids, wts):
    out = torch.zeros(T, H, dtype=torch.float64)
    for t in range(T):
        for j in range(K):
            e = int(ids[t, j])
            if 0 <= e < E:
                h = x[t].double() @ w1[e].double().T
                out[t] += wts[t, j].double() * ((torch.nn.functional.silu(h[:F]) * h[F:]) @ w2[e].double().T)
    return out


@pytest.mark.parametrize("placed", [False, True])
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_one_rank(placed, dtype):
    w1, w2, x, ids, wts = _case(0)
    w1[E - 1], w2[E - 1] = float("inf"), float("nan")       # what a wrapped index would have met
    want = _reference(w1, w2, x, ids, wts)
    if dtype == torch.int32:
        ids = ids.clamp(max=E).int()
    place = torch.randperm(E, generator=torch.Generator().manual_seed(1)).int() if placed else None
    if placed:
        order = torch.argsort(place)
        w1, w2 = w1[order], w2[order]
    out, plan = tbd.ExpertParallelMoE(w1, w2, E, grouped_fn=_grouped_cpu, expert_place=place).forward(x, ids, wts)
    live = (ids >= 0) & (ids < E)
    # fp32 sums of H and F terms around 1: 1e-5 covers (H + F) 2^-23 times their magnitudes
    assert torch.allclose(out.double(), want, atol=1e-5) and (out[2] == 0).all()
    assert int(plan.group_offsets[-1]) == int(live.sum()) == plan.sort_idx.numel()
    assert torch.equal(plan.pos >= 0, live.flatten())


def test_no_pair_at_all():
    w1, w2, x, ids, wts = _case(3)
    out, plan = tbd.ExpertParallelMoE(w1, w2, E, grouped_fn=_grouped_cpu).forward(x, ids * 0 - 1, wts)
    assert (out == 0).all() and out.shape == (T, H) and plan.sort_idx.numel() == 0


def _worker(rank, world, port, results):
    os.environ["MASTER_ADDR"], os.environ["MASTER_PORT"] = "127.0.0.1", str(port)
    dist.init_process_group("gloo", rank=rank, world_size=world)
    try:
        w1, w2, x, ids, wts = _case(0)
        x = x + rank                            # the same experts and choices, other rows
        epr = E // world
        moe = tbd.ExpertParallelMoE(w1[rank * epr:(rank + 1) * epr], w2[rank * epr:(rank + 1) * epr], E, grouped_fn=_grouped_cpu)
        out, _ = moe.forward(x, ids, wts)
        assert torch.allclose(out.double(), _reference(w1, w2, x, ids, wts), atol=1e-4)
        results[rank] = "ok"
    except Exception as exc:  # surfaced by the parent
        results[rank] = repr(exc)
    finally:
        dist.destroy_process_group()


def test_two_ranks():
    ctx = mp.get_context("spawn")
    results = ctx.Manager().dict()
    port = _free_port()
    procs = [ctx.Process(target=_worker, args=(r, 2, port, results)) for r in range(2)]
    for p in procs:
        p.start()
    for p in procs:
        p.join(120)
    assert dict(results) == {0: "ok", 1: "ok"}


@pytest.mark.parametrize("world", [1, 4])
def test_peer_plan(world):
    """Every routed pair has a row of its own inside the counts; the others have row -1."""
    g = torch.Generator().manual_seed(4)
    ids = [torch.randint(-1, E + 1, (T, K), generator=g) for _ in range(world)]
    live = [(i >= 0) & (i < E) for i in ids]
    counts = torch.stack([torch.bincount(i[m], minlength=E) for i, m in zip(ids, live)])
    epr = E // world
    landed = [torch.zeros(int(counts.sum()), dtype=torch.int32) for _ in range(world)]
    for r in range(world):
        plan = tbd.plan_peer_dispatch(ids[r], counts, r)
        m = live[r].flatten()
        assert (plan.pair_row[~m] == -1).all() and (plan.pair_rank[~m] == 0).all()
        assert torch.equal(plan.pair_rank[m].long(), ids[r].flatten()[m] // epr)
        n = int(m.sum())
        assert (plan.dest_row[:n] >= 0).all() and (plan.dest_row[n:] == -1).all()
        for d, row in zip(plan.pair_rank[m].tolist(), plan.pair_row[m].tolist()):
            landed[d][row] += 1
    for d in range(world):
        used = int(counts[:, d * epr:(d + 1) * epr].sum())
        assert (landed[d][:used] == 1).all() and (landed[d][used:] == 0).all()
