"""Pairs without an expert (the router's id -1) on the GPU: every expert path skips them, whatever the experts hold."""
import pytest
import torch

import tritonblas_b200 as tb
from tritonblas_b200 import distributed as tbd

pytestmark = pytest.mark.gpu

E, H, F = 8, 256, 128


def _case(T, K):
    g = torch.Generator(device="cuda").manual_seed(T)
    w1 = (torch.randn(E, 2 * F, H, device="cuda", generator=g) * H ** -0.5).bfloat16()
    w2 = (torch.randn(E, H, F, device="cuda", generator=g) * F ** -0.5).bfloat16()
    x = torch.randn(T, H, device="cuda", generator=g).bfloat16()
    logits = torch.randn(T, E, device="cuda", generator=g)
    logits[:, E - 1] = float("-inf")                # nobody chooses the last expert, which holds no numbers
    logits[: T // 3, 1:] = float("-inf")            # one live expert
    logits[T // 2] = float("-inf")                  # none
    w1[E - 1], w2[E - 1] = float("nan"), float("nan")
    return x, w1, w2, *tb.moe_route(logits, K)


def _reference(x, w1, w2, weights, ids):
    out = torch.zeros(x.shape, dtype=torch.float64, device="cuda")
    for e in range(E - 1):
        h = x.double() @ w1[e].double().T
        act = torch.nn.functional.silu(h[:, :F]) * h[:, F:]
        out += (weights.double() * (ids == e)).sum(1, keepdim=True) * (act @ w2[e].double().T)
    return out


def _check(out, ref, K):
    # three roundings to bf16 on the way (both projections, the activation), each half a step of values the size of the largest,
    # weighted with at most 1 in all and summed with random signs over F terms of size F^-0.5; one more at the end
    assert torch.isfinite(out).all() and (out.double() - ref).abs().max() <= 4 * 2.0 ** -8 * ref.abs().max()


@pytest.mark.parametrize("T,K", [(200, 2), (33, 5)])
def test_expert_parallel_layer(T, K):
    x, w1, w2, weights, ids = _case(T, K)
    assert (ids == -1).any()
    ref = _reference(x, w1, w2, weights, ids)
    for dtype in (torch.int32, torch.int64):
        out, plan = tbd.ExpertParallelMoE(w1, w2, E).forward(x, ids.to(dtype), weights)
        _check(out, ref, K)
        assert (out[T // 2] == 0).all() and plan.sort_idx.numel() == int((ids >= 0).sum())
    out, _ = tbd.ExpertParallelMoE(w1, w2, E).forward(x, ids * 0 - 1, weights)
    assert out.shape == x.shape and (out == 0).all()
    assert tb.device_status() == 0


@pytest.mark.parametrize("T,K", [(200, 2), (33, 5)])
def test_peer_memory_layer_counts_no_overflow(T, K):
    """The overflow counter tells a receive buffer that is too small; pairs without an expert need no row."""
    x, w1, w2, weights, ids = _case(T, K)
    live = int((ids >= 0).sum())
    moe = tbd.PeerMemoryMoE(w1, w2, E, live)
    out, _ = moe.forward(x, ids, weights)
    _check(out, _reference(x, w1, w2, weights, ids), K)
    assert int(moe.overflow) == 0
    small = tbd.PeerMemoryMoE(w1, w2, E, live - 7)
    small.forward(x, ids, weights)
    assert int(small.overflow) == 7 and tb.device_status() == 0
