"""Expert router and the expert feed-forward of a few tokens: thin marshalling over the C ABI (tb_moe_route, tb_moe_mlp).

``moe_route`` turns router logits into the ids and weights every expert path of this package takes; ``moe_mlp`` is the whole
expert layer of a decode batch in two launches. Batches of more than 128 tokens go through ``distributed.PeerMemoryMoE`` /
``distributed.ExpertParallelMoE``, whose grouped GEMMs work on 128-row tiles. The reference has no MoE path.
"""
import ctypes
from typing import Optional, Tuple

import torch

from . import _lib
from ._checks import on_device, require, require_cuda, rows16

MOE_MLP_MAX_TOKENS = 128
_MAX_EXPERTS, _MAX_TOPK = 1024, 32
_SCORING = {"softmax": 0, "sigmoid": 1}

# ------------------------------------------------------------------------------------------------------------- router
def _route_rows(logits):
    """The logits as rows with unit column stride and a row stride of at least their length."""
    if logits.stride(1) == 1 and (logits.shape[0] <= 1 or logits.stride(0) >= logits.shape[1]):
        return logits
    return logits.contiguous()


def _route_forward(logits, topk, sigmoid, renormalize):
    tokens, experts = logits.shape
    logits = _route_rows(logits)
    weights = torch.empty(tokens, topk, dtype=torch.float32, device=logits.device)
    ids = torch.empty(tokens, topk, dtype=torch.int32, device=logits.device)
    with on_device(logits.device):
        rc = _lib.lib.tb_moe_route(logits.data_ptr(), _lib.DTYPE_CODE[logits.dtype], logits.stride(0), tokens, experts, topk,
                                   sigmoid, renormalize, weights.data_ptr(), ids.data_ptr(),
                                   _lib.current_stream_ptr(logits.device))
    _lib.check(rc, "tb_moe_route")
    return weights, ids


@torch.library.custom_op("tritonblas::_moe_route", mutates_args=())
def _moe_route(logits: torch.Tensor, topk: int, sigmoid: bool, renormalize: bool) -> Tuple[torch.Tensor, torch.Tensor]:
    return _route_forward(logits, topk, int(sigmoid), int(renormalize))


@_moe_route.register_fake
def _(logits, topk, sigmoid, renormalize):
    shape = (logits.shape[0], topk)
    return logits.new_empty(shape, dtype=torch.float32), logits.new_empty(shape, dtype=torch.int32)


@torch.library.custom_op("tritonblas::_moe_route_backward", mutates_args=())
def _moe_route_backward(logits: torch.Tensor, weights: torch.Tensor, ids: torch.Tensor, grad: torch.Tensor, sigmoid: bool,
                        renormalize: bool) -> torch.Tensor:
    tokens, experts = logits.shape
    logits = _route_rows(logits)
    weights, ids, grad = weights.contiguous(), ids.contiguous(), grad.to(torch.float32).contiguous()
    out = torch.empty(tokens, experts, dtype=logits.dtype, device=logits.device)
    with on_device(logits.device):
        rc = _lib.lib.tb_moe_route_backward(logits.data_ptr(), _lib.DTYPE_CODE[logits.dtype], logits.stride(0), tokens, experts,
                                            ids.shape[1], int(sigmoid), int(renormalize), weights.data_ptr(), ids.data_ptr(),
                                            grad.data_ptr(), out.data_ptr(), _lib.current_stream_ptr(logits.device))
    _lib.check(rc, "tb_moe_route_backward")
    return out


@_moe_route_backward.register_fake
def _(logits, weights, ids, grad, sigmoid, renormalize):
    return logits.new_empty(logits.shape)


def _setup_context_route(ctx, inputs, output):
    logits, _, ctx.sigmoid, ctx.renormalize = inputs
    weights, ids = output
    ctx.mark_non_differentiable(ids)
    ctx.save_for_backward(logits, weights, ids)


def _route_backwards(ctx, grad_weights, _grad_ids):
    logits, weights, ids = ctx.saved_tensors
    return _moe_route_backward(logits, weights, ids, grad_weights, ctx.sigmoid, ctx.renormalize), None, None, None


_moe_route.register_autograd(_route_backwards, setup_context=_setup_context_route)


def moe_route(logits, topk, scoring="softmax", renormalize=True):
    """The ``topk`` experts of every token and their weights: ``(weights, ids)``, both (tokens, topk), float32 and int32.

    logits: (tokens, experts) in float16, bfloat16 or float32. The experts of a row are those with the largest logits, larger
    first, ties to the lowest index. A weight is the expert's softmax (``scoring="sigmoid"``: sigmoid) score, computed in
    float32; with ``renormalize`` a row's weights are divided by their sum. An expert whose logit is -inf (masked) or NaN is
    never chosen; a row with fewer than ``topk`` others gets id -1 and weight 0 in the remaining places, which every expert path
    of this package skips. At most 1024 experts and ``topk`` 32. The weights are differentiable in the logits.
    """
    require(logits.ndim == 2, "logits must be (tokens, experts)")
    require(logits.dtype in (torch.float16, torch.bfloat16, torch.float32), f"logits must be float16, bfloat16 or float32, got {logits.dtype}")
    require(scoring in _SCORING, f"scoring must be 'softmax' or 'sigmoid', got {scoring!r}")
    require(1 <= logits.shape[1] <= _MAX_EXPERTS, f"between 1 and {_MAX_EXPERTS} experts, got {logits.shape[1]}")
    topk = int(topk)
    require(1 <= topk <= min(_MAX_TOPK, logits.shape[1]), f"topk must be between 1 and min({_MAX_TOPK}, experts), got {topk}")
    sigmoid, renormalize = _SCORING[scoring], int(bool(renormalize))
    if torch.compiler.is_compiling() or (torch.is_grad_enabled() and logits.requires_grad):
        return _moe_route(logits, topk, bool(sigmoid), bool(renormalize))
    require_cuda(logits)
    return _route_forward(logits, topk, sigmoid, renormalize)    # no dispatcher round trip on the serving path


# -------------------------------------------------------------------------------------------------------- expert layer
def moe_mlp(x, w1, w2, topk_ids, topk_weights, out: Optional[torch.Tensor] = None):
    """Expert feed-forward of up to 128 tokens in two launches:
    ``out[t] = sum_j topk_weights[t, j] * (silu(x[t] @ gate.T) * (x[t] @ up.T)) @ w2[e].T`` with ``e = topk_ids[t, j]`` and
    ``w1[e] = [gate; up]``.

    x: (tokens, hidden); w1: (experts, 2*ffn, hidden) and w2: (experts, hidden, ffn), the layout ``PeerMemoryMoE`` takes; all
    float16 or all bfloat16, hidden and ffn multiples of 8. topk_ids: (tokens, topk) int32 or int64, topk_weights: (tokens, topk),
    as ``moe_route`` returns them. An id outside [0, experts) adds nothing; the same id twice counts twice. Sums, activation and
    weighting are float32 with one cast at the end. ``out`` may be given: (tokens, hidden), contiguous rows, no overlap with the
    weights. Inference only. More tokens: ``distributed.PeerMemoryMoE``.
    """
    require(x.ndim == 2 and w1.ndim == 3 and w2.ndim == 3 and topk_ids.ndim == 2, "x (tokens, hidden), w1 and w2 3-D, topk_ids 2-D")
    tokens, hidden = x.shape
    experts, ffn = w1.shape[0], w2.shape[2]
    require(w1.shape == (experts, 2 * ffn, hidden) and w2.shape == (experts, hidden, ffn),
             f"Incompatible Dimensions: x {tuple(x.shape)}, w1 {tuple(w1.shape)}, w2 {tuple(w2.shape)}")
    require(topk_ids.shape[0] == tokens and topk_weights.shape == topk_ids.shape, "topk_ids and topk_weights must be (tokens, topk)")
    require(x.dtype in (torch.float16, torch.bfloat16) and w1.dtype == x.dtype and w2.dtype == x.dtype,
             f"x, w1 and w2 must all be float16 or all bfloat16, got {x.dtype}, {w1.dtype}, {w2.dtype}")
    require(topk_ids.dtype in (torch.int32, torch.int64), "topk_ids must be int32 or int64")
    require(topk_weights.is_floating_point(), "topk_weights must be floating point")
    topk = topk_ids.shape[1]
    require(tokens <= MOE_MLP_MAX_TOKENS, f"moe_mlp takes at most {MOE_MLP_MAX_TOKENS} tokens, got {tokens}; use distributed.PeerMemoryMoE for more")
    require(1 <= topk <= _MAX_TOPK, f"topk must be between 1 and {_MAX_TOPK}, got {topk}")
    require(1 <= experts <= _MAX_EXPERTS, f"between 1 and {_MAX_EXPERTS} experts, got {experts}")
    require(hidden >= 8 and ffn >= 8 and hidden % 8 == 0 and ffn % 8 == 0, f"hidden and ffn must be multiples of 8, got {hidden} and {ffn}")
    require_cuda(x, w1, w2, topk_ids, topk_weights, out)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, w1, w2, topk_weights, out)):
        raise RuntimeError("tritonblas.moe_mlp(): inference only, but one of the arguments requires grad.")
    if out is None:
        out = torch.empty(tokens, hidden, dtype=x.dtype, device=x.device)
    else:
        require(out.shape == (tokens, hidden) and out.dtype == x.dtype, f"out must be {(tokens, hidden)} of {x.dtype}")
        require(out.stride(1) == 1 and (tokens <= 1 or out.stride(0) >= hidden), "out must have contiguous, non-overlapping rows")
    if tokens == 0:
        return out
    x, w1, w2 = (t if rows16(t) else t.clone(memory_format=torch.contiguous_format) for t in (x, w1, w2))
    ids, weights = topk_ids.contiguous(), topk_weights.to(torch.float32).contiguous()
    need = _lib.lib.tb_moe_mlp_workspace_bytes(tokens, topk, experts, hidden, ffn)
    # per call, from torch's allocator: calls on other streams and captured graphs never share it
    ws = torch.empty(need, dtype=torch.uint8, device=x.device)
    args = _lib.MoeMlpArgs(tokens, topk, experts, hidden, ffn, _lib.DTYPE_CODE[x.dtype], x.data_ptr(), x.stride(0),
                           w1.data_ptr(), w1.stride(0), w1.stride(1), w2.data_ptr(), w2.stride(0), w2.stride(1),
                           ids.data_ptr(), weights.data_ptr(), out.data_ptr(), out.stride(0), ws.data_ptr(), need,
                           int(ids.dtype == torch.int64), 0)
    with on_device(x.device):
        rc = _lib.lib.tb_moe_mlp(ctypes.byref(args), _lib.current_stream_ptr(x.device))
    _lib.check(rc, "tb_moe_mlp")
    return out
