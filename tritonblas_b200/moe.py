"""Expert router and the expert feed-forward of a few tokens: thin marshalling over the C ABI (tb_moe_route, tb_moe_mlp).

``moe_route`` turns router logits into the ids and weights every expert path of this package takes; ``moe_mlp`` is the whole
expert layer of a decode batch in two launches. Batches of more than 128 tokens go through ``distributed.PeerMemoryMoE`` /
``distributed.ExpertParallelMoE``, whose grouped GEMMs work on 128-row tiles. The reference has no MoE path.
"""
import ctypes
import operator
from typing import Optional, Tuple

import torch
from torch.autograd import forward_ad

from . import _lib
from ._checks import on_device, refuse, refuse_devices, refuse_tangents, rows16, traced

MOE_MLP_MAX_TOKENS = 128
_MAX_EXPERTS, _MAX_TOPK = 1024, 32
_SCORING = {"softmax": 0, "sigmoid": 1}
_ROUTE_TYPES = (torch.float16, torch.bfloat16, torch.float32)

# ------------------------------------------------------------------------------------------------------------- router
def _route_rows(logits):
    """The logits as rows with unit column stride and a row stride of at least their length."""
    if logits.stride(1) == 1 and (logits.shape[0] <= 1 or logits.stride(0) >= logits.shape[1]):
        return logits
    return logits.contiguous()


def _route_forward(logits, topk, sigmoid, renormalize):
    if not logits.is_cuda:
        refuse_devices(logits)
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


def _route_backward(logits, weights, ids, grad, sigmoid, renormalize):
    tokens, experts = logits.shape
    if not logits.is_cuda or not logits.device == weights.device == ids.device == grad.device:
        refuse_devices(logits, weights, ids, grad)
    if not (weights.shape == ids.shape == grad.shape and ids.ndim == 2 and ids.shape[0] == tokens):
        refuse("weights, ids and their gradient must be (tokens, topk)")
    logits = _route_rows(logits)
    weights, ids, grad = weights.contiguous(), ids.contiguous(), grad.to(torch.float32).contiguous()
    out = torch.empty(tokens, experts, dtype=logits.dtype, device=logits.device)
    with on_device(logits.device):
        rc = _lib.lib.tb_moe_route_backward(logits.data_ptr(), _lib.DTYPE_CODE[logits.dtype], logits.stride(0), tokens, experts,
                                            ids.shape[1], sigmoid, renormalize, weights.data_ptr(), ids.data_ptr(),
                                            grad.data_ptr(), out.data_ptr(), _lib.current_stream_ptr(logits.device))
    _lib.check(rc, "tb_moe_route_backward")
    return out


class _Route(torch.autograd.Function):
    """The eager path; traced code goes through the custom operators below, which are the same two calls."""

    @staticmethod
    def forward(ctx, logits, topk, sigmoid, renormalize):
        weights, ids = _route_forward(logits, topk, sigmoid, renormalize)
        ctx.mark_non_differentiable(ids)
        ctx.save_for_backward(logits, weights, ids)
        ctx.modes = sigmoid, renormalize
        return weights, ids

    @staticmethod
    def backward(ctx, grad_weights, _grad_ids):
        if torch.is_grad_enabled():     # create_graph=True
            raise RuntimeError("tritonblas.moe_route(): the gradient is not differentiable again.")
        return _route_backward(*ctx.saved_tensors, grad_weights, *ctx.modes), None, None, None


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
    return _route_backward(logits, weights, ids, grad, int(sigmoid), int(renormalize))


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
    of this package skips. A logit of +inf makes its row's softmax weights NaN, as the formula does. At most 1024 experts and
    ``topk`` 32. The weights are differentiable in the logits, once; a backward pass that is captured into a CUDA graph must not
    share leaves with the autograd graph of an earlier eager pass that is still referenced, as anywhere in torch.
    """
    if logits.ndim != 2:
        refuse("logits must be (tokens, experts)")
    if logits.dtype not in _ROUTE_TYPES:
        refuse(f"logits must be float16, bfloat16 or float32, got {logits.dtype}")
    if scoring not in _SCORING:
        refuse(f"scoring must be 'softmax' or 'sigmoid', got {scoring!r}")
    experts = logits.shape[1]
    if not 1 <= experts <= _MAX_EXPERTS:
        refuse(f"between 1 and {_MAX_EXPERTS} experts, got {experts}")
    topk = operator.index(topk)     # a whole number: 2.5 is not 2
    if not 1 <= topk <= min(_MAX_TOPK, experts):
        refuse(f"topk must be between 1 and min({_MAX_TOPK}, experts), got {topk}")
    sigmoid, renormalize = _SCORING[scoring], 1 if renormalize else 0
    if forward_ad._current_level >= 0:
        refuse_tangents("moe_route", logits)
    if traced(logits):
        return _moe_route(logits, topk, bool(sigmoid), bool(renormalize))
    if logits.requires_grad and torch.is_grad_enabled():
        return _Route.apply(logits, topk, sigmoid, renormalize)
    return _route_forward(logits, topk, sigmoid, renormalize)


# -------------------------------------------------------------------------------------------------------- expert layer
def _check_mlp(x, w1, w2, topk_ids, topk_weights, out):
    if x.ndim != 2 or w1.ndim != 3 or w2.ndim != 3 or topk_ids.ndim != 2:
        refuse("x must be (tokens, hidden), w1 and w2 3-D, topk_ids 2-D")
    tokens, hidden = x.shape
    experts, _, ffn = w2.shape
    dtype, device = x.dtype, x.device
    if w1.shape != (experts, 2 * ffn, hidden) or w2.shape[1] != hidden:
        refuse(f"Incompatible Dimensions: x {tuple(x.shape)}, w1 {tuple(w1.shape)}, w2 {tuple(w2.shape)}")
    topk = topk_ids.shape[1]
    if topk_ids.shape[0] != tokens or topk_weights.shape != topk_ids.shape:
        refuse("topk_ids and topk_weights must be (tokens, topk)")
    if (dtype is not torch.bfloat16 and dtype is not torch.float16) or w1.dtype is not dtype or w2.dtype is not dtype:
        refuse(f"x, w1 and w2 must all be float16 or all bfloat16, got {x.dtype}, {w1.dtype}, {w2.dtype}")
    if topk_ids.dtype not in (torch.int32, torch.int64):
        refuse("topk_ids must be int32 or int64")
    if not topk_weights.is_floating_point():
        refuse("topk_weights must be floating point")
    if tokens > MOE_MLP_MAX_TOKENS:
        refuse(f"moe_mlp takes at most {MOE_MLP_MAX_TOKENS} tokens, got {tokens}; use distributed.PeerMemoryMoE for more")
    if not 1 <= topk <= _MAX_TOPK:
        refuse(f"topk must be between 1 and {_MAX_TOPK}, got {topk}")
    if not 1 <= experts <= _MAX_EXPERTS:
        refuse(f"between 1 and {_MAX_EXPERTS} experts, got {experts}")
    if hidden < 8 or ffn < 8 or hidden % 8 or ffn % 8:
        refuse(f"hidden and ffn must be multiples of 8, got {hidden} and {ffn}")
    if not x.is_cuda or not device == w1.device == w2.device == topk_ids.device == topk_weights.device:
        refuse_devices(x, w1, w2, topk_ids, topk_weights)
    if torch.is_grad_enabled() and (x.requires_grad or w1.requires_grad or w2.requires_grad or topk_weights.requires_grad
                                    or (out is not None and out.requires_grad)):
        raise RuntimeError("tritonblas.moe_mlp(): inference only, but one of the arguments requires grad.")
    if out is not None:
        if out.shape != (tokens, hidden) or out.dtype is not dtype:
            refuse(f"out must be {(tokens, hidden)} of {dtype}")
        if out.device != device:
            refuse_devices(x, out)
        if out.stride(1) != 1 or (tokens > 1 and out.stride(0) < hidden):
            refuse("out must have contiguous, non-overlapping rows")
    return tokens, topk, experts, hidden, ffn, dtype, device


def _run_mlp(checked, x, w1, w2, topk_ids, topk_weights, out):
    tokens, topk, experts, hidden, ffn, dtype, device = checked
    if out is None:
        out = torch.empty(tokens, hidden, dtype=dtype, device=device)
    if tokens == 0:
        return out
    if not rows16(x):
        x = x.clone(memory_format=torch.contiguous_format)
    if not rows16(w1):
        w1 = w1.clone(memory_format=torch.contiguous_format)
    if not rows16(w2):
        w2 = w2.clone(memory_format=torch.contiguous_format)
    ids, weights = topk_ids.contiguous(), topk_weights.to(torch.float32).contiguous()
    need = _lib.lib.tb_moe_mlp_workspace_bytes(tokens, topk, experts, hidden, ffn)
    # per call, from torch's allocator: calls on other streams and captured graphs never share it
    ws = torch.empty(need, dtype=torch.uint8, device=device)
    w1_strides, w2_strides = w1.stride(), w2.stride()
    args = _lib.MoeMlpArgs(tokens, topk, experts, hidden, ffn, _lib.DTYPE_CODE[dtype], x.data_ptr(), x.stride(0),
                           w1.data_ptr(), w1_strides[0], w1_strides[1], w2.data_ptr(), w2_strides[0], w2_strides[1],
                           ids.data_ptr(), weights.data_ptr(), out.data_ptr(), out.stride(0), ws.data_ptr(), need,
                           int(ids.dtype is torch.int64), 0)
    with on_device(device):
        rc = _lib.lib.tb_moe_mlp(ctypes.byref(args), _lib.current_stream_ptr(device))
    _lib.check(rc, "tb_moe_mlp")
    return out


@torch.library.custom_op("tritonblas::_moe_mlp", mutates_args=())
def _moe_mlp(x: torch.Tensor, w1: torch.Tensor, w2: torch.Tensor, topk_ids: torch.Tensor, topk_weights: torch.Tensor) -> torch.Tensor:
    return _run_mlp(_check_mlp(x, w1, w2, topk_ids, topk_weights, None), x, w1, w2, topk_ids, topk_weights, None)


@_moe_mlp.register_fake
def _(x, w1, w2, topk_ids, topk_weights):
    return x.new_empty(x.shape)


@torch.library.custom_op("tritonblas::_moe_mlp_out", mutates_args={"out"})
def _moe_mlp_out(x: torch.Tensor, w1: torch.Tensor, w2: torch.Tensor, topk_ids: torch.Tensor, topk_weights: torch.Tensor,
                 out: torch.Tensor) -> None:
    _run_mlp(_check_mlp(x, w1, w2, topk_ids, topk_weights, out), x, w1, w2, topk_ids, topk_weights, out)


def moe_mlp(x, w1, w2, topk_ids, topk_weights, out: Optional[torch.Tensor] = None):
    """Expert feed-forward of up to 128 tokens in two launches:
    ``out[t] = sum_j topk_weights[t, j] * (silu(x[t] @ gate.T) * (x[t] @ up.T)) @ w2[e].T`` with ``e = topk_ids[t, j]`` and
    ``w1[e] = [gate; up]``.

    x: (tokens, hidden); w1: (experts, 2*ffn, hidden) and w2: (experts, hidden, ffn), the layout ``PeerMemoryMoE`` takes; all
    float16 or all bfloat16, hidden and ffn multiples of 8. topk_ids: (tokens, topk) int32 or int64, topk_weights: (tokens, topk),
    as ``moe_route`` returns them. An id outside [0, experts) adds nothing; the same id twice counts twice. Sums, activation and
    weighting are float32 with one cast at the end. silu(gate) * up is an operand of a tensor-core product and kept in two 16-bit
    halves: to 2^-16 relative in bfloat16; in float16 to 2^-22 relative or 2^-28 absolute, and infinite above 65504 * 256.
    ``out`` may be given: (tokens, hidden), contiguous rows, no overlap with the weights. Inference only. More tokens:
    ``distributed.PeerMemoryMoE``.
    """
    checked = _check_mlp(x, w1, w2, topk_ids, topk_weights, out)
    if forward_ad._current_level >= 0:
        refuse_tangents("moe_mlp", x, w1, w2, topk_weights)
    if traced(x):
        if out is None:
            return _moe_mlp(x, w1, w2, topk_ids, topk_weights)
        _moe_mlp_out(x, w1, w2, topk_ids, topk_weights, out)
        return out
    return _run_mlp(checked, x, w1, w2, topk_ids, topk_weights, out)
