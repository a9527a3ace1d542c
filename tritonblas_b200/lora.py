"""A shared projection beside the low-rank adapters of many requests: thin marshalling over the C ABI (tb_lora_gemm).

The reference has no adapters; ``lora_matmul`` stands beside ``matmul`` and ``addmm`` and takes the same weight layouts.
"""
import ctypes
from typing import Optional

import torch
from torch.autograd import forward_ad

from . import _lib
from ._checks import on_device, overlaps_itself, refuse, refuse_devices, refuse_tangents, rows16, traced
from .matmul import _repitch, _strides, _tma_loadable, _unit_stride_2d

_MAX_RANK = 128
# Rows of one launch pair are limited so that its workspace stays below this; a call with more of them makes several.
_MAX_WORKSPACE = 256 << 20


def _check(x, w, lora_a, lora_b, adapter_ids, scales, bias, out):
    if x.ndim != 2 or w.ndim != 2 or lora_a.ndim != 3 or lora_b.ndim != 3:
        refuse("x and w must be 2-D, lora_a and lora_b 3-D")
    tokens, k = x.shape
    n = w.shape[1]
    adapters, rank, _ = lora_a.shape
    dtype, device = x.dtype, x.device
    if w.shape[0] != k or lora_a.shape[2] != k or lora_b.shape != (adapters, n, rank):
        refuse(f"Incompatible Dimensions: x {tuple(x.shape)}, w {tuple(w.shape)}, lora_a {tuple(lora_a.shape)}, lora_b {tuple(lora_b.shape)}")
    if (dtype is not torch.bfloat16 and dtype is not torch.float16) or w.dtype is not dtype or lora_a.dtype is not dtype \
            or lora_b.dtype is not dtype:
        refuse(f"x, w, lora_a and lora_b must all be float16 or all bfloat16, got {x.dtype}, {w.dtype}, {lora_a.dtype}, {lora_b.dtype}")
    if k < 8 or k % 8:
        refuse(f"k must be a multiple of 8, got {k}")
    if not 8 <= rank <= _MAX_RANK or rank % 8:
        refuse(f"rank must be a multiple of 8 up to {_MAX_RANK}, got {rank}")
    if adapters < 1:
        refuse("at least one adapter")
    if adapter_ids.ndim != 1 or adapter_ids.shape[0] != tokens or adapter_ids.dtype not in (torch.int32, torch.int64):
        refuse("adapter_ids must be (tokens,) int32 or int64")
    if scales is not None and (scales.shape != (adapters,) or not scales.is_floating_point()):
        refuse("scales must be (adapters,) floating point")
    if bias is not None and (bias.shape != (n,) or bias.dtype not in (torch.float16, torch.bfloat16, torch.float32)):
        refuse("bias must be (n,) in float16, bfloat16 or float32")
    if out is not None and (out.shape != (tokens, n) or out.dtype is not dtype):
        refuse(f"out must be {(tokens, n)} of {dtype}")
    if out is not None and tokens and n and overlaps_itself(out):
        refuse("out must not overlap itself")
    if not x.is_cuda or not device == w.device == lora_a.device == lora_b.device == adapter_ids.device \
            or (scales is not None and scales.device != device) or (bias is not None and bias.device != device) \
            or (out is not None and out.device != device):
        refuse_devices(x, w, lora_a, lora_b, adapter_ids, scales, bias, out)
    if torch.is_grad_enabled() and (x.requires_grad or w.requires_grad or lora_a.requires_grad or lora_b.requires_grad
                                    or (scales is not None and scales.requires_grad) or (bias is not None and bias.requires_grad)
                                    or (out is not None and out.requires_grad)):
        raise RuntimeError("tritonblas.lora_matmul(): inference only, but one of the arguments requires grad.")
    return tokens, k, n, adapters, rank, dtype, device


def _run(checked, x, w, lora_a, lora_b, adapter_ids, scales, bias, out):
    tokens, k, n, adapters, rank, dtype, device = checked
    if out is None:
        out = torch.empty(tokens, n, dtype=dtype, device=device)
    if tokens == 0 or n == 0:
        return out
    if out.data_ptr() == x.data_ptr():
        refuse("out must not be x: other columns of its rows are still read while the first ones are written")
    if not rows16(x):
        x = x.clone(memory_format=torch.contiguous_format)
    if not rows16(lora_a):
        lora_a = lora_a.clone(memory_format=torch.contiguous_format)
    if not rows16(lora_b):
        lora_b = lora_b.clone(memory_format=torch.contiguous_format)
    w_k, w_n = w.stride()
    if w_k != 1 or w_n < k or w_n % 8 or w.data_ptr() % 16:     # anything but the fast layout
        w = _unit_stride_2d(w)
        w_k, w_n = _strides(w)
        if not _tma_loadable(w) or (w_n < k if w_k == 1 else w_k < n):     # or rows that overlap: an expanded w
            w = _repitch(w)
            w_k, w_n = _strides(w)
    ids = adapter_ids.contiguous()
    if scales is not None:
        scales = scales.to(torch.float32).contiguous()
    x_row, (o_m, o_n), a_strides, b_strides = x.stride(0), out.stride(), lora_a.stride(), lora_b.stride()
    es, id_size = x.element_size(), ids.element_size()
    args = _lib.LoraArgs(tokens, n, k, rank, adapters, _lib.DTYPE_CODE[dtype], x.data_ptr(), x_row, w.data_ptr(), w_k, w_n,
                         lora_a.data_ptr(), a_strides[0], a_strides[1], lora_b.data_ptr(), b_strides[0], b_strides[1],
                         ids.data_ptr(), None if scales is None else scales.data_ptr(),
                         None if bias is None else bias.data_ptr(), 0 if bias is None else bias.stride(0), out.data_ptr(), o_m, o_n,
                         None, 0, 0 if bias is None else _lib.DTYPE_CODE[bias.dtype], int(ids.dtype is torch.int64), 0)
    ref = ctypes.byref(args)
    # the plan behind both calls goes by the current device's SMs
    with on_device(device):
        need = _lib.lib.tb_lora_workspace_bytes(ref)
        rows = tokens
        while (need > _MAX_WORKSPACE or need == 0) and rows > 256:     # 0: more rows than one launch pair can number
            args.m = rows = max(256, (rows // 2 + 255) // 256 * 256)
            need = _lib.lib.tb_lora_workspace_bytes(ref)
        # per call, from torch's allocator: calls on other streams and captured graphs never share it
        ws = torch.empty(need, dtype=torch.uint8, device=device)
        args.workspace, args.workspace_bytes = ws.data_ptr(), need
        stream = _lib.current_stream_ptr(device)
        first = 0
        while True:
            rc = _lib.lib.tb_lora_gemm(ref, stream)
            _lib.check(rc, "tb_lora_gemm")
            first += rows
            if first >= tokens:
                return out
            rows = min(rows, tokens - first)
            args.m = rows
            args.x, args.adapter_ids = x.data_ptr() + first * x_row * es, ids.data_ptr() + first * id_size
            args.out = out.data_ptr() + first * o_m * es
            need = _lib.lib.tb_lora_workspace_bytes(ref)
            if need > ws.numel():       # the shorter last piece may be cut differently
                ws = torch.empty(need, dtype=torch.uint8, device=device)
                args.workspace, args.workspace_bytes = ws.data_ptr(), need


@torch.library.custom_op("tritonblas::_lora_matmul", mutates_args=())
def _lora_matmul(x: torch.Tensor, w: torch.Tensor, lora_a: torch.Tensor, lora_b: torch.Tensor, adapter_ids: torch.Tensor,
                 scales: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    return _run(_check(x, w, lora_a, lora_b, adapter_ids, scales, bias, None), x, w, lora_a, lora_b, adapter_ids, scales, bias, None)


@_lora_matmul.register_fake
def _(x, w, lora_a, lora_b, adapter_ids, scales=None, bias=None):
    return x.new_empty(x.shape[0], w.shape[1])


@torch.library.custom_op("tritonblas::_lora_matmul_out", mutates_args={"out"})
def _lora_matmul_out(x: torch.Tensor, w: torch.Tensor, lora_a: torch.Tensor, lora_b: torch.Tensor, adapter_ids: torch.Tensor,
                     out: torch.Tensor, scales: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None) -> None:
    _run(_check(x, w, lora_a, lora_b, adapter_ids, scales, bias, out), x, w, lora_a, lora_b, adapter_ids, scales, bias, out)


def lora_matmul(x, w, lora_a, lora_b, adapter_ids, scales=None, bias=None, out: Optional[torch.Tensor] = None):
    """``out[t] = x[t] @ w + scales[a] * (x[t] @ lora_a[a].T) @ lora_b[a].T (+ bias)`` with ``a = adapter_ids[t]``.

    x: (tokens, k); w: (k, n) in any of ``matmul``'s layouts (k contiguous, i.e. stored (n, k), is the fast one); lora_a:
    (adapters, rank, k); lora_b: (adapters, n, rank); all float16 or all bfloat16. adapter_ids: (tokens,) int32 or int64 on the
    GPU, in any order; an id outside [0, adapters), -1 for instance, leaves the row to the shared projection. scales: (adapters,)
    or None for 1; bias: (n,). k and rank multiples of 8, rank up to 128. The sum is float32 and rounded once. The rank-sized
    products ``scales[a] * x[t] @ lora_a[a].T`` are operands of a tensor-core product and kept in two 16-bit halves: to 2^-16
    relative in bfloat16; in float16 to 2^-22 relative or 2^-25 absolute, and infinite above 65504. ``out`` may be given:
    (tokens, n), any strides, no overlap with itself or the inputs. Inference only.

    Infinities and NaN in x, lora_a, lora_b and scales stay with the rows that use them; calls that meet some are slower.
    """
    checked = _check(x, w, lora_a, lora_b, adapter_ids, scales, bias, out)
    if forward_ad._current_level >= 0:
        refuse_tangents("lora_matmul", x, w, lora_a, lora_b, scales, bias)
    if traced(x):
        if out is None:
            return _lora_matmul(x, w, lora_a, lora_b, adapter_ids, scales, bias)
        _lora_matmul_out(x, w, lora_a, lora_b, adapter_ids, out, scales, bias)
        return out
    return _run(checked, x, w, lora_a, lora_b, adapter_ids, scales, bias, out)
