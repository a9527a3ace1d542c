"""A shared projection beside the low-rank adapters of many requests: thin marshalling over the C ABI (tb_lora_gemm).

The reference has no adapters; ``lora_matmul`` stands beside ``matmul`` and ``addmm`` and takes the same weight layouts.
"""
import ctypes
from typing import Optional

import torch

from . import _lib
from ._checks import on_device, require, require_cuda, rows16
from .matmul import _repitch, _strides, _tma_loadable, _unit_stride_2d

_MAX_RANK = 128
# Rows of one launch pair are limited so that its workspace stays below this; a call with more of them makes several.
_MAX_WORKSPACE = 256 << 20


def lora_matmul(x, w, lora_a, lora_b, adapter_ids, scales=None, bias=None, out: Optional[torch.Tensor] = None):
    """``out[t] = x[t] @ w + scales[a] * (x[t] @ lora_a[a].T) @ lora_b[a].T (+ bias)`` with ``a = adapter_ids[t]``.

    x: (tokens, k); w: (k, n) in any of ``matmul``'s layouts (k contiguous, i.e. stored (n, k), is the fast one); lora_a:
    (adapters, rank, k); lora_b: (adapters, n, rank); all float16 or all bfloat16. adapter_ids: (tokens,) int32 or int64 on the
    GPU, in any order; an id outside [0, adapters), -1 for instance, leaves the row to the shared projection. scales: (adapters,)
    or None for 1; bias: (n,). k and rank multiples of 8, rank up to 128. The sum is float32 and rounded once; the rank-sized
    products ``scales[a] * x[t] @ lora_a[a].T`` are rounded to the operands' type on the way. ``out`` may be given: (tokens, n),
    any strides, no overlap with the inputs. Inference only.
    """
    require(x.ndim == 2 and w.ndim == 2 and lora_a.ndim == 3 and lora_b.ndim == 3, "x and w must be 2-D, lora_a and lora_b 3-D")
    tokens, k = x.shape
    n = w.shape[1]
    adapters, rank = lora_a.shape[0], lora_a.shape[1]
    require(w.shape[0] == k and lora_a.shape[2] == k and lora_b.shape == (adapters, n, rank),
            f"Incompatible Dimensions: x {tuple(x.shape)}, w {tuple(w.shape)}, lora_a {tuple(lora_a.shape)}, lora_b {tuple(lora_b.shape)}")
    require(x.dtype in (torch.float16, torch.bfloat16) and w.dtype == x.dtype and lora_a.dtype == x.dtype and lora_b.dtype == x.dtype,
            f"x, w, lora_a and lora_b must all be float16 or all bfloat16, got {x.dtype}, {w.dtype}, {lora_a.dtype}, {lora_b.dtype}")
    require(k >= 8 and k % 8 == 0, f"k must be a multiple of 8, got {k}")
    require(8 <= rank <= _MAX_RANK and rank % 8 == 0, f"rank must be a multiple of 8 up to {_MAX_RANK}, got {rank}")
    require(adapters >= 1, "at least one adapter")
    require(adapter_ids.shape == (tokens,) and adapter_ids.dtype in (torch.int32, torch.int64), "adapter_ids must be (tokens,) int32 or int64")
    require(scales is None or (scales.shape == (adapters,) and scales.is_floating_point()), "scales must be (adapters,) floating point")
    require(bias is None or (bias.shape == (n,) and bias.dtype in (torch.float16, torch.bfloat16, torch.float32)),
            "bias must be (n,) in float16, bfloat16 or float32")
    require(out is None or (out.shape == (tokens, n) and out.dtype == x.dtype), f"out must be {(tokens, n)} of {x.dtype}")
    require_cuda(x, w, lora_a, lora_b, adapter_ids, scales, bias, out)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, w, lora_a, lora_b, scales, bias, out)):
        raise RuntimeError("tritonblas.lora_matmul(): inference only, but one of the arguments requires grad.")
    if out is None:
        out = torch.empty(tokens, n, dtype=x.dtype, device=x.device)
    if tokens == 0 or n == 0:
        return out
    x, lora_a, lora_b = (t if rows16(t) else t.clone(memory_format=torch.contiguous_format) for t in (x, lora_a, lora_b))
    w = _unit_stride_2d(w)
    w = w if _tma_loadable(w) else _repitch(w)
    ids = adapter_ids.contiguous()
    scales = None if scales is None else scales.to(torch.float32).contiguous()

    def args_for(rows, first):
        xs, os = x[first:first + rows], out[first:first + rows]
        w_k, w_n = _strides(w)
        o_m, o_n = os.stride()
        return _lib.LoraArgs(rows, n, k, rank, adapters, _lib.DTYPE_CODE[x.dtype], xs.data_ptr(), x.stride(0), w.data_ptr(), w_k, w_n,
                             lora_a.data_ptr(), lora_a.stride(0), lora_a.stride(1), lora_b.data_ptr(), lora_b.stride(0), lora_b.stride(1),
                             ids.data_ptr() + first * ids.element_size(), 0 if scales is None else scales.data_ptr(),
                             0 if bias is None else bias.data_ptr(), 0 if bias is None else bias.stride(0), os.data_ptr(), o_m, o_n,
                             0, 0, 0 if bias is None else _lib.DTYPE_CODE[bias.dtype], int(ids.dtype == torch.int64), 0)

    with on_device(x.device):
        stream = _lib.current_stream_ptr(x.device)
        rows, first, args = tokens, 0, args_for(tokens, 0)
        need = _lib.lib.tb_lora_workspace_bytes(ctypes.byref(args))
        while need > _MAX_WORKSPACE and rows > 256:
            rows = max(256, (rows // 2 + 255) // 256 * 256)
            args = args_for(rows, 0)
            need = _lib.lib.tb_lora_workspace_bytes(ctypes.byref(args))
        # per call, from torch's allocator: calls on other streams and captured graphs never share it
        ws = torch.empty(need, dtype=torch.uint8, device=x.device)
        while True:
            args.workspace, args.workspace_bytes = ws.data_ptr(), ws.numel()
            rc = _lib.lib.tb_lora_gemm(ctypes.byref(args), stream)
            _lib.check(rc, "tb_lora_gemm")
            first += rows
            if first >= tokens:
                return out
            rows = min(rows, tokens - first)
            args = args_for(rows, first)
            need = _lib.lib.tb_lora_workspace_bytes(ctypes.byref(args))
            if need > ws.numel():       # the shorter last piece may be cut differently
                ws = torch.empty(need, dtype=torch.uint8, device=x.device)
