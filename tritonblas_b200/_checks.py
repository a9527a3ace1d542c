"""Argument checks and small launch helpers shared by the per-token operators."""
import contextlib

import torch

_nullcontext = contextlib.nullcontext()


def require(ok, message):
    if not ok:
        raise ValueError(message)


def require_cuda(first, *others):
    if not first.is_cuda:
        raise RuntimeError("tritonblas_b200 runs on CUDA tensors only (no CPU path)")
    for t in others:
        if t is not None and t.device != first.device:
            raise RuntimeError(f"all tensors must be on one device, got {first.device} and {t.device}")


def on_device(device):
    """Context that makes ``device`` current; free when it already is."""
    return _nullcontext if device.index == torch.cuda.current_device() else torch.cuda.device(device)


def rows16(t):
    """True when the last axis is contiguous and rows start on 16-byte boundaries and do not overlap (TMA reads it in place)."""
    per16 = 16 // t.element_size()
    return t.stride(-1) == 1 and t.data_ptr() % 16 == 0 and all(
        n == 1 or (s >= t.shape[-1] and s % per16 == 0) for n, s in zip(t.shape[:-1], t.stride()[:-1]))
