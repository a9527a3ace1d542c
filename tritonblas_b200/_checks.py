"""Argument checks and small launch helpers shared by the per-token operators.

These operators run in microseconds, so their argument checks are plain ``if not ...: refuse(...)`` statements: nothing is
formatted unless a call is refused."""
import contextlib

import torch

_nullcontext = contextlib.nullcontext()


def refuse(message):
    raise ValueError(message)


def refuse_devices(*tensors):
    """Error for tensors that are not all on one CUDA device."""
    if not all(t.is_cuda for t in tensors if t is not None):
        raise RuntimeError("tritonblas_b200 runs on CUDA tensors only (no CPU path)")
    raise RuntimeError(f"all tensors must be on one device, got {[str(t.device) for t in tensors if t is not None]}")


def on_device(device):
    """Context that makes ``device`` current; free when it already is."""
    return _nullcontext if device.index == torch.cuda.current_device() else torch.cuda.device(device)


def rows16(t):
    """True when the last axis is contiguous and rows start on 16-byte boundaries and do not overlap (TMA reads it in place).
    For tensors whose last axis is a multiple of 16 bytes."""
    if t.data_ptr() % 16:
        return False
    if t.is_contiguous():
        return True
    strides, shape = t.stride(), t.shape
    if strides[-1] != 1:
        return False
    per16, row = 16 // t.element_size(), shape[-1]
    for n, s in zip(shape[:-1], strides[:-1]):
        if n != 1 and (s < row or s % per16):
            return False
    return True
