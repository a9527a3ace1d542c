"""Argument checks and small launch helpers shared by the per-token operators.

These operators run in microseconds, so their argument checks are plain ``if not ...: refuse(...)`` statements: nothing is
formatted unless a call is refused."""
import contextlib
import math

import torch
from torch.autograd import forward_ad

_nullcontext = contextlib.nullcontext()
_PLAIN = (torch.Tensor, torch.nn.Parameter)
_is_compiling = torch.compiler.is_compiling
_dispatch_modes = torch._C._len_torch_dispatch_stack
_transform = torch._C._functorch.peek_interpreter_stack


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


def overlaps_itself(t):
    """True when two elements of a 2-D tensor share memory: an expanded tensor, or a pitch shorter than a row."""
    if t.is_contiguous():
        return False
    (n0, n1), (s0, s1) = t.shape, t.stride()
    if (n0 > 1 and s0 == 0) or (n1 > 1 and s1 == 0):
        return True
    step = math.gcd(s0, s1)     # i s0 = j s1 for the first time at i = s1 / step, j = s0 / step
    return s1 // step < n0 and s0 // step < n1


def traced(t):
    """True where a call has to go through its registered operator because something looks at it or rewrites it: torch.compile, fake
    tensors and other subclasses, a dispatch mode (torch.export, make_fx, ...), a torch.func transform. Plain eager calls skip the
    dispatcher, which costs more than the operators run."""
    return _is_compiling() or type(t) not in _PLAIN or _dispatch_modes() > 0 or _transform() is not None


def refuse_tangents(name, *tensors):
    """Error for dual tensors of forward-mode differentiation: their tangents would be lost."""
    if forward_ad._current_level >= 0 and any(t is not None and t.is_floating_point() and forward_ad.unpack_dual(t).tangent is not None
                                              for t in tensors):
        raise RuntimeError(f"tritonblas.{name}(): no forward-mode derivative.")
