"""What the operators' bindings share: type codes, argument checks, the raw stream and the device guard."""
import contextlib

import torch

from .. import _lib

DTYPES = {torch.float32: _lib.OPE_F32, torch.bfloat16: _lib.OPE_BF16, torch.float16: _lib.OPE_F16}
E4M3 = torch.float8_e4m3fn
_NONE = contextlib.nullcontext()


def dtype_code(t, name):
    code = DTYPES.get(t.dtype)
    if code is None:
        raise TypeError("%s: float32, bfloat16 or float16 wanted, got %s" % (name, t.dtype))
    return code


def want(t, name, shape=None, dtype=None):
    """`t` is a tensor of that shape and type (None = not checked)."""
    if not isinstance(t, torch.Tensor):
        raise TypeError("%s: a tensor wanted, got %s" % (name, type(t).__name__))
    if shape is not None and tuple(t.shape) != tuple(shape):
        raise ValueError("%s: shape %s wanted, got %s" % (name, tuple(shape), tuple(t.shape)))
    if dtype is not None and t.dtype != dtype:
        raise TypeError("%s: %s wanted, got %s" % (name, dtype, t.dtype))


def on_device(first, *others):
    """All tensors live on one GPU; returns a context that makes it the current device (and costs nothing where it already is)."""
    if not first.is_cuda:
        raise ValueError("the operators run on the GPU only: got a tensor on %s" % first.device)
    for t in others:
        if t is not None and t.device != first.device:
            raise ValueError("tensors on %s and %s in one call" % (first.device, t.device))
    return _NONE if torch.cuda.current_device() == first.device.index else torch.cuda.device(first.device)


def inner(t):
    """`t` with its last axis contiguous (a copy where it is not)."""
    return t if t.stride(-1) == 1 or t.shape[-1] <= 1 else t.contiguous()


def rows_of(t, width):
    """`t` [..., width] as rows [n, width] at one stride, without a copy where its layout allows it. A stride below the width (an expanded
    axis) is fine for what is only read."""
    return inner(t.reshape(-1, width))


def like(t):
    """An empty tensor of t's shape, in t's order of axes where that keeps the last one contiguous."""
    out = torch.empty_like(t)
    return out if out.shape[-1] <= 1 or out.stride(-1) == 1 else torch.empty(t.shape, dtype=t.dtype, device=t.device)


def stream():
    return _lib.current_stream()


def wants_grad(*tensors):
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def scratch(nbytes, device, what):
    """Workspace of a call (None where it needs none); a negative size is the library's refusal of the configuration."""
    if nbytes < 0:
        _lib.check(nbytes, what)
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


def ptr(t):
    return None if t is None else t.data_ptr()
