"""What the operators' bindings share: type codes, argument checks, the raw stream and the device guard.

An agent acts one step at a time, so the host's share of a small call counts as much as the kernel's: what follows from sizes, strides and types
alone (the checks, the packed configuration, the workspaces' sizes) is worked out once for each combination and kept in an lru_cache; nothing
that depends on a tensor's place or contents is."""
import contextlib

import torch
from torch.autograd import forward_ad
from torch.fx.experimental import proxy_tensor

from .. import _lib

DTYPES = {torch.float32: _lib.OPE_F32, torch.bfloat16: _lib.OPE_BF16, torch.float16: _lib.OPE_F16}
E4M3 = torch.float8_e4m3fn
PLANS = 1024              # combinations of sizes and strides that are remembered for each entry point
_NONE = contextlib.nullcontext()
grad_enabled = torch.is_grad_enabled
stream = _lib.current_stream
_transforms = torch._C._functorch.peek_interpreter_stack


def dtype_code(dtype, name):
    code = DTYPES.get(dtype)
    if code is None:
        raise TypeError("%s: float32, bfloat16 or float16 wanted, got %s" % (name, dtype))
    return code


def tensors(*named):
    """Every (tensor, name) holds a tensor."""
    for t, name in named:
        if not isinstance(t, torch.Tensor):
            raise TypeError("%s: a tensor wanted, got %s" % (name, type(t).__name__))


def same_shape(shape, name, wanted):
    if tuple(shape) != tuple(wanted):
        raise ValueError("%s: shape %s wanted, got %s" % (name, tuple(wanted), tuple(shape)))


def same_dtype(dtype, name, wanted):
    if dtype != wanted:
        raise TypeError("%s: %s wanted, got %s" % (name, wanted, dtype))


def on_device(first, *others):
    """All tensors live on one GPU; returns a context that makes it the current device (and costs nothing where it already is)."""
    d = first.get_device()
    if d < 0:
        raise ValueError("the operators run on the GPU only: got a tensor on %s" % first.device)
    for t in others:
        if t is not None and t.get_device() != d:
            raise ValueError("tensors on %s and %s in one call" % (first.device, t.device))
    return _NONE if torch._C._cuda_getDevice() == d else torch.cuda.device(d)


def inner(t):
    """`t` with its last axis contiguous (a copy where it is not)."""
    return t if t.stride(-1) == 1 or t.shape[-1] <= 1 else t.contiguous()


def rows_of(t, width):
    """`t` [..., width] as rows at one stride, and that stride; a copy only where the layout has none. A stride below the width (an expanded axis)
    is fine for what is only read."""
    if t.is_contiguous():
        return t, width
    t = inner(t.reshape(-1, width))
    return t, t.stride(0)


def like(t):
    """An empty tensor of t's shape, in t's order of axes where that keeps the last one contiguous."""
    out = torch.empty_like(t)
    return out if out.shape[-1] <= 1 or out.stride(-1) == 1 else torch.empty(t.shape, dtype=t.dtype, device=t.device)


def plain_call(*ts):
    """Refuses what torch.autograd's tape alone would get right: the kernels are called by address, so a tracer would record the outputs' allocation and
    nothing that fills it (torch.jit.trace: untraced()), and a tangent (forward mode) or a batch axis (vmap) would be dropped."""
    if forward_ad._current_level < 0 and proxy_tensor._CURRENT_MAKE_FX_TRACER is None and _transforms() is None:
        return
    if proxy_tensor._CURRENT_MAKE_FX_TRACER is not None:
        raise RuntimeError("the memory operators cannot be recorded by make_fx")
    for t in ts:
        if t is None:
            continue
        if torch._C._functorch.is_functorch_wrapped_tensor(t):
            raise RuntimeError("the memory operators take no tensors inside torch.func transforms (vmap, grad, jvp): use torch.autograd")
        if forward_ad._current_level >= 0 and forward_ad.unpack_dual(t).tangent is not None:
            raise RuntimeError("the memory operators have no forward-mode derivative: a tensor with a tangent was given")


def untraced():
    """For what is worked out once for each combination of sizes: sizes are tensors while torch.jit.trace records, so such a call finds nothing kept and
    comes here."""
    if torch._C._get_tracing_state() is not None:
        raise RuntimeError("the memory operators cannot be recorded by torch.jit.trace")


def wants_grad(*ts):
    if grad_enabled():
        for t in ts:
            if t is not None and t.requires_grad:
                return True
    return False


def once(backward):
    """A backward pass that cannot be differentiated itself: refuses to be recorded (create_graph=True). torch's once_differentiable says it later,
    at the second differentiation, at three times the cost for every call."""
    def run(ctx, *grads):
        if grad_enabled():
            raise RuntimeError("the gradients of the memory operators cannot be differentiated again: no create_graph")
        plain_call(*grads)
        return backward(ctx, *grads)
    return staticmethod(run)


def size_or_raise(nbytes, what):
    """A negative size is the library's refusal of the configuration."""
    if nbytes < 0:
        _lib.check(nbytes, what)
    return nbytes


def scratch(nbytes, device):
    """Workspace of a call: (tensor, address, size); the tensor is held until the call has been enqueued."""
    if not nbytes:
        return None, None, 0
    t = torch.empty(nbytes, dtype=torch.uint8, device=device)
    return t, t.data_ptr(), nbytes


def ptr(t):
    return None if t is None else t.data_ptr()
