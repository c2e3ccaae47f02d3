"""RMS norm with the residual's addition, and rows in 8 bits (ope_rms_norm, ope_quantize_rows)."""
import struct

import torch
from torch.autograd.function import once_differentiable

from .. import _lib
from ._common import DTYPES, E4M3, dtype_code, on_device, ptr, rows_of, scratch, stream, want, wants_grad

_CFG = struct.Struct("qqqiiif")
_MAX_WIDTH = 1 << 20


def _cfg(rows, x_stride, r_stride, width, dtype, out_dtype, eps):
    return _CFG.pack(rows, x_stride, r_stride, width, dtype, out_dtype, eps)


def _check(x, weight, residual, eps):
    want(x, "x")
    code = dtype_code(x, "x")
    if x.dim() < 1 or not 1 <= x.shape[-1] <= _MAX_WIDTH:
        raise ValueError("x: at least one axis and a last one of 1 to %d wanted, got shape %s" % (_MAX_WIDTH, tuple(x.shape)))
    want(weight, "weight", (x.shape[-1],), x.dtype)
    if residual is not None:
        want(residual, "residual", x.shape, x.dtype)
    if not eps >= 0:
        raise ValueError("eps: zero or a positive number wanted, got %r" % (eps,))
    return code


def _forward(x, weight, residual, eps, code, fp8, rstd_too):
    """(y, scale, s, rstd), rows flattened."""
    D = x.shape[-1]
    rows, res = rows_of(x, D), None if residual is None else rows_of(residual, D)
    M, dev = rows.shape[0], x.device
    y = torch.empty(x.shape, dtype=E4M3 if fp8 else x.dtype, device=dev)
    scale = torch.empty(x.shape[:-1], dtype=torch.float32, device=dev) if fp8 else None
    s = None if residual is None else torch.empty(x.shape, dtype=x.dtype, device=dev)
    rstd = torch.empty(M, dtype=torch.float32, device=dev) if rstd_too else None
    weight = weight.contiguous()
    cfg = _cfg(M, rows.stride(0), 0 if res is None else res.stride(0), D, code, _lib.OPE_E4M3 if fp8 else code, eps)
    _lib.check(_lib.lib.ope_rms_norm(cfg, ptr(rows), ptr(res), ptr(weight), ptr(y), ptr(scale), ptr(s), ptr(rstd), stream()), "ope_rms_norm")
    return y, scale, s, rstd


class _RmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, residual, eps):
        code = DTYPES[x.dtype]
        with on_device(x, weight, residual):
            y, _, s, rstd = _forward(x, weight, residual, eps, code, False, True)
        ctx.save_for_backward(x if s is None else s, weight, rstd)
        ctx.eps, ctx.two = eps, s is not None
        ctx.set_materialize_grads(False)
        return y if s is None else (y, s)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dsum=None):
        s, weight, rstd = ctx.saved_tensors
        if dy is None and dsum is None:
            return None, None, None, None
        D = s.shape[-1]
        with on_device(s, weight, dy, dsum):
            dy = torch.zeros(s.shape, dtype=s.dtype, device=s.device) if dy is None else dy.contiguous()
            dsum = None if dsum is None else dsum.contiguous()
            rows = rows_of(s, D)
            dx = torch.empty(s.shape, dtype=s.dtype, device=s.device)
            dw = torch.empty(D, dtype=s.dtype, device=s.device)
            weight = weight.contiguous()
            code = DTYPES[s.dtype]
            cfg = _cfg(rows.shape[0], rows.stride(0), 0, D, code, code, ctx.eps)
            ws = scratch(_lib.lib.ope_rms_norm_backward_workspace_bytes(cfg), s.device, "ope_rms_norm_backward")
            _lib.check(_lib.lib.ope_rms_norm_backward(cfg, ptr(dy), ptr(dsum), ptr(rows), ptr(weight), ptr(rstd), ptr(dx), ptr(dw), ptr(ws),
                                                      0 if ws is None else ws.numel(), stream()), "ope_rms_norm_backward")
        return dx, dw, dx if ctx.two else None, None


def rms_norm(x, weight, residual=None, eps=1e-6):
    """y = s * weight / sqrt(mean(s^2) + eps) over the last axis, s = x + residual.

    x [..., D] float32, bfloat16 or float16, weight [D] and residual (x's shape) of the same type. Returns y, or (y, s) where a residual is
    given: s is what the next block adds to. The norm is taken of the float32 sum, in front of its rounding to x's type. Differentiable in x,
    weight and residual; the backward pass reads s as it was returned, so s must not be changed in place before it."""
    code = _check(x, weight, residual, eps)
    if wants_grad(x, weight, residual):
        on_device(x, weight, residual)
        return _RmsNorm.apply(x, weight, residual, float(eps))
    with on_device(x, weight, residual):
        y, _, s, _ = _forward(x, weight, residual, float(eps), code, False, False)
    return y if s is None else (y, s)


def rms_norm_fp8(x, weight, residual=None, eps=1e-6):
    """rms_norm with its output in 8 bits: returns (q, scale), or (q, scale, s) where a residual is given. q is float8_e4m3fn of x's shape, scale
    float32 of x.shape[:-1], y = q * scale; scale = max(max|y|, 448 * 2^-126) / 448 of the row. For acting: no gradients (a tensor that requires one
    is refused while gradients are recorded)."""
    code = _check(x, weight, residual, eps)
    if wants_grad(x, weight, residual):
        raise ValueError("rms_norm_fp8 has no gradients: call it under torch.no_grad(), or rms_norm")
    with on_device(x, weight, residual):
        y, scale, s, _ = _forward(x, weight, residual, float(eps), code, True, False)
    return (y, scale) if s is None else (y, scale, s)


def quantize_rows_fp8(x):
    """(q, scale) of the rows of x [..., D], by rms_norm_fp8's rule; for the weights of linear_fp8."""
    want(x, "x")
    code = dtype_code(x, "x")
    if x.dim() < 1 or not 1 <= x.shape[-1] <= _MAX_WIDTH:
        raise ValueError("x: at least one axis and a last one of 1 to %d wanted, got shape %s" % (_MAX_WIDTH, tuple(x.shape)))
    if wants_grad(x):
        raise ValueError("quantize_rows_fp8 has no gradients: call it under torch.no_grad()")
    D = x.shape[-1]
    with on_device(x):
        rows = rows_of(x, D)
        q = torch.empty(x.shape, dtype=E4M3, device=x.device)
        scale = torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device)
        cfg = _cfg(rows.shape[0], rows.stride(0), 0, D, code, _lib.OPE_E4M3, 0.0)
        _lib.check(_lib.lib.ope_quantize_rows(cfg, ptr(rows), ptr(q), ptr(scale), stream()), "ope_quantize_rows")
    return q, scale
