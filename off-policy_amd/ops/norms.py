"""RMS norm with the residual's addition, and rows in 8 bits (ope_rms_norm, ope_quantize_rows)."""
import functools
import struct

import torch

from .. import _lib
from ._common import DTYPES, E4M3, PLANS, dtype_code, on_device, once, plain_call, ptr, rows_of, same_dtype, same_shape, scratch, size_or_raise, stream, tensors, untraced, wants_grad

_CFG = struct.Struct("qqqiiif")
_MAX_WIDTH = 1 << 20
_lib_norm, _lib_norm_bwd, _lib_rows = _lib.lib.ope_rms_norm, _lib.lib.ope_rms_norm_backward, _lib.lib.ope_quantize_rows


@functools.lru_cache(PLANS)
def _pack(rows, x_stride, r_stride, width, dtype, out_dtype, eps):
    return _CFG.pack(rows, x_stride, r_stride, width, dtype, out_dtype, eps)


@functools.lru_cache(PLANS)
def _bwd_bytes(cfg):
    return size_or_raise(_lib.lib.ope_rms_norm_backward_workspace_bytes(cfg), "ope_rms_norm_backward")


@functools.lru_cache(PLANS)
def _plan(x, x_dtype, w, w_dtype, r, r_dtype, eps):
    """(type code, rows, width) of shapes and types that fit together."""
    untraced()
    code = dtype_code(x_dtype, "x")
    if len(x) < 1 or not 1 <= x[-1] <= _MAX_WIDTH:
        raise ValueError("x: at least one axis and a last one of 1 to %d wanted, got shape %s" % (_MAX_WIDTH, tuple(x)))
    if w is not None:
        same_shape(w, "weight", x[-1:])
        same_dtype(w_dtype, "weight", x_dtype)
    if r is not None:
        same_shape(r, "residual", x)
        same_dtype(r_dtype, "residual", x_dtype)
    if not eps >= 0:
        raise ValueError("eps: zero or a positive number wanted, got %r" % (eps,))
    return code, x.numel() // x[-1], x[-1]


def _check(x, weight, residual, eps):
    if residual is None:
        tensors((x, "x"), (weight, "weight"))
        return _plan(x.shape, x.dtype, weight.shape, weight.dtype, None, None, eps)
    tensors((x, "x"), (weight, "weight"), (residual, "residual"))
    return _plan(x.shape, x.dtype, weight.shape, weight.dtype, residual.shape, residual.dtype, eps)


def _forward(plan, x, weight, residual, eps, fp8, rstd_too):
    """(y, scale, s, rstd)"""
    code, M, D = plan
    dev = x.device
    rows, xs = rows_of(x, D)
    y = torch.empty(x.shape, dtype=E4M3 if fp8 else x.dtype, device=dev)
    scale = torch.empty(x.shape[:-1], dtype=torch.float32, device=dev) if fp8 else None
    rstd = torch.empty(M, dtype=torch.float32, device=dev) if rstd_too else None
    res = s = None
    rs = 0
    if residual is not None:
        res, rs = rows_of(residual, D)
        s = torch.empty(x.shape, dtype=x.dtype, device=dev)
    weight = weight.contiguous()
    rc = _lib_norm(_pack(M, xs, rs, D, code, _lib.OPE_E4M3 if fp8 else code, eps), rows.data_ptr(), ptr(res), weight.data_ptr(), y.data_ptr(), ptr(scale), ptr(s),
                   ptr(rstd), stream())
    if rc:
        _lib.check(rc, "ope_rms_norm")
    return y, scale, s, rstd


class _RmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, residual, call):
        plan, eps = call
        y, _, s, rstd = _forward(plan, x, weight, residual, eps, False, True)
        # float32 keeps every bit of the sum; 16-bit types form it again from what was added
        again = s is not None and x.dtype != torch.float32
        ctx.save_for_backward(x if s is None or again else s, residual if again else None, weight, rstd)
        ctx.two, ctx.call = s is not None, call
        ctx.set_materialize_grads(False)
        return y if s is None else (y, s)

    @once
    def backward(ctx, dy, dsum=None):
        if dy is None and dsum is None:
            return None, None, None, None
        x, residual, weight, rstd = ctx.saved_tensors
        (code, M, D), eps = ctx.call
        with on_device(x, dy, dsum):
            dev = x.device
            dy = torch.zeros(x.shape, dtype=x.dtype, device=dev) if dy is None else dy.contiguous()
            dsum = None if dsum is None else dsum.contiguous()
            rows, xs = rows_of(x, D)
            res, rs = (None, 0) if residual is None else rows_of(residual, D)
            dx = torch.empty(x.shape, dtype=x.dtype, device=dev)
            dw = torch.empty(D, dtype=x.dtype, device=dev)
            cfg = _pack(M, xs, rs, D, code, code, eps)
            hold, ws, nbytes = scratch(_bwd_bytes(cfg), dev)
            weight = weight.contiguous()
            rc = _lib_norm_bwd(cfg, dy.data_ptr(), ptr(dsum), rows.data_ptr(), ptr(res), weight.data_ptr(), rstd.data_ptr(), dx.data_ptr(), dw.data_ptr(), ws,
                               nbytes, stream())
            if rc:
                _lib.check(rc, "ope_rms_norm_backward")
        return dx, dw, dx if ctx.two else None, None


def rms_norm(x, weight, residual=None, eps=1e-6):
    """y = s * weight / sqrt(mean(s^2) + eps) over the last axis, s = x + residual.

    x [..., D] float32, bfloat16 or float16, weight [D] and residual (x's shape) of the same type. Returns y, or (y, s) where a residual is
    given: s is what the next block adds to. The norm is taken of the float32 sum, in front of its rounding to x's type. Differentiable in x,
    weight and residual, once (no create_graph)."""
    plain_call(x, weight, residual)
    eps = float(eps)
    plan = _check(x, weight, residual, eps)
    with on_device(x, weight, residual):
        if wants_grad(x, weight, residual):
            return _RmsNorm.apply(x, weight, residual, (plan, eps))
        y, _, s, _ = _forward(plan, x, weight, residual, eps, False, False)
    return y if s is None else (y, s)


def rms_norm_fp8(x, weight, residual=None, eps=1e-6):
    """rms_norm with its output in 8 bits: returns (q, scale), or (q, scale, s) where a residual is given. q is float8_e4m3fn of x's shape, scale
    float32 of x.shape[:-1], y = q * scale; scale = max(max|y|, 448 * 2^-126) / 448 of the row. For acting: no gradients (a tensor that requires one
    is refused while gradients are recorded)."""
    plain_call(x, weight, residual)
    eps = float(eps)
    plan = _check(x, weight, residual, eps)
    if wants_grad(x, weight, residual):
        raise ValueError("rms_norm_fp8 has no gradients: call it under torch.no_grad(), or rms_norm")
    with on_device(x, weight, residual):
        y, scale, s, _ = _forward(plan, x, weight, residual, eps, True, False)
    return (y, scale) if s is None else (y, scale, s)


def quantize_rows_fp8(x):
    """(q, scale) of the rows of x [..., D], by rms_norm_fp8's rule; for the weights of linear_fp8."""
    plain_call(x)
    tensors((x, "x"))
    code, M, D = _plan(x.shape, x.dtype, None, None, None, None, 0.0)
    if wants_grad(x):
        raise ValueError("quantize_rows_fp8 has no gradients: call it under torch.no_grad()")
    with on_device(x):
        rows, xs = rows_of(x, D)
        q = torch.empty(x.shape, dtype=E4M3, device=x.device)
        scale = torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device)
        _lib.check(_lib_rows(_pack(M, xs, 0, D, code, _lib.OPE_E4M3, 0.0), ptr(rows), ptr(q), ptr(scale), stream()), "ope_quantize_rows")
    return q, scale
