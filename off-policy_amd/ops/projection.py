"""Linear layer with bias, activation and residual in its epilogue (ope_linear, ope_linear_backward)."""
import functools
import struct

import torch

from .. import _lib
from ._common import DTYPES, E4M3, PLANS, dtype_code, on_device, once, plain_call, ptr, rows_of, same_dtype, same_shape, scratch, size_or_raise, stream, tensors, untraced, wants_grad

ACTIVATIONS = {"none": 0, "relu": 1, "tanh": 2, "silu": 3, "gelu": 4}
_CFG = struct.Struct("qqqiiiii4x")
_MAX_WIDTH = 1 << 20
_lib_linear, _lib_linear_bwd = _lib.lib.ope_linear, _lib.lib.ope_linear_backward


@functools.lru_cache(PLANS)
def _pack(rows, x_stride, r_stride, K, N, dtype, out_dtype, act):
    """(configuration, workspace bytes of the forward call)"""
    cfg = _CFG.pack(rows, x_stride, r_stride, K, N, dtype, out_dtype, act)
    return cfg, size_or_raise(_lib.lib.ope_linear_workspace_bytes(cfg), "ope_linear")


@functools.lru_cache(PLANS)
def _bwd_bytes(cfg):
    return size_or_raise(_lib.lib.ope_linear_backward_workspace_bytes(cfg), "ope_linear_backward")


@functools.lru_cache(PLANS)
def _plan(x, x_dtype, w, w_dtype, b, b_dtype, r, r_dtype, activation, out_dtype):
    """(rows, in, out, activation, type code, type code of the output) of shapes and types that fit together."""
    untraced()
    if out_dtype not in DTYPES:
        raise TypeError("out_dtype: float32, bfloat16 or float16 wanted, got %s" % (out_dtype,))
    same_dtype(w_dtype, "weight", x_dtype)
    if len(x) < 1 or len(w) != 2 or w[1] != x[-1]:
        raise ValueError("x [..., in] and weight [out, in] wanted, got %s and %s" % (tuple(x), tuple(w)))
    if not all(1 <= n <= _MAX_WIDTH for n in w):
        raise ValueError("weight: widths of 1 to %d wanted, got %s" % (_MAX_WIDTH, tuple(w)))
    if b is not None:
        same_shape(b, "bias", w[:1])
        same_dtype(b_dtype, "bias", out_dtype)
    if r is not None:
        same_shape(r, "residual", (*x[:-1], w[0]))
        same_dtype(r_dtype, "residual", out_dtype)
    if activation not in ACTIVATIONS:
        raise ValueError("activation: one of %s wanted, got %r" % (", ".join(ACTIVATIONS), activation))
    return x.numel() // w[1], w[1], w[0], ACTIVATIONS[activation], _lib.OPE_E4M3 if x_dtype == E4M3 else DTYPES[x_dtype], DTYPES[out_dtype]


def _check(x, weight, bias, residual, activation, out_dtype):
    tensors((x, "x"), (weight, "weight"))
    b = b_dtype = r = r_dtype = None
    if bias is not None:
        tensors((bias, "bias"))
        b, b_dtype = bias.shape, bias.dtype
    if residual is not None:
        tensors((residual, "residual"))
        r, r_dtype = residual.shape, residual.dtype
    return _plan(x.shape, x.dtype, weight.shape, weight.dtype, b, b_dtype, r, r_dtype, activation, out_dtype)


def _forward(plan, x, weight, x_scale, w_scale, bias, residual, out_dtype, keep_z):
    """(y, z or None)"""
    M, K, N, act, code, out_code = plan
    dev = x.device
    rows, xs = rows_of(x, K)
    res, rs = (None, 0) if residual is None else rows_of(residual, N)
    weight = weight.contiguous()
    bias = None if bias is None else bias.contiguous()
    y = torch.empty((*x.shape[:-1], N), dtype=out_dtype, device=dev)
    z = torch.empty((M, N), dtype=torch.float32, device=dev) if keep_z else None
    cfg, need = _pack(M, xs, rs, K, N, code, out_code, act)
    hold, ws, nbytes = scratch(need, dev)
    rc = _lib_linear(cfg, rows.data_ptr(), weight.data_ptr(), ptr(x_scale), ptr(w_scale), ptr(bias), ptr(res), y.data_ptr(), ptr(z), ws, nbytes, stream())
    if rc:
        _lib.check(rc, "ope_linear")
    return y, z


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, plan):
        y, z = _forward(plan, x, weight, None, None, bias, residual, x.dtype, plan[3] != 0)
        ctx.save_for_backward(x, weight, z)
        ctx.plan = plan
        return y

    @once
    def backward(ctx, dy):
        x, weight, z = ctx.saved_tensors
        M, K, N, act, code, _ = ctx.plan
        need_x, need_w, need_b, need_r, _ = ctx.needs_input_grad
        dx = dw = db = None
        with on_device(x, dy):
            dev = x.device
            dy = dy.contiguous()
            if need_x or need_w or need_b:
                rows, xs = rows_of(x, K)
                weight = weight.contiguous()
                if need_x:
                    dx = torch.empty(x.shape, dtype=x.dtype, device=dev)
                if need_w:
                    dw = torch.empty((N, K), dtype=x.dtype, device=dev)
                if need_b:
                    db = torch.empty(N, dtype=x.dtype, device=dev)
                cfg = _pack(M, xs, 0, K, N, code, code, act)[0]
                hold, ws, nbytes = scratch(_bwd_bytes(cfg), dev)
                rc = _lib_linear_bwd(cfg, dy.data_ptr(), ptr(z), rows.data_ptr(), weight.data_ptr(), ptr(dx), ptr(dw), ptr(db), ws, nbytes, stream())
                if rc:
                    _lib.check(rc, "ope_linear_backward")
        return dx, dw, db, dy if need_r else None, None


def linear(x, weight, bias=None, residual=None, activation="none"):
    """y = act(x weight^T + bias) + residual.

    x [..., in], weight [out, in] (torch.nn.Linear's), bias [out], residual [..., out], all of one type (float32, bfloat16 or float16); activation
    "none", "relu", "tanh", "silu" or "gelu" (z Phi(z)). Sums in float32, one rounding at the end. Differentiable in all four, once (no create_graph); the gradient of
    z = x weight^T + bias is rounded to x's type in front of the backward products."""
    plain_call(x, weight, bias, residual)
    tensors((x, "x"))
    dtype_code(x.dtype, "x")
    plan = _check(x, weight, bias, residual, activation, x.dtype)
    with on_device(x, weight, bias, residual):
        if wants_grad(x, weight, bias, residual):
            return _Linear.apply(x, weight, bias, residual, plan)
        return _forward(plan, x, weight, None, None, bias, residual, x.dtype, False)[0]


def linear_fp8(x, x_scale, weight, w_scale, bias=None, residual=None, activation="none", out_dtype=torch.bfloat16):
    """y = act((x weight^T) x_scale w_scale + bias) + residual with 8-bit operands, as rms_norm_fp8 and quantize_rows_fp8 return them: x [..., in]
    and weight [out, in] float8_e4m3fn, x_scale float32 of x.shape[:-1], w_scale float32 [out]; bias and residual of out_dtype. For acting: no gradients
    (an argument that requires one is refused while gradients are recorded)."""
    plain_call(x, x_scale, weight, w_scale, bias, residual)
    tensors((x, "x"), (x_scale, "x_scale"), (w_scale, "w_scale"))
    same_dtype(x.dtype, "x", E4M3)
    plan = _check(x, weight, bias, residual, activation, out_dtype)
    if x_scale.shape != x.shape[:-1] or w_scale.shape != weight.shape[:1]:
        raise ValueError("x_scale and w_scale: shapes %s and %s wanted, got %s and %s" % (tuple(x.shape[:-1]), tuple(weight.shape[:1]), tuple(x_scale.shape), tuple(w_scale.shape)))
    same_dtype(x_scale.dtype, "x_scale", torch.float32)
    same_dtype(w_scale.dtype, "w_scale", torch.float32)
    if wants_grad(x, x_scale, weight, w_scale, bias, residual):
        raise ValueError("linear_fp8 has no gradients: call it under torch.no_grad(), or linear")
    with on_device(x, x_scale, weight, w_scale, bias, residual):
        return _forward(plan, x, weight, x_scale.contiguous(), w_scale.contiguous(), bias, residual, out_dtype, False)[0]
