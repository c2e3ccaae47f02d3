"""Linear layer with bias, activation and residual in its epilogue (ope_linear, ope_linear_backward)."""
import struct

import torch
from torch.autograd.function import once_differentiable

from .. import _lib
from ._common import DTYPES, E4M3, dtype_code, on_device, ptr, rows_of, scratch, stream, want, wants_grad

ACTIVATIONS = {"none": 0, "relu": 1, "tanh": 2, "silu": 3, "gelu": 4}
_CFG = struct.Struct("qqqiiiii4x")
_MAX_WIDTH = 1 << 20


def _check(x, weight, bias, residual, activation, out_dtype):
    want(x, "x")
    want(weight, "weight")
    if x.dim() < 1 or weight.dim() != 2 or weight.shape[1] != x.shape[-1]:
        raise ValueError("x [..., in] and weight [out, in] wanted, got %s and %s" % (tuple(x.shape), tuple(weight.shape)))
    if not all(1 <= n <= _MAX_WIDTH for n in weight.shape):
        raise ValueError("weight: widths of 1 to %d wanted, got %s" % (_MAX_WIDTH, tuple(weight.shape)))
    if bias is not None:
        want(bias, "bias", (weight.shape[0],), out_dtype)
    if residual is not None:
        want(residual, "residual", (*x.shape[:-1], weight.shape[0]), out_dtype)
    if activation not in ACTIVATIONS:
        raise ValueError("activation: one of %s wanted, got %r" % (", ".join(ACTIVATIONS), activation))


def _forward(x, weight, x_scale, w_scale, bias, residual, act, code, out_dtype, keep_z):
    """(y, z or None)."""
    N, K = weight.shape
    rows, res = rows_of(x, K), None if residual is None else rows_of(residual, N)
    weight = weight.contiguous()
    bias = None if bias is None else bias.contiguous()
    M, dev = rows.shape[0], x.device
    y = torch.empty((*x.shape[:-1], N), dtype=out_dtype, device=dev)
    z = torch.empty((M, N), dtype=out_dtype, device=dev) if keep_z else None
    cfg = _CFG.pack(M, rows.stride(0), 0 if res is None else res.stride(0), K, N, code, DTYPES[out_dtype], act)
    ws = scratch(_lib.lib.ope_linear_workspace_bytes(cfg), dev, "ope_linear")
    _lib.check(_lib.lib.ope_linear(cfg, ptr(rows), ptr(weight), ptr(x_scale), ptr(w_scale), ptr(bias), ptr(res), ptr(y), ptr(z), ptr(ws),
                                   0 if ws is None else ws.numel(), stream()), "ope_linear")
    return y, z


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, act):
        with on_device(x, weight, bias, residual):
            y, z = _forward(x, weight, None, None, bias, residual, act, DTYPES[x.dtype], x.dtype, act != 0)
        ctx.save_for_backward(x, weight, z)
        ctx.act = act
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, z = ctx.saved_tensors
        N, K = weight.shape
        need = ctx.needs_input_grad
        with on_device(x, weight, dy):
            rows, weight, dy = rows_of(x, K), weight.contiguous(), dy.contiguous()
            dx = torch.empty(x.shape, dtype=x.dtype, device=x.device) if need[0] else None
            dw = torch.empty((N, K), dtype=x.dtype, device=x.device) if need[1] else None
            db = torch.empty(N, dtype=x.dtype, device=x.device) if need[2] else None
            if need[0] or need[1] or need[2]:
                code = DTYPES[x.dtype]
                cfg = _CFG.pack(rows.shape[0], rows.stride(0), 0, K, N, code, code, ctx.act)
                ws = scratch(_lib.lib.ope_linear_backward_workspace_bytes(cfg), x.device, "ope_linear_backward")
                _lib.check(_lib.lib.ope_linear_backward(cfg, ptr(dy), ptr(z), ptr(rows), ptr(weight), ptr(dx), ptr(dw), ptr(db), ptr(ws),
                                                        0 if ws is None else ws.numel(), stream()), "ope_linear_backward")
        return dx, dw, db, dy if need[3] else None, None


def linear(x, weight, bias=None, residual=None, activation="none"):
    """y = act(x weight^T + bias) + residual.

    x [..., in], weight [out, in] (torch.nn.Linear's), bias [out], residual [..., out], all of one type (float32, bfloat16 or float16); activation
    "none", "relu", "tanh", "silu" or "gelu" (z Phi(z)). Sums in float32, one rounding at the end. Differentiable in all four; the gradient of
    z = x weight^T + bias is rounded to x's type in front of the backward products."""
    want(x, "x")
    code = dtype_code(x, "x")
    want(weight, "weight", None, x.dtype)
    _check(x, weight, bias, residual, activation, x.dtype)
    if wants_grad(x, weight, bias, residual):
        on_device(x, weight, bias, residual)
        return _Linear.apply(x, weight, bias, residual, ACTIVATIONS[activation])
    with on_device(x, weight, bias, residual):
        return _forward(x, weight, None, None, bias, residual, ACTIVATIONS[activation], code, x.dtype, False)[0]


def linear_fp8(x, x_scale, weight, w_scale, bias=None, residual=None, activation="none", out_dtype=torch.bfloat16):
    """y = act((x weight^T) x_scale w_scale + bias) + residual with 8-bit operands, as rms_norm_fp8 and quantize_rows_fp8 return them: x [..., in]
    and weight [out, in] float8_e4m3fn, x_scale float32 of x.shape[:-1], w_scale float32 [out]; bias and residual of out_dtype. For acting: no gradients
    (a scale, bias or residual that requires one is refused while gradients are recorded)."""
    want(x, "x", None, E4M3)
    want(weight, "weight", None, E4M3)
    if out_dtype not in DTYPES:
        raise TypeError("out_dtype: float32, bfloat16 or float16 wanted, got %s" % (out_dtype,))
    _check(x, weight, bias, residual, activation, out_dtype)
    want(x_scale, "x_scale", x.shape[:-1], torch.float32)
    want(w_scale, "w_scale", (weight.shape[0],), torch.float32)
    if wants_grad(x_scale, w_scale, bias, residual):
        raise ValueError("linear_fp8 has no gradients: call it under torch.no_grad(), or linear")
    with on_device(x, x_scale, weight, w_scale, bias, residual):
        return _forward(x, weight, x_scale.contiguous(), w_scale.contiguous(), bias, residual, ACTIVATIONS[activation], _lib.OPE_E4M3, out_dtype, False)[0]
