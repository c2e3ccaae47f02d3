"""Gated delta rule: a state matrix per head as an agent's memory, chunked over whole episodes or one step at a time (ope_delta_*)."""
import struct

import torch
from torch.autograd.function import once_differentiable

from .. import _lib
from ._common import DTYPES, dtype_code, inner, like, on_device, ptr, scratch, stream, want, wants_grad

_CFG = struct.Struct("7if33q")
_NONE3 = (0, 0, 0)
MAX_KEY, MAX_VALUE = 128, 1024


def _check(q, k, v, log_decay, beta, scale, lead):
    """`lead` axes in front of the heads (2: batch and time, 1: batch)."""
    for t, name in ((q, "q"), (k, "k"), (v, "v")):
        want(t, name)
    code = dtype_code(q, "q")
    if q.dim() != lead + 2 or v.dim() != lead + 2 or v.shape[:lead] != q.shape[:lead]:
        raise ValueError("q and v: %d axes with the same first %d wanted, got %s and %s" % (lead + 2, lead, tuple(q.shape), tuple(v.shape)))
    want(k, "k", q.shape, q.dtype)
    want(v, "v", None, q.dtype)
    Hk, K, H, V = q.shape[-2], q.shape[-1], v.shape[-2], v.shape[-1]
    if Hk < 1 or H < 1 or H % Hk:
        raise ValueError("the value heads (%d) have to be a multiple of the query / key heads (%d)" % (H, Hk))
    if not 1 <= K <= MAX_KEY or not 1 <= V <= MAX_VALUE:
        raise ValueError("key widths of 1 to %d and value widths of 1 to %d wanted, got %d and %d" % (MAX_KEY, MAX_VALUE, K, V))
    want(log_decay, "log_decay", v.shape[:-1], torch.float32)
    want(beta, "beta", v.shape[:-1], torch.float32)
    return code, float(K ** -0.5 if scale is None else scale)


def _strides(*tensors):
    out = []
    for t in tensors:
        out += _NONE3 if t is None else t.stride()[:3]
    return out


def _pack(shape, code, scale, q, k, v, o, g, beta, *grads):
    """ope_delta_cfg of the call; the gradients' strides stay zero in a forward call."""
    return _CFG.pack(*shape, code, scale, *_strides(q, k, v, o, g, beta, *(grads or (None,) * 5)))


def _forward(q, k, v, g, beta, state, lengths, scale, code):
    (B, T, Hk, K), (H, V), dev = q.shape, v.shape[2:], q.device
    o, last = like(v), torch.empty((B, H, K, V), dtype=torch.float32, device=dev)
    cfg = _pack((B, T, H, Hk, K, V), code, scale, q, k, v, o, g, beta)
    saved = scratch(_lib.lib.ope_delta_saved_bytes(cfg), dev, "ope_delta_forward")
    ws = scratch(_lib.lib.ope_delta_workspace_bytes(cfg, 0), dev, "ope_delta_forward")
    _lib.check(_lib.lib.ope_delta_forward(cfg, ptr(q), ptr(k), ptr(v), ptr(g), ptr(beta), ptr(state), ptr(lengths), ptr(o), ptr(last), ptr(saved),
                                          0 if saved is None else saved.numel(), ptr(ws), 0 if ws is None else ws.numel(), stream()), "ope_delta_forward")
    return o, last, saved


class _GatedDelta(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, g, beta, state, lengths, scale):
        with on_device(q, k, v, g, beta, state, lengths):
            o, last, saved = _forward(q, k, v, g, beta, state, lengths, scale, DTYPES[q.dtype])
        ctx.save_for_backward(q, k, v, g, beta, lengths, saved)
        ctx.scale = scale
        ctx.set_materialize_grads(False)
        return o, last

    @staticmethod
    @once_differentiable
    def backward(ctx, do, dlast):
        if do is None and dlast is None:
            return (None,) * 8
        q, k, v, g, beta, lengths, saved = ctx.saved_tensors
        (B, T, Hk, K), (H, V), dev = q.shape, v.shape[2:], q.device
        with on_device(q, do, dlast):
            do = torch.zeros(v.shape, dtype=v.dtype, device=dev) if do is None else inner(do)
            dlast = None if dlast is None else dlast.contiguous()
            dq, dk, dv, dg, db = like(q), like(k), like(v), torch.empty_like(g), torch.empty_like(beta)
            dstate = torch.empty((B, H, K, V), dtype=torch.float32, device=dev) if ctx.needs_input_grad[5] else None
            cfg = _pack((B, T, H, Hk, K, V), DTYPES[q.dtype], ctx.scale, q, k, v, do, g, beta, dq, dk, dv, dg, db)
            ws = scratch(_lib.lib.ope_delta_workspace_bytes(cfg, 1), dev, "ope_delta_backward")
            _lib.check(_lib.lib.ope_delta_backward(cfg, ptr(q), ptr(k), ptr(v), ptr(g), ptr(beta), ptr(lengths), ptr(saved),
                                                   0 if saved is None else saved.numel(), ptr(do), ptr(dlast), ptr(dq), ptr(dk), ptr(dv), ptr(dg), ptr(db),
                                                   ptr(dstate), ptr(ws), 0 if ws is None else ws.numel(), stream()), "ope_delta_backward")
        return dq, dk, dv, dg, db, dstate, None, None


def gated_delta_rule(q, k, v, log_decay, beta, initial_state=None, lengths=None, scale=None):
    """The memory over whole sequences: per sequence and head a state S [K, V], and per token

        S <- exp(log_decay) S;  S <- S + beta k (v - S^T k)^T;  out = scale S^T q

    q, k [B, T, Hk, K], v [B, T, H, V] of one type (float32, bfloat16, float16), any strides with a contiguous last axis (a time-major batch is
    passed as x.transpose(0, 1)); H is a multiple of Hk and value head h reads query / key head h // (H // Hk). K up to 128, V up to 1024.
    log_decay, beta float32 [B, T, H]: log_decay is at most 0 in use; -inf clears the (finite) state in front of its token, as where a row of the
    batch goes on with another episode. initial_state float32 [B, H, K, V] (None: zeros). lengths int32 [B] (None: T): tokens at and behind
    lengths[b] are not read and change nothing, their outputs and gradients are 0. scale: 1 / sqrt(K) where None. Keys have unit length in use:
    the rule needs beta |k|^2 < 2 to stay bounded.

    Returns (out [B, T, H, V] of q's type, final state float32 [B, H, K, V]); differentiable in q, k, v, log_decay (0 at -inf), beta and
    initial_state. The backward pass keeps per 64 tokens and head one state and the tokens' updates in float32: (K V + 64 (K + V)) * 4 bytes."""
    code, scale = _check(q, k, v, log_decay, beta, scale, 2)
    B, K, H, V = q.shape[0], q.shape[-1], v.shape[-2], v.shape[-1]
    if initial_state is not None:
        want(initial_state, "initial_state", (B, H, K, V), torch.float32)
    if lengths is not None:
        want(lengths, "lengths", (B,), torch.int32)
        lengths = lengths.contiguous()
    guard = on_device(q, k, v, log_decay, beta, initial_state, lengths)
    grads = wants_grad(q, k, v, log_decay, beta, initial_state)
    q, k, v = inner(q), inner(k), inner(v)
    state = None if initial_state is None else initial_state.contiguous()
    if grads:
        return _GatedDelta.apply(q, k, v, log_decay, beta, state, lengths, scale)
    with guard:
        return _forward(q, k, v, log_decay, beta, state, lengths, scale, code)[:2]


def gated_delta_step(q, k, v, log_decay, beta, state, scale=None):
    """One token of gated_delta_rule for every row: q, k [B, Hk, K], v [B, H, V], log_decay, beta float32 [B, H]; `state` float32 [B, H, K, V], contiguous,
    is updated in place (log_decay = -inf: cleared first, whatever it holds). Returns out [B, H, V]. For acting: no gradients."""
    code, scale = _check(q, k, v, log_decay, beta, scale, 1)
    B, Hk, K = q.shape
    H, V = v.shape[1:]
    want(state, "state", (B, H, K, V), torch.float32)
    if not state.is_contiguous():
        raise ValueError("state: it is updated in place and has to be contiguous")
    if wants_grad(q, k, v, log_decay, beta, state):
        raise ValueError("gated_delta_step has no gradients: call it under torch.no_grad(), or gated_delta_rule")
    with on_device(q, k, v, log_decay, beta, state):
        q, k, v = inner(q), inner(k), inner(v)
        o = torch.empty((B, H, V), dtype=v.dtype, device=v.device)
        cfg = _CFG.pack(B, 1, H, Hk, K, V, code, scale, q.stride(0), 0, q.stride(1), k.stride(0), 0, k.stride(1), v.stride(0), 0, v.stride(1), H * V, 0, V,
                        log_decay.stride(0), 0, log_decay.stride(1), beta.stride(0), 0, beta.stride(1), *_NONE3 * 5)
        _lib.check(_lib.lib.ope_delta_step(cfg, ptr(q), ptr(k), ptr(v), ptr(log_decay), ptr(beta), ptr(state), ptr(o), stream()), "ope_delta_step")
    return o
