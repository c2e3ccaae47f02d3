"""Gated delta rule: a state matrix per head as an agent's memory, chunked over whole episodes or one step at a time (ope_delta_*)."""
import functools
import struct

import torch

from .. import _lib
from ._common import PLANS, dtype_code, inner, like, on_device, once, plain_call, ptr, same_dtype, same_shape, scratch, size_or_raise, stream, tensors, untraced, wants_grad

_CFG = struct.Struct("7if33q")
_NONE3 = (0, 0, 0)
MAX_KEY, MAX_VALUE = 128, 1024
_lib_forward, _lib_backward, _lib_step = _lib.lib.ope_delta_forward, _lib.lib.ope_delta_backward, _lib.lib.ope_delta_step


@functools.lru_cache(PLANS)
def _plan(q, k, v, g, beta, state, lengths, dtypes, lead):
    """(B, T, H, Hk, K, V, type code) of shapes and types that fit together; `lead` axes in front of the heads (2: batch and time, 1: batch)."""
    untraced()
    q_dtype, k_dtype, v_dtype, g_dtype, beta_dtype, state_dtype, lengths_dtype = dtypes
    code = dtype_code(q_dtype, "q")
    if len(q) != lead + 2 or len(v) != lead + 2 or v[:lead] != q[:lead]:
        raise ValueError("q and v: %d axes with the same first %d wanted, got %s and %s" % (lead + 2, lead, tuple(q), tuple(v)))
    same_shape(k, "k", q)
    same_dtype(k_dtype, "k", q_dtype)
    same_dtype(v_dtype, "v", q_dtype)
    Hk, K, H, V = q[-2], q[-1], v[-2], v[-1]
    if Hk < 1 or H < 1 or H % Hk:
        raise ValueError("the value heads (%d) have to be a multiple of the query / key heads (%d)" % (H, Hk))
    if not 1 <= K <= MAX_KEY or not 1 <= V <= MAX_VALUE:
        raise ValueError("key widths of 1 to %d and value widths of 1 to %d wanted, got %d and %d" % (MAX_KEY, MAX_VALUE, K, V))
    same_shape(g, "log_decay", v[:-1])
    same_dtype(g_dtype, "log_decay", torch.float32)
    same_shape(beta, "beta", v[:-1])
    same_dtype(beta_dtype, "beta", torch.float32)
    if state is not None:
        same_shape(state, "the state", (q[0], H, K, V))
        same_dtype(state_dtype, "the state", torch.float32)
    if lengths is not None:
        same_shape(lengths, "lengths", q[:1])
        same_dtype(lengths_dtype, "lengths", torch.int32)
    return q[0], q[1] if lead == 2 else 1, H, Hk, K, V, code


def _check(q, k, v, g, beta, state, lengths, lead):
    tensors((q, "q"), (k, "k"), (v, "v"), (g, "log_decay"), (beta, "beta"))
    s = s_dtype = n = n_dtype = None
    if state is not None:
        tensors((state, "the state"))
        s, s_dtype = state.shape, state.dtype
    if lengths is not None:
        tensors((lengths, "lengths"))
        n, n_dtype = lengths.shape, lengths.dtype
    return _plan(q.shape, k.shape, v.shape, g.shape, beta.shape, s, n, (q.dtype, k.dtype, v.dtype, g.dtype, beta.dtype, s_dtype, n_dtype), lead)


@functools.lru_cache(PLANS)
def _pack(plan, scale, *strides):
    """(configuration, bytes of `saved`, of the forward workspace, of the backward workspace); the gradients' strides are zeros in a forward call."""
    flat = [x for s in strides for x in s[:3]]
    cfg = _CFG.pack(*plan, scale, *flat, *(0,) * (33 - len(flat)))
    lib, what = _lib.lib, "ope_delta"
    return (cfg, size_or_raise(lib.ope_delta_saved_bytes(cfg), what), size_or_raise(lib.ope_delta_workspace_bytes(cfg, 0), what),
            size_or_raise(lib.ope_delta_workspace_bytes(cfg, 1), what))


def _forward(plan, q, k, v, g, beta, state, lengths, scale):
    B, _, H, _, K, V, _ = plan
    dev = q.device
    o, last = like(v), torch.empty((B, H, K, V), dtype=torch.float32, device=dev)
    cfg, saved_bytes, ws_bytes, _ = _pack(plan, scale, q.stride(), k.stride(), v.stride(), o.stride(), g.stride(), beta.stride())
    saved, saved_at, _ = scratch(saved_bytes, dev)
    hold, ws, _ = scratch(ws_bytes, dev)
    rc = _lib_forward(cfg, q.data_ptr(), k.data_ptr(), v.data_ptr(), g.data_ptr(), beta.data_ptr(), ptr(state), ptr(lengths), o.data_ptr(), last.data_ptr(),
                      saved_at, saved_bytes, ws, ws_bytes, stream())
    if rc:
        _lib.check(rc, "ope_delta_forward")
    return o, last, saved


class _GatedDelta(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, g, beta, state, lengths, call):
        plan, scale = call
        o, last, saved = _forward(plan, q, k, v, g, beta, state, lengths, scale)
        ctx.save_for_backward(q, k, v, g, beta, lengths, saved)
        ctx.call = call
        ctx.set_materialize_grads(False)
        return o, last

    @once
    def backward(ctx, do, dlast):
        if do is None and dlast is None:
            return (None,) * 8
        q, k, v, g, beta, lengths, saved = ctx.saved_tensors
        plan, scale = ctx.call
        B, _, H, _, K, V, _ = plan
        with on_device(q, do, dlast):
            dev = q.device
            do = torch.zeros(v.shape, dtype=v.dtype, device=dev) if do is None else inner(do)
            dlast = None if dlast is None else dlast.contiguous()
            dq, dk, dv, dg, db = like(q), like(k), like(v), torch.empty_like(g), torch.empty_like(beta)
            dstate = torch.empty((B, H, K, V), dtype=torch.float32, device=dev) if ctx.needs_input_grad[5] else None
            cfg, saved_bytes, _, ws_bytes = _pack(plan, scale, q.stride(), k.stride(), v.stride(), do.stride(), g.stride(), beta.stride(), dq.stride(),
                                                  dk.stride(), dv.stride(), dg.stride(), db.stride())
            hold, ws, _ = scratch(ws_bytes, dev)
            rc = _lib_backward(cfg, q.data_ptr(), k.data_ptr(), v.data_ptr(), g.data_ptr(), beta.data_ptr(), ptr(lengths), ptr(saved), saved_bytes, do.data_ptr(),
                               ptr(dlast), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), dg.data_ptr(), db.data_ptr(), ptr(dstate), ws, ws_bytes, stream())
            if rc:
                _lib.check(rc, "ope_delta_backward")
        return dq, dk, dv, dg, db, dstate, None, None


def gated_delta_rule(q, k, v, log_decay, beta, initial_state=None, lengths=None, scale=None):
    """The memory over whole sequences: per sequence and head a state S [K, V], and per token

        S <- exp(log_decay) S;  S <- S + beta k (v - S^T k)^T;  out = scale S^T q

    q, k [B, T, Hk, K], v [B, T, H, V] of one type (float32, bfloat16, float16), any strides with a contiguous last axis (a time-major batch is
    passed as x.transpose(0, 1)); H is a multiple of Hk and value head h reads query / key head h // (H // Hk). K up to 128, V up to 1024.
    log_decay, beta float32 [B, T, H]: log_decay is at most 0 in use; where exp(log_decay) is 0 in float32 (-inf, the type's lowest value, anything
    under -103.97) the state is cleared in front of its token, as where a row of the batch goes on with another episode: nothing of the one reaches the
    other, not even what is not finite (which inside its own episode may also reach tokens in front of it, within a chunk of 64). initial_state float32 [B, H, K, V] (None: zeros). lengths int32 [B] (None: T): tokens at and behind
    lengths[b] are not read and change nothing, their outputs and gradients are 0. scale: 1 / sqrt(K) where None. Keys have unit length in use:
    the rule needs beta |k|^2 < 2 to stay bounded.

    Returns (out [B, T, H, V] of q's type, final state float32 [B, H, K, V]); differentiable in q, k, v, log_decay (0 where it clears), beta and
    initial_state, once (no create_graph). Beside its inputs, the backward pass keeps per 64 tokens (or part of them) and head one state, the tokens' updates and
    their decays in float32: (Kp Vp + 64 (Kp + Vp) + 65) * 4 bytes, with Kp and Vp the widths rounded up to 16 (Kp: to 128 above 96)."""
    plain_call(q, k, v, log_decay, beta, initial_state)
    plan = _check(q, k, v, log_decay, beta, initial_state, lengths, 2)
    scale = float(plan[4] ** -0.5 if scale is None else scale)
    with on_device(q, k, v, log_decay, beta, initial_state, lengths):
        q, k, v = inner(q), inner(k), inner(v)
        state = None if initial_state is None else initial_state.contiguous()
        lengths = None if lengths is None else lengths.contiguous()
        if wants_grad(q, k, v, log_decay, beta, state):
            return _GatedDelta.apply(q, k, v, log_decay, beta, state, lengths, (plan, scale))
        return _forward(plan, q, k, v, log_decay, beta, state, lengths, scale)[:2]


@functools.lru_cache(PLANS)
def _pack_step(plan, scale, q, k, v, g, beta):
    _, _, H, _, _, V, _ = plan
    three = lambda s: (s[0], 0, s[1])       # noqa: E731
    return _CFG.pack(*plan, scale, *three(q), *three(k), *three(v), H * V, 0, V, *three(g), *three(beta), *_NONE3 * 5)


def gated_delta_step(q, k, v, log_decay, beta, state, scale=None):
    """One token of gated_delta_rule for every row: q, k [B, Hk, K], v [B, H, V], log_decay, beta float32 [B, H]; `state` float32 [B, H, K, V], contiguous,
    is updated in place and shares no memory with the other arguments (cleared first, whatever it holds, where exp(log_decay) is 0). Returns out [B, H, V]. For acting: no gradients."""
    plain_call(q, k, v, log_decay, beta, state)
    tensors((state, "the state"))
    plan = _check(q, k, v, log_decay, beta, state, None, 1)
    scale = float(plan[4] ** -0.5 if scale is None else scale)
    if not state.is_contiguous():
        raise ValueError("the state is updated in place and has to be contiguous")
    if wants_grad(q, k, v, log_decay, beta, state):
        raise ValueError("gated_delta_step has no gradients: call it under torch.no_grad(), or gated_delta_rule")
    with on_device(q, k, v, log_decay, beta, state):
        q, k, v = inner(q), inner(k), inner(v)
        o = torch.empty(v.shape, dtype=v.dtype, device=v.device)
        rc = _lib_step(_pack_step(plan, scale, q.stride(), k.stride(), v.stride(), log_decay.stride(), beta.stride()), q.data_ptr(), k.data_ptr(), v.data_ptr(),
                       log_decay.data_ptr(), beta.data_ptr(), state.data_ptr(), o.data_ptr(), stream())
        if rc:
            _lib.check(rc, "ope_delta_step")
    torch._C._increment_version((state,))          # a graph that holds the old state refuses to go on with the new one
    return o
