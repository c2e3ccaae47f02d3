"""Operators of a residual memory block for agents, on hand-written gfx950 kernels (include/ope.h, "Memory-block operators").

The engine's own networks are fixed to the reference's shape: LayerNorm, linear layers of width 64 and a GRU (offpolicy/algorithms/utils/
rnn.py:5-43). These operators are what a wider or longer memory is made of:

    s = x + residual, y = RMS norm of s        rms_norm, rms_norm_fp8 (8-bit output for acting)
    q, k, v = act(y W^T + bias)                linear, linear_fp8, quantize_rows_fp8
    o = memory(q, k, v, log decay, beta)       gated_delta_rule (whole episodes, with gradients), gated_delta_step (one step of acting)
    x = o Wo^T + s                             linear with a residual

float32, bfloat16 and float16; the gradients come through torch.autograd, backwards and once: forward mode, torch.func's transforms, torch.jit.trace and
make_fx are refused. Everything runs on the tensors' device and torch's current stream
there, allocates through torch's allocator (so it may be captured into a HIP graph) and keeps nothing between calls. There is no CPU path.
"""
from .memory import gated_delta_rule, gated_delta_step
from .projection import linear, linear_fp8
from .norms import quantize_rows_fp8, rms_norm, rms_norm_fp8

__all__ = ["gated_delta_rule", "gated_delta_step", "linear", "linear_fp8", "quantize_rows_fp8", "rms_norm", "rms_norm_fp8"]
