"""Plain 64-bit forms of the memory-block operators (offpolicy_amd.ops), differentiable through torch.autograd, and the tolerances their
tests hold the kernels to."""
import torch

U32 = 2.0 ** -24          # half a step of float32, relative to the value


def half_step(dtype):
    """The largest relative error of one rounding to `dtype`."""
    return torch.finfo(dtype).eps / 2


def delta_rule(q, k, v, g, beta, state=None, lengths=None, scale=None):
    """Token by token. q, k [B, T, Hk, K], v [B, T, H, V], g, beta [B, T, H]; float64 in, float64 out."""
    B, T, Hk, K = q.shape
    H, V = v.shape[2:]
    r = H // Hk
    q, k = q.repeat_interleave(r, 2) * (K ** -0.5 if scale is None else scale), k.repeat_interleave(r, 2)
    S = torch.zeros(B, H, K, V, dtype=q.dtype, device=q.device) if state is None else state
    n = torch.full((B,), T, device=q.device) if lengths is None else lengths.long().clamp(0, T)
    out = []
    for t in range(T):
        on = (t < n)[:, None, None]
        kt, qt, vt = (torch.where(on, x[:, t], 0.0) for x in (k, q, v))
        gt, bt = (torch.where(on[..., 0], x[:, t], 0.0) for x in (g, beta))
        F = gt.exp()[..., None, None] * S
        u = bt[..., None] * (vt - (F * kt[..., None]).sum(-2))
        S = F + kt[..., None] * u[..., None, :]
        out.append((S * qt[..., None]).sum(-2))
    o = torch.stack(out, 1) if T else torch.zeros(B, 0, H, V, dtype=q.dtype, device=q.device)
    return o, S


def rms_norm(x, weight, residual=None, eps=1e-6):
    s = x if residual is None else x + residual
    return s * weight / (s.square().mean(-1, keepdim=True) + eps).sqrt(), s


def activation(z, act):
    return {"none": lambda: z, "relu": lambda: z.clamp_min(0), "tanh": lambda: z.tanh(), "silu": lambda: z * torch.sigmoid(z),
            "gelu": lambda: z * torch.special.ndtr(z)}[act]()


def linear(x, weight, bias=None, residual=None, act="none"):
    z = x @ weight.t()
    y = activation(z if bias is None else z + bias, act)
    return y if residual is None else y + residual


def close(got, want, roundings, terms, name, scale=None):
    """|got - want| <= roundings * half_step(got's type) * |want| + terms * U32 * scale, element by element.

    `roundings`: how often a value of the result is rounded to its type. `terms`: the length of the float32 sums behind it (a sum of n terms is off
    by at most n half steps of its largest partial sum). `scale`: the size of those partial sums, the result's own largest value unless it is
    what is left of larger ones."""
    assert got.shape == want.shape, (name, got.shape, want.shape)
    if not want.numel():
        return
    if scale is None:
        scale = want.abs().max().item()
    off = (got.double() - want).abs()
    # the smallest step of the type is what subnormal results are rounded by
    bound = roundings * half_step(got.dtype) * want.abs() + terms * U32 * scale + torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps
    assert torch.isfinite(got.double()).all(), name
    worst = (off / bound).max().item()
    assert worst <= 1, "%s: %.3g times its tolerance (largest difference %.3g, largest value %.3g)" % (name, worst, off.max().item(), scale)
