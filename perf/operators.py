"""Cases of the memory-block operators: the gated delta rule (chunked training pass and one-token step), the RMS norm with the
residual's addition (and an 8-bit output), and the linear layer with bias, activation and residual in its epilogue.

`listed()` / `draw(rng)` give cases, `prepare(case, seed)` what a program has in hand before the call, `run(state)` one pass: with
`own` false in elementary torch operations, with `own` true through offpolicy_amd.ops. `exact(case, seed)` is the operator's definition
in 64 bits, `work(case)` the bytes and operations one pass cannot do without."""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
E4M3 = torch.float8_e4m3fn
E4M3_MAX = 448.0
TINY = 2.0 ** -126
EPS = 1e-6
CHUNK = 64


# ------------------------------------------------------------------------------------------------------------------------- the cases
def listed():
    return [
        # replayed episodes of 8 agents (32 episodes of up to 150 steps, time-major as the replay store hands them out), a memory of
        # width 64 in two heads, float32 as everything else in the training step; some rows hold two episodes one behind the other
        dict(name="memory, replayed episodes", op="delta", dtype="f32", B=256, T=150, H=2, Hk=2, K=32, V=32, train=True, ragged=True, resets=True, time_major=True),
        # the same memory with odd widths, shared query / key heads and bfloat16: a wider agent on long ragged episodes
        dict(name="memory, odd widths", op="delta", dtype="bf16", B=6, T=1003, H=8, Hk=4, K=72, V=100, train=True, ragged=True, resets=False, time_major=False),
        # few rows and a long history: the scan over time is all there is to split
        dict(name="memory, long history", op="delta", dtype="bf16", B=2, T=8192, H=8, Hk=8, K=128, V=128, train=False, ragged=False, resets=False, time_major=False),
        # training on long histories, the largest pass over the memory
        dict(name="memory, long training", op="delta", dtype="bf16", B=4, T=4096, H=8, Hk=8, K=128, V=128, train=True, ragged=False, resets=False, time_major=False),
        # acting: 8 environments of 8 agents take one step; latency
        dict(name="memory step, acting", op="delta_step", dtype="f32", B=64, H=2, Hk=2, K=32, V=32),
        # acting with a wide memory and many environments: the states are read and written once
        dict(name="memory step, wide", op="delta_step", dtype="bf16", B=512, H=8, Hk=4, K=128, V=128),
        # the norm in front of the agents' block on a replayed batch (151 steps of 256 rows, width 64), with its gradients
        dict(name="norm, replayed batch", op="norm", dtype="f32", M=38656, D=64, train=True, fp8=False, residual=True),
        # acting in 8 bits: a handful of rows
        dict(name="norm, acting, 8 bits", op="norm", dtype="bf16", M=64, D=256, train=False, fp8=True, residual=True),
        # a wide block's norm, 8-bit output
        dict(name="norm, wide, 8 bits", op="norm", dtype="bf16", M=8192, D=4096, train=False, fp8=True, residual=True),
        # the agents' first layer (observations of width 252 to width 64) on a replayed batch, forward and gradients, float32
        dict(name="linear, replayed batch", op="linear", dtype="f32", M=38656, K=252, N=64, act="relu", bias=True, residual=False, train=True, fp8=False),
        # a wide block's projection in training
        dict(name="linear, wide training", op="linear", dtype="bf16", M=4096, K=2048, N=4096, act="silu", bias=True, residual=True, train=True, fp8=False),
        # acting in 8 bits with a wide block: few rows, the weights are what is read
        dict(name="linear, acting, 8 bits", op="linear", dtype="bf16", M=64, K=2048, N=2048, act="silu", bias=True, residual=True, train=False, fp8=True),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["delta", "delta", "delta_step", "norm", "linear", "linear"])
    dtype = rng.choice(["f32", "bf16", "bf16", "f16"])
    if kind in ("delta", "delta_step"):
        Hk = rng.choice([1, 2, 3, 4])
        H = Hk * rng.choice([1, 1, 2, 3])
        K = rng.choice([16, 32, 64, 128, rng.randint(8, 128)])
        V = rng.choice([16, 32, 64, 128, rng.randint(8, 160)])
        if kind == "delta_step":
            B = _spread(rng, 4, max(4, min(2048, 512 * 8 * 128 * 128 // (H * K * V))))
            return dict(op=kind, dtype=dtype, B=B, H=H, Hk=Hk, K=K, V=V)
        train = rng.random() < 0.6
        T = _spread(rng, 32, 4096)
        B = _spread(rng, 1, max(1, min(512, 4 * 4096 * 8 * 128 * 128 // (2 * T * H * K * max(V, K)))))
        return dict(op=kind, dtype=dtype, B=B, T=T, H=H, Hk=Hk, K=K, V=V, train=train, ragged=rng.random() < 0.5, resets=rng.random() < 0.4, time_major=rng.random() < 0.5)
    if kind == "norm":
        fp8 = rng.random() < 0.4
        D = rng.choice([64, 256, 1024, 4096, _spread(rng, 16, 8192)])
        M = _spread(rng, 16, max(16, min(65536, 8192 * 4096 // (2 * D))))
        return dict(op=kind, dtype=dtype, M=M, D=D, train=not fp8 and rng.random() < 0.7, fp8=fp8, residual=rng.random() < 0.8)
    fp8 = rng.random() < 0.3
    K, N = _spread(rng, 32, 2048), _spread(rng, 32, 2048)
    if rng.random() < 0.6:
        K, N = max(32, K // 32 * 32), max(32, N // 32 * 32)
    M = _spread(rng, 16, max(16, min(40000, 4096 * 2048 * 4096 // (8 * K * N))))
    if fp8:
        K = max(32, K // 16 * 16)
        dtype = "bf16" if dtype == "f32" else dtype
    return dict(op=kind, dtype=dtype, M=M, K=K, N=N, act=rng.choice(["none", "relu", "tanh", "silu", "gelu"]), bias=rng.random() < 0.8, residual=rng.random() < 0.5,
                train=not fp8 and rng.random() < 0.7, fp8=fp8)


# ----------------------------------------------------------------------------------------------------------------------- the inputs
def _rows8(w):
    """Rows of `w` in e4m3 with one float32 scale each."""
    s = w.float().abs().amax(-1).clamp_min(E4M3_MAX * TINY) / E4M3_MAX
    return (w.float() / s[:, None]).clamp(-E4M3_MAX, E4M3_MAX).to(E4M3), s


def prepare(case, seed):
    c, dt = case, DTYPES[case["dtype"]]
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape, scale=1.0):
        return torch.randn(shape, generator=gen, device="cuda") * scale

    def rand(*shape):
        return torch.rand(shape, generator=gen, device="cuda")

    st = {"case": dict(c)}
    if c["op"] == "delta":
        B, T = (c["T"], c["B"]) if c["time_major"] else (c["B"], c["T"])     # the two leading axes as they lie in memory
        turn = (lambda x: x.transpose(0, 1)) if c["time_major"] else (lambda x: x)
        k = randn(B, T, c["Hk"], c["K"])
        k = k / k.norm(dim=-1, keepdim=True)                                # a delta rule's keys have unit length
        g = -0.3 * rand(B, T, c["H"]) ** 3 - 1e-4
        if c["resets"]:                                                     # an episode boundary about every 80 steps
            g = torch.where(rand(B, T, 1) < 0.0125, torch.full_like(g, -math.inf), g)
        st["leaves"] = [turn(x).detach().requires_grad_(c["train"]) for x in
                        (randn(B, T, c["Hk"], c["K"]).to(dt), k.to(dt), randn(B, T, c["H"], c["V"]).to(dt), g, torch.sigmoid(randn(B, T, c["H"])))]
        st["leaves"].append(randn(c["B"], c["H"], c["K"], c["V"], scale=0.3).requires_grad_(c["train"]))
        st["lengths"] = (1 + (rand(c["B"]) * c["T"]).int()).clamp_max(c["T"]) if c["ragged"] else None
        if c["train"]:
            st["grads"] = [turn(randn(B, T, c["H"], c["V"]).to(dt)), randn(c["B"], c["H"], c["K"], c["V"], scale=0.1)]
    elif c["op"] == "delta_step":
        k = randn(c["B"], c["Hk"], c["K"])
        st["inputs"] = [randn(c["B"], c["Hk"], c["K"]).to(dt), (k / k.norm(dim=-1, keepdim=True)).to(dt), randn(c["B"], c["H"], c["V"]).to(dt),
                        -0.3 * rand(c["B"], c["H"]) ** 3 - 1e-4, torch.sigmoid(randn(c["B"], c["H"]))]
        st["memory"] = randn(c["B"], c["H"], c["K"], c["V"], scale=0.3)
    elif c["op"] == "norm":
        st["x"] = randn(c["M"], c["D"]).to(dt).requires_grad_(c["train"])
        st["residual"] = randn(c["M"], c["D"], scale=2.0).to(dt).requires_grad_(c["train"]) if c["residual"] else None
        st["weight"] = (1 + randn(c["D"], scale=0.1)).to(dt).requires_grad_(c["train"])
        if c["train"]:
            st["grads"] = [randn(c["M"], c["D"]).to(dt) for _ in range(2 if c["residual"] else 1)]
    else:
        M, K, N = c["M"], c["K"], c["N"]
        x, w = randn(M, K), randn(N, K, scale=K ** -0.5)
        st["bias"] = randn(N, scale=0.2).to(dt).requires_grad_(c["train"]) if c["bias"] else None
        st["residual"] = randn(M, N).to(dt).requires_grad_(c["train"]) if c["residual"] else None
        if c["fp8"]:
            (st["x"], st["x_scale"]), (st["weight"], st["w_scale"]) = _rows8(x), _rows8(w)
        else:
            st["x"], st["weight"] = x.to(dt).requires_grad_(c["train"]), w.to(dt).requires_grad_(c["train"])
        if c["train"]:
            st["grads"] = [randn(M, N).to(dt)]
    return st


# ------------------------------------------------------------------------------------------------------------------ the plain forms
def _delta_plain(q, k, v, g, beta, S, lengths):
    """The chunked form: within a chunk a triangular system, between chunks one state. 32 bits; the decays' sums in 64."""
    B, T, H, V = v.shape
    K, dt = q.shape[-1], v.dtype
    if lengths is not None:
        live = torch.arange(T, device=q.device)[None, :] < lengths[:, None]
        beta, g = torch.where(live[..., None], beta, 0.0), torch.where(live[..., None], g, 0.0)
    n = -(-T // CHUNK)

    def chunks(x, heads):                                                   # [B, T, h, ...] -> [B, H, n, CHUNK, ...] float32
        x = torch.nn.functional.pad(x.float(), [0, 0] * (x.dim() - 2) + [0, n * CHUNK - T])
        x = x.reshape(B, n, CHUNK, *x.shape[2:]).movedim(3, 1)
        return x.repeat_interleave(heads // x.shape[1], 1)

    q, k, v = chunks(q, H) * K ** -0.5, chunks(k, H), chunks(v, H)
    g, beta = chunks(g[..., None], H)[..., 0], chunks(beta[..., None], H)[..., 0]
    cut = g == -math.inf
    G, R = torch.where(cut, 0.0, g).double().cumsum(-1), cut.long().cumsum(-1)
    lower = torch.ones(CHUNK, CHUNK, device=q.device, dtype=torch.bool).tril()
    D = torch.where(lower & (R[..., :, None] == R[..., None, :]), (G[..., :, None] - G[..., None, :]).clamp_max(0).exp(), 0.0).float()
    head = torch.where(R == 0, G.exp(), 0.0).float()                        # from the chunk's start to i
    tail = D[..., -1, :]                                                    # from i to the chunk's end
    kt = k.transpose(-1, -2).contiguous()
    P = (q @ kt) * D
    eye = torch.eye(CHUNK, device=q.device)
    X = -(beta[..., None] * (k @ kt) * D).tril(-1)                          # nilpotent: (I - X)^-1 = (I + X)(I + X^2)(I + X^4) ...
    inv = eye + X
    for _ in range(5):
        X = X @ X
        inv = inv + inv @ X
    W, U0 = inv @ ((beta * head)[..., None] * k), inv @ (beta[..., None] * v)
    Q, Kt = q * head[..., None], (k * tail[..., None]).transpose(-1, -2).contiguous()
    outs = []
    for i in range(n):
        U = U0[:, :, i] - W[:, :, i] @ S
        outs.append(Q[:, :, i] @ S + P[:, :, i] @ U)
        S = head[:, :, i, -1, None, None] * S + Kt[:, :, i] @ U
    o = torch.stack(outs, 2).reshape(B, H, n * CHUNK, V)[:, :, :T].transpose(1, 2)
    if lengths is not None:
        o = torch.where(live[..., None, None], o, 0.0)
    return o.to(dt), S


def _step_plain(q, k, v, g, beta, S):
    r = S.shape[1] // q.shape[1]
    qf, kf = q.float().repeat_interleave(r, 1) * q.shape[-1] ** -0.5, k.float().repeat_interleave(r, 1)
    S.mul_(g.exp()[..., None, None])
    u = beta[..., None] * (v.float() - (S * kf[..., None]).sum(-2))
    S.add_(kf[..., None] * u[..., None, :])
    return (S * qf[..., None]).sum(-2).to(v.dtype)


def _norm_plain(x, residual, weight):
    s = x.float() if residual is None else x.float() + residual.float()
    return s, s * torch.rsqrt(s.square().mean(-1, keepdim=True) + EPS) * weight.float()


def _act(z, act):
    if act == "relu":
        return torch.where(z > 0, z, 0.0)
    if act == "tanh":
        return torch.tanh(z)
    if act == "silu":
        return z / (1 + torch.exp(-z))
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * 2 ** -0.5))
    return z


def run(state):
    st, c = state, state["case"]
    if own:
        from offpolicy_amd import ops
    if c["op"] == "delta":
        if own:
            o, S = ops.gated_delta_rule(*st["leaves"][:5], initial_state=st["leaves"][5], lengths=st["lengths"])
        else:
            o, S = _delta_plain(*st["leaves"], st["lengths"])
        if not c["train"]:
            return o, S
        return (o.detach(), S.detach(), *torch.autograd.grad([o, S], st["leaves"], st["grads"]))
    if c["op"] == "delta_step":
        if own:
            return ops.gated_delta_step(*st["inputs"], st["memory"]), st["memory"]
        return _step_plain(*st["inputs"], st["memory"]), st["memory"]
    if c["op"] == "norm":
        if c["fp8"]:
            if own:
                return ops.rms_norm_fp8(st["x"], st["weight"], residual=st["residual"], eps=EPS)
            s, y = _norm_plain(st["x"], st["residual"], st["weight"])
            q, scale = _rows8(y)
            return (q, scale) if st["residual"] is None else (q, scale, s.to(st["x"].dtype))
        if own:
            got = ops.rms_norm(st["x"], st["weight"], residual=st["residual"], eps=EPS)
        else:
            s, y = _norm_plain(st["x"], st["residual"], st["weight"])
            got = y.to(st["x"].dtype) if st["residual"] is None else (y.to(st["x"].dtype), s.to(st["x"].dtype))
        got = got if isinstance(got, tuple) else (got,)
        if not c["train"]:
            return got
        leaves = [t for t in (st["x"], st["residual"], st["weight"]) if t is not None]
        return (*(t.detach() for t in got), *torch.autograd.grad(got, leaves, st["grads"]))
    if c["fp8"]:
        if own:
            return ops.linear_fp8(st["x"], st["x_scale"], st["weight"], st["w_scale"], bias=st["bias"], residual=st["residual"], activation=c["act"], out_dtype=DTYPES[c["dtype"]])
        z = (st["x"].float() @ st["weight"].float().t()) * st["x_scale"][:, None] * st["w_scale"]
    elif own:
        y = ops.linear(st["x"], st["weight"], bias=st["bias"], residual=st["residual"], activation=c["act"])
    else:
        z = st["x"].float() @ st["weight"].float().t()
    if not own:
        z = z if st["bias"] is None else z + st["bias"].float()
        y = _act(z, c["act"])
        y = (y if st["residual"] is None else y + st["residual"].float()).to(DTYPES[c["dtype"]])
    if not c["train"]:
        return y
    leaves = [t for t in (st["x"], st["weight"], st["bias"], st["residual"]) if t is not None]
    return (y.detach(), *torch.autograd.grad([y], leaves, st["grads"]))


# ------------------------------------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    c, e = case, SIZE[case["dtype"]]
    if c["op"] == "delta":
        n = c["B"] * c["T"]
        q, v, state = 2 * n * c["Hk"] * c["K"] * e, n * c["H"] * c["V"] * e, c["B"] * c["H"] * c["K"] * c["V"] * 4
        gates, flops = 2 * n * c["H"] * 4, 6 * n * c["H"] * c["K"] * c["V"]
        if not c["train"]:
            return {"bytes": q + 2 * v + gates + 2 * state, "flops": flops}
        return {"bytes": 2 * q + 4 * v + 2 * gates + 4 * state, "flops": 3 * flops}
    if c["op"] == "delta_step":
        rows = c["B"] * c["H"]
        return {"bytes": rows * (8 * c["K"] * c["V"] + 2 * c["V"] * e + 8) + 2 * c["B"] * c["Hk"] * c["K"] * e, "flops": 7 * rows * c["K"] * c["V"]}
    if c["op"] == "norm":
        n, two = c["M"] * c["D"], 2 if c["residual"] else 1
        out = n * (1 if c["fp8"] else e) + (c["M"] * 4 if c["fp8"] else 0) + (n * e if c["residual"] else 0)
        fwd = two * n * e + out + c["D"] * e
        return {"bytes": fwd + ((two + 1) * n * e + c["D"] * e if c["train"] else 0), "flops": 5 * n + (8 * n if c["train"] else 0)}
    M, K, N = c["M"], c["K"], c["N"]
    one = 1 if c["fp8"] else e
    fwd = (M * K + N * K) * one + M * N * e * (2 if c["residual"] else 1) + (N * e if c["bias"] else 0) + ((M + N) * 4 if c["fp8"] else 0)
    bwd = (M * N * (2 if c["residual"] else 1) + M * K + N * K) * e + (N * e if c["bias"] else 0)
    return {"bytes": fwd + (bwd if c["train"] else 0), "flops": 2 * M * K * N * (3 if c["train"] else 1)}


# ----------------------------------------------------------------------------------------------------- the definitions, in 64 bits
def _delta_exact(st):
    """Token by token, as the rule is written; the gradients by its adjoint, walked backwards."""
    c = st["case"]
    q, k, v, g, beta, S = [t.detach().double() for t in st["leaves"]]
    r, T, dev = c["H"] // c["Hk"], c["T"], q.device
    q, k = q.repeat_interleave(r, 2) * c["K"] ** -0.5, k.repeat_interleave(r, 2)
    n = st["lengths"].long() if st["lengths"] is not None else torch.full((c["B"],), T, device=dev)
    o, past, told = torch.zeros_like(v), [], []
    for t in range(T):
        on = (t < n).double()[:, None, None]
        a = torch.where((t < n)[:, None], g[:, t].exp(), 1.0)[..., None, None]
        b = on * beta[:, t, :, None]
        F = a * S
        e = v[:, t] - (F * k[:, t, :, :, None]).sum(-2)
        if c["train"]:
            past.append(S)
            told.append(e)
        S = F + k[:, t, :, :, None] * (b * e)[:, :, None, :]
        o[:, t] = on * (S * q[:, t, :, :, None]).sum(-2)
    if not c["train"]:
        return o, S
    do, dS = [t.double() for t in st["grads"]]
    dq, dk, dv, dg, db = [torch.zeros_like(t) for t in (q, k, v, g, beta)]
    end = S
    for t in reversed(range(T)):
        on = (t < n).double()[:, None, None]
        a = torch.where((t < n)[:, None], g[:, t].exp(), 1.0)[..., None, None]
        b, kt, e, d = on * beta[:, t, :, None], k[:, t], told[t], on * do[:, t]
        F = a * past[t]
        now = F + kt[..., None] * (b * e)[:, :, None, :]
        dq[:, t] = (now * d[:, :, None, :]).sum(-1)
        dS = dS + q[:, t, :, :, None] * d[:, :, None, :]
        du = (dS * kt[..., None]).sum(-2)                                   # the gradient of u = b e
        db[:, t] = (on * du[:, :, :] * e).sum(-1)
        dv[:, t] = b * du
        dk[:, t] = (dS * (b * e)[:, :, None, :]).sum(-1) - (F * (b * du)[:, :, None, :]).sum(-1)
        dF = dS - kt[..., None] * (b * du)[:, :, None, :]
        dg[:, t] = (dF * F).sum((-1, -2)) * on[:, 0]
        dS = a * dF
        dk[:, t] *= on
    share = lambda x: x.reshape(c["B"], T, c["Hk"], r, c["K"]).sum(3)       # noqa: E731
    return o, end, share(dq) * c["K"] ** -0.5, share(dk), dv, dg, db, dS


def exact(case, seed):
    c, st = case, prepare(case, seed)
    if c["op"] == "delta":
        if c["train"] and c["T"] * c["B"] * c["H"] * c["K"] * c["V"] * 8 > 60e9:
            return None
        return _delta_exact(st)
    if c["op"] == "delta_step":
        q, k, v, g, beta, S = [t.double() for t in (*st["inputs"], st["memory"])]
        r = c["H"] // c["Hk"]
        q, k = q.repeat_interleave(r, 1), k.repeat_interleave(r, 1)
        S = torch.exp(g)[..., None, None] * S
        S = S + torch.einsum("bhk,bhv->bhkv", k, beta[..., None] * (v - torch.einsum("bhkv,bhk->bhv", S, k)))
        return torch.einsum("bhkv,bhk->bhv", S, q) / math.sqrt(c["K"]), S
    if c["op"] == "norm":
        x, w = st["x"].detach().double(), st["weight"].detach().double()
        s = x if st["residual"] is None else x + st["residual"].detach().double()
        rstd = 1 / torch.sqrt((s * s).sum(-1, keepdim=True) / c["D"] + EPS)
        y = s * rstd * w
        if c["fp8"]:
            scale = y.abs().amax(-1) / E4M3_MAX
            return (y / scale[:, None], scale) if st["residual"] is None else (y / scale[:, None], scale, s)
        got = (y,) if st["residual"] is None else (y, s)
        if not c["train"]:
            return got
        d = [t.double() for t in st["grads"]]
        h = w * d[0]
        ds = rstd * h - s * rstd ** 3 * (h * s).sum(-1, keepdim=True) / c["D"]
        if st["residual"] is None:
            return (*got, ds, (d[0] * s * rstd).sum(0))
        return (*got, ds + d[1], ds + d[1], (d[0] * s * rstd).sum(0))
    x, w = st["x"].detach().double(), st["weight"].detach().double()
    if c["fp8"]:
        x, w = x * st["x_scale"].double()[:, None], w * st["w_scale"].double()[:, None]
    z = torch.mm(x, w.t())
    if st["bias"] is not None:
        z += st["bias"].detach().double()
    sig = torch.sigmoid(z)
    cdf = torch.special.ndtr(z)
    a, slope = {"none": (z, torch.ones_like(z)), "relu": (z.clamp_min(0), (z > 0).double()), "tanh": (z.tanh(), 1 - z.tanh() ** 2),
                "silu": (z * sig, sig * (1 + z * (1 - sig))), "gelu": (z * cdf, cdf + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi))}[c["act"]]
    y = a if st["residual"] is None else a + st["residual"].detach().double()
    if not c["train"]:
        return y
    dy = st["grads"][0].double()
    dz = dy * slope
    got = [y, torch.mm(dz, w), torch.mm(dz.t(), x)]
    if st["bias"] is not None:
        got.append(dz.sum(0))
    if st["residual"] is not None:
        got.append(dy)
    return tuple(got)
