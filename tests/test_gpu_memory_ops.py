"""The memory-block operators (offpolicy_amd.ops) against their definitions in 64 bits (memory_ops_reference.py)."""
import math

import pytest
import torch

import memory_ops_reference as R

pytestmark = pytest.mark.gpu
F32, BF16, F16, E4M3 = torch.float32, torch.bfloat16, torch.float16, torch.float8_e4m3fn
INF = math.inf


@pytest.fixture(scope="module")
def ops():
    from offpolicy_amd import ops
    return ops


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape, dtype=F32, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def rand(g, *shape):
    return torch.rand(shape, generator=g, device="cuda")


# ------------------------------------------------------------------------------------------------------------------ gated delta rule
def delta_inputs(g, B, T, H, Hk, K, V, dtype, resets=0.0, decay=0.3, time_major=False):
    a, b = (T, B) if time_major else (B, T)
    k = randn(g, a, b, Hk, K)
    k = k / k.norm(dim=-1, keepdim=True).clamp_min(1e-6)
    gate = -decay * rand(g, a, b, H) ** 2
    gate = torch.where(rand(g, a, b, 1) < resets, torch.full_like(gate, -INF), gate)
    t = [randn(g, a, b, Hk, K, dtype=dtype), k.to(dtype), randn(g, a, b, H, V, dtype=dtype), gate, torch.sigmoid(randn(g, a, b, H))]
    return [x.transpose(0, 1) if time_major else x for x in t]


def delta_terms(K, V, T):
    """Length of the float32 sums behind an output: over the keys, over the values and over a chunk's tokens, a chunk's triangular solve and the
    state's way through the chunks (two products each)."""
    return K + V + 2 * 64 + 2 * (-(-T // 64)) * 4


def check_delta(ops, inputs, state=None, lengths=None, grads=True, scale=None, g=None):
    q, k, v, gate, beta = inputs
    (B, T, Hk, K), (H, V) = q.shape, v.shape[2:]
    n = delta_terms(K, V, T)
    leaves = [x.detach().requires_grad_() for x in inputs] + ([] if state is None else [state.detach().requires_grad_()])
    o, S = ops.gated_delta_rule(*leaves[:5], initial_state=leaves[5] if state is not None else None, lengths=lengths, scale=scale)
    wide = [x.detach().double().requires_grad_() for x in leaves]
    o64, S64 = R.delta_rule(*wide[:5], wide[5] if state is not None else None, lengths, scale)
    assert o.dtype == v.dtype and S.dtype == F32
    R.close(o.detach(), o64.detach(), 1, n, "out")
    R.close(S.detach(), S64.detach(), 0, n, "state")
    with torch.no_grad():                 # the call that keeps nothing for a backward pass
        o2, S2 = ops.gated_delta_rule(*inputs, initial_state=state, lengths=lengths, scale=scale)
    assert torch.equal(o2, o.detach()) and torch.equal(S2, S.detach())
    if not grads:
        return
    g = g or gen(77)
    do, dS = randn(g, B, T, H, V, dtype=v.dtype), randn(g, B, H, K, V, scale=0.3)
    got = torch.autograd.grad([o, S], leaves, [do, dS])
    want = torch.autograd.grad([o64, S64], wide, [do.double(), dS.double()])
    names = ["dq", "dk", "dv", "dlog_decay", "dbeta", "dstate"]
    # dlog_decay is the difference of sums the size of q.dq and k.dk; every gradient passes through the forward's sums and the adjoint's
    wq, wk = (want[i].detach() * wide[i].detach() for i in (0, 1))
    for i, (x, w) in enumerate(zip(got, want)):
        assert x.dtype == leaves[i].dtype and x.shape == leaves[i].shape
        size = None
        if names[i] in ("dlog_decay", "dbeta"):
            size = max(w.abs().max().item(), wq.abs().sum(-1).max().item(), wk.abs().sum(-1).max().item())
        R.close(x, torch.nan_to_num(w, nan=0.0), 1 if x.dtype != F32 else 0, 4 * n, names[i], size)
    return got


DELTA = [
    # B, T, H, Hk, K, V, dtype, resets, time-major
    (1, 1, 1, 1, 1, 1, F32, 0, False),
    (2, 2, 1, 1, 16, 16, BF16, 0, False),
    (2, 63, 2, 1, 5, 3, BF16, 0, False),
    (3, 64, 2, 2, 16, 16, F32, 0, False),
    (2, 65, 4, 2, 17, 33, F16, 0, True),
    (2, 130, 3, 1, 72, 100, BF16, 0.05, False),
    (1, 300, 2, 2, 128, 128, F32, 0.02, False),
    (2, 200, 2, 2, 64, 40, F32, 0, True),
    (5, 150, 2, 2, 32, 32, F32, 0.03, True),
    (1, 129, 1, 1, 127, 257, F16, 0, False),
    (2, 140, 2, 1, 33, 20, F32, 0.03, False),
    (3, 131, 2, 2, 48, 48, BF16, 0, True),
    (2, 190, 4, 2, 48, 17, F16, 0, False),
    (2, 260, 2, 2, 96, 96, F32, 0.02, False),
    (1, 130, 2, 1, 96, 64, F16, 0, True),
    (2, 70, 2, 2, 65, 130, BF16, 0, False),
    (1, 200, 1, 1, 97, 30, F32, 0, False),
    (2, 150, 2, 1, 80, 36, F32, 0.02, True),
    (1, 260, 2, 2, 112, 112, BF16, 0, False),
    (2, 129, 2, 2, 103, 20, F32, 0, False),
]


@pytest.mark.parametrize("B,T,H,Hk,K,V,dtype,resets,time_major", DELTA)
def test_delta_rule_and_its_gradients(ops, B, T, H, Hk, K, V, dtype, resets, time_major):
    g = gen(1)
    check_delta(ops, delta_inputs(g, B, T, H, Hk, K, V, dtype, resets, time_major=time_major), randn(g, B, H, K, V, scale=0.3))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_delta_rule_on_ragged_rows(ops, dtype):
    """Lengths of zero, one, a chunk and past the batch's length; what lies behind them is NaN and is not read."""
    g = gen(2)
    lengths = torch.tensor([0, 1, 64, 65, 97, 130, 500, -3], dtype=torch.int32, device="cuda")
    B, T = len(lengths), 130
    inputs = delta_inputs(g, B, T, 2, 1, 24, 20, dtype, 0.03)
    dead = torch.arange(T, device="cuda")[None] >= lengths[:, None]
    state = randn(g, B, 2, 24, 20, scale=0.3)
    poisoned = [x.masked_fill(dead.reshape(B, T, *[1] * (x.dim() - 2)), math.nan) for x in inputs]
    got = check_delta(ops, poisoned, state, lengths)
    for x in got[:5]:
        assert (x[dead] == 0).all()
    with torch.no_grad():
        o, S = ops.gated_delta_rule(*poisoned, initial_state=state, lengths=lengths)
    assert (o[dead] == 0).all() and torch.equal(S[0], state[0]) and torch.equal(S[7], state[7])


@pytest.mark.parametrize("value", [math.nan, INF])
@pytest.mark.parametrize("Hk,dtype", [(2, F32), (1, BF16)])
def test_behind_the_length_all_is_zero_whatever_the_state_holds(ops, Hk, dtype, value):
    g = gen(55)
    lengths = torch.tensor([0, 1, 40, 64, 70, 100], dtype=torch.int32, device="cuda")
    B, T = len(lengths), 100
    inputs = delta_inputs(g, B, T, 2, Hk, 24, 20, dtype)
    state = randn(g, B, 2, 24, 20)
    state[:, 0, 3] = value
    leaves = [x.detach().requires_grad_() for x in inputs] + [state.requires_grad_()]
    o, S = ops.gated_delta_rule(*leaves[:5], initial_state=state, lengths=lengths)
    grads = torch.autograd.grad([o, S], leaves, [randn(g, B, T, 2, 20, dtype=dtype), randn(g, B, 2, 24, 20)])
    dead = torch.arange(T, device="cuda")[None] >= lengths[:, None]
    for x in (o, *grads[:5]):
        assert (x[dead] == 0).all()
    assert torch.equal(S[0].isnan(), state[0].isnan()) and not o[1:, 0, 0].isfinite().all()


def test_delta_rule_resets_are_exact(ops):
    """A row that holds two episodes gives, behind the reset, bit for bit what the second one gives at the same place of its chunk after another first."""
    g = gen(3)
    a, b = (delta_inputs(g, 1, 140, 2, 2, 32, 32, F32) for _ in range(2))
    at = 70
    for x, y in zip(a, b):
        y[:, at:] = x[:, at:]
    for x in (a, b):
        x[3][:, at] = -INF
    state = randn(g, 1, 2, 32, 32)
    (oa, Sa), (ob, Sb) = (ops.gated_delta_rule(*x, initial_state=state) for x in (a, b))
    assert torch.equal(oa[:, at:], ob[:, at:]) and torch.equal(Sa, Sb)
    leaves = [x.detach().requires_grad_() for x in a]
    o, S = ops.gated_delta_rule(*leaves, initial_state=state)
    grads = torch.autograd.grad(o[:, at:].sum() + S.sum(), leaves)
    for x in grads:
        assert (x[:, :at] == 0).all()                    # nothing reaches over the reset
    assert (grads[3][:, at] == 0).all()
    first = ops.gated_delta_rule(*[x[:, at:at + 58] for x in a])[0]
    R.close(first, oa[:, at:at + 58].double(), 0, 2 * delta_terms(32, 32, 140), "second episode alone")


@pytest.mark.parametrize("low", [-INF, torch.finfo(F32).min])
@pytest.mark.parametrize("H,Hk,K,V,dtype", [(2, 1, 24, 20, F32), (2, 2, 128, 40, BF16), (1, 1, 96, 130, F16), (2, 2, 64, 64, F32)])
def test_what_is_not_finite_stays_in_its_episode(ops, H, Hk, K, V, dtype, low):
    """A NaN or an infinity in any input or gradient of one episode of a row leaves the other episodes' outputs and gradients what they are, to the bit.
    Episodes of one chunk, of parts of chunks, of several, and one of three tokens; the initial state is the first's, the final one the last's."""
    g = gen(56)
    B, T, starts = 2, 200, [0, 20, 64, 90, 93, 150]
    ends = starts[1:] + [T]
    clean = delta_inputs(g, B, T, H, Hk, K, V, dtype)
    clean[3][:, starts[1:]] = low
    clean += [randn(g, B, H, K, V), randn(g, B, T, H, V, dtype=dtype), randn(g, B, H, K, V)]

    def run(x):
        leaves = [t.clone().requires_grad_() for t in x[:6]]
        o, S = ops.gated_delta_rule(*leaves[:5], initial_state=leaves[5])
        return (o.detach(), S.detach(), *torch.autograd.grad([o, S], leaves, [x[6], x[7]]))

    want = run(clean)
    assert all(t.isfinite().all() for t in want)
    for e, (a, b) in enumerate(zip(starts, ends)):
        for i, name in enumerate(("q", "k", "v", "log_decay", "beta", "initial_state", "dout", "dstate")):
            for value in (math.nan, INF):
                if name == "initial_state" and e or name == "dstate" and e < len(starts) - 1:
                    continue
                x = [t.clone() for t in clean]
                if name in ("initial_state", "dstate"):
                    x[i][0, :, K // 2, V // 2] = value
                else:
                    x[i][0, (a + b) // 2] = value
                others = torch.ones(B, T, dtype=torch.bool, device="cuda")
                others[0, a:b] = False
                for j, (got, ref) in enumerate(zip(run(x), want)):
                    if j == 1 or j == 7:             # the final state, the initial state's gradient
                        same = got, ref
                        if e == (len(starts) - 1 if j == 1 else 0):
                            same = got[1], ref[1]
                    else:
                        same = got[others], ref[others]
                    assert torch.equal(*same), (name, e, value, j)


def test_a_reset_clears_whatever_the_state_holds(ops):
    """At the first token of a row, of a chunk, and of a row whose state leaves the range of float32; huge finite keys and queries are no NaN."""
    g = gen(57)
    inputs = delta_inputs(g, 2, 140, 2, 2, 32, 32, F32)
    inputs[3][:, 0] = inputs[3][:, 128] = -INF
    bad = torch.full((2, 2, 32, 32), math.nan, device="cuda")
    leaves = [[x.clone().requires_grad_() for x in (*inputs, s)] for s in (bad, torch.zeros_like(bad))]
    runs = [(*(out := ops.gated_delta_rule(*x[:5], initial_state=x[5])), *torch.autograd.grad(out[0].sum() + out[1].sum(), x)) for x in leaves]
    for a, b in zip(*runs):
        assert a.isfinite().all() and torch.equal(a, b)
    over = [x.clone() for x in inputs]
    over[4][:, 100:110] = 1e30                       # the state grows past float32 within a few of these
    o, S = ops.gated_delta_rule(*over)
    assert not o[:, 100:128].isfinite().all() and torch.equal(o[:, 128:], runs[0][0][:, 128:]) and torch.equal(S, runs[0][1])
    huge = [x.clone() for x in inputs]
    huge[0][:, 5], huge[4][:, 5] = 1.2e38, 0.0
    x = [t.requires_grad_() for t in huge]
    dk = torch.autograd.grad(ops.gated_delta_rule(*x, scale=1e-38)[0][:, 10:].sum(), x[1])[0]
    assert dk.isfinite().all()


def test_delta_rule_on_repeated_keys_and_full_writes(ops):
    """All keys the same and beta = 1: the triangular system at its worst, every token overwrites the last."""
    g = gen(4)
    inputs = delta_inputs(g, 2, 150, 2, 2, 32, 32, F32, decay=0.0)
    inputs[1] = inputs[1][:, :1].expand(-1, 150, -1, -1)
    inputs[4] = torch.ones_like(inputs[4])
    check_delta(ops, inputs, randn(g, 2, 2, 32, 32))


@pytest.mark.parametrize("decay", [3.0, 60.0, 400.0])
def test_delta_rule_on_strong_decays(ops, decay):
    g = gen(5)
    check_delta(ops, delta_inputs(g, 2, 130, 2, 2, 32, 32, F32, decay=decay), randn(g, 2, 2, 32, 32))


@pytest.mark.parametrize("low", [-103.0, -104.5, -200.0, -1e15, -1e30, torch.finfo(F32).min])
@pytest.mark.parametrize("at", [(10,), (0, 70), (20, 40), (20, 21, 63, 64)])
def test_delta_rule_on_finite_stand_ins_for_a_reset(ops, low, at):
    """A gate whose exponential is 0 (or nearly) clears the state like -inf and leaves the gates behind it what they are; the one-token step agrees."""
    g = gen(51)
    inputs = delta_inputs(g, 2, 100, 2, 1, 24, 20, F32)
    for t in at:
        inputs[3][:, t, 0] = low
    state = randn(g, 2, 2, 24, 20)
    got = check_delta(ops, inputs, state)
    if low < -104:
        assert (got[3][:, list(at), 0] == 0).all()
        as_inf = [x.clone() for x in inputs]
        as_inf[3][as_inf[3] == low] = -INF
        for x, y in zip(ops.gated_delta_rule(*inputs, initial_state=state), ops.gated_delta_rule(*as_inf, initial_state=state)):
            assert torch.equal(x, y)
    S, want = state.clone(), R.delta_rule(*[x.double() for x in inputs], state.double())
    for t in range(100):
        o = ops.gated_delta_step(*[x[:, t] for x in inputs], S)
        R.close(o, want[0][:, t], 0, 4 * (t + 4) + 24 + 20, "step %d" % t, want[0].abs().max().item())
    R.close(S, want[1], 0, 4 * 100 + 44, "state")


def test_delta_rule_takes_slices_and_expanded_inputs(ops):
    """q, k and v as slices of one projection (rows of odd stride and start), gates expanded over the heads."""
    g = gen(6)
    B, T, H, K, V = 2, 70, 3, 20, 24
    both = randn(g, B, T, H * (2 * K + V) + 1, dtype=BF16)[..., 1:]
    q, k, v = both[..., :H * K].unflatten(-1, (H, K)), both[..., H * K:2 * H * K].unflatten(-1, (H, K)) * 0.2, both[..., 2 * H * K:].unflatten(-1, (H, V))
    gate, beta = (-0.1 * rand(g, B, T, 1)).expand(-1, -1, H), rand(g, B, 1, H).expand(-1, T, -1)
    check_delta(ops, [q, k, v, gate, beta])
    tilted = randn(g, B, T, K, H, dtype=BF16).transpose(-1, -2)              # last axis not contiguous
    check_delta(ops, [tilted, k, v, gate, beta], scale=0.7)


def test_delta_rule_on_nothing(ops):
    for B, T in ((0, 5), (2, 0), (0, 0)):
        inputs = [x.requires_grad_() for x in delta_inputs(gen(7), B, T, 2, 1, 8, 6, F32)]
        state = randn(gen(7), B, 2, 8, 6).requires_grad_()
        o, S = ops.gated_delta_rule(*inputs, initial_state=state)
        assert o.shape == (B, T, 2, 6) and torch.equal(S, state)
        grads = torch.autograd.grad([S], [*inputs, state], [torch.full_like(S, 2.0)], allow_unused=True)
        assert (grads[5] == 2).all()
        assert (ops.gated_delta_rule(*[x.detach() for x in inputs])[1] == 0).all()


@pytest.mark.parametrize("through", ["out", "state"])
def test_delta_gradients_through_one_output_alone(ops, through):
    g = gen(12)
    inputs = delta_inputs(g, 2, 90, 2, 1, 20, 24, F32, 0.02)
    leaves = [x.requires_grad_() for x in inputs] + [randn(g, 2, 2, 20, 24, scale=0.3).requires_grad_()]
    wide = [x.detach().double().requires_grad_() for x in leaves]
    i = 0 if through == "out" else 1
    y, y64 = ops.gated_delta_rule(*leaves[:5], initial_state=leaves[5])[i], R.delta_rule(*wide[:5], wide[5])[i]
    dy = randn(g, *y.shape)
    got, want = torch.autograd.grad(y, leaves, dy), torch.autograd.grad(y64, wide, dy.double(), allow_unused=True)
    size = max((want[j] * wide[j]).detach().abs().sum(-1).max().item() for j in (0, 1) if want[j] is not None)
    for j, (a, b) in enumerate(zip(got, want)):
        b = torch.zeros_like(wide[j]) if b is None else torch.nan_to_num(b, nan=0.0)
        R.close(a, b, 0, 4 * delta_terms(20, 24, 90), "gradient %d" % j, max(size, b.abs().max().item()) if j in (3, 4) else None)


def test_time_major_block_as_documented(ops):
    """The block over a time-major batch is the block over the turned one, and its output comes back time-major without a copy."""
    g = gen(13)
    T, rows, D, H, K, V = 70, 6, 48, 2, 16, 24
    x, res, lengths = randn(g, T, rows, D), randn(g, T, rows, D), torch.tensor([70, 1, 0, 64, 33, 70], dtype=torch.int32, device="cuda")
    nw, w, wo = 1 + randn(g, D, scale=0.1), randn(g, H * (2 * K + V), D, scale=D ** -0.5), randn(g, D, H * V, scale=0.1)
    decay, beta = -0.1 * rand(g, T, rows, H), rand(g, T, rows, H)
    turn = lambda t: t.transpose(0, 1)                                                   # noqa: E731

    def block(x, res, decay, beta, major):
        y, s = ops.rms_norm(x, nw, residual=res)
        q, k, v = (t.unflatten(-1, (H, -1)) for t in ops.linear(y, w, activation="silu").split([H * K, H * K, H * V], -1))
        k = torch.nn.functional.normalize(k, dim=-1)
        o, S = ops.gated_delta_rule(*(turn(t) if major else t for t in (q, k, v, decay, beta)), lengths=lengths)
        o = turn(o) if major else o
        assert o.is_contiguous()
        return ops.linear(o.flatten(-2), wo, residual=s), S
    leaf = x.requires_grad_()
    y, S = block(leaf, res, decay, beta, True)
    leaf2 = turn(x.detach()).contiguous().requires_grad_()
    y2, S2 = block(leaf2, turn(res).contiguous(), turn(decay).contiguous(), turn(beta).contiguous(), False)
    assert torch.equal(turn(y), y2) and torch.equal(S, S2)
    dy = randn(g, T, rows, D)
    assert torch.equal(turn(torch.autograd.grad(y, leaf, dy)[0]), torch.autograd.grad(y2, leaf2, turn(dy))[0])


def test_delta_gradient_agrees_with_differences(ops):
    g = gen(8)
    inputs = delta_inputs(g, 2, 100, 2, 1, 16, 12, F32) + [randn(g, 2, 2, 16, 12, scale=0.3)]
    wo, ws = randn(g, 2, 100, 2, 12).double(), randn(g, 2, 2, 16, 12).double()

    def loss(xs):
        o, S = ops.gated_delta_rule(*xs[:5], initial_state=xs[5])
        return (o.double() * wo).sum() + (S.double() * ws).sum()
    leaves = [x.detach().requires_grad_() for x in inputs]
    grads = torch.autograd.grad(loss(leaves), leaves)
    for i, x in enumerate(inputs):
        way, h = randn(g, *x.shape), 2.0 ** -7
        if i == 3:
            way = -way.abs()
        with torch.no_grad():
            up, down = (loss([y + (s * h * way if j == i else 0) for j, y in enumerate(inputs)]).item() for s in (1, -1))
        slope, want = (up - down) / (2 * h), (grads[i].double() * way.double()).sum().item()
        # the loss sums 4800 + 768 float32 values of size up to 10, off by 2^-24 * 200 each at random: under 1e-2 in all; the cubic term under 2 %
        assert abs(slope - want) <= 0.02 * abs(want) + 1e-2 / h * 0.05 + 0.5, (i, slope, want)


@pytest.mark.parametrize("B,H,Hk,K,V,dtype", [(1, 1, 1, 1, 1, F32), (3, 4, 2, 17, 5, F16), (64, 2, 2, 32, 32, F32), (5, 3, 1, 64, 66, BF16), (7, 8, 4, 128, 128, BF16),
                                              (2, 2, 2, 100, 300, F32)])
def test_delta_step(ops, B, H, Hk, K, V, dtype):
    g = gen(9)
    state = randn(g, B, H, K, V, scale=0.5)
    mine, S64 = state.clone(), state.double()
    n = K + 16
    for t in range(3):
        q, k, v, gate, beta = (x[:, 0] for x in delta_inputs(g, B, 1, H, Hk, K, V, dtype))
        if t == 1:
            gate = gate.clone()
            gate[0] = -INF                                  # one row's episode begins: whatever its state holds is gone
            mine[0], S64[0] = math.nan, 0.0
        o64, S64 = R.delta_rule(*(x[:, None].double() for x in (q, k, v, gate, beta)), S64)
        o = ops.gated_delta_step(q, k, v, gate, beta, mine)
        R.close(o, o64[:, 0], 1, 3 * n, "out")
        R.close(mine, S64, 0, 3 * n, "state")


def test_delta_step_reads_its_scale_in_every_call(ops):
    """A scale that is a tensor is taken by its value, not by which tensor it is."""
    a = [x[:, 0] for x in delta_inputs(gen(53), 2, 1, 2, 2, 16, 16, F32)]
    scale, S = torch.tensor(0.5), torch.zeros(2, 2, 16, 16, device="cuda")
    one = ops.gated_delta_step(*a, S.clone(), scale=scale)
    scale.fill_(2.0)
    assert torch.equal(ops.gated_delta_step(*a, S.clone(), scale=scale), 4 * one) and torch.equal(ops.gated_delta_step(*a, S.clone(), scale=2), 4 * one)


def test_delta_steps_follow_the_chunked_pass(ops):
    g = gen(10)
    inputs = delta_inputs(g, 3, 90, 2, 1, 48, 40, F32, 0.03)
    o, S = ops.gated_delta_rule(*inputs)
    state = torch.zeros(3, 2, 48, 40, device="cuda")
    steps = torch.stack([ops.gated_delta_step(*(x[:, t] for x in inputs), state) for t in range(90)], 1)
    n = 2 * delta_terms(48, 40, 90)
    R.close(steps, o.double(), 0, n, "out")
    R.close(state, S.double(), 0, n, "state")


def test_delta_offsets_past_32_bits(ops):
    """A strided batch whose last row starts more than 2^31 elements behind its first."""
    g = gen(11)
    rows, K = 5, 16
    big = torch.empty((rows, (1 << 29) + 64), dtype=BF16, device="cuda")
    inputs = delta_inputs(g, rows, 3, 1, 1, K, K, BF16)
    far = []
    for i, x in enumerate(inputs[:3]):
        view = big.as_strided(x.shape, (big.stride(0), K, K, 1), i * 64)
        view.copy_(x)
        far.append(view)
    a, b = ops.gated_delta_rule(*inputs), ops.gated_delta_rule(*far, *inputs[3:])
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


# ------------------------------------------------------------------------------------------------------------------------- RMS norm
WIDTHS = [1, 3, 7, 8, 9, 63, 64, 65, 250, 513, 1003, 2050, 4096, 5000, 9001]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("D", WIDTHS)
def test_norm_and_its_gradients(ops, D, dtype):
    g = gen(20)
    for M, residual in ((1, True), (37, False), (131, True)):
        x, w = randn(g, M, D, dtype=dtype), (1 + randn(g, D, scale=0.2)).to(dtype)
        r = randn(g, M, D, dtype=dtype, scale=2.0) if residual else None
        leaves = [t.requires_grad_() for t in (x, w, r) if t is not None]
        got = ops.rms_norm(x, w, residual=r, eps=1e-5)
        wide = [t.detach().double().requires_grad_() for t in leaves]
        y64, s64 = R.rms_norm(wide[0], wide[1], wide[2] if residual else None, 1e-5)
        y, s = got if residual else (got, None)
        # mean of D squares, its root, two products: D + 8 half steps of the value itself (no cancellation)
        R.close(y.detach(), y64.detach(), 1, 8 + D ** 0.5, "y")
        if residual:
            R.close(s.detach(), s64.detach(), 1, 0 if dtype != F32 else 1, "s")
        dy, ds = randn(g, M, D, dtype=dtype), randn(g, M, D, dtype=dtype)
        grads = torch.autograd.grad(got, leaves, [dy, ds] if residual else [dy])
        want = torch.autograd.grad([y64, s64] if residual else [y64], wide, [dy.double(), ds.double()] if residual else [dy.double()])
        rstd = (s64.detach().square().mean(-1, keepdim=True) + 1e-5).rsqrt()
        size = ((wide[1].abs() * dy.double().abs()).max() * rstd.max() * 2).item() + (ds.abs().max().item() if residual else 0)
        R.close(grads[0], want[0], 1, 16 + D ** 0.5, "dx", size)
        part = (dy.double() * s64.detach() * rstd).abs().sum(0).max().item()
        R.close(grads[1], want[1], 1, M + 16, "dweight", part)
        if residual:
            assert torch.equal(grads[0], grads[2])
        with torch.no_grad():
            again = ops.rms_norm(x, w, residual=r, eps=1e-5)
        assert torch.equal(again[0] if residual else again, y.detach())


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_norm_of_rows_past_the_registers(ops, dtype):
    """Widths over 4096 packs: the row is walked again for each pass."""
    g = gen(21)
    D = 4096 * (4 if dtype == F32 else 8) + 5
    x, w, r = randn(g, 3, D, dtype=dtype), (1 + randn(g, D, scale=0.2)).to(dtype), randn(g, 3, D, dtype=dtype)
    leaves = [t.requires_grad_() for t in (x, w, r)]
    y, s = ops.rms_norm(*leaves[:2], residual=r)
    wide = [t.detach().double().requires_grad_() for t in leaves]
    y64, s64 = R.rms_norm(*wide)
    R.close(y.detach(), y64.detach(), 1, 64, "y")
    R.close(s.detach(), s64.detach(), 1, 1, "s")
    dy = randn(g, 3, D, dtype=dtype)
    for name, a, b in zip(("dx", "dw", "dr"), torch.autograd.grad(y, leaves, dy), torch.autograd.grad(y64, wide, dy.double())):
        R.close(a, b, 1, 64, name, 2 * b.abs().max().item())
    with torch.no_grad():
        check_fp8(*ops.rms_norm_fp8(x, w, residual=r)[:2], y64.detach())


def check_fp8(q, scale, y):
    """q * scale against y in 64 bits: half a step of e4m3 (2^-4 of the value, 2^-10 of the scale among its subnormals), and float32's own."""
    assert q.dtype == E4M3 and scale.dtype == F32 and q.shape == y.shape and scale.shape == y.shape[:-1]
    want = y.abs().amax(-1).clamp_min(448 * 2.0 ** -126) / 448
    assert ((scale.double() - want).abs() <= 64 * R.U32 * want).all()
    s = scale.double()[..., None]
    off = (q.float().double() * s - y).abs()
    assert (off <= (2.0 ** -4 * y.abs() + 2.0 ** -10 * s) * (1 + 1e-5) + 64 * R.U32 * y.abs()).all(), (off / s).max()
    assert (q.float().abs().amax(-1) == 448).logical_or(y.abs().amax(-1) < 448 * 2.0 ** -126).all()     # the row's largest value uses the whole range


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("D", [1, 5, 8, 65, 250, 1003, 4096, 9001])
def test_norm_in_8_bits(ops, D, dtype):
    g = gen(22)
    x, w, r = randn(g, 19, D, dtype=dtype), (1 + randn(g, D, scale=0.2)).to(dtype), randn(g, 19, D, dtype=dtype)
    q, scale, s = ops.rms_norm_fp8(x, w, residual=r)
    y64, s64 = R.rms_norm(x.double(), w.double(), r.double())
    check_fp8(q, scale, y64)
    R.close(s, s64, 1, 1, "s")
    q, scale = ops.rms_norm_fp8(x, w)
    check_fp8(q, scale, R.rms_norm(x.double(), w.double())[0])
    q, scale = ops.quantize_rows_fp8(x)
    check_fp8(q, scale, x.double())


def test_8_bits_of_rows_without_a_size(ops):
    """Rows of zeros, of subnormals, with one huge value, with an infinity and with a NaN."""
    x = torch.zeros(6, 40, device="cuda")
    x[1] = 1e-42
    x[2, 3], x[2, 4] = 3e38, 1.0
    x[3, 7] = INF
    x[4, 9] = math.nan
    x[5] = torch.linspace(-1, 1, 40)
    q, scale = ops.quantize_rows_fp8(x)
    assert (q[0].float() == 0).all() and scale[0] == 2.0 ** -126
    assert torch.isfinite(q[1].float()).all() and scale[1] == 2.0 ** -126
    assert q[2, 3].float() == 448 and q[2, 4].float() == 0
    assert scale[3] == INF and torch.isnan(q[3, 7].float()) and (q[3, :7].float() == 0).all()
    assert torch.isnan(scale[4]) and torch.isnan(q[4].float()).all()
    check_fp8(q[5:], scale[5:], x[5:].double())


def test_norm_of_values_that_are_no_numbers(ops):
    """A NaN or an infinity stays in its row."""
    g = gen(23)
    x, w = randn(g, 70, 64), randn(g, 64)
    clean = ops.rms_norm(x, w)
    bad = x.clone()
    bad[3, 5], bad[40, 0] = math.nan, INF
    y = ops.rms_norm(bad, w)
    assert torch.isnan(y[3]).all() and torch.isnan(y[40, 0]) and (y[40, 1:] == 0).all()
    keep = [i for i in range(70) if i not in (3, 40)]
    assert torch.equal(y[keep], clean[keep])
    zero = ops.rms_norm(torch.zeros(4, 64, device="cuda"), w, eps=1e-6)
    assert (zero == 0).all()


def test_norm_takes_rows_of_any_stride(ops):
    g = gen(24)
    wide, w = randn(g, 33, 401, dtype=BF16), randn(g, 100, dtype=BF16)
    x, r = wide[:, 1:101], wide[:, 200:300]
    y, s = ops.rms_norm(x, w, residual=r)
    y2, s2 = ops.rms_norm(x.contiguous(), w, residual=r.contiguous())
    assert torch.equal(y, y2) and torch.equal(s, s2)
    same = x[:1].expand(33, -1)
    assert torch.equal(ops.rms_norm(same, w), ops.rms_norm(same.contiguous(), w))
    turned = randn(g, 100, 6, 4, dtype=BF16).permute(2, 1, 0)
    assert torch.equal(ops.rms_norm(turned, w), ops.rms_norm(turned.contiguous(), w))
    leaf = wide[:, 1:101].detach().requires_grad_()
    a = torch.autograd.grad(ops.rms_norm(leaf, w).sum(), leaf)[0]         # an expanded gradient
    leaf2 = leaf.detach().contiguous().requires_grad_()
    assert torch.equal(a, torch.autograd.grad(ops.rms_norm(leaf2, w).sum(), leaf2)[0])


def test_norm_of_no_rows(ops):
    x, w = torch.zeros(0, 8, device="cuda").requires_grad_(), torch.ones(8, device="cuda").requires_grad_()
    y, s = ops.rms_norm(x, w, residual=torch.zeros(0, 8, device="cuda"))
    dx, dw = torch.autograd.grad(y.sum() + s.sum(), [x, w])
    assert y.shape == (0, 8) and dx.shape == (0, 8) and (dw == 0).all()
    with torch.no_grad():
        assert ops.rms_norm_fp8(x, w)[0].shape == (0, 8)


# --------------------------------------------------------------------------------------------------------------------------- linear
def check_linear(ops, g, M, K, N, dtype, act, bias=True, residual=True, x=None):
    x = randn(g, M, K, dtype=dtype) if x is None else x
    w = randn(g, N, K, dtype=dtype, scale=K ** -0.5)
    b = randn(g, N, dtype=dtype, scale=0.3) if bias else None
    r = randn(g, M, N, dtype=dtype) if residual else None
    leaves = [t.detach().requires_grad_() for t in (x, w, b, r) if t is not None]
    args = dict(zip([n for n, t in (("x", x), ("weight", w), ("bias", b), ("residual", r)) if t is not None], leaves))
    y = ops.linear(activation=act, **args)
    wide = {n: t.detach().double().requires_grad_() for n, t in args.items()}
    y64 = R.linear(wide["x"], wide["weight"], wide.get("bias"), wide.get("residual"), act)
    size = (x.double().abs() @ w.double().abs().t()).max().item() + 4 if M else 1
    R.close(y.detach(), y64.detach(), 1, K + 8, "y", size)
    with torch.no_grad():
        assert torch.equal(ops.linear(activation=act, **{n: t.detach() for n, t in args.items()}), y.detach())
    dy = randn(g, M, N, dtype=dtype)
    got = dict(zip(args, torch.autograd.grad(y, leaves, dy)))
    want = dict(zip(args, torch.autograd.grad(y64, list(wide.values()), dy.double())))
    # dz = dy act'(z) is rounded to its type in front of the products
    more = (R.half_step(dtype) / R.U32 if dtype != F32 else 0) + K + 8
    d = dy.double().abs()
    sizes = {"x": (d @ w.double().abs()).max().item() if M else 0, "weight": (d.t() @ x.double().abs()).max().item() if M else 0, "bias": d.sum(0).max().item() if M else 0}
    terms = {"x": N, "weight": M, "bias": M}
    for n in ("x", "weight", "bias"):
        if n in got:
            R.close(got[n], want[n], 1, 1.2 * (terms[n] + more), "d" + n, 1.1 * sizes[n])
    if residual:
        assert torch.equal(got["residual"], dy)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("M,K,N", [(1, 1, 1), (1, 64, 64), (3, 5, 7), (16, 128, 48), (17, 33, 65), (64, 252, 64), (65, 252, 64), (130, 100, 259), (300, 520, 130), (1000, 64, 192)])
def test_linear_and_its_gradients(ops, M, K, N, dtype):
    check_linear(ops, gen(30), M, K, N, dtype, "silu")


@pytest.mark.parametrize("act", ["none", "tanh", "silu", "gelu"])
@pytest.mark.parametrize("bias,residual", [(False, False), (True, False), (False, True)])
def test_linear_activations(ops, act, bias, residual):
    check_linear(ops, gen(31), 70, 48, 40, F32, act, bias, residual)
    check_linear(ops, gen(31), 70, 48, 40, BF16, act, bias, residual)


def test_linear_relu(ops):
    """Whole numbers: every product and sum is exact, so the slope's jump at 0 is hit on the same side."""
    g = gen(32)
    for dtype in (F32, BF16, F16):
        x, w, b, dy = (torch.randint(-3, 4, s, generator=g, device="cuda").to(dtype) for s in ((90, 20), (30, 20), (30,), (90, 30)))
        leaves = [t.requires_grad_() for t in (x, w, b)]
        wide = [t.detach().double().requires_grad_() for t in leaves]
        y, y64 = ops.linear(*leaves, activation="relu"), R.linear(*wide, act="relu")
        assert torch.equal(y.double(), y64)
        for a, c in zip(torch.autograd.grad(y, leaves, dy), torch.autograd.grad(y64, wide, torch.where(y64 > 0, dy.double(), 0.0))):
            R.close(a, c, 1, 0, "gradient")


@pytest.mark.parametrize("act", ["none", "relu"])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("M,K,N", [(5, 7, 3), (64, 252, 64), (65, 33, 70), (300, 520, 130), (1203, 1101, 1003), (4090, 601, 4090), (4090, 2045, 600), (601, 4090, 4090)])
def test_linear_loses_nothing_of_whole_numbers(ops, M, K, N, dtype, act):
    """Products and sums of small whole numbers are exact, so every result is the exact one rounded once: a row, a column or a tail that is left out shows.
    Few rows, tiles of 64, 128 and 256 with and without splits, in y, dx and dw, all in odd sizes."""
    g = gen(58)
    x, w, b, r, dy = (torch.randint(-n, n + 1, s, generator=g, device="cuda").to(dtype) for n, s in ((3, (M, K)), (2, (N, K)), (3, (N,)), (3, (M, N)), (2, (M, N))))
    leaves = [t.requires_grad_() for t in (x, w, b, r)]
    y = ops.linear(x, w, bias=b, residual=r, activation=act)
    x64, w64, b64, r64, dy64 = (t.detach().double() for t in (x, w, b, r, dy))
    z = x64 @ w64.t() + b64
    assert z.abs().max() < 2 ** 20
    dz = dy64 if act == "none" else torch.where(z > 0, dy64, 0.0)
    want = ((z if act == "none" else z.clamp_min(0)) + r64, dz @ w64, dz.t() @ x64, dz.sum(0), dy64)
    for name, got, exact in zip(("y", "dx", "dw", "db", "dr"), (y.detach(), *torch.autograd.grad(y, leaves, dy)), want):
        assert torch.equal(got, exact.float().to(dtype)), name


@pytest.mark.parametrize("out", [F32, BF16])
@pytest.mark.parametrize("M,K,N", [(5, 16, 3), (64, 2048, 96), (65, 130, 70), (300, 1003, 260), (2050, 1040, 2050)])
def test_linear_on_8_bits_loses_nothing_of_whole_numbers(ops, M, K, N, out):
    g = gen(59)
    x, w = (torch.randint(-n, n + 1, s, generator=g, device="cuda").float() for n, s in ((3, (M, K)), (2, (N, K))))
    xs, ws = (2.0 ** torch.randint(-2, 3, (n,), generator=g, device="cuda").float() for n in (M, N))
    y = ops.linear_fp8(x.to(E4M3), xs, w.to(E4M3), ws, out_dtype=out)
    assert torch.equal(y, ((x.double() @ w.double().t()) * xs.double()[:, None] * ws.double()).float().to(out))


@pytest.mark.parametrize("M,K,N,dtype,act", [(4090, 600, 2045, BF16, "silu"), (4090, 600, 2045, BF16, "none"), (4090, 520, 4090, F16, "gelu"), (601, 1030, 2050, BF16, "tanh")])
def test_linear_errors_in_16_bits_are_those_of_their_roundings(ops, M, K, N, dtype, act):
    """By the norm, where roundings of independent values add up as their squares: one of each dz (none without an activation) and one of each result, each at most
    half a step u, make at most sqrt(2) u and u of a result whose terms are as independent; 1.6 u and 1.1 u leave room for the sums in float32 and for
    chance (3 % over some 10^6 values). A single row left out of M = 4090 would be 1.6 % of dw, 4 u in bfloat16."""
    g = gen(60)
    x, w, dy = randn(g, M, K, dtype=dtype).requires_grad_(), randn(g, N, K, dtype=dtype, scale=K ** -0.5).requires_grad_(), randn(g, M, N, dtype=dtype)
    y = ops.linear(x, w, activation=act)
    x64, w64 = (t.detach().double().requires_grad_() for t in (x, w))
    y64 = R.linear(x64, w64, act=act)
    u = R.half_step(dtype)
    off = lambda a, b: ((a.double() - b).norm() / b.norm()).item()                    # noqa: E731
    assert off(y.detach(), y64.detach()) <= 1.1 * u
    for name, a, b in zip(("dx", "dw"), torch.autograd.grad(y, (x, w), dy), torch.autograd.grad(y64, (x64, w64), dy.double())):
        assert off(a, b) <= (1.1 if act == "none" else 1.6) * u, name


def test_linear_wide_tiles(ops):
    """Enough tiles of 128 that the large tile is taken, in whole and in odd sizes."""
    g = gen(33)
    for M, K, N, dtype in ((2048, 256, 2048, BF16), (2100, 200, 2050, F16), (2048, 96, 2048, F32)):
        check_linear(ops, g, M, K, N, dtype, "none", True, False)


def test_linear_wide_outputs_whose_contraction_is_split(ops):
    """Two splits of float32 tiles of 128 (forward), and of tiles of 64 (gradients), in odd sizes, joined with the whole epilogue."""
    g = gen(41)
    check_linear(ops, g, 2100, 1030, 2050, F32, "gelu")
    check_linear(ops, g, 2040, 1030, 2045, F32, "gelu")
    check_linear(ops, g, 1203, 1101, 1003, BF16, "tanh")


@pytest.mark.parametrize("M,K,N,dtype", [(4090, 300, 2045, F32), (4090, 600, 2045, BF16), (4090, 520, 4090, F16)])
def test_linear_tiles_of_every_size(ops, M, K, N, dtype):
    """The tiles of 128 (float32, 16 bits) and of 256 in odd sizes, with the whole epilogue."""
    check_linear(ops, gen(48), M, K, N, dtype, "silu")


@pytest.mark.parametrize("rows", [64, 60001])
def test_silu_and_its_slope_keep_their_bits_in_float32(ops, rows):
    """z passes through unchanged (a width of 1, weight 1). e^-z is off by 2 half steps (one step of the exponential) and its correction's rounding, 1 + e^-z
    by one more, the reciprocal by 2, the product by 1: 7; the slope s (1 + z (1 - s)) twice that of the size of its two terms. Down to -87: the
    sigmoid is subnormal below."""
    g = gen(54)
    z = torch.cat([torch.linspace(-87, 87, rows // 2, device="cuda"), randn(g, rows - rows // 2, scale=4.0).clamp(-87, 87)])[:, None].requires_grad_()
    y = ops.linear(z, torch.ones(1, 1, device="cuda"), activation="silu")
    z64 = z.detach().double()
    s64 = torch.sigmoid(z64)
    assert ((y.double() - z64 * s64).abs() <= 8 * R.U32 * (z64 * s64).abs()).all()
    slope = torch.autograd.grad(y, z, torch.ones_like(y))[0].double()
    assert ((slope - s64 * (1 + z64 * (1 - s64))).abs() <= 16 * R.U32 * (s64 + (z64 * s64 * (1 - s64)).abs())).all()
    far = torch.tensor([[100.0], [1e30], [INF], [-100.0], [-1e30], [math.nan]], device="cuda", requires_grad=True)
    y = ops.linear(far, torch.ones(1, 1, device="cuda"), activation="silu")
    assert torch.equal(y[:3], far[:3]) and (y[3:5].abs() < 1e-36).all() and torch.isnan(y[5])
    slope = torch.autograd.grad(y, far, torch.ones_like(y))[0]
    assert (slope[:2] == 1).all() and (slope[3:5].abs() < 1e-36).all()


def in_order(x, w, order):
    """x w^T in float32, one fused multiply-add for each k of `order` (a product of two float32 values is exact in 64 bits)."""
    acc = torch.zeros(x.shape[0], w.shape[0], device="cuda")
    for k in order:
        acc = (acc.double() + x.double()[:, k, None] * w.double()[None, :, k]).float()
    return acc


@pytest.mark.parametrize("M,K,N", [(200, 30, 70), (200, 125, 70), (200, 128, 70), (32768, 252, 64)])
def test_linear_float32_adds_up_in_the_stated_order(ops, M, K, N):
    """Whole steps of 32 values by k = 16 s + 4 g + r (g innermost), what is left of the row in ascending order: a relu's gate at z = 0 hangs on it."""
    g = gen(50)
    x, w = randn(g, M, K), randn(g, N, K, scale=K ** -0.5)
    whole = K // 32 * 32
    order = [s + 4 * q + r for s in range(0, whole, 16) for r in range(4) for q in range(4)] + list(range(whole, K))
    want = in_order(x[:96], w, order)
    y = ops.linear(x, w)
    assert torch.equal(y[:96], want)
    leaf = x.detach().requires_grad_()
    z = ops.linear(leaf, w, activation="relu")
    assert torch.equal(z[:96], want.clamp_min(0))
    dx = torch.autograd.grad(z, leaf, torch.ones_like(z))[0][:96]
    R.close(dx, (want > 0).double() @ w.double(), 0, N + 2, "dx", w.abs().sum(0).max().item())


def test_linear_takes_rows_of_any_stride_and_no_rows(ops):
    g = gen(34)
    wide = randn(g, 90, 301, dtype=BF16)
    check_linear(ops, g, 90, 77, 50, BF16, "silu", x=wide[:, 3:80])
    check_linear(ops, g, 90, 77, 50, BF16, "silu", x=wide[:1, 3:80].expand(90, -1))
    check_linear(ops, g, 0, 16, 24, F32, "silu")
    x = randn(g, 2, 3, 4, 16)
    w = randn(g, 8, 16)
    y = ops.linear(x.permute(1, 0, 2, 3), w)
    assert y.shape == (3, 2, 4, 8)
    R.close(y, (x.double() @ w.double().t()).permute(1, 0, 2, 3), 1, 24, "y", 40.0)
    one = ops.linear(x[0, 0, 0], w, residual=torch.ones(8, device="cuda"))
    assert one.shape == (8,)


def test_linear_gradients_that_are_not_wanted(ops):
    g = gen(35)
    x, w, b = randn(g, 70, 32), randn(g, 40, 32), randn(g, 40)
    for i in range(3):
        leaves = [t.detach().requires_grad_(j == i) for j, t in enumerate((x, w, b))]
        all_three = [t.detach().requires_grad_() for t in (x, w, b)]
        dy = randn(g, 70, 40)
        one = torch.autograd.grad(ops.linear(*leaves, activation="tanh"), leaves[i], dy)[0]
        assert torch.equal(one, torch.autograd.grad(ops.linear(*all_three, activation="tanh"), all_three, dy)[i])


@pytest.mark.parametrize("out", [F32, BF16, F16])
@pytest.mark.parametrize("M,K,N", [(1, 1, 1), (5, 40, 33), (16, 256, 512), (64, 2048, 96), (65, 130, 70), (300, 512, 260), (2050, 128, 2050), (20, 37, 45), (70, 333, 129)])
def test_linear_on_8_bits(ops, M, K, N, out):
    g = gen(36)
    xq, xs = ops.quantize_rows_fp8(randn(g, M, K))
    wq, ws = ops.quantize_rows_fp8(randn(g, N, K, scale=K ** -0.5))
    b, r = randn(g, N, dtype=out), randn(g, M, N, dtype=out)
    y = ops.linear_fp8(xq, xs, wq, ws, bias=b, residual=r, activation="silu", out_dtype=out)
    x64, w64 = xq.float().double() * xs.double()[:, None], wq.float().double() * ws.double()[:, None]
    size = (x64.abs() @ w64.abs().t()).max().item() + 4
    # (a product of two e4m3 values is exact in float32)
    R.close(y, R.linear(x64, w64, b.double(), r.double(), "silu"), 1, K + 8, "y", size)


def test_every_8_bit_value_is_read_for_what_it_is(ops):
    codes = torch.arange(256, device="cuda", dtype=torch.uint8).view(E4M3)
    fine = codes[~torch.isnan(codes.float())]
    n = len(fine)
    eye, one = torch.eye(n, device="cuda").to(E4M3), torch.ones(n, device="cuda")
    for m in (n, 64, 3):
        assert torch.equal(ops.linear_fp8(fine.expand(m, n).contiguous(), one[:m], eye, one, out_dtype=F32), fine.float().expand(m, n))
    assert torch.isnan(ops.linear_fp8(codes[127:128, None], one[:1], codes[56:57, None], one[:1], out_dtype=F32)).all()


# ------------------------------------------------------------------------------------------------------------------ used together
class Block:
    """One residual memory block, as an agent would have it."""

    def __init__(self, g, D, H, K, V, dtype):
        self.H, self.K, self.V = H, K, V
        self.p = [(1 + randn(g, D, scale=0.1)).to(dtype), randn(g, H * (2 * K + V), D, dtype=dtype, scale=D ** -0.5), randn(g, D, H * V, dtype=dtype, scale=(H * V) ** -0.5),
                  randn(g, 2 * H, D, scale=D ** -0.5)]

    def __call__(self, ops, x, residual, p=None, state=None):
        nw, wi, wo, wg = p or self.p
        H, K, V = self.H, self.K, self.V
        y, s = ops.rms_norm(x, nw, residual=residual)
        q, k, v = ops.linear(y, wi, activation="silu").split([H * K, H * K, H * V], -1)
        gates = ops.linear(y.float(), wg)
        decay, beta = -torch.nn.functional.softplus(gates[..., :H]) * 0.1, torch.sigmoid(gates[..., H:])
        k = torch.nn.functional.normalize(k.unflatten(-1, (H, K)).float(), dim=-1).to(x.dtype)
        q, v = q.unflatten(-1, (H, K)), v.unflatten(-1, (H, V))
        if state is None:
            o, state = ops.gated_delta_rule(q, k, v, decay, beta)
        else:
            o = ops.gated_delta_step(q, k, v, decay, beta, state)
        return ops.linear(o.flatten(-2), wo, residual=s), state


class Plain:
    """The same operators in 64 bits."""
    @staticmethod
    def rms_norm(x, w, residual):
        return R.rms_norm(x, w, residual)

    @staticmethod
    def linear(x, w, bias=None, residual=None, activation="none"):
        return R.linear(x, w.double(), bias, residual, activation)

    gated_delta_rule = staticmethod(R.delta_rule)


def test_block_of_all_of_them(ops):
    g = gen(40)
    block = Block(g, 48, 2, 16, 20, F32)
    x, r = randn(g, 3, 100, 48), randn(g, 3, 100, 48)
    leaves = [t.detach().requires_grad_() for t in (x, r, *block.p)]
    y, S = block(ops, leaves[0], leaves[1], leaves[2:])

    class Wide(Plain):
        pass
    wide = [t.detach().double().requires_grad_() for t in leaves]
    torch_float = torch.Tensor.float
    try:
        torch.Tensor.float = torch.Tensor.double            # the block's own casts, in 64 bits
        y64, S64 = block(Wide, wide[0], wide[1], wide[2:])
    finally:
        torch.Tensor.float = torch_float
    # five operators one behind the other, each within (K + V + 128 + ..) half steps of float32
    n = 5 * delta_terms(16, 20, 100)
    R.close(y.detach(), y64.detach(), 0, n, "y")
    R.close(S.detach(), S64.detach(), 0, n, "state")
    dy = randn(g, 3, 100, 48)
    for i, (a, b) in enumerate(zip(torch.autograd.grad(y, leaves, dy), torch.autograd.grad(y64, wide, dy.double()))):
        R.close(a, b, 0, 8 * n, "gradient %d" % i)


def test_block_acts_step_by_step_in_8_bits(ops):
    """Acting: one step at a time with 8-bit projections, against the same steps with the float ones on the values the 8 bits stand for."""
    g = gen(41)
    D, H, K, V, B = 64, 2, 16, 16, 9
    w = randn(g, H * (2 * K + V), D, scale=D ** -0.5)
    nw = 1 + randn(g, D, scale=0.1)
    wq, ws = ops.quantize_rows_fp8(w)
    state, state64 = torch.zeros(B, H, K, V, device="cuda"), torch.zeros(B, H, K, V, device="cuda", dtype=torch.float64)
    r = torch.zeros(B, D, device="cuda")
    for t in range(4):
        q8, sc, r = ops.rms_norm_fp8(randn(g, B, D), nw, residual=r)
        p = ops.linear_fp8(q8, sc, wq, ws, activation="tanh", out_dtype=F32)
        p64 = torch.tanh((q8.float().double() * sc.double()[:, None]) @ (wq.float().double() * ws.double()[:, None]).t())
        gate, beta = -0.1 * rand(g, B, H), rand(g, B, H)
        split = lambda a: (a[:, :H * K].unflatten(-1, (H, K)), a[:, H * K:2 * H * K].unflatten(-1, (H, K)) * 0.3, a[:, 2 * H * K:].unflatten(-1, (H, V)))   # noqa: E731
        o = ops.gated_delta_step(*split(p), gate, beta, state)
        o64, state64 = R.delta_rule(*(a[:, None] for a in split(p64)), gate.double()[:, None], beta.double()[:, None], state64)
        R.close(o, o64[:, 0], 0, 500, "out")
    R.close(state, state64, 0, 500, "state")


def test_captured_training_pass_replays(ops):
    """Forward and backward of a block in a HIP graph, replayed on new inputs with eager work between the replays; two graphs side by side."""
    g = gen(42)
    block = Block(g, 64, 2, 32, 32, F32)
    made = []
    for k in range(2):
        leaves = [t.detach().clone().requires_grad_() for t in (randn(g, 4, 70, 64), randn(g, 4, 70, 64), *block.p)]
        dy = randn(g, 4, 70, 64)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for _ in range(2):
                y, S = block(ops, leaves[0], leaves[1], leaves[2:])
                torch.autograd.grad([y], leaves, [dy])
            del y, S
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y, S = block(ops, leaves[0], leaves[1], leaves[2:])
            grads = torch.autograd.grad([y], leaves, [dy])
        made.append((graph, leaves, dy, y.detach(), S.detach(), grads))
        del y, S
    for turn in range(3):
        for graph, leaves, dy, *_ in made:
            with torch.no_grad():
                leaves[0].copy_(randn(g, 4, 70, 64))
            graph.replay()
        torch.cuda.synchronize()
        for graph, leaves, dy, y, S, grads in made:
            fresh = [t.detach().clone().requires_grad_() for t in leaves]
            y2, S2 = block(ops, fresh[0], fresh[1], fresh[2:])
            assert torch.equal(y, y2) and torch.equal(S, S2)
            for a, b in zip(grads, torch.autograd.grad([y2], fresh, [dy])):
                assert torch.equal(a, b)


def test_a_step_is_seen_by_graphs_that_hold_the_state(ops):
    """The step changes the state in place: as after any in-place change, a graph that saved it refuses its backward pass."""
    g = gen(47)
    args = [x[:, 0].contiguous() for x in delta_inputs(g, 4, 1, 2, 2, 32, 32, F32)]
    state, w = randn(g, 4, 2, 32, 32), randn(g, 4, 2, 32, 32).requires_grad_()
    loss = (state * w).sum()
    with torch.no_grad():
        ops.gated_delta_step(*args, state)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    with torch.inference_mode():
        ops.gated_delta_step(*args, state.clone())


def test_captured_step_replays(ops):
    g = gen(43)
    args = [x[:, 0].contiguous() for x in delta_inputs(g, 8, 1, 2, 2, 32, 32, F32)]
    state = randn(g, 8, 2, 32, 32)
    start = state.clone()
    ops.gated_delta_step(*args, state)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = ops.gated_delta_step(*args, state)
    state.copy_(start)
    mine = start.clone()
    for _ in range(3):
        graph.replay()
        want = ops.gated_delta_step(*args, mine)
        torch.cuda.synchronize()
        assert torch.equal(o, want) and torch.equal(state, mine)


def test_on_another_stream_and_twice_at_once(ops):
    g = gen(44)
    inputs = [delta_inputs(g, 2, 200, 2, 2, 32, 32, BF16) for _ in range(2)]
    want = [ops.gated_delta_rule(*x) for x in inputs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [None, None]
    for _ in range(3):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i] = ops.gated_delta_rule(*inputs[i])
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_the_same_call_gives_the_same_bits(ops):
    """Sums are split by the sizes alone and added in a fixed order."""
    g = gen(45)
    x, w = randn(g, 5000, 252).requires_grad_(), randn(g, 64, 252).requires_grad_()
    dy = randn(g, 5000, 64)
    first = torch.autograd.grad(ops.linear(x, w, activation="silu"), [x, w], dy)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, torch.autograd.grad(ops.linear(x, w, activation="silu"), [x, w], dy)))


def test_gradients_twice_from_one_graph_and_never_of_gradients(ops):
    """retain_graph gives the same bits again; a graph of the gradients themselves is refused, not silently wrong."""
    g = gen(46)
    block = Block(g, 32, 2, 16, 16, BF16)
    leaves = [t.detach().requires_grad_() for t in (randn(g, 2, 70, 32, dtype=BF16), randn(g, 2, 70, 32, dtype=BF16), *block.p)]
    y, _ = block(ops, leaves[0], leaves[1], leaves[2:])
    dy = randn(g, 2, 70, 32, dtype=BF16)
    first = torch.autograd.grad(y, leaves, dy, retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(first, torch.autograd.grad(y, leaves, dy)))
    x, w = randn(g, 4, 8).requires_grad_(), randn(g, 8).requires_grad_()
    for out in (ops.rms_norm(x, w), ops.linear(x, randn(g, 5, 8)), ops.gated_delta_rule(*[t.requires_grad_() for t in delta_inputs(g, 1, 3, 1, 1, 4, 4, F32)])[0]):
        with pytest.raises(RuntimeError, match="differentiated again"):
            torch.autograd.grad(out.sum(), x if out.shape != (1, 3, 1, 4) else out, create_graph=True) if out.shape != (1, 3, 1, 4) else out.sum().backward(create_graph=True)


def test_changed_inputs_are_noticed(ops):
    """What the backward pass reads and somebody changed in between is an error, as everywhere in torch."""
    g = gen(47)
    for dtype in (F32, BF16):
        x, w, r = randn(g, 4, 8, dtype=dtype).requires_grad_(), randn(g, 8, dtype=dtype).requires_grad_(), randn(g, 4, 8, dtype=dtype)
        y, s = ops.rms_norm(x, w, residual=r)
        (s.detach() if dtype == F32 else r).add_(1)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.sum().backward()


def test_a_compiled_program_calls_the_kernels(ops):
    """torch.compile leaves the calls to Python: same results, new inputs seen, gradients too."""
    torch._dynamo.reset()
    g = gen(52)
    w, n = randn(g, 24, 16), randn(g, 16)

    def f(x, r):
        y, s = ops.rms_norm(x * 2, n, residual=r)
        return ops.linear(y, w, activation="silu") + s.sum(-1, keepdim=True)

    c = torch.compile(f, backend="eager")
    for _ in range(3):
        x, r = randn(g, 70, 16), randn(g, 70, 16)
        with torch.no_grad():
            assert torch.equal(c(x, r), f(x, r))
        a, b = x.clone().requires_grad_(), x.clone().requires_grad_()
        assert torch.equal(torch.autograd.grad(c(a, r).sum(), a)[0], torch.autograd.grad(f(b, r).sum(), b)[0])
    torch._dynamo.reset()


def test_tangents_in_the_gradients_are_refused(ops):
    from torch.autograd import forward_ad
    x, w = torch.ones(70, 8, device="cuda", requires_grad=True), torch.ones(5, 8, device="cuda")
    y = ops.linear(x, w)
    with forward_ad.dual_level():
        dy = forward_ad.make_dual(torch.ones_like(y), torch.ones_like(y))
        with pytest.raises(RuntimeError, match="forward-mode"):
            torch.autograd.grad(y, x, dy)


def test_tensors_on_two_devices_are_refused(ops):
    x, w = torch.zeros(3, 8, device="cuda"), torch.zeros(8)
    with pytest.raises(ValueError, match="in one call"):
        ops.rms_norm(x, w)
    with pytest.raises(ValueError, match="in one call"):
        ops.linear(x, torch.zeros(5, 8))
