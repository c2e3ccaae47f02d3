"""CPU-only checks of offpolicy_amd.ops: what the entry points refuse, and the C entries' own checks of their arguments."""
import ctypes as C

import pytest
import torch

from offpolicy_amd import _lib, ops

F32, BF16, E4M3 = torch.float32, torch.bfloat16, torch.float8_e4m3fn


def delta_args(B=2, T=5, Hk=2, H=4, K=8, V=6, dtype=F32, step=False):
    lead = (B,) if step else (B, T)
    return [torch.zeros(*lead, Hk, K, dtype=dtype), torch.zeros(*lead, Hk, K, dtype=dtype), torch.zeros(*lead, H, V, dtype=dtype), torch.zeros(*lead, H), torch.zeros(*lead, H)]


def test_struct_sizes_match_the_library():
    for name, cls in _lib.OPERATOR_MIRRORS.items():
        assert _lib.lib.ope_abi_sizeof(name.encode()) == C.sizeof(cls), name
    from offpolicy_amd.ops import memory, norms, projection
    for mod, cls in ((norms, _lib.NormCfg), (memory, _lib.DeltaCfg), (projection, _lib.LinearCfg)):
        assert mod._CFG.size == C.sizeof(cls)


@pytest.mark.parametrize("change, error", [
    (dict(H=3), ValueError),                                     # 3 value heads on 2 query / key heads
    (dict(K=129), ValueError), (dict(V=1025), ValueError),
    (dict(dtype=torch.float64), TypeError), (dict(dtype=torch.int32), TypeError),
])
def test_delta_rule_refuses_sizes_and_types(change, error):
    for step in (False, True):
        a = delta_args(step=step, **change)
        with pytest.raises(error):
            if step:
                ops.gated_delta_step(*a, torch.zeros(a[2].shape[0], a[2].shape[1], a[0].shape[-1], a[2].shape[-1]))
            else:
                ops.gated_delta_rule(*a)


def test_delta_rule_refuses_what_does_not_fit_together():
    q, k, v, g, b = delta_args()
    bad = [
        (q, k[:, :4], v, g, b), (q, k, v[:, :4], g, b), (q, k, v, g[:, :4], b), (q, k, v, g, b[..., :3]), (q, k.to(BF16), v, g, b), (q, k, v.to(BF16), g, b),
        (q, k, v, g.to(BF16), b), (q, k, v, g, b.double()), (q[0], k[0], v[0], g[0], b[0]), (q, k, v, g, 1.0),
    ]
    for a in bad:
        with pytest.raises((ValueError, TypeError)):
            ops.gated_delta_rule(*a)
    for more in (dict(initial_state=torch.zeros(2, 4, 6, 8)), dict(initial_state=torch.zeros(2, 4, 8, 6, dtype=BF16)), dict(lengths=torch.zeros(3, dtype=torch.int32)),
                 dict(lengths=torch.zeros(2, dtype=torch.int64)), dict(lengths=[5, 5])):
        with pytest.raises((ValueError, TypeError)):
            ops.gated_delta_rule(q, k, v, g, b, **more)


def test_delta_step_refuses_states_it_cannot_update():
    a = delta_args(step=True)
    for state in (torch.zeros(2, 4, 6, 8), torch.zeros(2, 4, 8, 6, dtype=BF16), torch.zeros(2, 4, 6, 8).transpose(-1, -2)):
        with pytest.raises((ValueError, TypeError)):
            ops.gated_delta_step(*a, state)
    a[2].requires_grad_()
    with pytest.raises(ValueError, match="no gradients"):
        ops.gated_delta_step(*a, torch.zeros(2, 4, 8, 6))


def test_norm_refuses():
    x, w = torch.zeros(3, 8), torch.zeros(8)
    for a, more in (((x, w[:7]), {}), ((x, w.to(BF16)), {}), ((x, w), dict(residual=torch.zeros(3, 7))), ((x, w), dict(residual=x.to(BF16))), ((x, w), dict(eps=-1.0)),
                    ((x, w), dict(eps=float("nan"))), ((x.double(), w.double()), {}), ((torch.zeros(3, 0), torch.zeros(0)), {}), ((torch.zeros(()), w), {})):
        for f in (ops.rms_norm, ops.rms_norm_fp8):
            with pytest.raises((ValueError, TypeError)):
                f(*a, **more)
    with pytest.raises(ValueError, match="no gradients"):
        ops.rms_norm_fp8(x.clone().requires_grad_(), w)
    with pytest.raises(TypeError):
        ops.quantize_rows_fp8(x.double())


def test_linear_refuses():
    x, w = torch.zeros(3, 8), torch.zeros(5, 8)
    for a, more in (((x, w[:, :7]), {}), ((x, w[0]), {}), ((x, w.to(BF16)), {}), ((x, w), dict(bias=torch.zeros(8))), ((x, w), dict(bias=torch.zeros(5, dtype=BF16))),
                    ((x, w), dict(residual=torch.zeros(3, 8))), ((x, w), dict(activation="swish")), ((x.double(), w.double()), {}), ((x, torch.zeros(0, 8)), {})):
        with pytest.raises((ValueError, TypeError)):
            ops.linear(*a, **more)
    x8, w8, xs, ws = x.to(E4M3), w.to(E4M3), torch.ones(3), torch.ones(5)
    for a, more in (((x, xs, w8, ws), {}), ((x8, xs, w, ws), {}), ((x8, xs[:2], w8, ws), {}), ((x8, xs, w8, ws[:4]), {}), ((x8, xs.to(BF16), w8, ws), {}),
                    ((x8, xs, w8, ws), dict(out_dtype=torch.float64)), ((x8, xs, w8, ws), dict(bias=torch.zeros(5))), ((x8, xs, w8, ws), dict(activation="exp"))):
        with pytest.raises((ValueError, TypeError)):
            ops.linear_fp8(*a, **more)


def test_acting_forms_refuse_arguments_that_want_gradients():
    x8, w8, xs, ws = torch.zeros(3, 8).to(E4M3), torch.zeros(5, 8).to(E4M3), torch.ones(3), torch.ones(5)
    for i in range(4):
        a = [t.clone().requires_grad_(i == j) for j, t in enumerate((x8, xs, w8, ws))]
        with pytest.raises(ValueError, match="no gradients"):
            ops.linear_fp8(*a)
    with pytest.raises(ValueError, match="no gradients"):
        ops.quantize_rows_fp8(torch.zeros(3, 8, requires_grad=True))


def entries():
    """Every entry point as a function of one float32 tensor [3, 8] that it reads, on the CPU: a call that is not refused first ends with "GPU only"."""
    w, xs, ws = torch.zeros(5, 8), torch.ones(3), torch.ones(5)
    d, s = delta_args(B=1, T=3, Hk=1, H=1, K=8, V=8), delta_args(B=3, Hk=1, H=1, K=8, V=8, step=True)
    return {
        "rms_norm": lambda x: ops.rms_norm(x, w[0]), "rms_norm, residual": lambda x: ops.rms_norm(w[:3], w[0], residual=x), "rms_norm_fp8": lambda x: ops.rms_norm_fp8(x, w[0]),
        "quantize_rows_fp8": lambda x: ops.quantize_rows_fp8(x), "linear": lambda x: ops.linear(x, w), "linear, weight": lambda x: ops.linear(w, x),
        "linear, residual": lambda x: ops.linear(w[:3], torch.zeros(8, 8), residual=x),
        "linear_fp8, residual": lambda x: ops.linear_fp8(w[:3].to(E4M3), xs, torch.zeros(8, 8).to(E4M3), torch.ones(8), residual=x, out_dtype=F32),
        "linear_fp8, scale": lambda x: ops.linear_fp8(w[:3].to(E4M3), x[:, 0], w.to(E4M3), ws),
        "gated_delta_rule": lambda x: ops.gated_delta_rule(d[0], d[1], x[None, :, None], d[3], d[4]),
        "gated_delta_rule, state": lambda x: ops.gated_delta_rule(*d, initial_state=x[None, None, :1].expand(1, 1, 8, 8)),
        "gated_delta_step": lambda x: ops.gated_delta_step(x[:, None], s[1], s[2], s[3], s[4], torch.zeros(3, 1, 8, 8)),
    }


@pytest.mark.parametrize("name", list(entries()))
def test_what_the_tape_does_not_see_is_refused(name):
    from torch.autograd import forward_ad
    from torch.fx.experimental.proxy_tensor import make_fx
    f, x = entries()[name], torch.zeros(3, 8)
    first = lambda y: y[0] if isinstance(y, tuple) else y         # noqa: E731
    with pytest.raises(ValueError, match="GPU only"):              # an ordinary call passes these checks
        f(x)
    with torch.no_grad(), forward_ad.dual_level():
        with pytest.raises(ValueError, match="GPU only"):          # no tangent, no harm
            f(x)
    with forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="forward-mode"):
            f(forward_ad.make_dual(x, torch.ones_like(x)))
    with pytest.raises(RuntimeError, match="jit.trace"), torch.no_grad():
        torch.jit.trace(lambda x: first(f(x)), (x,), check_trace=False)
    for pre in (False, True):
        with pytest.raises(RuntimeError, match="make_fx"):
            make_fx(lambda x: first(f(x)), pre_dispatch=pre)(x)
    for transform in (lambda: torch.func.vmap(f)(torch.zeros(2, 3, 8)), lambda: torch.func.grad(lambda x: first(f(x)).sum())(x),
                      lambda: torch.func.jvp(f, (x,), (x,)), lambda: torch.func.functionalize(f)(x)):
        with pytest.raises(RuntimeError, match="torch.func"):
            transform()


def test_a_tangent_in_the_gradients_is_refused():
    """Forward over reverse: the backward pass would drop it."""
    from torch.autograd import forward_ad
    from offpolicy_amd.ops import _common
    seen = []
    backward = _common.once(lambda ctx, *grads: seen.append(grads)).__func__
    x = torch.ones(3)
    with torch.no_grad(), forward_ad.dual_level():
        backward(None, x, None)
        with pytest.raises(RuntimeError, match="forward-mode"):
            backward(None, None, forward_ad.make_dual(x, x))
    assert len(seen) == 1


def test_there_is_no_cpu_path():
    with pytest.raises(ValueError, match="GPU only"):
        ops.gated_delta_rule(*delta_args())
    with pytest.raises(ValueError, match="GPU only"):
        ops.gated_delta_step(*delta_args(step=True), torch.zeros(2, 4, 8, 6))
    with pytest.raises(ValueError, match="GPU only"):
        ops.rms_norm(torch.zeros(3, 8), torch.zeros(8).requires_grad_())
    with pytest.raises(ValueError, match="GPU only"):
        ops.linear(torch.zeros(3, 8), torch.zeros(5, 8))


def test_c_entries_check_before_they_launch():
    lib, EINVAL, ENOSPC = _lib.lib, -1, -3
    norm = lambda **k: C.byref(_lib.NormCfg(**{**dict(rows=2, x_stride=8, width=8, eps=1e-6), **k}))                  # noqa: E731
    some = C.c_void_p(16)                                     # never dereferenced: every call below is refused first
    assert lib.ope_rms_norm(None, *[some] * 8) == EINVAL
    for k in (dict(width=0), dict(rows=-1), dict(dtype=3), dict(dtype=7), dict(out_dtype=1), dict(eps=-1.0), dict(eps=float("nan")), dict(x_stride=-8), dict(width=(1 << 20) + 1), dict(rows=1 << 31), dict(rows=1 << 28), dict(rows=1 << 23, width=8192)):
        assert lib.ope_rms_norm(norm(**k), *[some] * 8) == EINVAL, k
    assert lib.ope_rms_norm(norm(), None, *[some] * 7) == EINVAL
    assert lib.ope_rms_norm(norm(out_dtype=3), some, some, some, some, None, some, some, some) == EINVAL      # 8 bits without a place for the scales
    assert lib.ope_rms_norm(norm(rows=0), *[None] * 8) == 0
    assert lib.ope_quantize_rows(norm(), some, some, None, some) == EINVAL
    need = lib.ope_rms_norm_backward_workspace_bytes(norm())
    assert need > 0 and lib.ope_rms_norm_backward_workspace_bytes(norm(width=0)) == EINVAL
    assert lib.ope_rms_norm_backward(norm(), *[some] * 9, need - 1, some) == ENOSPC
    assert lib.ope_rms_norm_backward(norm(), None, *[some] * 8, need, some) == EINVAL

    sizes = dict(batch=2, seq_len=5, n_heads=4, n_qk_heads=2, key_dim=8, value_dim=6)
    delta = lambda **k: C.byref(_lib.DeltaCfg(**{**sizes, **k}))                                                      # noqa: E731
    for k in (dict(batch=-1), dict(seq_len=-1), dict(n_heads=0), dict(n_qk_heads=0), dict(n_qk_heads=3), dict(key_dim=0), dict(key_dim=129), dict(value_dim=0),
              dict(value_dim=1025), dict(dtype=3), dict(batch=1 << 20, n_heads=1 << 12, seq_len=1 << 20), dict(batch=1 << 30, n_heads=1 << 30),
              dict(batch=1 << 22), dict(batch=1 << 14, seq_len=1 << 14, n_heads=4, key_dim=128)):
        assert lib.ope_delta_saved_bytes(delta(**k)) == EINVAL and lib.ope_delta_workspace_bytes(delta(**k), 1) == EINVAL, k
        assert lib.ope_delta_forward(delta(**k), *[some] * 10, 1 << 40, some, 1 << 40, some) == EINVAL, k
        assert lib.ope_delta_step(delta(**k), *[some] * 8) == EINVAL, k
    saved, ws, wb = lib.ope_delta_saved_bytes(delta()), lib.ope_delta_workspace_bytes(delta(), 0), lib.ope_delta_workspace_bytes(delta(), 1)
    assert min(saved, ws, wb) > 0
    assert lib.ope_delta_forward(delta(), *[some] * 10, saved - 1, some, ws, some) == ENOSPC
    assert lib.ope_delta_forward(delta(), *[some] * 10, saved, some, ws - 1, some) == ENOSPC
    assert lib.ope_delta_forward(delta(), None, *[some] * 9, saved, some, ws, some) == EINVAL
    assert lib.ope_delta_backward(delta(), *[some] * 7, saved, *[some] * 9, wb - 1, some) == ENOSPC
    assert lib.ope_delta_backward(delta(), *[some] * 7, saved - 1, *[some] * 9, wb, some) == ENOSPC
    assert lib.ope_delta_backward(delta(), *[some] * 7, saved, None, *[some] * 8, wb, some) == EINVAL
    assert lib.ope_delta_step(delta(), *[some] * 5, None, some, some) == EINVAL
    assert lib.ope_delta_forward(delta(batch=0), *[None] * 10, 0, None, 0, None) == 0

    lin = lambda **k: C.byref(_lib.LinearCfg(**{**dict(rows=100, x_stride=8, in_width=8, out_width=5), **k}))          # noqa: E731
    for k in (dict(rows=-1), dict(in_width=0), dict(out_width=0), dict(in_width=(1 << 20) + 1), dict(dtype=1), dict(dtype=3, out_dtype=3), dict(dtype=9), dict(activation=5),
              dict(activation=-1), dict(x_stride=-1), dict(rows=1 << 31), dict(rows=1 << 30, out_width=1 << 14), dict(in_width=1 << 20, out_width=1 << 13)):
        assert lib.ope_linear_workspace_bytes(lin(**k)) == EINVAL and lib.ope_linear(lin(**k), *[some] * 9, 1 << 40, some) == EINVAL, k
    assert lib.ope_linear(lin(), some, some, some, None, *[some] * 5, 1 << 40, some) == EINVAL                  # scales are for 8-bit operands
    assert lib.ope_linear(lin(dtype=3), some, some, some, None, *[some] * 5, 1 << 40, some) == EINVAL
    assert lib.ope_linear_backward_workspace_bytes(lin(dtype=3)) == EINVAL
    need = lib.ope_linear_backward_workspace_bytes(lin(activation=1))
    assert lib.ope_linear_backward(lin(activation=1), *[some] * 8, need - 1, some) == ENOSPC
    assert lib.ope_linear_backward(lin(activation=1), some, None, *[some] * 6, need, some) == EINVAL            # the activation's slope needs z
    assert lib.ope_linear_workspace_bytes(lin(rows=0)) == 0 and lib.ope_linear_backward_workspace_bytes(lin(rows=0, activation=1)) >= 0
    assert lib.ope_linear(lin(rows=0), *[None] * 9, 0, None) == 0
    split = dict(rows=512, in_width=4096, out_width=64)
    assert lib.ope_linear_workspace_bytes(lin(**split)) > 0
    assert lib.ope_linear(lin(**split), some, some, None, None, *[some] * 4, None, 0, some) == ENOSPC
