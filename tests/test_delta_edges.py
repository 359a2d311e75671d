"""The gated delta rule and the layer norm at the edges of what their calls allow: the largest launches, empty axes,
values that a padded lane turns into NaN, and gradients that are zero by the formulas."""

import ctypes

import pytest
import torch

from test_gated_delta import DEV, NAMES, U, _params, gradients, problem, rel, to_dev


# --------------------------------------------------------------------------- CPU: the largest calls


@pytest.mark.parametrize("name", ["mko_delta_fwd", "mko_delta_bwd"])
@pytest.mark.parametrize("kw", [{"batch": 1 << 13, "heads": 1 << 10}, {"batch": 1 << 10, "length": 64 << 13},
                                {"batch": 1 << 9, "heads": 2, "value": 16 << 13}])
def test_c_entries_refuse_more_threads_than_a_launch_has(name, kw):
    """Workgroups have up to 512 threads and a launch below 2^32, so it has room for fewer than 2^23 of them; one
    sequence less and the next check is reached."""
    from metal_kernelops import _native as nat
    lib = nat.lib()
    kw = {"length": 64, "heads": 1, "value": 16, "workspace_bytes": 64, **kw}
    assert getattr(lib, name)(ctypes.byref(_params(**kw)), None) == 3  # MKO_EUNSUPPORTED
    assert b"2^23" in lib.mko_last_error()
    kw["batch"] -= 1
    assert getattr(lib, name)(ctypes.byref(_params(**kw)), None) == 4  # MKO_EWORKSPACE


@pytest.mark.parametrize("name", ["mko_delta_fwd", "mko_delta_bwd"])
def test_c_entries_refuse_wide_values(name):
    from metal_kernelops import _native as nat
    assert getattr(nat.lib(), name)(ctypes.byref(_params(value=1 << 20)), None) == 3
    assert b"2^20" in nat.lib().mko_last_error()


def test_calls_refuse_what_the_launches_do_not_take(monkeypatch):
    from metal_kernelops import _native as nat
    from metal_kernelops.cv import gated_delta, gated_delta_rule
    monkeypatch.setattr(gated_delta, "_require_gpu", lambda t: None)
    monkeypatch.setattr(nat, "launch", lambda *args: pytest.fail("launched"))
    monkeypatch.setattr(torch, "empty", lambda *args, **kw: pytest.fail("allocated"))
    one = torch.zeros(1)
    for batch, length, heads, value, text in [(1 << 13, 1, 1 << 10, 1, r"2\^23"), (1, 1 << 29, 1, 1, r"2\^23"),
                                              (1, 1, 1, 1 << 20, r"2\^20")]:
        q, v, gate = (one.expand(s) for s in ((batch, length, 1, 1), (batch, length, heads, value), (batch, length, heads)))
        with pytest.raises(ValueError, match=text):
            gated_delta_rule(q, q, v, gate, gate)


# --------------------------------------------------------------------------- CPU: what a trace is told


@pytest.mark.parametrize("sizes", [(0, 5, 1, 2, 8, 8), (2, 0, 1, 2, 8, 8), (2, 5, 1, 2, 8, 0), (2, 5, 1, 0, 8, 8)])
@pytest.mark.parametrize("carried", [False, True])
def test_fakes_of_empty_calls_have_the_shapes_of_the_ops(sizes, carried):
    """Calls without outputs launch nothing, so what the ops return can be seen here."""
    from metal_kernelops.cv import gated_delta
    from torch._subclasses.fake_tensor import FakeTensorMode
    b, l, hk, h, k, v = sizes

    def inputs(device):
        shapes = ((b, l, hk, k), (b, l, hk, k), (b, l, h, v), (b, l, h), (b, l, h), (b, h, v, k))
        return [torch.zeros(s, device=device) for s in shapes[:5]] + [torch.zeros(shapes[5], device=device) if carried else None]

    args = inputs("cpu")
    outs = gated_delta._delta_fwd_op(*args, 1.0, True, True)
    grads = gated_delta._delta_bwd_op(outs[0], outs[1], *args, outs[2], 1.0, carried)
    with FakeTensorMode():
        args = inputs(DEV)
        fakes = torch.ops.mko.delta_fwd(*args, 1.0, True, True)
        fake_grads = torch.ops.mko.delta_bwd(fakes[0], fakes[1], *args, fakes[2], 1.0, carried)
    assert [(t.shape, t.dtype) for t in fakes] == [(t.shape, t.dtype) for t in outs]
    assert [(t.shape, t.dtype) for t in fake_grads] == [(t.shape, t.dtype) for t in grads]


# --------------------------------------------------------------------------- GPU


@pytest.mark.gpu
def test_gradients_of_a_norm_of_67_million_features():
    """The sums of the parameters' gradients have more columns than one axis of a launch has room for.  One row: dbias is
    dout, and dweight's error is that of the variance, whose threads add 65537 squares each: at most 65537 * 2^-24 of it,
    and half of that of its root."""
    from metal_kernelops.cv import layernorm_residual
    g = torch.Generator(device=DEV).manual_seed(0)
    n = (1 << 26) + 100
    x = torch.randn(1, n, generator=g, device=DEV).half()
    dout = torch.randn(1, n, generator=g, device=DEV).half()
    w, b = (torch.ones(n, device=DEV, requires_grad=True) for _ in range(2))
    dw, db = torch.autograd.grad(layernorm_residual(x, w, b)[0], (w, b), dout)
    assert torch.equal(db, dout[0].float())
    wide = x[0].double()
    wide = (wide - wide.mean()) / wide.std(correction=0)
    wide *= dout[0].double()
    assert (dw.double() - wide).norm() <= 65537 * 2.0 ** -25 * wide.norm()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("features", [96, 100, 1000])
def test_a_norm_of_large_equal_features_has_finite_gradients(features, dtype):
    """mu / sqrt(eps) passes float32's largest number, and so does the zero of a lane without features normalised.  The
    sums are exact: the row's differences from its mean are zero, and dx is (gw - mean(gw)) / sqrt(eps)."""
    from metal_kernelops.cv import layernorm_residual
    g = torch.Generator().manual_seed(features)
    x = torch.full((3, features), 2.0 ** (120 if features < 128 else 117), dtype=dtype, device=DEV, requires_grad=True)
    w = torch.ones(features, device=DEV, requires_grad=True)
    dout = torch.randn(3, features, generator=g).to(dtype)
    eps = 1e-5 if features < 128 else 1e-8
    dx, dw = torch.autograd.grad(layernorm_residual(x, w, eps=eps)[0], (x, w), dout.to(DEV))
    want = (dout.double() - dout.double().mean(-1, keepdim=True)) * eps ** -0.5
    assert (dw == 0).all()
    assert (dx.cpu().double() - want).norm() <= (1e-6 + torch.finfo(dtype).eps / 2) * want.norm()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("cleared", [-float("inf"), -2e4, -1e4, -150.0])
@pytest.mark.parametrize("heads", [1, 4])
def test_a_decay_that_clears_the_state_has_a_gradient_of_zero(cleared, dtype, heads):
    """It is exp(log_decay) times something, and float32 has no number for exp(-104) and below."""
    p = problem(2, 150, 1, heads, 32, 24, dtype, gates=torch.float32)
    at = [0, 1, 63, 64, 100, 149]
    p["log_decay"][:, at] = cleared
    _, grads = gradients(to_dev(p))
    assert (grads["log_decay"][:, at] == 0).all()
    rest = [t for t in range(150) if t not in at]
    assert (grads["log_decay"][:, rest] != 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_an_update_with_a_gradient_is_a_rule_of_length_one(dtype):
    """Its values are the rule's, to the bit, and beside the update's without a gradient off by the rule's eight roundings
    to the activations' type, which the update does not make, and by the stored output's of both: 10 u."""
    from metal_kernelops.cv import gated_delta_rule, gated_delta_rule_update
    d = to_dev(problem(2, 1, 2, 4, 64, 48, dtype, state=torch.float32))
    args = [d[n] for n in NAMES[:5]]
    one = [t[:, 0] for t in args]
    plain = gated_delta_rule_update(d["initial"], *one)
    recorded = gated_delta_rule_update(d["initial"].clone().requires_grad_(True), *one)
    y, final = gated_delta_rule(*args, initial_state=d["initial"], return_final_state=True)
    assert torch.equal(recorded[0], y[:, 0]) and torch.equal(recorded[1], final)
    for a, b in zip(recorded, plain):
        assert rel(a, b) <= (1e-5 if dtype == torch.float32 else 10 * U[dtype])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("length", [1, 2, 65])
@pytest.mark.parametrize("heads", [1, 3])
def test_a_decay_that_meets_no_state_has_a_gradient_of_zero(length, heads, dtype):
    """The first token's without an initial state."""
    for carried in (False, True):
        p = problem(2, length, 1, heads, 32, 24, dtype, initial=carried)
        _, grads = gradients(to_dev(p), use=("y",))
        assert ((grads["log_decay"][:, 0] != 0) == carried).all()
        assert (grads["log_decay"][:, 1:] != 0).all()
