"""Operators under what watches a call: a trace holds the operators themselves, not
only the allocation of their outputs, and its replay on other inputs gives the eager results; modes and
a recording profiler see them by name.  The CPU tests trace fake GPU tensors and launch nothing."""

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx
from torch.utils._python_dispatch import TorchDispatchMode

DEV = "cuda"


class Seen(TorchDispatchMode):
    def __init__(self):
        super().__init__()
        self.ops = []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        self.ops.append(str(func))
        return func(*args, **(kwargs or {}))


def _recurrence(x, ig, rg, decay, h0):
    from metal_kernelops.cv import gated_recurrence
    return gated_recurrence(x, ig, rg, decay, initial_state=h0, return_final_state=True)


def _recurrence_alone(x, ig, rg, decay):
    from metal_kernelops.cv import gated_recurrence
    return (gated_recurrence(x, ig, rg, decay),)


def _update(state, x, ig, rg, decay):
    from metal_kernelops.cv import gated_recurrence_update
    return gated_recurrence_update(state, x, ig, rg, decay)


def _norm(x, weight, residual):
    from metal_kernelops.cv import rmsnorm_residual
    return rmsnorm_residual(x, weight, residual)


def _norm_first(x, weight):
    from metal_kernelops.cv import rmsnorm_residual
    return rmsnorm_residual(x, weight)[:1]


def _norm_int8(x, weight, residual):
    from metal_kernelops.cv import rmsnorm_residual_int8
    return rmsnorm_residual_int8(x, weight, residual)


def _quantise(x):
    from metal_kernelops.cv import quantize_int8
    return quantize_int8(x)


def _linear(q, qs, w, ws, bias):
    from metal_kernelops.cv import int8_linear
    return (int8_linear(q, qs, w, ws, bias, out_dtype=torch.float32),)


def _ssm_update(state, x, dt, A, B):
    from metal_kernelops.cv import mamba2_state_update
    return mamba2_state_update(state, x, dt, A, B, B, dt_softplus=True)


def _gated_norm(x, weight, bias, z):
    from metal_kernelops.cv import rmsnorm_gated
    return (rmsnorm_gated(x, weight, bias, z),)


def _ss2d(u, dt, A, B, C):
    from metal_kernelops.cv import ss2d_scan
    return (ss2d_scan(u, dt.abs(), -A.abs(), B, C, merge="mean"),)


def _normal(*shape, dtype=torch.float32):
    return lambda g: torch.randn(shape, generator=g).to(dtype)


def _bytes(*shape):
    return lambda g: torch.randint(-127, 128, shape, generator=g, dtype=torch.int8)


BF16 = torch.bfloat16
# name: the call, its inputs, the op that a trace holds, whether it is differentiable
CALLS = {
    "recurrence": (_recurrence, [_normal(2, 70, 24, dtype=BF16)] * 3 + [_normal(24), _normal(2, 24)], "recur_fwd", True),
    "recurrence alone": (_recurrence_alone, [_normal(2, 70, 24)] * 3 + [_normal(24)], "recur_fwd", True),
    "update": (_update, [_normal(3, 40)] + [_normal(3, 40, dtype=BF16)] * 3 + [_normal(40)], "recur_update", False),
    "norm": (_norm, [_normal(5, 50, dtype=BF16), _normal(50), _normal(5, 50)], "resnorm_fwd", True),
    "norm one type": (_norm, [_normal(2, 3, 50), _normal(50, dtype=BF16), _normal(2, 3, 50)], "resnorm_fwd", True),
    "norm first": (_norm_first, [_normal(5, 50), _normal(50)], "resnorm_fwd", True),
    "norm int8": (_norm_int8, [_normal(5, 50, dtype=BF16), _normal(50), _normal(5, 50)], "resnorm_int8", False),
    "quantise": (_quantise, [_normal(2, 3, 50)], "quantize_int8", False),
    "ssm update": (_ssm_update, [_normal(2, 4, 8, 16), _normal(2, 4, 8), _normal(2, 4), _normal(4), _normal(2, 1, 16)],
                   "state_update_fwd", True),
    "gated norm": (_gated_norm, [_normal(2, 5, 48), _normal(48), _normal(48), _normal(2, 5, 48)], "gated_norm_fwd", True),
    "ss2d": (_ss2d, [_normal(1, 4, 5, 6), _normal(1, 4, 5, 6), _normal(4, 8), _normal(1, 2, 8, 5, 6), _normal(1, 2, 8, 5, 6)],
             "selscan_fwd", True),
    "linear": (_linear, [_bytes(20, 64), _normal(20), _bytes(30, 64), _normal(30), _normal(30)], "int8_linear", False),
}


def inputs(name, seed):
    g = torch.Generator().manual_seed(seed)
    return [make(g) for make in CALLS[name][1]]


def traced_ops(graph):
    return [str(n.target) for n in graph.graph.nodes if n.op == "call_function"]


def with_gradients(call):
    """The call's outputs and the gradients of its inputs, as one function of the inputs."""
    def run(*args):
        leaves = [a.detach().requires_grad_(True) for a in args]
        outs = call(*leaves)
        return (*outs, *torch.autograd.grad(outs, leaves, [torch.ones_like(o) for o in outs]))

    return run


# --------------------------------------------------------------------------- CPU: fake GPU tensors


@pytest.mark.parametrize("name", CALLS)
def test_a_trace_holds_the_operator(name):
    call, _, op, _ = CALLS[name]
    with FakeTensorMode():
        args = [t.to(DEV) for t in inputs(name, 0)]
        with torch.no_grad():
            graph = make_fx(call)(*args)
            outs = call(*args)
        assert any(f"mko.{op}." in o for o in traced_ops(graph)), traced_ops(graph)
        assert all(o.device.type == "cuda" for o in outs)


def test_the_backward_ops_know_their_outputs():
    f32, bf16 = dict(device=DEV), dict(device=DEV, dtype=BF16)
    with FakeTensorMode():
        x, decay, h0 = torch.empty(2, 70, 24, **bf16), torch.empty(24, **f32), torch.empty(2, 24, **f32)
        grads = torch.ops.mko.recur_bwd(x, None, x, x, x, decay, h0, None, None, 8.0, True, True)
        assert [(g.shape, g.dtype) for g in grads] == [(t.shape, t.dtype) for t in (x, x, x, decay, h0)]
        assert [g.numel() for g in torch.ops.mko.recur_bwd(x, h0, x, x, x, decay, None, None, None, 8.0, False, False)
                ][3:] == [0, 0]
        rstd = torch.empty(2, 70, **f32)
        dx, dres, dw = torch.ops.mko.resnorm_bwd(x, None, x.float(), decay, rstd, BF16, True)
        assert (dx.dtype, dres.dtype) == (BF16, torch.float32) and dx.shape == dres.shape == x.shape
        assert dw.shape == decay.shape and torch.ops.mko.resnorm_bwd(x, None, x, decay, rstd, BF16, False)[1].numel() == 0


def test_a_traced_update_writes_its_destination():
    from metal_kernelops.cv import gated_recurrence_update
    with FakeTensorMode():
        args = [t.to(DEV) for t in inputs("update", 0)]
        graph = make_fx(lambda s, *rest: gated_recurrence_update(s, *rest, out_state=s))(*args)
    ops = traced_ops(graph)
    assert any("mko.recur_update." in o for o in ops) and any("copy_" in o for o in ops), ops


# --------------------------------------------------------------------------- GPU


def on_gpu(name, seed):
    return [t.to(DEV) for t in inputs(name, seed)]


def same(got, want):
    return len(got) == len(want) and all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
@pytest.mark.parametrize("name", CALLS)
@pytest.mark.parametrize("how", ["jit.trace", "make_fx", "compile"])
def test_replays_give_the_eager_results(how, name):
    call, args = CALLS[name][0], on_gpu(name, 1)
    with torch.no_grad():
        if how == "jit.trace":
            traced = torch.jit.trace(call, tuple(args), check_trace=False)
        elif how == "make_fx":
            traced = make_fx(call)(*args)
        else:
            torch._dynamo.reset()
            traced = torch.compile(call, backend="aot_eager")
        for seed in (1, 2, 3):
            args = on_gpu(name, seed)
            assert same(traced(*args), call(*args))


@pytest.mark.gpu
@pytest.mark.parametrize("name", [n for n in CALLS if CALLS[n][3]])
@pytest.mark.parametrize("how", ["jit.trace", "make_fx", "compile"])
def test_replayed_gradients_are_the_eager_ones(how, name):
    call, args = CALLS[name][0], on_gpu(name, 1)
    if how == "make_fx":
        run = make_fx(with_gradients(call))(*args)
        op = CALLS[name][2]
        assert any("mko." + op in o for o in traced_ops(run))
        assert any("mko." + op.replace("fwd", "bwd") in o for o in traced_ops(run))
    elif how == "compile":
        torch._dynamo.reset()
        run = with_gradients(torch.compile(call, backend="aot_eager"))
    else:
        leaves = tuple(a.clone().requires_grad_(True) for a in args)
        run = with_gradients(torch.jit.trace(call, leaves, check_trace=False))
    for seed in (1, 2):
        args = on_gpu(name, seed)
        assert same(run(*args), with_gradients(call)(*args))


@pytest.mark.gpu
@pytest.mark.parametrize("name", CALLS)
def test_modes_and_profilers_see_the_operator(name):
    call, _, op, differentiable = CALLS[name]
    args = on_gpu(name, 4)
    with torch.no_grad():
        plain = call(*args)
        with Seen() as mode:
            seen = call(*args)
        with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CPU]) as prof:
            profiled = call(*args)
    assert any(f"mko.{op}" in o for o in mode.ops), mode.ops
    assert f"mko::{op}" in [e.key for e in prof.key_averages()]
    assert same(seen, plain) and same(profiled, plain)
    if differentiable:
        want = with_gradients(call)(*args)
        with torch.autograd.set_multithreading_enabled(False), Seen() as mode:
            assert same(with_gradients(call)(*args), want)
        assert any("mko." + op.replace("fwd", "bwd") in o for o in mode.ops), mode.ops


@pytest.mark.gpu
@pytest.mark.parametrize("name", CALLS)
def test_negated_views_and_zero_tensors_are_materialised(name):
    call, args = CALLS[name][0], on_gpu(name, 5)
    at = 1 if name == "linear" else 0
    with torch.no_grad():
        zero = torch._efficientzerotensor(tuple(args[at].shape), dtype=args[at].dtype, device=DEV)
        for odd, dense in ((torch._neg_view(args[at]), -args[at]), (zero, torch.zeros_like(args[at]))):
            assert same(call(*args[:at], odd, *args[at + 1:]), call(*args[:at], dense, *args[at + 1:]))
    if CALLS[name][3]:
        leaves = [a.clone().requires_grad_(True) for a in args]
        outs = call(*leaves)
        ones = [torch.randn_like(o) for o in outs]
        got = torch.autograd.grad(outs, leaves, [torch._neg_view(o) for o in ones], retain_graph=True)
        assert same(got, torch.autograd.grad(outs, leaves, [-o for o in ones]))


@pytest.mark.gpu
def test_a_traced_update_in_place_replays():
    from metal_kernelops.cv import gated_recurrence_update

    def call(state, *rest):
        return gated_recurrence_update(state, *rest, out_state=state)

    args = on_gpu("update", 1)
    with torch.no_grad():
        graph = make_fx(call)(*[a.clone() for a in args])
        for seed in (1, 2):
            args = on_gpu("update", seed)
            states = args[0].clone(), args[0].clone()
            got, want = graph(states[0], *args[1:]), call(states[1], *args[1:])
            assert same(got, want) and torch.equal(*states)


@pytest.mark.gpu
def test_conv1d_update_materialises_negated_views_and_zero_tensors():
    from metal_kernelops.cv import causal_conv1d_update
    g = torch.Generator().manual_seed(6)
    x, window, weight, bias = (torch.randn(s, generator=g).to(DEV) for s in ((2, 40), (2, 40, 3), (40, 4), (40,)))

    def call(x, weight, bias):
        state = window.clone()
        return causal_conv1d_update(x, state, weight, bias, activation="silu"), state

    def zero(t):
        return torch._efficientzerotensor(tuple(t.shape), device=DEV)

    assert same(call(torch._neg_view(x), weight, bias), call(-x, weight, bias))
    assert same(call(zero(x), weight, bias), call(torch.zeros_like(x), weight, bias))
    assert same(call(x, zero(weight), zero(bias)), call(x, torch.zeros_like(weight), torch.zeros_like(bias)))


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["selscan", "ssd", "conv1d", "conv1d update", "state update", "gated norm", "ss2d"])
def test_forward_mode_derivatives_are_refused(name):
    """The dispatcher drops the tangent of an op that has no formula for it; the calls refuse it."""
    import torch.autograd.forward_ad as fwd
    from metal_kernelops import cv, selective_scan
    g = torch.Generator().manual_seed(7)

    def r(*shape):
        return torch.randn(shape, generator=g).to(DEV)

    calls = {
        "selscan": (lambda u, *a: selective_scan(u, u.abs(), *a), [r(1, 8, 20), -r(8, 4).abs(), r(1, 1, 4, 20), r(1, 1, 4, 20)]),
        "ssd": (cv.mamba2_chunk_scan, [r(1, 20, 2, 8), r(1, 20, 2).abs(), -r(2).abs(), r(1, 20, 1, 8), r(1, 20, 1, 8)]),
        "conv1d": (cv.causal_conv1d_fn, [r(1, 8, 20), r(8, 4), r(8)]),
        "conv1d update": (cv.causal_conv1d_update, [r(2, 8), r(2, 8, 3), r(8, 4)]),
        "state update": (_ssm_update, on_gpu("ssm update", 7)),
        "gated norm": (_gated_norm, on_gpu("gated norm", 7)),
        "ss2d": (_ss2d, on_gpu("ss2d", 7)),
    }
    call, args = calls[name]
    call(*args)
    with fwd.dual_level():
        call(*args)  # no tangent, nothing to refuse
        dual = fwd.make_dual(args[0], torch.ones_like(args[0]))
        with pytest.raises((RuntimeError, NotImplementedError)):
            call(dual, *args[1:])


@pytest.mark.gpu
@pytest.mark.parametrize("name", [*CALLS, "update in place"])
def test_compiles_without_a_graph_break(name):
    torch._dynamo.reset()
    if name == "update in place":
        from metal_kernelops.cv import gated_recurrence_update

        def call(state, *rest):
            return (gated_recurrence_update(state, *rest, out_state=state)[0],)

        args = on_gpu("update", 8)
    else:
        call, args = CALLS[name][0], on_gpu(name, 8)
    compiled = torch.compile(call, backend="aot_eager", fullgraph=True)
    with torch.no_grad():
        mine, theirs = [a.clone() for a in args], [a.clone() for a in args]
        assert same(compiled(*mine), call(*theirs)) and same(mine, theirs)
    if CALLS.get(name, (None,) * 4)[3]:
        assert same(with_gradients(compiled)(*args), with_gradients(call)(*args))
