"""The delta-rule layer's operators together, as ``examples/delta_layer.py`` runs them, and what watches
their calls: training gradients against a float64 composition of the oracles, prompts and tokens against
the whole sequence, traces, modes and profilers.

Tolerances.  Training, float32: the operators' own 1e-5 and 1e-6 through two layers, 5e-5.  Serving in
bfloat16: a layer rounds about ten activations (norm, projection, convolution, q, k, v, gates, the rule's
own eight, the gated norm, projection), each by at most 2^-8 of its norm and independent of the others, and
the last norm divides by what two layers left: 2 sqrt(2 * 18) * 2^-8 = 5%.  Tokens against a prompt over
the same steps differ by the same roundings: 5%.
"""

import importlib.util
import os

import copy
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx

import oracle
from oracle import delta_rule, layer_norm
from test_traced_calls import Seen, same, traced_ops, with_gradients

DEV = "cuda"
BF16, F32 = torch.bfloat16, torch.float32
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def example():
    spec = importlib.util.spec_from_file_location("delta_layer_example", os.path.join(ROOT, "examples", "delta_layer.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def oracle_stack(stack, x, first=None):
    """The example's training pass in float64 on the CPU."""
    stream = None
    for p in stack.layers:
        out, stream = layer_norm.layernorm_residual(x, p.norm, p.norm_bias, stream)
        mixed, gate, step, beta = (out @ p.in_proj.t()).split((p.mixed, p.heads * p.value, p.heads, p.heads), -1)
        mixed, _ = oracle.causal_conv1d(mixed.transpose(1, 2), p.conv, p.conv_bias, "silu")
        q, k, v = p.split(mixed.transpose(1, 2))
        decay = -torch.exp(p.rate) * torch.nn.functional.softplus(step)
        if first is not None:
            decay = decay.masked_fill(first[..., None], -float("inf"))
        y, _ = delta_rule.gated_delta_rule(q, k, v, decay, torch.sigmoid(beta))
        y, _ = oracle.rmsnorm_gated(y, p.out_norm, z=gate.unflatten(-1, (p.heads, p.value)))
        x = y.flatten(-2) @ p.out_proj.t()
    return layer_norm.layernorm_residual(x, stack.norm, stack.norm_bias, stream)[0]


def rel(got, want):
    got, want = got.detach().double().cpu(), want.detach().double().cpu()
    return ((got - want).norm() / want.norm()).item()


@pytest.mark.gpu
@pytest.mark.parametrize("length", [50, 200])
def test_training_gradients(length):
    module = example()
    torch.manual_seed(length)
    hip = module.Stack(64, 2)
    ref = copy.deepcopy(hip).double()
    hip = hip.to(DEV)
    x = torch.randn(2, length, 64, dtype=torch.float64)
    first = torch.zeros(2, length, dtype=torch.bool)
    first[:, length // 2] = True
    want = oracle_stack(ref, x, first)
    got = hip(x.float().to(DEV), first.to(DEV))
    assert rel(got, want) <= 5e-5
    dy = torch.randn(want.shape, dtype=torch.float64)
    want.backward(dy)
    got.backward(dy.float().to(DEV))
    for (name, a), (_, b) in zip(ref.named_parameters(), hip.named_parameters()):
        assert rel(b.grad, a.grad) <= 5e-5, name


@pytest.mark.gpu
def test_serving_follows_the_whole_sequence():
    module = example()
    torch.manual_seed(4)
    stack = module.Stack(128, 2, key_heads=2, heads=4, key=64, value=64).to(DEV)
    x = torch.randn(3, 150, 128, device=DEV)
    with torch.no_grad():
        want = stack(x)
    whole = module.Served(stack, 3).prompt(x)
    assert rel(whole, want) <= 0.05
    served = module.Served(stack, 3)
    parts = [served.prompt(x[:, :1]), served.prompt(x[:, 1:130])] + [served.token(x[:, t])[:, None] for t in range(130, 150)]
    assert rel(torch.cat(parts, 1), want) <= 0.05 and rel(torch.cat(parts, 1), whole) <= 0.05
    exact = module.Served(stack, 3, dtype=F32)
    parts = [exact.prompt(x[:, :100])] + [exact.token(x[:, t])[:, None] for t in range(100, 150)]
    assert rel(torch.cat(parts, 1), want) <= 5e-5


# --------------------------------------------------------------------------- what watches a call


def _rule(q, k, v, decay, beta, h0):
    from metal_kernelops.cv import gated_delta_rule
    return gated_delta_rule(q, k, v, -decay.abs(), torch.sigmoid(beta), initial_state=h0, return_final_state=True)


def _rule_alone(q, k, v, decay, beta):
    from metal_kernelops.cv import gated_delta_rule
    return (gated_delta_rule(q, k, v, -decay.abs(), torch.sigmoid(beta)),)


def _step(state, q, k, v, decay, beta):
    from metal_kernelops.cv import gated_delta_rule_update
    return gated_delta_rule_update(state, q, k, v, -decay.abs(), torch.sigmoid(beta))


def _norm(x, weight, bias, residual):
    from metal_kernelops.cv import layernorm_residual
    return layernorm_residual(x, weight, bias, residual)


def _norm_first(x, weight):
    from metal_kernelops.cv import layernorm_residual
    return layernorm_residual(x, weight)[:1]


def _some(*shape, dtype=F32, std=1.0):
    return lambda g: (std * torch.randn(shape, generator=g)).to(dtype)


# name: the call, its inputs, the op that a trace holds, whether it is differentiable
CALLS = {
    "rule": (_rule, [_some(2, 70, 1, 16, dtype=BF16, std=0.25)] * 2 + [_some(2, 70, 2, 8, dtype=BF16)]
             + [_some(2, 70, 2)] * 2 + [_some(2, 2, 8, 16)], "delta_fwd", True),
    "rule alone": (_rule_alone, [_some(2, 70, 2, 16, std=0.25)] * 2 + [_some(2, 70, 2, 8)] + [_some(2, 70, 2)] * 2,
                   "delta_fwd", True),
    "step": (_step, [_some(3, 2, 8, 16)] + [_some(3, 1, 16, dtype=BF16, std=0.25)] * 2 + [_some(3, 2, 8, dtype=BF16)]
             + [_some(3, 2)] * 2, "delta_update", False),
    "norm": (_norm, [_some(5, 50, dtype=BF16), _some(50), _some(50), _some(5, 50)], "layernorm_fwd", True),
    "norm one type": (_norm, [_some(2, 3, 50), _some(50, dtype=BF16), _some(50), _some(2, 3, 50)], "layernorm_fwd", True),
    "norm first": (_norm_first, [_some(5, 50), _some(50)], "layernorm_fwd", True),
}


def inputs(name, seed):
    g = torch.Generator().manual_seed(seed)
    return [make(g) for make in CALLS[name][1]]


def on_gpu(name, seed):
    return [t.to(DEV) for t in inputs(name, seed)]


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
    with FakeTensorMode():
        q, v, gate, s = (torch.empty(n, device=DEV) for n in ((2, 70, 1, 16), (2, 70, 2, 8), (2, 70, 2), (2, 2, 8, 16)))
        saved = torch.empty(10, device=DEV, dtype=torch.uint8)
        grads = torch.ops.mko.delta_bwd(v, s, q, q, v, gate, gate, s, saved, 1.0, True)
        assert [g.shape for g in grads] == [t.shape for t in (q, q, v, gate, gate, s)]
        assert torch.ops.mko.delta_bwd(v, None, q, q, v, gate, gate, None, saved, 1.0, False)[5].numel() == 0
        x, w, stats = torch.empty(2, 70, 24, device=DEV, dtype=BF16), torch.empty(24, device=DEV), torch.empty(2, 70, 2, device=DEV)
        dx, dres, dw, db = torch.ops.mko.layernorm_bwd(x, None, x.float(), w, stats, BF16, True, True)
        assert (dx.dtype, dres.dtype) == (BF16, F32) and dx.shape == dres.shape == x.shape and dw.shape == db.shape == w.shape
        assert [t.numel() for t in torch.ops.mko.layernorm_bwd(x, None, x, w, stats, BF16, False, False)[1:]] == [0, 0, 0]


def test_a_traced_update_writes_its_destination():
    from metal_kernelops.cv import gated_delta_rule_update
    with FakeTensorMode():
        args = [t.to(DEV) for t in inputs("step", 0)]
        graph = make_fx(lambda s, *rest: gated_delta_rule_update(s, *rest, out_state=s))(*args)
    ops = traced_ops(graph)
    assert any("mko.delta_update." in o for o in ops) and any("copy_" in o for o in ops), ops


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
            traced = torch.compile(call, backend="aot_eager", fullgraph=True)
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
        assert any("mko." + CALLS[name][2].replace("fwd", "bwd") in o for o in traced_ops(run))
    elif how == "compile":
        torch._dynamo.reset()
        run = with_gradients(torch.compile(call, backend="aot_eager", fullgraph=True))
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
    with torch.no_grad():
        zero = torch._efficientzerotensor(tuple(args[0].shape), dtype=args[0].dtype, device=DEV)
        for odd, dense in ((torch._neg_view(args[0]), -args[0]), (zero, torch.zeros_like(args[0]))):
            assert same(call(odd, *args[1:]), call(dense, *args[1:]))
    if CALLS[name][3]:
        leaves = [a.clone().requires_grad_(True) for a in args]
        outs = call(*leaves)
        ones = [torch.randn_like(o) for o in outs]
        got = torch.autograd.grad(outs, leaves, [torch._neg_view(o) for o in ones], retain_graph=True)
        assert same(got, torch.autograd.grad(outs, leaves, [-o for o in ones]))


@pytest.mark.gpu
def test_a_traced_update_in_place_replays():
    from metal_kernelops.cv import gated_delta_rule_update

    def call(state, *rest):
        return gated_delta_rule_update(state, *rest, out_state=state)

    args = on_gpu("step", 1)
    with torch.no_grad():
        graph = make_fx(call)(*[a.clone() for a in args])
        for seed in (1, 2):
            args = on_gpu("step", seed)
            states = args[0].clone(), args[0].clone()
            assert same(graph(states[0], *args[1:]), call(states[1], *args[1:])) and torch.equal(*states)
