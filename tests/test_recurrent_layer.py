"""The recurrent layer's operators together, as ``examples/recurrent_layer.py`` runs them: training
gradients against a float64 composition of the oracles, prompts and tokens served in 8 bits against the
float layer, and results that do not depend on what memory held.

Tolerances.  Training, float32: the operators' own 1e-5 and 1e-6 through two layers, 5e-5.  Serving:
an 8-bit value of a row with its largest magnitude near 4 standard deviations is off by a step / sqrt(12),
4 / 127 / sqrt(12) = 0.9% of the row's deviation; two operands of two projections in each of two
layers make sqrt(8) * 0.9% = 2.6%, beside bfloat16 activations of 0.2% in ten places; 5%.  Tokens
against a prompt over the same steps differ by roundings of the bfloat16 outputs alone, and by the 8-bit
steps that those move: 2%.
"""

import copy
import importlib.util
import os

import pytest
import torch

import oracle
from oracle import recurrent_layer as layer_oracle

DEV = "cuda"
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def example():
    spec = importlib.util.spec_from_file_location("recurrent_layer_example",
                                                  os.path.join(ROOT, "examples", "recurrent_layer.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def oracle_stack(stack, x, reset=None):
    """The example's training pass in float64 on the CPU."""
    stream = None
    for p in stack.layers:
        out, stream = layer_oracle.rmsnorm_residual(x, p.norm, stream)
        v, z, ig, rg = (out @ p.in_proj.t()).split(p.inner, -1)
        v, _ = oracle.causal_conv1d(v.transpose(1, 2), p.conv, p.conv_bias, "silu")
        y, _ = layer_oracle.gated_recurrence(v.transpose(1, 2), ig, rg, p.decay, None, reset)
        y, _ = oracle.rmsnorm_gated(y, p.out_norm, z=z, norm_before_gate=False)
        x = y @ p.out_proj.t()
    return layer_oracle.rmsnorm_residual(x, stack.norm, stream)[0]


def rel(got, want):
    got, want = got.detach().double().cpu(), want.detach().double().cpu()
    return ((got - want).norm() / want.norm()).item()


@pytest.mark.gpu
@pytest.mark.parametrize("width,length", [(24, 19), (64, 150)])
def test_training_matches_the_oracles(width, length):
    module = example()
    torch.manual_seed(3)
    ref = module.Stack(width, 2).double()
    hip = copy.deepcopy(ref).float().to(DEV)
    x = torch.randn(2, length, width, dtype=torch.float64)
    reset = torch.zeros(2, length, dtype=torch.bool)
    reset[:, length // 2] = True
    want = oracle_stack(ref, x, reset)
    got = hip(x.float().to(DEV), reset.to(DEV))
    assert rel(got, want) <= 5e-5
    dy = torch.randn(want.shape, dtype=torch.float64)
    want.backward(dy)
    got.backward(dy.float().to(DEV))
    for (name, a), (_, b) in zip(ref.named_parameters(), hip.named_parameters()):
        assert rel(b.grad, a.grad) <= 5e-5, name


@pytest.mark.gpu
def test_serving_follows_the_float_layer_and_tokens_follow_the_prompt():
    module = example()
    torch.manual_seed(4)
    stack = module.Stack(128, 2).to(DEV)
    x = torch.randn(3, 60, 128, device=DEV)
    with torch.no_grad():
        want = stack(x)
    whole = module.Served(stack, 3).prompt(x)
    assert rel(whole, want) <= 0.05
    served = module.Served(stack, 3)
    parts = [served.prompt(x[:, :1]), served.prompt(x[:, 1:50])]
    parts += [served.token(x[:, t])[:, None] for t in range(50, 60)]
    assert rel(torch.cat(parts, 1), want) <= 0.05
    assert rel(torch.cat(parts, 1), whole) <= 0.02


def _recurrence(batch, length, channels, dtype, reset):
    g = torch.Generator().manual_seed(length)
    leaves = [torch.randn(batch, length, channels, generator=g).to(dtype) for _ in range(3)]
    leaves += [torch.randn(channels, generator=g) - 4, torch.randn(batch, channels, generator=g)]
    cuts = torch.rand(batch, length, generator=g) < 0.02 if reset else None

    def call(x, ig, rg, decay, h0):
        from metal_kernelops.cv import gated_recurrence
        return gated_recurrence(x, ig, rg, decay, initial_state=h0, reset=None if cuts is None else cuts.to(DEV),
                                return_final_state=True)

    return leaves, call


def _norm(rows, features, dtype, stream):
    g = torch.Generator().manual_seed(rows)
    leaves = [torch.randn(rows, features, generator=g).to(dtype), torch.randn(features, generator=g),
              torch.randn(rows, features, generator=g).to(stream)]

    def call(x, w, r):
        from metal_kernelops.cv import rmsnorm_residual
        return rmsnorm_residual(x, w, r)

    return leaves, call


def _projections(rows, inner, outer):
    g = torch.Generator().manual_seed(rows)
    leaves = [torch.randn(rows, inner, generator=g).to(torch.bfloat16), torch.randn(outer, inner, generator=g)]

    def call(x, w):
        from metal_kernelops.cv import int8_linear, quantize_int8, rmsnorm_residual_int8
        q, s, _ = rmsnorm_residual_int8(x, w[0])
        packed = quantize_int8(w)
        return (int8_linear(q, s, *packed), int8_linear(*quantize_int8(x), *packed, out_dtype=torch.float32))

    return leaves, call


CASES = {
    "recurrence one chunk": _recurrence(2, 40, 70, torch.float32, False),
    "recurrence": _recurrence(2, 700, 130, torch.bfloat16, False),
    "recurrence resets": _recurrence(3, 331, 128, torch.float32, True),
    "recurrence many chains": _recurrence(8, 200, 1024, torch.bfloat16, False),
    "norm": _norm(37, 320, torch.bfloat16, torch.bfloat16), "norm ragged": _norm(600, 77, torch.float16, torch.float32),
    "norm wide": _norm(3, 40000, torch.float32, torch.float32),
    "projections few": _projections(5, 100, 70), "projections": _projections(130, 512, 300),
}


@pytest.mark.gpu
@pytest.mark.parametrize("name", CASES)
def test_results_do_not_depend_on_old_memory(name):
    leaves, call = CASES[name]
    grads = not name.startswith("projections")

    def run(fill):
        args = [t.to(DEV).requires_grad_(grads) for t in leaves]
        before = torch.are_deterministic_algorithms_enabled(), torch.utils.deterministic.fill_uninitialized_memory
        # deterministic mode fills what torch.empty allocates: NaN, or the largest value of an integer type
        torch.use_deterministic_algorithms(fill)
        torch.utils.deterministic.fill_uninitialized_memory = fill
        try:
            outs = call(*args)
            more = torch.autograd.grad(outs, args, [torch.ones_like(o) for o in outs]) if grads else ()
        finally:
            torch.use_deterministic_algorithms(before[0])
            torch.utils.deterministic.fill_uninitialized_memory = before[1]
        return [t.detach() for t in outs] + list(more)

    for k, (a, b) in enumerate(zip(run(False), run(True))):
        assert torch.isfinite(b.float()).all(), k
        assert torch.equal(a, b), k


@pytest.mark.gpu
def test_forward_mode_derivatives_are_refused_not_dropped():
    import torch.autograd.forward_ad as fwd
    from metal_kernelops.cv import (gated_recurrence, gated_recurrence_update, int8_linear, quantize_int8,
                                    rmsnorm_residual, rmsnorm_residual_int8)
    x, d = torch.randn(2, 5, 8, device=DEV), torch.randn(8, device=DEV)
    q, s = quantize_int8(x[0])
    with fwd.dual_level():
        dual = fwd.make_dual(x, torch.ones_like(x))
        calls = [lambda: gated_recurrence(dual, x, x, d),
                 lambda: gated_recurrence_update(x[:, 0], dual[:, 0], x[:, 0], x[:, 0], d),
                 lambda: rmsnorm_residual(dual, d, x), lambda: rmsnorm_residual_int8(dual, d, x),
                 lambda: quantize_int8(dual), lambda: int8_linear(q, s, q, s)]
        for call in calls:
            with pytest.raises((RuntimeError, ValueError, NotImplementedError)):
                call()


@pytest.mark.gpu
def test_a_negated_destination_is_refused():
    from metal_kernelops.cv import gated_recurrence_update
    x, d = torch.randn(2, 8, device=DEV), torch.randn(8, device=DEV)
    with pytest.raises(ValueError, match="contiguous"):
        gated_recurrence_update(x, x, x, x, d, out_state=torch._neg_view(torch.zeros(2, 8, device=DEV)))


@pytest.mark.gpu
def test_offsets_past_32_bits():
    """Tensors of more than 2^32 bytes: their last rows against the same rows alone.  The scan's
    channels forget (0.8 a step), so that 2048 steps before them are all that its last rows hold."""
    from metal_kernelops.cv import gated_recurrence, int8_linear, quantize_int8, rmsnorm_residual
    g = torch.Generator(device=DEV).manual_seed(0)
    length, channels = 900_000, 2560
    x = torch.empty(1, length, channels, dtype=torch.bfloat16, device=DEV).normal_(generator=g)
    gate = torch.zeros(1, 1, channels, dtype=torch.bfloat16, device=DEV).expand(1, length, channels)
    decay = torch.full((channels,), 0.0, device=DEV)  # a = exp(-scale log(2) / 2) = 0.8
    scale = 2 * 0.2231 / 0.6931
    y = gated_recurrence(x, gate, gate, decay, scale=scale)
    tail = slice(length - 2048, length)
    want = gated_recurrence(x[:, tail], gate[:, tail], gate[:, tail], decay, scale=scale)
    assert rel(y[:, -500:], want[:, -500:]) <= 2.0 ** -8
    leaf = x.requires_grad_(True)
    (dx,) = torch.autograd.grad(gated_recurrence(leaf, gate, gate, decay, scale=scale), leaf, y)
    part = x[:, :2048].detach().requires_grad_(True)
    (dpart,) = torch.autograd.grad(gated_recurrence(part, gate[:, :2048], gate[:, :2048], decay, scale=scale), part,
                                   y[:, :2048])
    assert rel(dx[:, :500], dpart[:, :500]) <= 2.0 ** -8
    del y, dx, want
    rows = x.detach()[0]
    weight = torch.ones(channels, device=DEV)
    out, stream = rmsnorm_residual(rows, weight, rows)
    last, last_stream = rmsnorm_residual(rows[-3:], weight, rows[-3:])
    assert torch.equal(out[-3:], last) and torch.equal(stream[-3:], last_stream)
    del out, stream
    q, s = quantize_int8(rows[:, :2048])
    q2 = torch.cat([q, q, q])  # 2.7 million rows of 2048 bytes
    wq, ws = quantize_int8(torch.randn(20, 2048, generator=g, device=DEV))
    whole = int8_linear(q2, torch.cat([s, s, s]), wq, ws, out_dtype=torch.float32)
    assert torch.equal(whole[-5:], int8_linear(q[-5:], s[-5:], wq, ws, out_dtype=torch.float32))
    assert torch.equal(whole[:70], int8_linear(q[:70], s[:70], wq, ws, out_dtype=torch.float32))
