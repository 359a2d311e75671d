"""One tensor in several roles of a call, and inputs broadcast by their callers: each role's gradient
reaches it.  Tolerances as in the operators' own tests, once for each role that is summed."""

import pytest
import torch

from oracle import recurrent_layer as oracle

DEV = "cuda"


def rel(got, want):
    got, want = got.detach().double().cpu(), want.detach().double().cpu()
    return ((got - want).norm() / want.norm()).item()


@pytest.mark.gpu
@pytest.mark.parametrize("features", [77, 512])
@pytest.mark.parametrize("use", ["out", "both"])
def test_norm_of_a_tensor_added_to_itself(features, use):
    from metal_kernelops.cv import rmsnorm_residual
    g = torch.Generator().manual_seed(features)
    x, w, dout, dstream = (torch.randn(s, generator=g) for s in ((9, features), (features,), (9, features), (9, features)))
    leaf, weight = x.to(DEV).requires_grad_(True), w.to(DEV).requires_grad_(True)
    out, stream = rmsnorm_residual(leaf, weight, leaf)
    outs, grads = ([out], [dout]) if use == "out" else ([out, stream], [dout, dstream])
    torch.autograd.backward(outs, [t.to(DEV) for t in grads])
    ds, dw = oracle.rmsnorm_residual_bwd(dout, dstream if use == "both" else None, 2 * x, w)
    assert rel(leaf.grad, 2 * ds) <= 2e-6 and rel(weight.grad, dw) <= 1e-6
    # the sum of the two roles through an intermediate, and a weight broadcast from one value
    leaf2, one = x.to(DEV).requires_grad_(True), torch.full((1,), 0.5, device=DEV, requires_grad=True)
    mid = leaf2 * 1.0
    rmsnorm_residual(mid, one.expand(features), mid)[0].backward(dout.to(DEV))
    ds, dw = oracle.rmsnorm_residual_bwd(dout, None, 2 * x, torch.full((features,), 0.5))
    assert rel(leaf2.grad, 2 * ds) <= 2e-6
    assert abs(one.grad.item() - dw.sum().item()) <= 1e-6 * dw.norm().item() * features ** 0.5


@pytest.mark.gpu
@pytest.mark.parametrize("channels", [65, 128])
def test_recurrence_gated_by_its_own_input(channels):
    from metal_kernelops.cv import gated_recurrence
    g = torch.Generator().manual_seed(channels)
    x, decay, dy = (torch.randn(s, generator=g) for s in ((2, 130, channels), (channels,), (2, 130, channels)))
    decay -= 3
    leaf = x.to(DEV).requires_grad_(True)
    gated_recurrence(leaf, leaf, leaf, decay.to(DEV)).backward(dy.to(DEV))
    dx, dig, drg, _, _ = oracle.gated_recurrence_bwd(dy, None, x, x, x, decay)
    assert rel(leaf.grad, dx + dig + drg) <= 3e-5
    # gates broadcast over the sequence, a decay over the channels
    gate, one = x[:, :1].to(DEV).requires_grad_(True), torch.full((1,), -3.0, device=DEV, requires_grad=True)
    wide = gate.expand(-1, 130, -1)
    gated_recurrence(x.to(DEV), wide, wide, one.expand(channels)).backward(dy.to(DEV))
    dense = x[:, :1].expand(-1, 130, -1)
    _, dig, drg, dd, _ = oracle.gated_recurrence_bwd(dy, None, x, dense, dense, torch.full((channels,), -3.0))
    terms = (dig.norm() ** 2 + drg.norm() ** 2) ** 0.5
    assert (gate.grad.double().cpu() - (dig + drg).sum(1, keepdim=True)).norm() <= 1e-5 * terms * 130 ** 0.5
    assert abs(one.grad.item() - dd.sum().item()) <= 1e-5 * dd.norm().item() * channels ** 0.5
