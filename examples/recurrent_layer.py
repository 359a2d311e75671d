"""A stack of gated recurrent layers, trained in floating point and served with 8-bit projections.

One layer, on the residual stream::

    norm(stream + x) -> in_proj -> causal conv1d -> gated recurrence -> gated norm -> out_proj -> x

Training runs ``rmsnorm_residual``, ``causal_conv1d_fn``, ``gated_recurrence`` and
``rmsnorm_gated`` with their gradients around plain float projections.  ``Served`` takes a trained
stack, lays its projections out in 8 bits once, and runs prompts (``rmsnorm_residual_int8`` ->
``int8_linear`` -> ... -> ``quantize_int8`` -> ``int8_linear``) and single tokens
(``causal_conv1d_update``, ``gated_recurrence_update``) on carried states.

    python examples/recurrent_layer.py [--width 256] [--layers 2] [--steps 20]

trains on a synthetic sequence to predict (each step's input, delayed), serves a prompt and then
single tokens, and prints how far the 8-bit outputs are from the float ones.
"""

from __future__ import annotations

import argparse
import math
import os
import sys

import torch
from torch import nn

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "metal-kernelops_amd"))

from metal_kernelops.cv import (  # noqa: E402
    causal_conv1d_fn,
    causal_conv1d_update,
    gated_recurrence,
    gated_recurrence_update,
    int8_linear,
    quantize_int8,
    rmsnorm_gated,
    rmsnorm_residual,
    rmsnorm_residual_int8,
)


class Layer(nn.Module):
    """The parameters of a layer and its training pass."""

    def __init__(self, width, inner, taps=4):
        super().__init__()
        self.inner = inner
        self.norm = nn.Parameter(torch.ones(width))
        self.in_proj = nn.Parameter(torch.randn(4 * inner, width) / math.sqrt(width))
        self.conv = nn.Parameter(torch.randn(inner, taps) / math.sqrt(taps))
        self.conv_bias = nn.Parameter(torch.zeros(inner))
        # at a full gate a channel keeps 0.9 to 0.999 of its state a step
        rate = -torch.log(torch.rand(inner) * 0.099 + 0.9) / 8.0
        self.decay = nn.Parameter(torch.log(torch.expm1(rate)))
        self.out_norm = nn.Parameter(torch.ones(inner))
        self.out_proj = nn.Parameter(torch.randn(width, inner) / math.sqrt(inner))

    def forward(self, x, stream, reset=None):
        """``(x, stream)`` of the layer before, ``(batch, length, width)``; None for no stream yet."""
        out, stream = rmsnorm_residual(x, self.norm, stream)
        x, z, input_gate, decay_gate = (out @ self.in_proj.to(out.dtype).t()).split(self.inner, -1)
        x = causal_conv1d_fn(x.transpose(1, 2), self.conv, self.conv_bias, activation="silu").transpose(1, 2)
        y = gated_recurrence(x, input_gate, decay_gate, self.decay, reset=reset)
        y = rmsnorm_gated(y, self.out_norm, z=z, norm_before_gate=False)
        return y @ self.out_proj.to(y.dtype).t(), stream


class Stack(nn.Module):
    """Layers and the norm after the last."""

    def __init__(self, width, layers, inner=None):
        super().__init__()
        self.layers = nn.ModuleList(Layer(width, inner or 2 * width) for _ in range(layers))
        self.norm = nn.Parameter(torch.ones(width))

    def forward(self, x, reset=None):
        stream = None
        for layer in self.layers:
            x, stream = layer(x, stream, reset)
        return rmsnorm_residual(x, self.norm, stream)[0]


class Served:
    """A trained stack with its projections in 8 bits, and the states of a batch of users."""

    @torch.no_grad()
    def __init__(self, stack, batch, dtype=torch.bfloat16):
        self.dtype, self.norm = dtype, stack.norm.detach()
        self.layers = []
        for layer in stack.layers:
            parameters = {n: p.detach() for n, p in layer.named_parameters()}
            conv = parameters["conv"].to(dtype)
            self.layers.append({
                **parameters, "inner": layer.inner, "conv": conv, "conv_bias": parameters["conv_bias"].to(dtype),
                "in": quantize_int8(parameters["in_proj"]), "out": quantize_int8(parameters["out_proj"]),
                "state": torch.zeros(batch, layer.inner, device=conv.device),
                "window": torch.zeros(batch, layer.inner, conv.shape[1] - 1, dtype=dtype, device=conv.device)})

    def _layer(self, p, x, stream, mix):
        q, scale, stream = rmsnorm_residual_int8(x, p["norm"], stream)
        x, z, input_gate, decay_gate = int8_linear(q, scale, *p["in"], out_dtype=self.dtype).split(p["inner"], -1)
        y = rmsnorm_gated(mix(x, input_gate, decay_gate), p["out_norm"], z=z, norm_before_gate=False)
        return int8_linear(*quantize_int8(y), *p["out"], out_dtype=self.dtype), stream

    @torch.no_grad()
    def prompt(self, x):
        """Outputs of ``(batch, length, width)``; the states move to the prompt's end."""
        x, stream = x.to(self.dtype), None
        for p in self.layers:
            def mix(v, input_gate, decay_gate):
                v, p["window"] = causal_conv1d_fn(v.transpose(1, 2), p["conv"], p["conv_bias"], activation="silu",
                                                  initial_state=p["window"], return_final_state=True)
                y, p["state"] = gated_recurrence(v.transpose(1, 2), input_gate, decay_gate, p["decay"],
                                                 initial_state=p["state"], return_final_state=True)
                return y

            x, stream = self._layer(p, x, stream, mix)
        return rmsnorm_residual(x, self.norm, stream)[0]

    @torch.no_grad()
    def token(self, x):
        """Outputs of one token of each user, ``(batch, width)``; the states move on in place."""
        x, stream = x.to(self.dtype), None
        for p in self.layers:
            def mix(v, input_gate, decay_gate):
                v = causal_conv1d_update(v, p["window"], p["conv"], p["conv_bias"], activation="silu")
                return gated_recurrence_update(p["state"], v, input_gate, decay_gate, p["decay"],
                                               out_state=p["state"])[0]

            x, stream = self._layer(p, x, stream, mix)
        return rmsnorm_residual(x, self.norm, stream)[0]


def main():
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--width", type=int, default=256)
    ap.add_argument("--layers", type=int, default=2)
    ap.add_argument("--steps", type=int, default=20)
    args = ap.parse_args()
    torch.manual_seed(0)
    stack = Stack(args.width, args.layers).cuda()
    optimiser = torch.optim.Adam(stack.parameters(), lr=1e-3)
    reset = torch.zeros(4, 256, dtype=torch.bool, device="cuda")
    reset[:, 128] = True  # two documents a row
    for step in range(args.steps):
        x = torch.randn(4, 256, args.width, device="cuda")
        target = torch.roll(x, 1, 1)
        loss = (stack(x, reset) - target).square().mean()
        optimiser.zero_grad()
        loss.backward()
        optimiser.step()
        if step % 5 == 0 or step + 1 == args.steps:
            print(f"step {step}: loss {loss.item():.4f}", flush=True)
    x = torch.randn(2, 40, args.width, device="cuda")
    with torch.no_grad():
        want = stack(x)
    served = Served(stack, 2)
    got = torch.cat([served.prompt(x[:, :32])] + [served.token(x[:, t])[:, None] for t in range(32, 40)], 1)
    for name, part in (("prompt", slice(0, 32)), ("tokens", slice(32, 40))):
        off = (got[:, part].float() - want[:, part]).norm() / want[:, part].norm()
        print(f"8-bit {name}: off the float outputs by {off.item():.4f} of their norm")


if __name__ == "__main__":
    main()
