"""A stack of gated delta-rule layers, trained on whole sequences and served a token at a time.

One layer, on the residual stream::

    layer norm(stream + x) -> in_proj -> causal conv1d -> gated delta rule -> gated norm -> out_proj -> x

Training runs ``layernorm_residual``, ``causal_conv1d_fn``, ``gated_delta_rule`` and ``rmsnorm_gated``
with their gradients around plain float projections; documents packed in one row are separated by a log
decay of ``-inf``.  ``Served`` takes a trained stack and runs prompts (``gated_delta_rule`` with the state
carried in and out) and single tokens (``causal_conv1d_update``, ``gated_delta_rule_update``) on a batch's
states.

    python examples/delta_layer.py [--width 256] [--layers 2] [--steps 20]

trains on a synthetic sequence to recall (each step's input, delayed), serves a prompt and then single
tokens, and prints how far they are from the outputs of the whole sequence.
"""

from __future__ import annotations

import argparse
import math
import os
import sys

import torch
from torch import nn
from torch.nn import functional as F

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "metal-kernelops_amd"))

from metal_kernelops.cv import (  # noqa: E402
    causal_conv1d_fn,
    causal_conv1d_update,
    gated_delta_rule,
    gated_delta_rule_update,
    layernorm_residual,
    rmsnorm_gated,
)


class Layer(nn.Module):
    """The parameters of a layer, and its parts between the operators."""

    def __init__(self, width, key_heads=2, heads=4, key=32, value=32, taps=4):
        super().__init__()
        self.key_heads, self.heads, self.key, self.value = key_heads, heads, key, value
        self.mixed = 2 * key_heads * key + heads * value  # q, k and v, which pass the convolution
        self.norm = nn.Parameter(torch.ones(width))
        self.norm_bias = nn.Parameter(torch.zeros(width))
        self.in_proj = nn.Parameter(torch.randn(self.mixed + heads * value + 2 * heads, width) / math.sqrt(width))
        self.conv = nn.Parameter(torch.randn(self.mixed, taps) / math.sqrt(taps))
        self.conv_bias = nn.Parameter(torch.zeros(self.mixed))
        self.rate = nn.Parameter(torch.log(torch.rand(heads) * 0.1 + 0.01))  # of forgetting, at a step of one
        self.out_norm = nn.Parameter(torch.ones(value))
        self.out_proj = nn.Parameter(torch.randn(width, heads * value) / math.sqrt(heads * value))

    def project(self, out):
        """q, k and v before the convolution, the gate, the log decay and beta."""
        mixed, gate, step, beta = (out @ self.in_proj.to(out.dtype).t()).split(
            (self.mixed, self.heads * self.value, self.heads, self.heads), -1)
        return mixed, gate, -torch.exp(self.rate) * F.softplus(step.float()), torch.sigmoid(beta)

    def split(self, mixed):
        """q and k of norm one and v, by heads."""
        n = self.key_heads * self.key
        q, k, v = mixed.split((n, n, self.heads * self.value), -1)
        q, k = (F.normalize(t.unflatten(-1, (self.key_heads, self.key)), dim=-1) for t in (q, k))
        return q, k, v.unflatten(-1, (self.heads, self.value))

    def finish(self, y, gate):
        y = rmsnorm_gated(y, self.out_norm, z=gate.unflatten(-1, (self.heads, self.value)))
        return y.flatten(-2) @ self.out_proj.to(y.dtype).t()

    def forward(self, x, stream, first=None):
        """``(x, stream)`` of the layer before, ``(batch, length, width)``; None for no stream yet.
        ``first`` is true at the first token of each packed document."""
        out, stream = layernorm_residual(x, self.norm, self.norm_bias, stream)
        mixed, gate, decay, beta = self.project(out)
        mixed = causal_conv1d_fn(mixed.transpose(1, 2), self.conv, self.conv_bias, activation="silu").transpose(1, 2)
        if first is not None:
            decay = decay.masked_fill(first[..., None], -math.inf)
        return self.finish(gated_delta_rule(*self.split(mixed), decay, beta), gate), stream


class Stack(nn.Module):
    """Layers and the norm after the last."""

    def __init__(self, width, layers, **sizes):
        super().__init__()
        self.layers = nn.ModuleList(Layer(width, **sizes) for _ in range(layers))
        self.norm = nn.Parameter(torch.ones(width))
        self.norm_bias = nn.Parameter(torch.zeros(width))

    def forward(self, x, first=None):
        stream = None
        for layer in self.layers:
            x, stream = layer(x, stream, first)
        return layernorm_residual(x, self.norm, self.norm_bias, stream)[0]


class Served:
    """A trained stack in ``dtype``, and the states of a batch of users, in float32."""

    @torch.no_grad()
    def __init__(self, stack, batch, dtype=torch.bfloat16):
        self.stack, self.dtype = stack, dtype
        device = stack.norm.device
        self.convs = [(p.conv.detach().to(dtype), p.conv_bias.detach().to(dtype)) for p in stack.layers]
        self.states = [torch.zeros(batch, p.heads, p.value, p.key, device=device) for p in stack.layers]
        self.windows = [torch.zeros(batch, p.mixed, p.conv.shape[1] - 1, dtype=dtype, device=device) for p in stack.layers]

    def _run(self, x, mix):
        x, stream = x.to(self.dtype), None
        for i, p in enumerate(self.stack.layers):
            out, stream = layernorm_residual(x, p.norm, p.norm_bias, stream)
            mixed, gate, decay, beta = p.project(out)
            x = p.finish(mix(i, p, mixed, decay, beta), gate)
        return layernorm_residual(x, self.stack.norm, self.stack.norm_bias, stream)[0]

    @torch.no_grad()
    def prompt(self, x):
        """Outputs of ``(batch, length, width)``; the states move to the prompt's end."""
        def mix(i, p, mixed, decay, beta):
            mixed, self.windows[i] = causal_conv1d_fn(mixed.transpose(1, 2), *self.convs[i], activation="silu",
                                                      initial_state=self.windows[i], return_final_state=True)
            y, self.states[i] = gated_delta_rule(*p.split(mixed.transpose(1, 2)), decay, beta,
                                                 initial_state=self.states[i], return_final_state=True)
            return y

        return self._run(x, mix)

    @torch.no_grad()
    def token(self, x):
        """Outputs of one token of each user, ``(batch, width)``; the states move on in place."""
        def mix(i, p, mixed, decay, beta):
            mixed = causal_conv1d_update(mixed, self.windows[i], *self.convs[i], activation="silu")
            return gated_delta_rule_update(self.states[i], *p.split(mixed), decay, beta, out_state=self.states[i])[0]

        return self._run(x, mix)


def main():
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--width", type=int, default=256)
    ap.add_argument("--layers", type=int, default=2)
    ap.add_argument("--steps", type=int, default=20)
    args = ap.parse_args()
    torch.manual_seed(0)
    stack = Stack(args.width, args.layers).cuda()
    optimiser = torch.optim.Adam(stack.parameters(), lr=1e-3)
    first = torch.zeros(4, 256, dtype=torch.bool, device="cuda")
    first[:, 128] = True  # two documents a row
    for step in range(args.steps):
        x = torch.randn(4, 256, args.width, device="cuda")
        target = torch.roll(x, 1, 1)
        loss = (stack(x, first) - target).square().mean()
        optimiser.zero_grad()
        loss.backward()
        optimiser.step()
        if step % 5 == 0 or step + 1 == args.steps:
            print(f"step {step}: loss {loss.item():.4f}", flush=True)
    x = torch.randn(2, 100, args.width, device="cuda")
    with torch.no_grad():
        want = stack(x)
    served = Served(stack, 2)
    got = torch.cat([served.prompt(x[:, :90])] + [served.token(x[:, t])[:, None] for t in range(90, 100)], 1)
    for name, part in (("prompt", slice(0, 90)), ("tokens", slice(90, 100))):
        off = (got[:, part].float() - want[:, part]).norm() / want[:, part].norm()
        print(f"bfloat16 {name}: off the float32 outputs by {off.item():.4f} of their norm")


if __name__ == "__main__":
    main()
