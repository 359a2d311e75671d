"""Float64 CPU statements of the recurrent layer's operators (test oracle): the gated linear
recurrence with its analytic gradients, the RMS norm of the residual stream with its own, the
quantisation of rows and the integer product.  Nothing here is imported by the product."""

from __future__ import annotations

import torch

F64 = torch.float64


def _coefficients(x, input_gate, decay_gate, decay, reset, scale):
    si, sr = torch.sigmoid(input_gate.to(F64)), torch.sigmoid(decay_gate.to(F64))
    v = scale * torch.log1p(torch.exp(decay.to(F64))) * sr
    a, m = torch.exp(-v), torch.sqrt(-torch.expm1(-2 * v))
    if reset is not None:
        a = torch.where(reset[..., None], torch.zeros_like(a), a)
        m = torch.where(reset[..., None], torch.ones_like(m), m)
    return x.to(F64), si, sr, v, a, m


def gated_recurrence(x, input_gate, decay_gate, decay, initial=None, reset=None, scale=8.0):
    """``(y, final)`` in float64, step by step; differentiable."""
    x, si, _, _, a, m = _coefficients(x, input_gate, decay_gate, decay, reset, scale)
    h = torch.zeros_like(x[:, 0]) if initial is None else initial.to(F64)
    out = []
    for t in range(x.shape[1]):
        carried = a[:, t] * h
        if reset is not None:  # a dropped state is not read, be it NaN
            carried = torch.where(reset[:, t, None], torch.zeros_like(h), carried)
        h = carried + m[:, t] * si[:, t] * x[:, t]
        out.append(h)
    return torch.stack(out, 1), h


def gated_recurrence_bwd(dy, dfinal, x, input_gate, decay_gate, decay, initial=None, reset=None, scale=8.0):
    """``(dx, dinput_gate, ddecay_gate, ddecay, dinitial)`` from the formulas."""
    y, _ = gated_recurrence(x, input_gate, decay_gate, decay, initial, reset, scale)
    x, si, sr, v, a, m = _coefficients(x, input_gate, decay_gate, decay, reset, scale)
    h0 = torch.zeros_like(x[:, 0]) if initial is None else initial.to(F64)
    g = torch.zeros_like(h0) if dfinal is None else dfinal.to(F64)
    dx, dig, drg = torch.empty_like(x), torch.empty_like(x), torch.empty_like(x)
    ddecay = torch.zeros(x.shape[2], dtype=F64)
    for t in reversed(range(x.shape[1])):
        g = g + dy[:, t].to(F64)
        before = y[:, t - 1] if t else h0
        u = si[:, t] * x[:, t]
        slope = torch.where(m[:, t] > 0, a[:, t] ** 2 / m[:, t].clamp_min(1e-300), torch.zeros_like(u))
        dv = g * (u * slope - a[:, t] * before)
        back = g * a[:, t]
        if reset is not None:
            cut = reset[:, t, None]
            dv, back = (torch.where(cut, torch.zeros_like(q), q) for q in (dv, back))
        dx[:, t] = g * m[:, t] * si[:, t]
        dig[:, t] = g * m[:, t] * x[:, t] * si[:, t] * (1 - si[:, t])
        drg[:, t] = dv * v[:, t] * (1 - sr[:, t])
        ddecay += (dv * sr[:, t]).sum(0)
        g = back
    return dx, dig, drg, ddecay * scale * torch.sigmoid(decay.to(F64)), g


def rmsnorm_residual(x, weight, residual=None, eps=1e-5):
    """``(out, stream)`` in float64, the stream rounded to the residual's dtype."""
    stream = x.to(F64) if residual is None else (x.to(F64) + residual.to(F64)).to(residual.dtype).to(F64)
    return stream / torch.sqrt(stream.square().mean(-1, keepdim=True) + eps) * weight.to(F64), stream


def rmsnorm_residual_bwd(dout, dstream, stream, weight, eps=1e-5):
    """``(dstream_in, dweight)``: the gradient of ``x`` and of the residual, and the weight's."""
    s = stream.to(F64)
    r = 1 / torch.sqrt(s.square().mean(-1, keepdim=True) + eps)
    gw = dout.to(F64) * weight.to(F64)
    ds = r * (gw - s * r * (gw * s * r).mean(-1, keepdim=True))
    if dstream is not None:
        ds = ds + dstream.to(F64)
    return ds, (dout.to(F64) * s * r).reshape(-1, s.shape[-1]).sum(0)


def quantize_int8(x):
    """Rows in 8 bits with the two float32 roundings of the definition: ``(q, scale)``."""
    v = x.float()
    amax = v.abs().amax(-1)
    most = torch.full_like(amax, 127.0)  # number / tensor would be a reciprocal and a product
    inv = torch.where(amax > 0, most / amax, torch.zeros_like(amax))
    return torch.round(v * inv[..., None]).to(torch.int8), amax / most


def int8_linear(q, q_scale, weight, weight_scale, bias=None):
    """The integer product scaled in float64."""
    acc = torch.matmul(q.to(F64), weight.to(F64).t())
    out = acc * q_scale.to(F64)[..., None] * weight_scale.to(F64)
    return out if bias is None else out + bias.to(F64)
