"""Float64 CPU statement of the layer norm of the residual stream (test oracle), with its analytic
gradients.  Nothing here is imported by the product."""

from __future__ import annotations

import torch

F64 = torch.float64


def _parts(stream, eps):
    n = stream.shape[-1]
    d = stream - stream.sum(-1, keepdim=True) / n
    r = (d.pow(2).sum(-1, keepdim=True) / n + eps).pow(-0.5)
    return d * r, r


def layernorm_residual(x, weight, bias=None, residual=None, eps=1e-5):
    """``(out, stream)`` in float64, the stream rounded as it is stored."""
    stream = x.to(F64)
    if residual is not None:
        stream = stream + residual.to(F64)
        stream = stream.to(residual.dtype).to(F64)
    out = _parts(stream, eps)[0] * weight.to(F64)
    return out if bias is None else out + bias.to(F64), stream


def layernorm_residual_bwd(dout, dstream, stream, weight, eps=1e-5):
    """``(dstream_in, dweight, dbias)``: the first is x's and the residual's gradient."""
    dout, n = dout.to(F64), stream.shape[-1]
    xh, r = _parts(stream.to(F64), eps)
    gw = dout * weight.to(F64)
    ds = r * (gw - gw.sum(-1, keepdim=True) / n - xh * ((gw * xh).sum(-1, keepdim=True) / n))
    if dstream is not None:
        ds = ds + dstream.to(F64)
    return ds, (dout * xh).flatten(0, -2).sum(0), dout.flatten(0, -2).sum(0)
