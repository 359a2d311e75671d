"""RMS norm of the residual stream on MI355X, with an output in the activations' type or in 8 bits.

Per row of the last axis::

    stream = x + residual            rounded to the residual's dtype (x itself without a residual)
    out    = stream * rsqrt(mean(stream^2) + eps) * weight

:func:`rmsnorm_residual` returns ``(out, stream)`` and is differentiable;
:func:`rmsnorm_residual_int8` returns ``(q, scale, stream)``, the norm's output in 8-bit integers
with ``out ~ q * scale[..., None]``, which :func:`~metal_kernelops.cv.int8_linear` reads.

The norm is that of the stream as it is stored, the value that the next layer adds to, so the
backward, which reads the stored stream, differentiates exactly what the forward computed.  The
residual has ``x``'s dtype, or float32 beside 16-bit ``x``.  Sums are float32, and ``dweight`` is
summed over rows in a fixed order.  There is no counterpart in dbydd/metal-kernelops (its gated
RMSNorm, :func:`~metal_kernelops.cv.rmsnorm_gated`, has no residual).
"""

from __future__ import annotations

import ctypes

import torch
from torch.autograd.function import once_differentiable

from .. import _native as nat
from .._contract import Rules
from ..scan import _require_gpu
from .int8_linear import ALIGN, quantize_int8_reference

__all__ = ["rmsnorm_residual", "rmsnorm_residual_int8", "rmsnorm_residual_int8_reference",
           "rmsnorm_residual_reference"]

_FLOATS = (torch.float32, torch.float16, torch.bfloat16)


def _params(x, weight, residual, eps):
    p = nat.ResnormParams()
    p.x, p.weight, p.residual = x.data_ptr(), weight.data_ptr(), nat.ptr(residual)
    p.rows, p.features = x.shape
    p.x_stride, p.residual_stride = x.stride(0), 0 if residual is None else residual.stride(0)
    p.eps, p.dtype, p.wdtype = eps, nat.code(x.dtype), nat.code(weight.dtype)
    p.stream_dtype = nat.code(x.dtype if residual is None else residual.dtype)
    return p


def _launch_fwd(p, x):
    with nat.on_device(x.device):
        nat.check(nat.lib().mko_resnorm_fwd(ctypes.byref(p), nat.stream_of(x.device)), "mko_resnorm_fwd")


def _rows(t):
    return nat.rows(t.reshape(-1, t.shape[-1]))


def _forward(x, weight, residual, eps, want_rstd):
    """``(out, stream, rstd)``; stream is None without a residual."""
    out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    stream = None if residual is None else torch.empty(x.shape, dtype=residual.dtype, device=x.device)
    rstd = torch.empty(x.shape[:-1].numel(), dtype=torch.float32, device=x.device) if want_rstd else None
    if x.numel():
        x2 = _rows(x)
        p = _params(x2, weight, None if residual is None else _rows(residual), eps)
        p.out, p.stream, p.rstd = out.data_ptr(), nat.ptr(stream), nat.ptr(rstd)
        _launch_fwd(p, x)
    return out, stream, rstd


def _backward(dout, dstream, stream, weight, rstd, dtype, need_weight):
    """``(dx, dresidual, dweight)`` of dense operands; one tensor for both where the types agree."""
    dx = torch.empty(stream.shape, dtype=dtype, device=stream.device)
    dres = dx if stream.dtype == dtype else torch.empty(stream.shape, dtype=stream.dtype, device=stream.device)
    dweight = torch.zeros(weight.shape, dtype=torch.float32, device=stream.device) if need_weight else None
    if stream.numel():
        lib = nat.lib()
        p = nat.ResnormParams()
        at = ctypes.byref(p)
        p.stream, p.weight, p.rstd = stream.data_ptr(), weight.data_ptr(), rstd.data_ptr()
        p.dout, p.dstream, p.dx = dout.data_ptr(), nat.ptr(dstream), dx.data_ptr()
        p.dresidual, p.dweight = None if dres is dx else dres.data_ptr(), nat.ptr(dweight)
        p.features = stream.shape[-1]
        p.rows = stream.numel() // p.features
        p.dtype, p.stream_dtype, p.wdtype = nat.code(dtype), nat.code(stream.dtype), nat.code(weight.dtype)
        size = lib.mko_resnorm_bwd_workspace_size(at)
        ws = nat.workspace(size, stream.device) if size else None
        p.workspace, p.workspace_bytes = nat.ptr(ws), size
        with nat.on_device(stream.device):
            nat.check(lib.mko_resnorm_bwd(at, nat.stream_of(stream.device)), "mko_resnorm_bwd")
    return dx, dres, dweight


class _ResidualNorm(torch.autograd.Function):
    """Forward and analytic first-order backward through the C ABI.  It takes and returns whole
    shapes: x and the residual get one gradient tensor where their types agree, and autograd
    copies a tensor that two leaves receive but not one that reaches them as two views."""

    @staticmethod
    def forward(ctx, x, weight, residual, eps):
        out, stream, rstd = _forward(x, weight, residual, eps, True)
        ctx.save_for_backward(x if stream is None else stream, weight, rstd)
        ctx.dtype = x.dtype
        ctx.set_materialize_grads(False)  # an unused output reaches backward as None
        return out, stream

    @staticmethod
    @once_differentiable
    def backward(ctx, dout, dstream):
        stream, weight, rstd = ctx.saved_tensors
        need = ctx.needs_input_grad
        dstream = None if dstream is None else nat.values(dstream).contiguous()
        if dout is None:  # only the stream was used
            return (None if dstream is None else dstream.to(ctx.dtype), None, dstream if need[2] else None, None)
        dx, dres, dweight = _backward(nat.values(dout).contiguous(), dstream, nat.values(stream).contiguous(), weight,
                                      rstd, ctx.dtype, need[1])
        return dx, None if dweight is None else dweight.to(weight.dtype), dres if need[2] else None, None


def _checked(op, x, weight, residual):
    """The argument rules, in their order; returns the weight as the kernels read it."""
    rules = Rules(op)
    rules.require(x.dim() >= 1, "x needs a feature axis")
    rules.shape("weight", weight, (x.shape[-1],))
    rules.shape("residual", residual, tuple(x.shape))
    _require_gpu(x)
    rules.same_device(x.device, weight=weight, residual=residual)
    rules.dtype_in(_FLOATS, x=x, weight=weight)
    if residual is not None:
        rules.dtype_in((x.dtype, torch.float32), residual=residual)
    rows = x.shape[:-1].numel()
    rules.require(rows < 1 << 22, f"at most 2^22 - 1 rows (got {rows})")
    return nat.values(weight).contiguous()


def _wants_grad(*tensors):
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def rmsnorm_residual(x, weight, residual=None, eps=1e-5):
    """Add ``x`` to the residual stream and normalise it; returns ``(out, stream)``.

    Args:
        x: ``(..., features)``, float32, float16 or bfloat16 on the ROCm GPU, any row stride.
        weight: ``(features,)`` scale in one of those dtypes; its gradient has its dtype.
        residual: the stream so far, shaped like ``x``, of its dtype or float32; None for a first
            layer, where the stream is ``x`` and is returned as it is.
        eps: added to the mean square before the reciprocal square root.

    Returns:
        ``out`` in ``x.dtype`` and ``stream`` in the residual's.
    """
    w = _checked("rmsnorm_residual", x, weight, residual)
    if _wants_grad(x, weight, residual):
        out, stream = _ResidualNorm.apply(x, w, residual, float(eps))
    else:
        out, stream, _ = _forward(x, w, residual, float(eps), False)
    return out, x if residual is None else stream


def rmsnorm_residual_int8(x, weight, residual=None, eps=1e-5):
    """The same with the norm's output in 8 bits; returns ``(q, scale, stream)``.

    ``q`` is int8 ``(..., features)`` and ``scale`` float32 ``(...)``: per row
    ``scale = amax / 127`` and ``q = rint(v * 127 / amax)`` with ``v`` the float32 output before
    any rounding and ``amax`` its largest magnitude.  A row of zeros has scale 0; a row with an
    infinity or a NaN has a scale that is not finite.  Rows of ``q`` start at multiples of 16 bytes.
    For inference: arguments that require grad are refused while grad mode is on.
    """
    w = _checked("rmsnorm_residual_int8", x, weight, residual)
    Rules("rmsnorm_residual_int8").require(not _wants_grad(x, weight, residual),
                                           "8-bit outputs have no gradient; call it under torch.no_grad()")
    lead, features = x.shape[:-1], x.shape[-1]
    pitch = -(-features // ALIGN) * ALIGN
    q = torch.empty((*lead, pitch), dtype=torch.int8, device=x.device)
    scale = torch.empty(lead, dtype=torch.float32, device=x.device)
    stream = x if residual is None else torch.empty(x.shape, dtype=residual.dtype, device=x.device)
    if x.numel():
        p = _params(_rows(x), w, None if residual is None else _rows(residual), float(eps))
        p.q, p.q_scale, p.q_stride = q.data_ptr(), scale.data_ptr(), pitch
        p.stream = None if residual is None else stream.data_ptr()
        _launch_fwd(p, x)
    elif not features:
        scale.zero_()
    return q[..., :features], scale, stream


def rmsnorm_residual_reference(x, weight, residual=None, eps=1e-5):
    """The definition in float64 torch ops on any device: ``(out, stream)``; differentiable."""
    stream = x if residual is None else (x.double() + residual.double()).to(residual.dtype)
    s = stream.double()
    out = s * torch.rsqrt(s.square().mean(-1, keepdim=True) + eps) * weight.double()
    return out.to(x.dtype), stream


def rmsnorm_residual_int8_reference(x, weight, residual=None, eps=1e-5):
    """The definition in float64 torch ops on any device: ``(q, scale, stream)``."""
    stream = x if residual is None else (x.double() + residual.double()).to(residual.dtype)
    s = stream.double()
    q, scale = quantize_int8_reference(s * torch.rsqrt(s.square().mean(-1, keepdim=True) + eps) * weight.double())
    return q, scale, stream
