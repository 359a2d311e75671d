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
import functools
from typing import Optional, Tuple

import torch
from torch import Tensor

from .. import _native as nat
from .._contract import Rules
from ..scan import _require_gpu
from .int8_linear import ALIGN, quantize_int8_reference

__all__ = ["rmsnorm_residual", "rmsnorm_residual_int8", "rmsnorm_residual_int8_reference",
           "rmsnorm_residual_reference"]

_FLOATS = (torch.float32, torch.float16, torch.bfloat16)


def _rows(t):
    """The rows of ``t`` at one stride: ``t`` itself where it has them, as a 2-d view or a copy."""
    if t.is_contiguous():
        return t, t.shape[-1]
    t = nat.rows(t if t.dim() == 2 else t.reshape(-1, t.shape[-1]))
    return t, t.stride(0)


def _launch_fwd(x, weight, residual, out, q, scale, stream, rstd, pitch, eps):
    (x, xs), (r, rs) = _rows(x), (None, 0) if residual is None else _rows(residual)
    features = x.shape[-1]
    nat.launch("mko_resnorm_fwd", nat.ResnormParams(
        x.data_ptr(), nat.ptr(r), weight.data_ptr(), nat.ptr(out), nat.ptr(q), nat.ptr(scale), nat.ptr(stream),
        nat.ptr(rstd), None, None, None, None, None, None, 0, x.numel() // features, features, xs, rs, pitch, eps,
        nat.code(x.dtype), nat.code(x.dtype if r is None else r.dtype), nat.code(weight.dtype)), x.device)


def _forward(x, weight, residual, eps, want_rstd):
    """``(out, stream, rstd)``; stream is None without a residual."""
    out = nat.empty_as(x)
    stream = None if residual is None else nat.empty_as(residual)
    rstd = torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device) if want_rstd else None
    if x.numel():
        _launch_fwd(x, weight, residual, out, None, None, stream, rstd, 0, eps)
    return out, stream, rstd


@functools.lru_cache(maxsize=256)
def _workspace(rows, features, dtype, stream_dtype):
    """Bytes of the backward's partial sums of dweight."""
    p = nat.ResnormParams(rows=rows, features=features, dtype=dtype, stream_dtype=stream_dtype, dweight=1)
    return nat.lib().mko_resnorm_bwd_workspace_size(ctypes.byref(p))


def _backward(dout, dstream, stream, weight, rstd, dtype, need_weight):
    """``(dx, dresidual, dweight)``; one tensor for both where the types agree."""
    dout, dstream, stream = nat.dense(dout), nat.dense(dstream), nat.dense(stream)
    device, dres = stream.device, nat.empty_as(stream)
    dx = dres if stream.dtype == dtype else torch.empty(stream.shape, dtype=dtype, device=device)
    dweight = torch.empty(weight.shape, dtype=torch.float32, device=device) if need_weight else None
    if stream.numel():
        features = stream.shape[-1]
        rows, code, scode = stream.numel() // features, nat.code(dtype), nat.code(stream.dtype)
        space = None
        if need_weight:
            space = torch.empty(_workspace(rows, features, code, scode), dtype=torch.uint8, device=device)
        nat.launch("mko_resnorm_bwd", nat.ResnormParams(
            None, None, weight.data_ptr(), None, None, None, stream.data_ptr(), rstd.data_ptr(), dout.data_ptr(),
            nat.ptr(dstream), dx.data_ptr(), None if dres is dx else dres.data_ptr(), nat.ptr(dweight), nat.ptr(space),
            0 if space is None else space.numel(), rows, features, 0, 0, 0, 0.0, code, scode, nat.code(weight.dtype)),
            device)
    elif need_weight:
        dweight.zero_()
    return dx, dres, dweight


def _grads(ctx, dout, dstream, _drstd=None):
    """The gradients of the inputs of :class:`_ResidualNorm` and of the custom op."""
    stream, weight, rstd = ctx.saved_tensors
    need = ctx.needs_input_grad
    if dout is None:  # only the stream was used
        return (None if dstream is None else dstream.to(ctx.dtype), None, dstream if need[2] else None, None)
    # a backward that is itself recorded goes through the op, which refuses to be differentiated
    op = ctx.through_op or torch.is_grad_enabled() or nat.watched(dout, dstream)
    backward = torch.ops.mko.resnorm_bwd if op else _backward
    dx, dres, dweight = backward(dout, dstream, stream, weight, rstd, ctx.dtype, need[1])
    if stream.dtype == ctx.dtype:
        dres = dx
    if not need[1]:
        dweight = None
    elif weight.dtype != torch.float32:
        dweight = dweight.to(weight.dtype)
    return dx, dweight, dres if need[2] else None, None


class _ResidualNorm(torch.autograd.Function):
    """Forward and analytic first-order backward through the C ABI.  It takes and returns whole
    shapes: x and the residual get one gradient tensor where their types agree, and autograd
    copies a tensor that two leaves receive but not one that reaches them as two views."""

    @staticmethod
    def forward(ctx, x, weight, residual, eps):
        out, stream, rstd = _forward(x, weight, residual, eps, True)
        ctx.save_for_backward(x if stream is None else stream, weight, rstd)
        ctx.dtype, ctx.through_op = x.dtype, False
        ctx.set_materialize_grads(False)  # an unused output reaches backward as None
        return out, stream

    backward = staticmethod(_grads)


def _resnorm_fwd_op(x: Tensor, weight: Tensor, residual: Optional[Tensor], eps: float
                    ) -> Tuple[Tensor, Tensor, Tensor]:
    out, stream, rstd = _forward(x, nat.dense(weight), residual, eps, True)
    return out, nat.absent(stream, x), rstd


_resnorm_fwd = torch.library.custom_op("mko::resnorm_fwd", _resnorm_fwd_op, mutates_args=(), device_types="cuda")


@_resnorm_fwd.register_fake
def _(x, weight, residual, eps):
    return (x.new_empty(x.shape), x.new_empty(0) if residual is None else residual.new_empty(residual.shape),
            x.new_empty(x.shape[:-1], dtype=torch.float32))


def _resnorm_bwd_op(dout: Tensor, dstream: Optional[Tensor], stream: Tensor, weight: Tensor, rstd: Tensor,
                    dtype: torch.dtype, need_weight: bool) -> Tuple[Tensor, Tensor, Tensor]:
    dx, dres, dweight = _backward(dout, dstream, stream, nat.dense(weight), nat.dense(rstd), dtype, need_weight)
    return dx, nat.absent(None if dres is dx else dres, dx), nat.absent(dweight, rstd)


_resnorm_bwd = torch.library.custom_op("mko::resnorm_bwd", _resnorm_bwd_op, mutates_args=(), device_types="cuda")


@_resnorm_bwd.register_fake
def _(dout, dstream, stream, weight, rstd, dtype, need_weight):
    return (stream.new_empty(stream.shape, dtype=dtype),
            stream.new_empty(0 if stream.dtype == dtype else stream.shape),
            rstd.new_empty(weight.shape if need_weight else 0))


def _setup(ctx, inputs, output):
    x, weight, residual, _ = inputs
    ctx.save_for_backward(x if residual is None else output[1], weight, output[2])
    ctx.dtype, ctx.through_op = x.dtype, True
    ctx.set_materialize_grads(False)


torch.library.register_autograd("mko::resnorm_fwd", _grads, setup_context=_setup)


def _int8(x, weight, residual, eps):
    """``(q, scale, stream)``, q with its rows' padding; stream is None without a residual."""
    lead, features = x.shape[:-1], x.shape[-1]
    pitch = -(-features // ALIGN) * ALIGN
    q = torch.empty((*lead, pitch), dtype=torch.int8, device=x.device)
    scale = torch.empty(lead, dtype=torch.float32, device=x.device)
    stream = None if residual is None else nat.empty_as(residual)
    if x.numel():
        _launch_fwd(x, weight, residual, None, q, scale, stream, None, pitch, eps)
    elif not features:
        scale.zero_()
    return q, scale, stream


def _resnorm_int8_op(x: Tensor, weight: Tensor, residual: Optional[Tensor], eps: float
                     ) -> Tuple[Tensor, Tensor, Tensor]:
    q, scale, stream = _int8(x, nat.dense(weight), residual, eps)
    return q, scale, nat.absent(stream, x)


_resnorm_int8 = torch.library.custom_op("mko::resnorm_int8", _resnorm_int8_op, mutates_args=(), device_types="cuda")


@_resnorm_int8.register_fake
def _(x, weight, residual, eps):
    lead, features = x.shape[:-1], x.shape[-1]
    return (x.new_empty((*lead, -(-features // ALIGN) * ALIGN), dtype=torch.int8),
            x.new_empty(lead, dtype=torch.float32),
            x.new_empty(0) if residual is None else residual.new_empty(residual.shape))


def _checked(op, x, weight, residual):
    """The argument rules, in their order; returns the weight as the kernels read it.  Messages are
    formed only for an argument that breaks a rule: the checks are host time."""
    rules = Rules(op)
    if x.dim() < 1:
        rules.fail("x needs a feature axis")
    shape, device = x.shape, x.device
    if weight.shape != shape[-1:] or (residual is not None and residual.shape != shape):
        rules.shape("weight", weight, shape[-1:])
        rules.shape("residual", residual, shape)
    _require_gpu(x)
    if weight.device != device or (residual is not None and residual.device != device):
        rules.same_device(device, weight=weight, residual=residual)
    if x.dtype not in _FLOATS or weight.dtype not in _FLOATS:
        rules.dtype_in(_FLOATS, x=x, weight=weight)
    if residual is not None and residual.dtype != x.dtype:
        rules.dtype_in((x.dtype, torch.float32), residual=residual)
    if shape[:-1].numel() >= 1 << 22:
        rules.fail(f"at most 2^22 - 1 rows (got {shape[:-1].numel()})")
    return nat.dense(weight)


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
    eps = float(eps)
    if nat.watched(x, w, residual):
        out, stream, _ = nat.through(torch.ops.mko.resnorm_fwd, x, w, residual, eps)
    elif nat.wants_grad(x, w, residual):
        out, stream = _ResidualNorm.apply(x, w, residual, eps)
    else:
        out, stream, _ = _forward(x, w, residual, eps, False)
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
    if nat.wants_grad(x, weight, residual):
        Rules("rmsnorm_residual_int8").fail("8-bit outputs have no gradient; call it under torch.no_grad()")
    if nat.watched(x, w, residual):
        q, scale, stream = nat.through(torch.ops.mko.resnorm_int8, x, w, residual, float(eps))
    else:
        q, scale, stream = _int8(x, w, residual, float(eps))
    features = x.shape[-1]
    return q if q.shape[-1] == features else q[..., :features], scale, x if residual is None else stream


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
