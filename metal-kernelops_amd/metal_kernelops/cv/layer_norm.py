"""Layer norm of the residual stream on MI355X.

Per row of the last axis::

    stream = x + residual            rounded to the residual's dtype (x itself without a residual)
    mu     = mean(stream)
    out    = (stream - mu) * rsqrt(mean((stream - mu)^2) + eps) * weight + bias

:func:`layernorm_residual` returns ``(out, stream)`` and is differentiable.  As in
:func:`~metal_kernelops.cv.rmsnorm_residual` the norm is that of the stream as it is stored, and the
backward, which reads the stored stream, differentiates exactly what the forward computed.  The
residual has ``x``'s dtype, or float32 beside 16-bit ``x``.  Sums are float32, the variance is that of
the differences from the mean, and ``dweight`` and ``dbias`` are summed over rows in a fixed order.  There
is no counterpart in dbydd/metal-kernelops.
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
from .residual_norm import _rows

__all__ = ["layernorm_residual", "layernorm_residual_reference"]

_FLOATS = (torch.float32, torch.float16, torch.bfloat16)


def _forward(x, weight, bias, residual, eps, want_stats):
    """``(out, stream, stats)``; stream is None without a residual."""
    out = nat.empty_as(x)
    stream = None if residual is None else nat.empty_as(residual)
    stats = torch.empty((*x.shape[:-1], 2), dtype=torch.float32, device=x.device) if want_stats else None
    if x.numel():
        (x, xs), (r, rs) = _rows(x), (None, 0) if residual is None else _rows(residual)
        features, code = x.shape[-1], nat.code(x.dtype)
        nat.launch("mko_layernorm_fwd", nat.LayernormParams(
            x.data_ptr(), nat.ptr(r), weight.data_ptr(), nat.ptr(bias), out.data_ptr(), nat.ptr(stream), nat.ptr(stats),
            None, None, None, None, None, None, None, 0, x.numel() // features, features, xs, rs, eps, code,
            code if r is None else nat.code(r.dtype), nat.code(weight.dtype),
            nat.F32 if bias is None else nat.code(bias.dtype)), x.device)
    return out, stream, stats


@functools.lru_cache(maxsize=256)
def _workspace(rows, features, dtype, stream_dtype):
    """Bytes of the backward's partial sums of dweight and dbias."""
    p = nat.LayernormParams(rows=rows, features=features, dtype=dtype, stream_dtype=stream_dtype, dweight=1)
    return nat.lib().mko_layernorm_bwd_workspace_size(ctypes.byref(p))


def _backward(dout, dstream, stream, weight, stats, dtype, need_weight, need_bias):
    """``(dx, dresidual, dweight, dbias)``; one tensor for the first two where the types agree, the last
    two None if unwanted."""
    dout, dstream, stream = nat.dense(dout), nat.dense(dstream), nat.dense(stream)
    device, dres = stream.device, nat.empty_as(stream)
    dx = dres if stream.dtype == dtype else torch.empty(stream.shape, dtype=dtype, device=device)
    dweight = torch.empty(weight.shape, dtype=torch.float32, device=device) if need_weight else None
    dbias = torch.empty(weight.shape, dtype=torch.float32, device=device) if need_bias else None
    if stream.numel():
        features = stream.shape[-1]
        rows, code, scode = stream.numel() // features, nat.code(dtype), nat.code(stream.dtype)
        space = None
        if need_weight or need_bias:
            space = torch.empty(_workspace(rows, features, code, scode), dtype=torch.uint8, device=device)
        nat.launch("mko_layernorm_bwd", nat.LayernormParams(
            None, None, weight.data_ptr(), None, None, stream.data_ptr(), stats.data_ptr(), dout.data_ptr(),
            nat.ptr(dstream), dx.data_ptr(), None if dres is dx else dres.data_ptr(), nat.ptr(dweight), nat.ptr(dbias),
            nat.ptr(space), 0 if space is None else space.numel(), rows, features, 0, 0, 0.0, code, scode,
            nat.code(weight.dtype), nat.F32), device)
    else:
        for t in (dweight, dbias):
            if t is not None:
                t.zero_()
    return dx, dres, dweight, dbias


def _grads(ctx, dout, dstream, _dstats=None):
    """The gradients of the inputs of :class:`_LayerNorm` and of the custom op."""
    stream, weight, stats = ctx.saved_tensors
    need = ctx.needs_input_grad
    if dout is None:  # only the stream was used
        return (None if dstream is None else dstream.to(ctx.dtype), None, None, dstream if need[3] else None, None)
    need_weight, need_bias = need[1], ctx.bias_dtype is not None and need[2]
    # a backward that is itself recorded goes through the op, which refuses to be differentiated
    op = ctx.through_op or torch.is_grad_enabled() or nat.watched(dout, dstream)
    backward = torch.ops.mko.layernorm_bwd if op else _backward
    dx, dres, dweight, dbias = backward(dout, dstream, stream, weight, stats, ctx.dtype, need_weight, need_bias)
    if stream.dtype == ctx.dtype:
        dres = dx
    dweight = dweight.to(weight.dtype) if need_weight else None
    dbias = dbias.to(ctx.bias_dtype) if need_bias else None
    return dx, dweight, dbias, dres if need[3] else None, None


class _LayerNorm(torch.autograd.Function):
    """Forward and analytic first-order backward through the C ABI.  It takes and returns whole
    shapes: x and the residual get one gradient tensor where their types agree, and autograd
    copies a tensor that two leaves receive but not one that reaches them as two views."""

    @staticmethod
    def forward(ctx, x, weight, bias, residual, eps):
        out, stream, stats = _forward(x, weight, bias, residual, eps, True)
        ctx.save_for_backward(x if stream is None else stream, weight, stats)
        ctx.dtype, ctx.bias_dtype, ctx.through_op = x.dtype, None if bias is None else bias.dtype, False
        ctx.set_materialize_grads(False)  # an unused output reaches backward as None
        return out, stream

    backward = staticmethod(_grads)


def _layernorm_fwd_op(x: Tensor, weight: Tensor, bias: Optional[Tensor], residual: Optional[Tensor], eps: float
                      ) -> Tuple[Tensor, Tensor, Tensor]:
    out, stream, stats = _forward(x, nat.dense(weight), nat.dense(bias), residual, eps, True)
    return out, nat.absent(stream, x), stats


_layernorm_fwd = torch.library.custom_op("mko::layernorm_fwd", _layernorm_fwd_op, mutates_args=(), device_types="cuda")


@_layernorm_fwd.register_fake
def _(x, weight, bias, residual, eps):
    return (x.new_empty(x.shape), x.new_empty(0) if residual is None else residual.new_empty(residual.shape),
            x.new_empty((*x.shape[:-1], 2), dtype=torch.float32))


def _layernorm_bwd_op(dout: Tensor, dstream: Optional[Tensor], stream: Tensor, weight: Tensor, stats: Tensor,
                      dtype: torch.dtype, need_weight: bool, need_bias: bool) -> Tuple[Tensor, Tensor, Tensor, Tensor]:
    dx, dres, dweight, dbias = _backward(dout, dstream, stream, nat.dense(weight), nat.dense(stats), dtype, need_weight,
                                         need_bias)
    return dx, nat.absent(None if dres is dx else dres, dx), nat.absent(dweight, stats), nat.absent(dbias, stats)


_layernorm_bwd = torch.library.custom_op("mko::layernorm_bwd", _layernorm_bwd_op, mutates_args=(), device_types="cuda")


@_layernorm_bwd.register_fake
def _(dout, dstream, stream, weight, stats, dtype, need_weight, need_bias):
    return (stream.new_empty(stream.shape, dtype=dtype), stream.new_empty(0 if stream.dtype == dtype else stream.shape),
            stats.new_empty(weight.shape if need_weight else 0), stats.new_empty(weight.shape if need_bias else 0))


def _setup(ctx, inputs, output):
    x, weight, bias, residual, _ = inputs
    ctx.save_for_backward(x if residual is None else output[1], weight, output[2])
    ctx.dtype, ctx.bias_dtype, ctx.through_op = x.dtype, None if bias is None else bias.dtype, True
    ctx.set_materialize_grads(False)


torch.library.register_autograd("mko::layernorm_fwd", _grads, setup_context=_setup)


def _checked(x, weight, bias, residual):
    """The argument rules, in their order.  Messages are formed only for an argument that breaks a rule:
    the checks are host time."""
    rules = Rules("layernorm_residual")
    if x.dim() < 1:
        rules.fail("x needs a feature axis")
    shape, device = x.shape, x.device
    if weight.shape != shape[-1:] or (bias is not None and bias.shape != shape[-1:]) \
            or (residual is not None and residual.shape != shape):
        rules.shape("weight", weight, shape[-1:])
        rules.shape("bias", bias, shape[-1:])
        rules.shape("residual", residual, shape)
    _require_gpu(x)
    if weight.device != device or (bias is not None and bias.device != device) \
            or (residual is not None and residual.device != device):
        rules.same_device(device, weight=weight, bias=bias, residual=residual)
    if x.dtype not in _FLOATS or weight.dtype not in _FLOATS or (bias is not None and bias.dtype not in _FLOATS):
        rules.dtype_in(_FLOATS, x=x, weight=weight, bias=bias)
    if residual is not None and residual.dtype != x.dtype:
        rules.dtype_in((x.dtype, torch.float32), residual=residual)
    if shape[:-1].numel() >= 1 << 22:
        rules.fail(f"at most 2^22 - 1 rows (got {shape[:-1].numel()})")
    if shape[-1] >= 1 << 30:
        rules.fail(f"at most 2^30 - 1 features (got {shape[-1]})")


def layernorm_residual(x, weight, bias=None, residual=None, eps=1e-5):
    """Add ``x`` to the residual stream and normalise it; returns ``(out, stream)``.

    Args:
        x: ``(..., features)``, float32, float16 or bfloat16 on the ROCm GPU, any row stride.
        weight: ``(features,)`` scale in one of those dtypes; its gradient has its dtype.
        bias: ``(features,)`` in one of those dtypes, or None.
        residual: the stream so far, shaped like ``x``, of its dtype or float32; None for a first
            layer, where the stream is ``x`` and is returned as it is.
        eps: added to the variance before the reciprocal square root.

    Returns:
        ``out`` in ``x.dtype`` and ``stream`` in the residual's.
    """
    _checked(x, weight, bias, residual)
    weight, bias, eps = nat.dense(weight), nat.dense(bias), float(eps)
    if nat.watched(x, weight, bias, residual):
        out, stream, _ = nat.through(torch.ops.mko.layernorm_fwd, x, weight, bias, residual, eps)
    elif nat.wants_grad(x, weight, bias, residual):
        out, stream = _LayerNorm.apply(x, weight, bias, residual, eps)
    else:
        out, stream, _ = _forward(x, weight, bias, residual, eps, False)
    return out, x if residual is None else stream


def layernorm_residual_reference(x, weight, bias=None, residual=None, eps=1e-5):
    """The definition in float64 torch ops on any device: ``(out, stream)``; differentiable."""
    stream = x if residual is None else (x.double() + residual.double()).to(residual.dtype)
    s = stream.double()
    s = s - s.mean(-1, keepdim=True)
    out = s * torch.rsqrt(s.square().mean(-1, keepdim=True) + eps) * weight.double()
    if bias is not None:
        out = out + bias.double()
    return out.to(x.dtype), stream
