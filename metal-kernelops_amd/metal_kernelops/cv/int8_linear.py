"""Projections in 8-bit integers on MI355X: quantisation of rows, and the matrix product.

A row (a token's activations, or an output channel's weights) is held as int8 with one float32
scale: ``scale = amax / 127`` and ``q = rint(x * (127 / amax))`` with ``amax`` the row's largest
magnitude.  The product of tokens ``(..., inner)`` and weights ``(outer, inner)`` is

    out[m, n] = q_scale[m] * weight_scale[n] * sum_k q[m, k] * weight[n, k] + bias[n]

on the int8 matrix cores.  The sum is exact in int32 (``inner`` below 2^17); the scales and the
bias are applied in float32 and the result is rounded once.  A row of zeros, or of magnitudes below
2^-100, has scale 0; a row with an infinity or a NaN has a scale that is not finite, and so are its
outputs.  There is no
counterpart in dbydd/metal-kernelops.
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch
from torch import Tensor

from .. import _native as nat
from .._contract import Rules
from ..scan import _require_gpu

__all__ = ["int8_linear", "int8_linear_reference", "quantize_int8", "quantize_int8_reference"]

ALIGN = 16
"""Bytes that the rows of quantised tensors start at multiples of: the product's widest loads."""

MAX_INNER = 131071
"""Longest sum of products of two bytes that stays inside int32."""

_FLOATS = (torch.float32, torch.float16, torch.bfloat16)


def _quantize(x: Tensor) -> Tuple[Tensor, Tensor]:
    """``(q, scale)``, q with its rows' padding."""
    features, lead = x.shape[-1], x.shape[:-1]
    pitch = -(-features // ALIGN) * ALIGN
    q = torch.empty((*lead, pitch), dtype=torch.int8, device=x.device)
    scale = torch.empty(lead, dtype=torch.float32, device=x.device)
    if scale.numel():
        if x.dim() != 2 and not x.is_contiguous():
            x = x.reshape(scale.numel(), features)
        x = nat.rows(x)
        nat.launch("mko_quantize_int8", nat.QuantizeParams(
            x.data_ptr(), q.data_ptr(), scale.data_ptr(), scale.numel(), features,
            x.stride(0) if x.dim() == 2 else features, pitch, nat.code(x.dtype)), x.device)
    return q, scale


_quantize_op = torch.library.custom_op("mko::quantize_int8", _quantize, mutates_args=(), device_types="cuda")


@_quantize_op.register_fake
def _(x):
    pitch = -(-x.shape[-1] // ALIGN) * ALIGN
    return x.new_empty((*x.shape[:-1], pitch), dtype=torch.int8), x.new_empty(x.shape[:-1], dtype=torch.float32)


def _linear(q: Tensor, q_scale: Tensor, weight: Tensor, weight_scale: Tensor, bias: Optional[Tensor],
            out_dtype: torch.dtype) -> Tensor:
    outer, inner = weight.shape
    out = torch.empty((*q.shape[:-1], outer), dtype=out_dtype, device=q.device)
    if out.numel():
        if inner:
            if q.dim() != 2 and not q.is_contiguous():
                q = q.reshape(-1, inner)
            q, weight = nat.rows(q), nat.rows(weight)
        qs, ws, b = nat.dense_f32(q_scale), nat.dense_f32(weight_scale), nat.dense_f32(bias)
        nat.launch("mko_int8_linear", nat.Int8LinearParams(
            q.data_ptr(), qs.data_ptr(), weight.data_ptr(), ws.data_ptr(), nat.ptr(b), out.data_ptr(),
            out.numel() // outer, inner, outer, q.stride(0) if q.dim() == 2 else inner, weight.stride(0),
            nat.code(out_dtype)), q.device)
    return out


_linear_op = torch.library.custom_op("mko::int8_linear", _linear, mutates_args=(), device_types="cuda")


@_linear_op.register_fake
def _(q, q_scale, weight, weight_scale, bias, out_dtype):
    return q.new_empty((*q.shape[:-1], weight.shape[0]), dtype=out_dtype)


def quantize_int8(x):
    """Rows of the last axis in 8 bits; returns ``(q, scale)``.

    ``x`` is ``(..., features)`` in float32, float16 or bfloat16 on the ROCm GPU, with any row
    stride; ``q`` is int8 of its shape, its rows at multiples of 16 bytes, and ``scale`` float32
    ``(...)``.  Used for activations that another operator produced, and once for weights
    ``(outer, inner)`` when a model is loaded.  There is no gradient: an ``x`` that requires grad
    is refused while grad mode is on.
    """
    rules = Rules("quantize_int8")
    if x.dim() < 1:
        rules.fail("x needs a feature axis")
    _require_gpu(x)
    if x.dtype not in _FLOATS:
        rules.dtype_in(_FLOATS, x=x)
    if nat.wants_grad(x):
        rules.fail("8-bit outputs have no gradient; call it under torch.no_grad()")
    features = x.shape[-1]
    if x.numel() >= features << 22 and x.shape[:-1].numel() >= 1 << 22:
        rules.fail(f"at most 2^22 - 1 rows (got {x.shape[:-1].numel()})")
    if nat.watched(x):
        q, scale = nat.through(torch.ops.mko.quantize_int8, x)
    else:
        q, scale = _quantize(x)
    return q if q.shape[-1] == features else q[..., :features], scale


def int8_linear(q, q_scale, weight, weight_scale, bias=None, out_dtype=torch.bfloat16):
    """Product of quantised tokens and quantised weights, scaled back.

    Args:
        q: int8 ``(..., inner)`` tokens on the ROCm GPU, any row stride; ``inner`` at most 131071.
        q_scale: ``(...)``, one scale for each token.
        weight: int8 ``(outer, inner)``, any row stride.
        weight_scale: ``(outer,)``, one scale for each output channel.
        bias: ``(outer,)`` added after the scales, or None.
        out_dtype: float32, float16 or bfloat16.

    Scales and bias are read as float32.  Returns ``(..., outer)``.  For inference: a scale or
    bias that requires grad is refused while grad mode is on.
    """
    rules = Rules("int8_linear")
    if q.dim() < 1:
        rules.fail("q needs an inner axis")
    if weight.dim() != 2:
        rules.dims("weight", weight, 2, "(outer, inner)")
    outer, inner = weight.shape
    lead = q.shape[:-1]
    if q.shape[-1] != inner:
        rules.fail(f"q has {q.shape[-1]} inner features, weight has {inner}")
    if q_scale.shape != lead or weight_scale.shape != (outer,) or (bias is not None and bias.shape != (outer,)):
        rules.shape("q_scale", q_scale, lead)
        rules.shape("weight_scale", weight_scale, (outer,))
        rules.shape("bias", bias, (outer,))
    _require_gpu(q)
    rules.same_device(q.device, q_scale=q_scale, weight=weight, weight_scale=weight_scale, bias=bias)
    if q.dtype != torch.int8 or weight.dtype != torch.int8:
        rules.dtype_in((torch.int8,), q=q, weight=weight)
    for name, t in (("q_scale", q_scale), ("weight_scale", weight_scale), ("bias", bias)):
        if t is not None:
            if not t.is_floating_point():
                rules.fail(f"{name} should be a floating tensor; it is {t.dtype}")
            if nat.wants_grad(t):
                rules.fail(f"{name} requires grad, and this product has no gradient; call it under torch.no_grad()")
    if out_dtype not in _FLOATS:
        rules.fail(f"out_dtype should be float32, float16 or bfloat16; it is {out_dtype}")
    if inner > MAX_INNER:
        rules.fail(f"inner is at most {MAX_INNER} here (got {inner})")
    if nat.watched(q, q_scale, weight, weight_scale, bias):
        return nat.through(torch.ops.mko.int8_linear, q, q_scale, weight, weight_scale, bias, out_dtype)
    return _linear(q, q_scale, weight, weight_scale, bias, out_dtype)


def quantize_int8_reference(x):
    """The definition in float64 torch ops on any device: ``(q, scale)``."""
    v = x.double()
    amax = v.abs().amax(-1) if x.shape[-1] else v.new_zeros(x.shape[:-1])
    safe = torch.where(amax > 0, amax, torch.ones_like(amax))
    return torch.round(v * (127.0 / safe)[..., None]).to(torch.int8), (amax / 127.0).float()


def int8_linear_reference(q, q_scale, weight, weight_scale, bias=None, out_dtype=torch.bfloat16):
    """The definition in float64 torch ops on any device."""
    out = (q.double() @ weight.double().t()) * q_scale.double()[..., None] * weight_scale.double()
    return (out if bias is None else out + bias.double()).to(out_dtype)
