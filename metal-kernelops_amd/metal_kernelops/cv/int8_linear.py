"""Projections in 8-bit integers on MI355X: quantisation of rows, and the matrix product.

A row (a token's activations, or an output channel's weights) is held as int8 with one float32
scale: ``scale = amax / 127`` and ``q = rint(x * (127 / amax))`` with ``amax`` the row's largest
magnitude.  The product of tokens ``(..., inner)`` and weights ``(outer, inner)`` is

    out[m, n] = q_scale[m] * weight_scale[n] * sum_k q[m, k] * weight[n, k] + bias[n]

on the int8 matrix cores.  The sum is exact in int32 (``inner`` below 2^17); the scales and the
bias are applied in float32 and the result is rounded once.  A row of zeros has scale 0; a row
with an infinity or a NaN has a scale that is not finite, and so are its outputs.  There is no
counterpart in dbydd/metal-kernelops.
"""

from __future__ import annotations

import ctypes

import torch

from .. import _native as nat
from .._contract import Rules
from ..scan import _require_gpu

__all__ = ["int8_linear", "int8_linear_reference", "quantize_int8", "quantize_int8_reference"]

ALIGN = 16
"""Bytes that the rows of quantised tensors start at multiples of: the product's widest loads."""

MAX_INNER = 131071
"""Longest sum of products of two bytes that stays inside int32."""

_FLOATS = (torch.float32, torch.float16, torch.bfloat16)


def quantize_int8(x):
    """Rows of the last axis in 8 bits; returns ``(q, scale)``.

    ``x`` is ``(..., features)`` in float32, float16 or bfloat16 on the ROCm GPU, with any row
    stride; ``q`` is int8 of its shape, its rows at multiples of 16 bytes, and ``scale`` float32
    ``(...)``.  Used for activations that another operator produced, and once for weights
    ``(outer, inner)`` when a model is loaded.  There is no gradient: an ``x`` that requires grad
    is refused while grad mode is on.
    """
    rules = Rules("quantize_int8")
    rules.require(x.dim() >= 1, "x needs a feature axis")
    _require_gpu(x)
    rules.dtype_in(_FLOATS, x=x)
    rules.require(not (torch.is_grad_enabled() and x.requires_grad),
                  "8-bit outputs have no gradient; call it under torch.no_grad()")
    features, lead = x.shape[-1], x.shape[:-1]
    x2 = nat.rows(x.reshape(-1, features)) if features else x.reshape(lead.numel(), 0)
    rows = x2.shape[0]
    rules.require(rows < 1 << 22, f"at most 2^22 - 1 rows (got {rows})")
    pitch = -(-features // ALIGN) * ALIGN
    q = torch.empty((rows, pitch), dtype=torch.int8, device=x.device)
    if not features:
        return q.view(*lead, 0), x.new_zeros(lead, dtype=torch.float32)
    scale = torch.empty(rows, dtype=torch.float32, device=x.device)
    if rows:
        p = nat.QuantizeParams(x2.data_ptr(), q.data_ptr(), scale.data_ptr(), rows, features, x2.stride(0), pitch,
                               nat.code(x.dtype))
        with nat.on_device(x.device):
            nat.check(nat.lib().mko_quantize_int8(ctypes.byref(p), nat.stream_of(x.device)), "mko_quantize_int8")
    return q.view(*lead, pitch)[..., :features], scale.view(lead)


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
    rules.require(q.dim() >= 1, "q needs an inner axis")
    rules.dims("weight", weight, 2, "(outer, inner)")
    outer, inner = weight.shape
    lead = q.shape[:-1]
    rules.require(q.shape[-1] == inner, f"q has {q.shape[-1]} inner features, weight has {inner}")
    rules.shape("q_scale", q_scale, tuple(lead))
    rules.shape("weight_scale", weight_scale, (outer,))
    rules.shape("bias", bias, (outer,))
    _require_gpu(q)
    rules.same_device(q.device, q_scale=q_scale, weight=weight, weight_scale=weight_scale, bias=bias)
    rules.dtype_in((torch.int8,), q=q, weight=weight)
    for name, t in (("q_scale", q_scale), ("weight_scale", weight_scale), ("bias", bias)):
        if t is not None:
            rules.require(t.is_floating_point(), f"{name} should be a floating tensor; it is {t.dtype}")
            rules.require(not (torch.is_grad_enabled() and t.requires_grad),
                          f"{name} requires grad, and this product has no gradient; call it under torch.no_grad()")
    rules.require(out_dtype in _FLOATS, f"out_dtype should be float32, float16 or bfloat16; it is {out_dtype}")
    rules.require(inner <= MAX_INNER, f"inner is at most {MAX_INNER} here (got {inner})")
    q2 = nat.rows(q.reshape(-1, inner)) if inner else q.reshape(lead.numel(), 0)
    rows = q2.shape[0]
    out = torch.empty((rows, outer), dtype=out_dtype, device=q.device)
    if rows and outer:
        weight, qs, ws, b = nat.rows(weight) if inner else weight, _f32(q_scale), _f32(weight_scale), _f32(bias)
        lib = nat.lib()
        p = nat.Int8LinearParams(q2.data_ptr(), qs.data_ptr(), weight.data_ptr(), ws.data_ptr(), nat.ptr(b),
                                 out.data_ptr(), None, 0, rows, inner, outer, q2.stride(0), weight.stride(0),
                                 nat.code(out_dtype))
        size = lib.mko_int8_linear_workspace_size(ctypes.byref(p))
        if size:
            space = nat.workspace(size, q.device)
            p.workspace, p.workspace_bytes = space.data_ptr(), size
        with nat.on_device(q.device):
            nat.check(lib.mko_int8_linear(ctypes.byref(p), nat.stream_of(q.device)), "mko_int8_linear")
    return out.view(*lead, outer)


def _f32(t):
    return None if t is None else nat.values(t if t.dtype == torch.float32 else t.float()).contiguous()


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
