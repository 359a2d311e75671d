"""Gated linear recurrence on MI355X: the scan over a sequence, its gradients, and one decode step.

Per channel, with ``rate = scale * softplus(decay)``::

    v = rate * sigmoid(decay_gate)
    a = exp(-v),  m = sqrt(1 - exp(-2 v))
    h[t] = a[t] * h[t-1] + m[t] * sigmoid(input_gate[t]) * x[t],   y = h

``m`` keeps the state's variance at that of its input: ``a^2 + m^2 = 1``.  At a step marked in
``reset`` the state before it is dropped (``a = 0``, ``m = 1``), so documents packed in one row do
not see each other.

Layouts: ``x`` and both gates ``(batch, length, channels)`` in one of float32, float16 and
bfloat16, with any batch and step strides (slices of one projection are read in place); ``decay``
``(channels,)``; states ``(batch, channels)``, float32 in :func:`gated_recurrence`.  The state is
float32 throughout and ``y`` is rounded once.  The gradients are analytic, once-differentiable and
summed in a fixed order, so repeated runs give the same bits.  There is no counterpart in
dbydd/metal-kernelops.
"""

from __future__ import annotations

import ctypes

import torch
from torch.autograd.function import once_differentiable

from .. import _native as nat
from .._contract import Rules
from ..scan import _require_gpu

__all__ = ["gated_recurrence", "gated_recurrence_reference", "gated_recurrence_update",
           "gated_recurrence_update_reference"]

_FLOATS = (torch.float32, torch.float16, torch.bfloat16)


def _params(x, input_gate, decay_gate, decay, initial, reset, scale):
    p = nat.RecurParams()
    p.x, p.input_gate, p.decay_gate = x.data_ptr(), input_gate.data_ptr(), decay_gate.data_ptr()
    p.decay, p.initial, p.reset = decay.data_ptr(), nat.ptr(initial), nat.ptr(reset)
    p.batch, p.length, p.channels = x.shape
    p.x_stride_b, p.x_stride_t = x.stride(0), x.stride(1)
    p.ig_stride_b, p.ig_stride_t = input_gate.stride(0), input_gate.stride(1)
    p.rg_stride_b, p.rg_stride_t = decay_gate.stride(0), decay_gate.stride(1)
    p.scale, p.dtype = scale, nat.code(x.dtype)
    return p


def _forward(x, input_gate, decay_gate, decay, initial, reset, scale, want_final):
    """``(y, final, states)``; ``states`` is what the backward reads, ``final`` None if unwanted."""
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    final = None
    if x.shape[1] == 0:
        if want_final:
            final = initial.clone() if initial is not None else x.new_zeros((x.shape[0], x.shape[2]),
                                                                            dtype=torch.float32)
        return y, final, None
    if want_final:
        final = torch.empty((x.shape[0], x.shape[2]), dtype=torch.float32, device=x.device)
    if y.numel() == 0:
        return y, final, None
    lib = nat.lib()
    p = _params(x, input_gate, decay_gate, decay, initial, reset, scale)
    at = ctypes.byref(p)
    states = nat.workspace(lib.mko_recur_states_size(at), x.device)
    size = lib.mko_recur_fwd_workspace_size(at)
    ws = nat.workspace(size, x.device) if size else None
    p.y, p.final_state, p.states = y.data_ptr(), nat.ptr(final), states.data_ptr()
    p.workspace, p.workspace_bytes = nat.ptr(ws), size
    with nat.on_device(x.device):
        nat.check(lib.mko_recur_fwd(at, nat.stream_of(x.device)), "mko_recur_fwd")
    return y, final, states


class _Recurrence(torch.autograd.Function):
    """Forward and analytic first-order backward through the C ABI."""

    @staticmethod
    def forward(ctx, x, input_gate, decay_gate, decay, initial, reset, scale):
        y, final, states = _forward(x, input_gate, decay_gate, decay, initial, reset, scale, True)
        ctx.save_for_backward(x, input_gate, decay_gate, decay, initial, reset, states)
        ctx.scale = scale
        ctx.set_materialize_grads(False)  # an unused output reaches backward as None
        return y, final

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dfinal):
        x, input_gate, decay_gate, decay, initial, reset, states = ctx.saved_tensors
        need = ctx.needs_input_grad
        dfinal = None if dfinal is None else nat.values(dfinal).contiguous()
        dx, dig, drg = (torch.empty(x.shape, dtype=x.dtype, device=x.device) for _ in range(3))
        ddecay = torch.zeros_like(decay) if need[3] else None
        dinitial = None
        if initial is not None and need[4]:
            dinitial = torch.zeros_like(initial) if dfinal is None else dfinal.clone()
        if x.numel():
            dy = torch.zeros_like(dx) if dy is None else nat.values(dy).contiguous()
            lib = nat.lib()
            p = _params(x, input_gate, decay_gate, decay, initial, reset, ctx.scale)
            at = ctypes.byref(p)
            p.states, p.dy, p.dfinal = states.data_ptr(), dy.data_ptr(), nat.ptr(dfinal)
            p.dx, p.dinput_gate, p.ddecay_gate = dx.data_ptr(), dig.data_ptr(), drg.data_ptr()
            p.ddecay, p.dinitial = nat.ptr(ddecay), nat.ptr(dinitial)
            size = lib.mko_recur_bwd_workspace_size(at)
            ws = nat.workspace(size, x.device) if size else None
            p.workspace, p.workspace_bytes = nat.ptr(ws), size
            with nat.on_device(x.device):
                nat.check(lib.mko_recur_bwd(at, nat.stream_of(x.device)), "mko_recur_bwd")
        return dx, dig, drg, ddecay, dinitial, None, None


def _check(op, x, input_gate, decay_gate, decay, scale, layout):
    """The argument rules that the scan and the update share, in their order."""
    rules = Rules(op)
    rules.dims("x", x, len(layout), f"({', '.join(layout)})")
    rules.shape("input_gate", input_gate, tuple(x.shape))
    rules.shape("decay_gate", decay_gate, tuple(x.shape))
    rules.shape("decay", decay, (x.shape[-1],))
    _require_gpu(x)
    rules.same_device(x.device, input_gate=input_gate, decay_gate=decay_gate, decay=decay)
    rules.dtype_in(_FLOATS, x=x)
    rules.dtype_in((x.dtype,), input_gate=input_gate, decay_gate=decay_gate)
    rules.require(decay.is_floating_point(), f"decay should be a floating tensor; it is {decay.dtype}")
    rules.require(scale > 0, f"scale should be positive; it is {scale}")
    return rules


def _f32(t):
    return None if t is None else nat.values(t if t.dtype == torch.float32 else t.float()).contiguous()


def gated_recurrence(x, input_gate, decay_gate, decay, initial_state=None, reset=None, scale=8.0,
                     return_final_state=False):
    """The gated linear recurrence over a sequence (the module notes have the formulas).

    Args:
        x: ``(batch, length, channels)``, float32, float16 or bfloat16 on the ROCm GPU.
        input_gate: its shape and dtype; the input's gate before the logistic function.
        decay_gate: its shape and dtype; the decay's gate before the logistic function.
        decay: ``(channels,)``, any float dtype (read as float32); ``scale * softplus(decay)`` is
            the channel's largest log decay a step.
        initial_state: ``(batch, channels)`` state before the first step, or None for zeros.
        reset: ``(batch, length)`` bool, True where a step drops the state before it, or None.
        scale: the factor of the log decay.
        return_final_state: also return the float32 state after the last step.

    Returns:
        ``y`` in ``x.dtype``, or ``(y, final_state)``.
    """
    rules = _check("gated_recurrence", x, input_gate, decay_gate, decay, scale, ("batch", "length", "channels"))
    batch, length, channels = x.shape
    rules.require(batch <= 65535, f"batch is at most 65535 (got {batch})")
    rules.shape("initial_state", initial_state, (batch, channels))
    rules.shape("reset", reset, (batch, length))
    rules.same_device(x.device, initial_state=initial_state, reset=reset)
    if initial_state is not None:
        rules.require(initial_state.is_floating_point(),
                      f"initial_state should be a floating tensor; it is {initial_state.dtype}")
    if reset is not None:
        rules.dtype_in((torch.bool,), reset=reset)
        reset = reset.contiguous()
    decay, initial = _f32(decay), _f32(initial_state)
    x, input_gate, decay_gate = nat.rows(x), nat.rows(input_gate), nat.rows(decay_gate)
    if torch.is_grad_enabled() and (x.requires_grad or input_gate.requires_grad or decay_gate.requires_grad
                                    or decay.requires_grad or (initial is not None and initial.requires_grad)):
        y, final = _Recurrence.apply(x, input_gate, decay_gate, decay, initial, reset, float(scale))
    else:
        y, final, _ = _forward(x, input_gate, decay_gate, decay, initial, reset, float(scale), return_final_state)
    return (y, final) if return_final_state else y


def gated_recurrence_update(state, x, input_gate, decay_gate, decay, scale=8.0, out_state=None):
    """Advance a state by one token; returns ``(y, new_state)``.

    ``state`` is ``(batch, channels)`` in float32, float16 or bfloat16 and is read, never written,
    unless it is passed again as ``out_state``; ``x`` and the gates are ``(batch, channels)`` in
    one of those dtypes, with any row stride, and ``y`` has theirs.  With ``out_state``
    (contiguous, the state's shape and dtype, not requiring grad) the new state is written there
    and returned as that tensor, outside the autograd graph; the state may be its own destination.
    The step is computed in float32; ``new_state`` and ``y`` are each rounded once.

    Where a gradient is wanted the step is a :func:`gated_recurrence` of length one.
    """
    rules = _check("gated_recurrence_update", x, input_gate, decay_gate, decay, scale, ("batch", "channels"))
    rules.shape("state", state, tuple(x.shape))
    rules.same_device(x.device, state=state, out_state=out_state)
    rules.dtype_in(_FLOATS, state=state)
    rules.require(x.shape[0] <= 65535, f"batch is at most 65535 (got {x.shape[0]})")
    if out_state is not None:
        rules.require(out_state.shape == state.shape and out_state.dtype == state.dtype,
                      "out_state should have the shape and dtype of state")
        rules.require(out_state.is_contiguous(), "out_state should be contiguous")
        rules.require(not out_state.requires_grad, "out_state is overwritten in place, so it may not require grad")
    if torch.is_grad_enabled() and any(t.requires_grad for t in (state, x, input_gate, decay_gate, decay)):
        y, final = gated_recurrence(x[:, None], input_gate[:, None], decay_gate[:, None], decay, initial_state=state,
                                    scale=scale, return_final_state=True)
        final = final.to(state.dtype)
        if out_state is None:
            return y[:, 0], final
        with torch.no_grad():
            out_state.copy_(final)
        return y[:, 0], out_state
    x, input_gate, decay_gate = nat.rows(x), nat.rows(input_gate), nat.rows(decay_gate)
    state, decay = nat.values(state).contiguous(), _f32(decay)
    new_state = out_state if out_state is not None else torch.empty_like(state)
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    if y.numel():
        p = nat.RecurUpdateParams(x.data_ptr(), input_gate.data_ptr(), decay_gate.data_ptr(), decay.data_ptr(),
                                  state.data_ptr(), new_state.data_ptr(), y.data_ptr(), x.shape[0], x.shape[1],
                                  x.stride(0), input_gate.stride(0), decay_gate.stride(0), scale,
                                  nat.code(x.dtype), nat.code(state.dtype))
        with nat.on_device(x.device):
            nat.check(nat.lib().mko_recur_update(ctypes.byref(p), nat.stream_of(x.device)), "mko_recur_update")
    return y, new_state


def _step(x, input_gate, decay_gate, decay, scale):
    v = scale * torch.nn.functional.softplus(decay) * torch.sigmoid(decay_gate)
    return torch.exp(-v), torch.sqrt(-torch.expm1(-2 * v)), torch.sigmoid(input_gate) * x


def gated_recurrence_reference(x, input_gate, decay_gate, decay, initial_state=None, reset=None, scale=8.0,
                               return_final_state=False):
    """The recurrence step by step in torch ops, on any device and float dtype; differentiable."""
    a, m, u = _step(x, input_gate, decay_gate, decay, scale)
    if reset is not None:
        a = torch.where(reset[..., None], torch.zeros_like(a), a)
        m = torch.where(reset[..., None], torch.ones_like(m), m)
    h = initial_state if initial_state is not None else torch.zeros_like(x[:, 0]) if x.shape[1] else \
        x.new_zeros((x.shape[0], x.shape[2]))
    out = []
    for t in range(x.shape[1]):
        h = a[:, t] * h + m[:, t] * u[:, t]
        out.append(h)
    y = torch.stack(out, 1) if out else torch.zeros_like(x)
    return (y, h) if return_final_state else y


def gated_recurrence_update_reference(state, x, input_gate, decay_gate, decay, scale=8.0):
    """One step in torch ops, on any device and float dtype; returns ``(y, new_state)``."""
    a, m, u = _step(x, input_gate, decay_gate, decay, scale)
    h = a * state + m * u
    return h, h
