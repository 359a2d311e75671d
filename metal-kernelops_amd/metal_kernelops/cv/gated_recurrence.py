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
import functools
from typing import Optional, Tuple

import torch
from torch import Tensor

from .. import _native as nat
from .._contract import Rules
from ..scan import _require_gpu

__all__ = ["gated_recurrence", "gated_recurrence_reference", "gated_recurrence_update",
           "gated_recurrence_update_reference"]

_FLOATS = (torch.float32, torch.float16, torch.bfloat16)

CHUNK = 64
"""MKO_RECUR_CHUNK: steps between the saved states."""


@functools.lru_cache(maxsize=256)
def _sizes(batch, length, channels):
    """Bytes of the saved states and of the forward's and the backward's workspaces."""
    p = nat.RecurParams(batch=batch, length=length, channels=channels, ddecay=1)
    lib, at = nat.lib(), ctypes.byref(p)
    return lib.mko_recur_states_size(at), lib.mko_recur_fwd_workspace_size(at), lib.mko_recur_bwd_workspace_size(at)


def _params(x, input_gate, decay_gate, decay, initial, reset, scale, y, final, states, dy, dfinal, dx, dig, drg, ddecay,
            dinitial, space):
    batch, length, channels = x.shape
    return nat.RecurParams(
        x.data_ptr(), input_gate.data_ptr(), decay_gate.data_ptr(), decay.data_ptr(), nat.ptr(initial), nat.ptr(reset),
        nat.ptr(y), nat.ptr(final), states.data_ptr(), nat.ptr(dy), nat.ptr(dfinal), nat.ptr(dx), nat.ptr(dig),
        nat.ptr(drg), nat.ptr(ddecay), nat.ptr(dinitial), nat.ptr(space), 0 if space is None else space.numel(),
        batch, length, channels, x.stride(0), x.stride(1), input_gate.stride(0), input_gate.stride(1),
        decay_gate.stride(0), decay_gate.stride(1), scale, nat.code(x.dtype))


def _forward(x, input_gate, decay_gate, decay, initial, reset, scale, want_final):
    """``(y, final, states)``; ``states`` is what the backward reads, ``final`` None if unwanted."""
    batch, length, channels = x.shape
    y = nat.empty_as(x)
    final = None
    if want_final:
        final = torch.empty((batch, channels), dtype=torch.float32, device=x.device)
        if length == 0:
            final.zero_() if initial is None else final.copy_(initial)
    if y.numel() == 0:
        return y, final, None
    saved, size, _ = _sizes(batch, length, channels)
    states = torch.empty(saved, dtype=torch.uint8, device=x.device)
    space = torch.empty(size, dtype=torch.uint8, device=x.device) if size else None
    nat.launch("mko_recur_fwd", _params(x, input_gate, decay_gate, decay, initial, reset, scale, y, final, states, None,
                                        None, None, None, None, None, None, space), x.device)
    return y, final, states


def _backward(dy, dfinal, x, input_gate, decay_gate, decay, initial, reset, states, scale, need_decay, need_initial):
    """``(dx, dinput_gate, ddecay_gate, ddecay, dinitial)``, the last two None if unwanted."""
    dfinal = nat.dense(dfinal)
    dx, dig, drg = nat.empty_as(x), nat.empty_as(x), nat.empty_as(x)
    ddecay = nat.empty_as(decay) if need_decay else None
    dinitial = nat.empty_as(initial) if need_initial else None
    if x.numel():
        dy = torch.zeros_like(dx) if dy is None else nat.dense(dy)
        space = torch.empty(_sizes(*x.shape)[2], dtype=torch.uint8, device=x.device)
        nat.launch("mko_recur_bwd", _params(x, input_gate, decay_gate, decay, initial, reset, scale, None, None,
                                            states, dy, dfinal, dx, dig, drg, ddecay, dinitial, space), x.device)
    else:
        if ddecay is not None:
            ddecay.zero_()
        if dinitial is not None:
            dinitial.zero_() if dfinal is None else dinitial.copy_(dfinal)
    return dx, dig, drg, ddecay, dinitial


def _grads(ctx, dy, dfinal, _states=None):
    """The gradients of the inputs of :class:`_Recurrence` and of the custom op."""
    x, input_gate, decay_gate, decay, initial, reset, states = ctx.saved_tensors
    need = ctx.needs_input_grad
    need_decay, need_initial = need[3], initial is not None and need[4]
    if not ctx.want_final:
        dfinal = None
    # a backward that is itself recorded goes through the op, which refuses to be differentiated
    op = ctx.through_op or torch.is_grad_enabled() or nat.watched(dy, dfinal)
    backward = torch.ops.mko.recur_bwd if op else _backward
    dx, dig, drg, ddecay, dinitial = backward(dy, dfinal, x, input_gate, decay_gate, decay, initial, reset, states,
                                              ctx.scale, need_decay, need_initial)
    return dx, dig, drg, ddecay if need_decay else None, dinitial if need_initial else None, None, None, None


class _Recurrence(torch.autograd.Function):
    """Forward and analytic first-order backward through the C ABI."""

    @staticmethod
    def forward(ctx, x, input_gate, decay_gate, decay, initial, reset, scale, want_final):
        y, final, states = _forward(x, input_gate, decay_gate, decay, initial, reset, scale, want_final)
        ctx.save_for_backward(x, input_gate, decay_gate, decay, initial, reset, states)
        ctx.scale, ctx.want_final, ctx.through_op = scale, want_final, False
        ctx.set_materialize_grads(False)  # an unused output reaches backward as None
        return y, final

    backward = staticmethod(_grads)


def _recur_fwd_op(x: Tensor, input_gate: Tensor, decay_gate: Tensor, decay: Tensor, initial: Optional[Tensor],
                  reset: Optional[Tensor], scale: float, want_final: bool) -> Tuple[Tensor, Tensor, Tensor]:
    y, final, states = _forward(nat.rows(x), nat.rows(input_gate), nat.rows(decay_gate), nat.dense(decay),
                                nat.dense(initial), nat.dense(reset), scale, want_final)
    return y, nat.absent(final, decay), nat.absent(states, decay, torch.uint8)


_recur_fwd = torch.library.custom_op("mko::recur_fwd", _recur_fwd_op, mutates_args=(), device_types="cuda")


@_recur_fwd.register_fake
def _(x, input_gate, decay_gate, decay, initial, reset, scale, want_final):
    batch, length, channels = x.shape
    saved = -(-(batch * -(-length // CHUNK) * channels * 4) // 16) * 16
    return (x.new_empty(x.shape), x.new_empty((batch, channels) if want_final else 0, dtype=torch.float32),
            x.new_empty(saved, dtype=torch.uint8))


def _recur_bwd_op(dy: Optional[Tensor], dfinal: Optional[Tensor], x: Tensor, input_gate: Tensor, decay_gate: Tensor,
                  decay: Tensor, initial: Optional[Tensor], reset: Optional[Tensor], states: Optional[Tensor],
                  scale: float, need_decay: bool, need_initial: bool
                  ) -> Tuple[Tensor, Tensor, Tensor, Tensor, Tensor]:
    dx, dig, drg, ddecay, dinitial = _backward(
        dy, dfinal, nat.rows(x), nat.rows(input_gate), nat.rows(decay_gate), nat.dense(decay), nat.dense(initial),
        nat.dense(reset), nat.dense(states), scale, need_decay, need_initial)
    return dx, dig, drg, nat.absent(ddecay, decay), nat.absent(dinitial, decay)


_recur_bwd = torch.library.custom_op("mko::recur_bwd", _recur_bwd_op, mutates_args=(), device_types="cuda")


@_recur_bwd.register_fake
def _(dy, dfinal, x, input_gate, decay_gate, decay, initial, reset, states, scale, need_decay, need_initial):
    return (*(x.new_empty(x.shape) for _ in range(3)), decay.new_empty(decay.shape if need_decay else 0),
            decay.new_empty(initial.shape if need_initial else 0))


def _setup(ctx, inputs, output):
    x, input_gate, decay_gate, decay, initial, reset, ctx.scale, ctx.want_final = inputs
    ctx.save_for_backward(x, input_gate, decay_gate, decay, initial, reset, output[2])
    ctx.through_op = True  # whatever the forward's tensors were
    ctx.set_materialize_grads(False)


torch.library.register_autograd("mko::recur_fwd", _grads, setup_context=_setup)


def _update(state, x, input_gate, decay_gate, decay, scale, new_state, y):
    batch, channels = x.shape
    if batch and channels:
        nat.launch("mko_recur_update", nat.RecurUpdateParams(
            x.data_ptr(), input_gate.data_ptr(), decay_gate.data_ptr(), decay.data_ptr(), state.data_ptr(),
            new_state.data_ptr(), y.data_ptr(), batch, channels, x.stride(0), input_gate.stride(0), decay_gate.stride(0),
            scale, nat.code(x.dtype), nat.code(state.dtype)), x.device)
    return y, new_state


def _recur_update_op(state: Tensor, x: Tensor, input_gate: Tensor, decay_gate: Tensor, decay: Tensor, scale: float
                     ) -> Tuple[Tensor, Tensor]:
    return _update(nat.dense(state), nat.rows(x), nat.rows(input_gate), nat.rows(decay_gate), nat.dense(decay), scale,
                   nat.empty_as(state), nat.empty_as(x))


_recur_update = torch.library.custom_op("mko::recur_update", _recur_update_op, mutates_args=(), device_types="cuda")


@_recur_update.register_fake
def _(state, x, input_gate, decay_gate, decay, scale):
    return x.new_empty(x.shape), state.new_empty(state.shape)


def _check(op, x, input_gate, decay_gate, decay, scale, layout):
    """The argument rules that the scan and the update share, in their order.  Messages are formed
    only for an argument that breaks a rule: a decode step's checks are host time."""
    rules = Rules(op)
    shape = x.shape
    if len(shape) != layout.count(",") + 1:
        rules.dims("x", x, layout.count(",") + 1, layout)
    if input_gate.shape != shape or decay_gate.shape != shape or decay.shape != shape[-1:]:
        rules.shape("input_gate", input_gate, shape)
        rules.shape("decay_gate", decay_gate, shape)
        rules.shape("decay", decay, shape[-1:])
    _require_gpu(x)
    device, dtype = x.device, x.dtype
    if input_gate.device != device or decay_gate.device != device or decay.device != device:
        rules.same_device(device, input_gate=input_gate, decay_gate=decay_gate, decay=decay)
    if dtype not in _FLOATS or input_gate.dtype != dtype or decay_gate.dtype != dtype:
        rules.dtype_in(_FLOATS, x=x)
        rules.dtype_in((dtype,), input_gate=input_gate, decay_gate=decay_gate)
    if not decay.is_floating_point():
        rules.fail(f"decay should be a floating tensor; it is {decay.dtype}")
    if not scale > 0:
        rules.fail(f"scale should be positive; it is {scale}")
    if shape[0] > 65535:
        rules.fail(f"batch is at most 65535 (got {shape[0]})")
    return rules


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
    rules = _check("gated_recurrence", x, input_gate, decay_gate, decay, scale, "(batch, length, channels)")
    batch, length, channels = x.shape
    if initial_state is not None:
        rules.shape("initial_state", initial_state, (batch, channels))
        rules.same_device(x.device, initial_state=initial_state)
        if not initial_state.is_floating_point():
            rules.fail(f"initial_state should be a floating tensor; it is {initial_state.dtype}")
    if reset is not None:
        rules.shape("reset", reset, (batch, length))
        rules.same_device(x.device, reset=reset)
        rules.dtype_in((torch.bool,), reset=reset)
        reset = reset.contiguous()
    decay, initial = nat.dense_f32(decay), nat.dense_f32(initial_state)
    scale, want_final = float(scale), bool(return_final_state)
    if nat.watched(x, input_gate, decay_gate, decay, initial, reset):
        y, final, _ = nat.through(torch.ops.mko.recur_fwd, x, input_gate, decay_gate, decay, initial, reset, scale,
                                  want_final)
        return (y, final) if want_final else y
    x, input_gate, decay_gate = nat.rows(x), nat.rows(input_gate), nat.rows(decay_gate)
    if nat.wants_grad(x, input_gate, decay_gate, decay, initial):
        y, final = _Recurrence.apply(x, input_gate, decay_gate, decay, initial, reset, scale, want_final)
    else:
        y, final, _ = _forward(x, input_gate, decay_gate, decay, initial, reset, scale, want_final)
    return (y, final) if want_final else y


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
    rules = _check("gated_recurrence_update", x, input_gate, decay_gate, decay, scale, "(batch, channels)")
    if state.shape != x.shape or state.device != x.device or state.dtype not in _FLOATS:
        rules.shape("state", state, x.shape)
        rules.same_device(x.device, state=state)
        rules.dtype_in(_FLOATS, state=state)
    if out_state is not None:
        if out_state.shape != state.shape or out_state.dtype != state.dtype or out_state.device != state.device:
            rules.fail("out_state should have the shape, dtype and device of state")
        if not out_state.is_contiguous():
            rules.fail("out_state should be contiguous")
        if out_state.requires_grad:
            rules.fail("out_state is overwritten in place, so it may not require grad")
    if nat.wants_grad(state, x, input_gate, decay_gate, decay):
        if out_state is not None and out_state.untyped_storage()._cdata == state.untyped_storage()._cdata:
            state = state.clone()  # the backward reads the entering state, which its destination overwrites
        y, final = gated_recurrence(x[:, None], input_gate[:, None], decay_gate[:, None], decay, initial_state=state,
                                    scale=scale, return_final_state=True)
        final = final.to(state.dtype)
        if out_state is None:
            return y[:, 0], final
        with torch.no_grad():
            out_state.copy_(final)
        return y[:, 0], out_state
    decay = nat.dense_f32(decay)
    if nat.watched(state, x, input_gate, decay_gate, decay, out_state):
        if out_state is not None and not torch.compiler.is_compiling() and out_state.is_neg():
            rules.fail("out_state should be contiguous, and not a negated view")
        y, new_state = nat.through(torch.ops.mko.recur_update, state, x, input_gate, decay_gate, decay, float(scale))
        return y, new_state if out_state is None else out_state.copy_(new_state)
    state = nat.dense(state)
    if out_state is not None and out_state is not state:
        state = nat.unshifted(state, out_state)
    y, new_state = _update(state, nat.rows(x), nat.rows(input_gate), nat.rows(decay_gate), decay, scale,
                           nat.empty_as(state) if out_state is None else out_state, nat.empty_as(x))
    if out_state is not None:
        nat.written(out_state)
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
