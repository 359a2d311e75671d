"""Gated delta rule on MI355X: the recurrence over a sequence, its gradients, and one decode step.

Per value head, with a matrix state ``S`` (value x key) that first forgets and then corrects what a
key reads from it::

    e[t] = v[t] - exp(log_decay[t]) * S[t-1] k[t]
    S[t] = exp(log_decay[t]) * S[t-1] + beta[t] * outer(e[t], k[t])
    y[t] = scale * S[t] q[t]

Layouts: ``q``, ``k`` ``(batch, length, key_heads, key)`` and ``v`` ``(batch, length, heads, value)`` in
one of float32, float16 and bfloat16, with any strides but the last (slices of one projection are read
in place); value head ``h`` reads key head ``h // (heads // key_heads)``.  ``log_decay`` and ``beta``
``(batch, length, heads)``; states ``(batch, heads, value, key)``, as ``mamba2_state_update`` has them.

The rule is stable for keys of norm one (``beta * |k|^2`` below two) and log decays of at most zero; a
log decay of ``-inf`` drops the state before it, so documents packed in one row do not see each other.

Kernels (``libmko.so``): chunks of 64 tokens on the matrix cores, their operands rounded to the
activations' type (float32 products for float32), with the state, the decays and all sums in float32
and the triangular systems of the chunks solved in float32.  The gradients are analytic,
once-differentiable and summed in a fixed order, so repeated runs give the same bits.  Few long sequences
are cut into segments that run side by side; whether goes by the sizes of the call, so a sequence alone and
the same one in a batch may differ by roundings.  A value that is
not finite reaches its whole chunk and what follows it.  There is no counterpart in dbydd/metal-kernelops.
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

__all__ = ["gated_delta_rule", "gated_delta_rule_reference", "gated_delta_rule_update",
           "gated_delta_rule_update_reference"]

_FLOATS = (torch.float32, torch.float16, torch.bfloat16)

CHUNK = 64
"""MKO_DELTA_CHUNK: tokens that are worked on together."""

MAX_KEY = 256
"""MKO_DELTA_MAX_KEY: the longest key."""

_TOKENS = CHUNK * (8 + 4 * 4)  # bytes of a chunk's decays
_SQUARES = 2 * 6 * 512  # elements of its two triangular operands


@functools.lru_cache(maxsize=256)
def _sizes(batch, length, key_heads, heads, key, value, dtype, save):
    """Bytes of what the forward saves and of its and the backward's workspaces."""
    p = nat.DeltaParams(batch=batch, length=length, key_heads=key_heads, heads=heads, key=key, value=value, dtype=dtype,
                        saved=1 if save else None)
    lib, at = nat.lib(), ctypes.byref(p)
    return (lib.mko_delta_saved_size(at) if save else 0, lib.mko_delta_fwd_workspace_size(at),
            lib.mko_delta_bwd_workspace_size(at))


def _params(q, k, v, log_decay, beta, initial, y, final, saved, grads, space, scale, state_dtype):
    batch, length, key_heads, key = q.shape
    dy, dfinal, dq, dk, dv, dg, dbeta, dinitial = grads
    return nat.DeltaParams(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), log_decay.data_ptr(), beta.data_ptr(), nat.ptr(initial), nat.ptr(y),
        nat.ptr(final), nat.ptr(saved), nat.ptr(dy), nat.ptr(dfinal), nat.ptr(dq), nat.ptr(dk), nat.ptr(dv), nat.ptr(dg),
        nat.ptr(dbeta), nat.ptr(dinitial), nat.ptr(space), 0 if space is None else space.numel(), batch, length, key_heads,
        v.shape[2], key, v.shape[3], *q.stride()[:3], *k.stride()[:3], *v.stride()[:3], scale, nat.code(q.dtype),
        nat.code(log_decay.dtype), nat.code(beta.dtype), nat.code(state_dtype))


def _forward(q, k, v, log_decay, beta, initial, scale, want_final, save):
    """``(y, final, saved)``; the last two None if unwanted."""
    batch, length, key_heads, key = q.shape
    heads, value = v.shape[2:]
    state_dtype = v.dtype if initial is None else initial.dtype
    y = nat.empty_as(v)
    final = None
    if want_final:
        final = torch.empty((batch, heads, value, key), dtype=state_dtype, device=v.device)
        if length == 0:
            final.zero_() if initial is None else final.copy_(initial)
    if y.numel() == 0:
        return y, final, None
    kept, size, _ = _sizes(batch, length, key_heads, heads, key, value, nat.code(q.dtype), save)
    saved = torch.empty(kept, dtype=torch.uint8, device=v.device) if save else None
    space = torch.empty(size, dtype=torch.uint8, device=v.device)
    nat.launch("mko_delta_fwd", _params(q, k, v, log_decay, beta, initial, y, final, saved, (None,) * 8, space, scale,
                                        state_dtype), v.device)
    return y, final, saved


def _backward(dy, dfinal, q, k, v, log_decay, beta, initial, saved, scale, need_initial):
    """``(dq, dk, dv, dlog_decay, dbeta, dinitial)``, the last None if unwanted."""
    batch, length, key_heads, key = q.shape
    heads, value = v.shape[2:]
    dfinal = nat.dense(dfinal)
    dq, dk, dv, dg, dbeta = (nat.empty_as(t) for t in (q, k, v, log_decay, beta))
    dinitial = nat.empty_as(initial) if need_initial else None
    if v.numel():
        dy = torch.zeros_like(dv) if dy is None else nat.dense(dy)
        size = _sizes(batch, length, key_heads, heads, key, value, nat.code(q.dtype), True)[2]
        space = torch.empty(size, dtype=torch.uint8, device=v.device)
        nat.launch("mko_delta_bwd", _params(q, k, v, log_decay, beta, initial, None, None, saved,
                                            (dy, dfinal, dq, dk, dv, dg, dbeta, dinitial), space, scale,
                                            v.dtype if initial is None else initial.dtype), v.device)
    else:
        for t in (dq, dk, dg, dbeta):  # tokens without values
            t.zero_()
        if dinitial is not None:
            dinitial.zero_() if dfinal is None else dinitial.copy_(dfinal)
    return dq, dk, dv, dg, dbeta, dinitial


def _grads(ctx, dy, dfinal, _saved=None):
    """The gradients of the inputs of :class:`_Delta` and of the custom op."""
    q, k, v, log_decay, beta, initial, saved = ctx.saved_tensors
    need = ctx.needs_input_grad
    need_initial = initial is not None and need[5]
    if not ctx.want_final:
        dfinal = None
    # a backward that is itself recorded goes through the op, which refuses to be differentiated
    op = ctx.through_op or torch.is_grad_enabled() or nat.watched(dy, dfinal)
    backward = torch.ops.mko.delta_bwd if op else _backward
    *grads, dinitial = backward(dy, dfinal, q, k, v, log_decay, beta, initial, saved, ctx.scale, need_initial)
    return (*(t if n else None for t, n in zip(grads, need)), dinitial if need_initial else None, None, None, None)


class _Delta(torch.autograd.Function):
    """Forward and analytic first-order backward through the C ABI."""

    @staticmethod
    def forward(ctx, q, k, v, log_decay, beta, initial, scale, want_final, save):
        y, final, saved = _forward(q, k, v, log_decay, beta, initial, scale, want_final, save)
        ctx.save_for_backward(q, k, v, log_decay, beta, initial, saved)
        ctx.scale, ctx.want_final, ctx.through_op = scale, want_final, False
        ctx.set_materialize_grads(False)  # an unused output reaches backward as None
        return y, final

    backward = staticmethod(_grads)


def _delta_fwd_op(q: Tensor, k: Tensor, v: Tensor, log_decay: Tensor, beta: Tensor, initial: Optional[Tensor], scale: float,
                  want_final: bool, save: bool) -> Tuple[Tensor, Tensor, Tensor]:
    y, final, saved = _forward(nat.rows(q), nat.rows(k), nat.rows(v), nat.dense(log_decay), nat.dense(beta),
                               nat.dense(initial), scale, want_final, save)
    return y, nat.absent(final, v, v.dtype if initial is None else initial.dtype), nat.absent(saved, v, torch.uint8)


_delta_fwd = torch.library.custom_op("mko::delta_fwd", _delta_fwd_op, mutates_args=(), device_types="cuda")


@_delta_fwd.register_fake
def _(q, k, v, log_decay, beta, initial, scale, want_final, save):
    batch, length, heads, value = v.shape
    key, size = q.shape[3], 4 if v.dtype == torch.float32 else 2
    cells = batch * heads * -(-length // CHUNK)
    kept = sum(-(-cells * n // 256) * 256 for n in (_TOKENS, _SQUARES * size, value * key * size, CHUNK * value * size))
    return (v.new_empty(v.shape),
            (v if initial is None else initial).new_empty((batch, heads, value, key) if want_final else 0),
            v.new_empty(kept if save and value else 0, dtype=torch.uint8))  # without values nothing is launched


def _delta_bwd_op(dy: Optional[Tensor], dfinal: Optional[Tensor], q: Tensor, k: Tensor, v: Tensor, log_decay: Tensor,
                  beta: Tensor, initial: Optional[Tensor], saved: Optional[Tensor], scale: float, need_initial: bool
                  ) -> Tuple[Tensor, Tensor, Tensor, Tensor, Tensor, Tensor]:
    *grads, dinitial = _backward(dy, dfinal, nat.rows(q), nat.rows(k), nat.rows(v), nat.dense(log_decay), nat.dense(beta),
                                 nat.dense(initial), nat.dense(saved), scale, need_initial)
    return (*grads, nat.absent(dinitial, v, v.dtype if initial is None else initial.dtype))


_delta_bwd = torch.library.custom_op("mko::delta_bwd", _delta_bwd_op, mutates_args=(), device_types="cuda")


@_delta_bwd.register_fake
def _(dy, dfinal, q, k, v, log_decay, beta, initial, saved, scale, need_initial):
    return (*(t.new_empty(t.shape) for t in (q, k, v, log_decay, beta)),
            (v if initial is None else initial).new_empty(initial.shape if need_initial else 0))


def _setup(ctx, inputs, output):
    q, k, v, log_decay, beta, initial, ctx.scale, ctx.want_final, _ = inputs
    ctx.save_for_backward(q, k, v, log_decay, beta, initial, output[2])
    ctx.through_op = True  # whatever the forward's tensors were
    ctx.set_materialize_grads(False)


torch.library.register_autograd("mko::delta_fwd", _grads, setup_context=_setup)


def _update(state, q, k, v, log_decay, beta, scale, new_state, y):
    batch, key_heads, key = q.shape
    if y.numel():
        nat.launch("mko_delta_update", nat.DeltaUpdateParams(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), log_decay.data_ptr(), beta.data_ptr(), state.data_ptr(),
            new_state.data_ptr(), y.data_ptr(), batch, key_heads, v.shape[1], key, v.shape[2], q.stride(0), q.stride(1),
            k.stride(0), k.stride(1), v.stride(0), v.stride(1), scale, nat.code(q.dtype), nat.code(log_decay.dtype),
            nat.code(beta.dtype), nat.code(state.dtype)), v.device)
    return y, new_state


def _delta_update_op(state: Tensor, q: Tensor, k: Tensor, v: Tensor, log_decay: Tensor, beta: Tensor, scale: float
                     ) -> Tuple[Tensor, Tensor]:
    return _update(nat.dense(state), nat.rows(q), nat.rows(k), nat.rows(v), nat.dense(log_decay), nat.dense(beta), scale,
                   nat.empty_as(state), nat.empty_as(v))


_delta_update = torch.library.custom_op("mko::delta_update", _delta_update_op, mutates_args=(), device_types="cuda")


@_delta_update.register_fake
def _(state, q, k, v, log_decay, beta, scale):
    return v.new_empty(v.shape), state.new_empty(state.shape)


def _check(op, q, k, v, log_decay, beta, scale, lead):
    """The argument rules that the scan and the update share, in their order; returns them with the
    scale.  Messages are formed only for an argument that breaks a rule: a decode step's checks are
    host time."""
    rules = Rules(op)
    shape, vshape, n = q.shape, v.shape, lead.count(",") + 3
    if len(shape) != n or len(vshape) != n:
        rules.dims("q", q, n, f"({lead}, key_heads, key)")
        rules.dims("v", v, n, f"({lead}, heads, value)")
    if k.shape != shape or vshape[:-2] != shape[:-2] or log_decay.shape != vshape[:-1] or beta.shape != vshape[:-1]:
        rules.shape("k", k, shape)
        if vshape[:-2] != shape[:-2]:
            rules.fail(f"v should lead with ({lead}) = {tuple(shape[:-2])}; its shape is {tuple(vshape)}")
        rules.shape("log_decay", log_decay, vshape[:-1])
        rules.shape("beta", beta, vshape[:-1])
    key_heads, key, heads = shape[-2], shape[-1], vshape[-2]
    if key_heads < 1 or heads % key_heads:
        rules.fail(f"{heads} heads do not split evenly over {key_heads} key heads")
    if not 1 <= key <= MAX_KEY:
        rules.fail(f"the key axis has 1 to {MAX_KEY} elements (got {key})")
    _require_gpu(q)
    device, dtype = q.device, q.dtype
    if k.device != device or v.device != device or log_decay.device != device or beta.device != device:
        rules.same_device(device, k=k, v=v, log_decay=log_decay, beta=beta)
    if dtype not in _FLOATS or k.dtype != dtype or v.dtype != dtype:
        rules.dtype_in(_FLOATS, q=q)
        rules.dtype_in((dtype,), k=k, v=v)
    if log_decay.dtype not in _FLOATS or beta.dtype not in _FLOATS:
        rules.dtype_in(_FLOATS, log_decay=log_decay, beta=beta)
    return rules, key ** -0.5 if scale is None else float(scale)


def _limit(rules, n, bits, text):
    if n >= 1 << bits:
        rules.fail(f"{text} should be below 2^{bits} (got {n})")


def gated_delta_rule(q, k, v, log_decay, beta, scale=None, initial_state=None, return_final_state=False):
    """The gated delta rule over a sequence (the module notes have the formulas).

    Args:
        q, k: ``(batch, length, key_heads, key)``, float32, float16 or bfloat16 on the ROCm GPU, ``key``
            up to 256.  Keys are used as they are; normalise them first.
        v: ``(batch, length, heads, value)`` in their dtype; ``heads`` is a multiple of ``key_heads``, and
            ``batch * heads`` times the chunks of 64 tokens, or the tiles of 16 values, is below 2^23.
        log_decay: ``(batch, length, heads)`` logarithm of what the state keeps at a step, at most 0, in
            one of those dtypes.  Below ``-1e4`` it counts as ``-1e4``, which clears the state.
        beta: ``(batch, length, heads)`` strength of the correction, in one of those dtypes.
        scale: of the output; ``key ** -0.5`` by default.
        initial_state: ``(batch, heads, value, key)`` state before the first token in one of those
            dtypes, or None for zeros.
        return_final_state: also return the state after the last token, in ``initial_state``'s dtype, or
            ``v``'s without one.

    Returns:
        ``y`` ``(batch, length, heads, value)`` in ``v.dtype``, or ``(y, final_state)``.
    """
    rules, scale = _check("gated_delta_rule", q, k, v, log_decay, beta, scale, "batch, length")
    batch, length, heads, value = v.shape
    if initial_state is not None:
        rules.shape("initial_state", initial_state, (batch, heads, value, q.shape[3]))
        rules.same_device(q.device, initial_state=initial_state)
        rules.dtype_in(_FLOATS, initial_state=initial_state)
    _limit(rules, value, 20, "the value axis")
    _limit(rules, batch * heads * max(-(-length // CHUNK), -(-value // 16)), 23,
           "batch * heads * (chunks of 64 tokens, or tiles of 16 values)")
    initial, want_final = nat.dense(initial_state), bool(return_final_state)
    log_decay, beta = nat.dense(log_decay), nat.dense(beta)
    if nat.watched(q, k, v, log_decay, beta, initial):
        save = nat.wants_grad(q, k, v, log_decay, beta, initial)
        y, final, _ = nat.through(torch.ops.mko.delta_fwd, q, k, v, log_decay, beta, initial, scale, want_final, save)
        return (y, final) if want_final else y
    q, k, v = nat.rows(q), nat.rows(k), nat.rows(v)
    if nat.wants_grad(q, k, v, log_decay, beta, initial):
        y, final = _Delta.apply(q, k, v, log_decay, beta, initial, scale, want_final, True)
    else:
        y, final, _ = _forward(q, k, v, log_decay, beta, initial, scale, want_final, False)
    return (y, final) if want_final else y


def gated_delta_rule_update(state, q, k, v, log_decay, beta, scale=None, out_state=None):
    """Advance a state by one token; returns ``(y, new_state)``.

    ``state`` is ``(batch, heads, value, key)`` in float32, float16 or bfloat16 and is read, never
    written, unless it is passed again as ``out_state``; ``q`` and ``k`` are ``(batch, key_heads, key)``
    and ``v`` ``(batch, heads, value)`` in one of those dtypes, ``log_decay`` and ``beta``
    ``(batch, heads)``, and ``y`` is ``(batch, heads, value)`` in ``v.dtype``.  With ``out_state``
    (contiguous, the state's shape and dtype, not requiring grad) the new state is written there and
    returned as that tensor, outside the autograd graph; the state may be its own destination.

    Without a gradient the step is computed in float32; ``new_state`` and ``y`` are each rounded once.  Where
    one is wanted it is a :func:`gated_delta_rule` of length one, whose operands (the state that it reads, the
    error, the correction) are rounded to the activations' type: 16-bit calls differ by those roundings, float32 ones
    by the order of their sums.
    """
    rules, scale = _check("gated_delta_rule_update", q, k, v, log_decay, beta, scale, "batch")
    shape = (*v.shape, q.shape[2])
    if state.shape != shape or state.device != q.device or state.dtype not in _FLOATS:
        rules.shape("state", state, shape)
        rules.same_device(q.device, state=state)
        rules.dtype_in(_FLOATS, state=state)
    if out_state is not None:
        if out_state.shape != state.shape or out_state.dtype != state.dtype or out_state.device != state.device:
            rules.fail("out_state should have the shape, dtype and device of state")
        if not out_state.is_contiguous():
            rules.fail("out_state should be contiguous")
        if out_state.requires_grad:
            rules.fail("out_state is overwritten in place, so it may not require grad")
    _limit(rules, shape[0] * shape[1] * -(-shape[2] // 8), 24, "batch * heads * (groups of 8 values)")
    if nat.wants_grad(state, q, k, v, log_decay, beta):
        if out_state is not None and out_state.untyped_storage()._cdata == state.untyped_storage()._cdata:
            state = state.clone()  # the backward reads the entering state, which its destination overwrites
        y, final = gated_delta_rule(q[:, None], k[:, None], v[:, None], log_decay[:, None], beta[:, None], scale,
                                    initial_state=state, return_final_state=True)
        if out_state is None:
            return y[:, 0], final
        with torch.no_grad():
            out_state.copy_(final)
        return y[:, 0], out_state
    log_decay, beta = nat.dense(log_decay), nat.dense(beta)
    if nat.watched(state, q, k, v, log_decay, beta, out_state):
        if out_state is not None and not torch.compiler.is_compiling() and out_state.is_neg():
            rules.fail("out_state should be contiguous, and not a negated view")
        y, new_state = nat.through(torch.ops.mko.delta_update, state, q, k, v, log_decay, beta, scale)
        return y, new_state if out_state is None else out_state.copy_(new_state)
    state = nat.dense(state)
    if out_state is not None and out_state is not state:
        state = nat.unshifted(state, out_state)
    y, new_state = _update(state, nat.rows(q), nat.rows(k), nat.rows(v), log_decay, beta, scale,
                           nat.empty_as(state) if out_state is None else out_state, nat.empty_as(v))
    if out_state is not None:
        nat.written(out_state)
    return y, new_state


def gated_delta_rule_reference(q, k, v, log_decay, beta, scale=None, initial_state=None, return_final_state=False):
    """The rule token by token in torch ops, on any device and float dtype; differentiable."""
    batch, length, heads, value = v.shape
    state = initial_state if initial_state is not None else v.new_zeros(batch, heads, value, q.shape[3])
    out = []
    for t in range(length):
        y, state = gated_delta_rule_update_reference(state, q[:, t], k[:, t], v[:, t], log_decay[:, t], beta[:, t], scale)
        out.append(y)
    y = torch.stack(out, 1) if out else torch.zeros_like(v)
    return (y, state) if return_final_state else y


def gated_delta_rule_update_reference(state, q, k, v, log_decay, beta, scale=None):
    """One step in torch ops, on any device and float dtype; returns ``(y, new_state)``."""
    rep = v.shape[1] // q.shape[1]
    q, k = q.repeat_interleave(rep, 1), k.repeat_interleave(rep, 1)
    kept = torch.exp(log_decay)[..., None, None] * state
    error = v - (kept * k[:, :, None]).sum(-1)
    state = kept + (beta[..., None] * error)[..., None] * k[:, :, None]
    return (state * q[:, :, None]).sum(-1) * (q.shape[-1] ** -0.5 if scale is None else scale), state
