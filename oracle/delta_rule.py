"""Float64 CPU statements of the gated delta rule (test oracle), token by token: the recurrence and its
analytic gradients.  Nothing here is imported by the product."""

from __future__ import annotations

import torch

F64 = torch.float64


def _wide(q, k, v, log_decay, beta):
    rep = v.shape[2] // q.shape[2]
    q, k = (t.to(F64).repeat_interleave(rep, 2) for t in (q, k))
    return q, k, v.to(F64), log_decay.to(F64).exp(), beta.to(F64)


def _start(v, q, initial):
    return v.new_zeros(v.shape[0], v.shape[2], v.shape[3], q.shape[3], dtype=F64) if initial is None else initial.to(F64)


def _scale(q, scale):
    return q.shape[-1] ** -0.5 if scale is None else scale


def gated_delta_rule(q, k, v, log_decay, beta, scale=None, initial=None):
    """``(y, final)`` in float64; differentiable."""
    S = _start(v, q, initial)
    scale, out = _scale(q, scale), []
    q, k, v, a, beta = _wide(q, k, v, log_decay, beta)
    for t in range(v.shape[1]):
        P = a[:, t, :, None, None] * S
        e = v[:, t] - torch.einsum("bhvk,bhk->bhv", P, k[:, t])
        S = P + torch.einsum("bhv,bhk->bhvk", beta[:, t, :, None] * e, k[:, t])
        out.append(scale * torch.einsum("bhvk,bhk->bhv", S, q[:, t]))
    return torch.stack(out, 1) if out else torch.zeros_like(v), S


def gated_delta_rule_bwd(dy, dfinal, q, k, v, log_decay, beta, scale=None, initial=None):
    """``(dq, dk, dv, dlog_decay, dbeta, dinitial)`` from the formulas, the state's gradient walked back."""
    key_heads, scale, S = q.shape[2], _scale(q, scale), _start(v, q, initial)
    q, k, v, a, beta = _wide(q, k, v, log_decay, beta)
    kept = []
    for t in range(v.shape[1]):
        P = a[:, t, :, None, None] * S
        e = v[:, t] - torch.einsum("bhvk,bhk->bhv", P, k[:, t])
        S = P + torch.einsum("bhv,bhk->bhvk", beta[:, t, :, None] * e, k[:, t])
        kept.append((P, e, S))
    G = torch.zeros_like(S) if dfinal is None else dfinal.to(F64)
    dq, dk, dv, dg, db = (torch.zeros_like(t) for t in (q, k, v, a, beta))
    for t in reversed(range(v.shape[1])):
        P, e, S = kept[t]
        d = dy[:, t].to(F64)
        dq[:, t] = scale * torch.einsum("bhvk,bhv->bhk", S, d)
        G = G + scale * torch.einsum("bhv,bhk->bhvk", d, q[:, t])
        Gk = torch.einsum("bhvk,bhk->bhv", G, k[:, t])
        db[:, t] = (Gk * e).sum(-1)
        de = beta[:, t, :, None] * Gk
        dv[:, t] = de
        dk[:, t] = torch.einsum("bhvk,bhv->bhk", G, beta[:, t, :, None] * e) - torch.einsum("bhvk,bhv->bhk", P, de)
        G = G - torch.einsum("bhv,bhk->bhvk", de, k[:, t])
        dg[:, t] = (G * P).sum((-1, -2))
        G = a[:, t, :, None, None] * G
    shared = (*dq.shape[:2], key_heads, -1, dq.shape[3])
    return dq.reshape(shared).sum(3), dk.reshape(shared).sum(3), dv, dg, db, G
