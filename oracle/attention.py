"""Attention of a generating decoder in 64 bits: per-head norm and rotation, and attention under a causal mask, a sliding window and
first tokens that stay visible.  Written from the definitions, one query at a time where that is the plainest form."""

from __future__ import annotations

import torch


def norm_rope(x, weight, eps, cos, sin):
    """x [tokens, heads, head_dim], cos / sin [tokens, rotary / 2]: (y behind the norm, z behind the rotation), float64."""
    y = x.double()
    if weight is not None:
        y = y / (y.square().mean(-1, keepdim=True) + eps).sqrt() * weight.double()
    r = 2 * cos.shape[1]
    c, s = cos.double()[:, None], sin.double()[:, None]
    a, b = y[..., : r // 2], y[..., r // 2 : r]
    return y, torch.cat([a * c - b * s, b * c + a * s, y[..., r:]], dim=-1)


def visible(pos, window, sinks):
    """The keys that the query at this position sees, in order."""
    return [j for j in range(pos + 1) if window <= 0 or j > pos - window or j < sinks]


def attend(q, k, v, pos, window, sinks, scale):
    """q [heads, d] at position ``pos`` against k, v [keys, d] of the kv head they share: (out, sum of weight * |v|, largest sum of
    |q_d k_d| * scale), float64.  Rows that see nothing, or nothing but minus infinity, are zeros."""
    seen = visible(pos, window, sinks)
    out = torch.zeros(q.shape, dtype=torch.float64)
    if not seen:
        return out, out.clone(), torch.zeros(q.shape[0], dtype=torch.float64)
    q, k, v = q.double(), k[seen].double(), v[seen].double()
    x = q @ k.t() * scale
    top = x.amax(-1, keepdim=True)
    w = (x - top.masked_fill(top == -torch.inf, 0.0)).exp()
    total = w.sum(-1, keepdim=True)
    w = torch.where(total == 0, 0.0, w / total)
    size = (q.abs() @ k.abs().t()).amax(-1) * scale
    none = total == 0  # zeros, whatever the values hold
    return (w[:, :, None] * v).sum(1).masked_fill(none, 0.0), (w[:, :, None] * v.abs()).sum(1).masked_fill(none, 0.0), size
