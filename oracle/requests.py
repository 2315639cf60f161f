"""What a head says about given tokens, and low-rank adapters on a projection, in 64 bits from the definitions."""

from __future__ import annotations

import torch


def score(x, tokens, top):
    """Rows x [rows, vocab]: a dict of float64 logprobs (0 for negative tokens), entropy, top ids and their log probabilities, and the mean distance of a
    logit from the largest, which the entropy's rounding goes by."""
    x = x.double()
    m = x.amax(-1, keepdim=True)
    d = x - m
    log_s = torch.where(d == -torch.inf, 0.0, d.exp()).sum(-1, keepdim=True).log()
    log_p = d - log_s
    p = log_p.exp()
    known = tokens >= 0
    ids = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :top]
    weighted = lambda v: torch.where(p == 0, 0.0, p * v).sum(-1)  # noqa: E731
    return dict(logprobs=torch.where(known, log_p.gather(1, tokens.clamp(min=0)[:, None])[:, 0], 0.0), entropy=-weighted(log_p), top_ids=ids,
                top_logprobs=log_p.gather(1, ids), distance=weighted(d.abs()), log_p=log_p)  # fmt: skip


def score_gradient(x, tokens, d_logprobs, d_entropy):
    """The gradient of sum(d_logprobs * logprobs + d_entropy * entropy) by x, float64, and the sum of the magnitudes of its terms."""
    s = score(x, tokens, 0)
    log_p, p = s["log_p"], s["log_p"].exp()
    dl = torch.where(tokens >= 0, d_logprobs.double(), 0.0)[:, None]
    dh = d_entropy.double()[:, None]
    term = torch.where(p == 0, 0.0, p * (log_p + s["entropy"][:, None]))
    one = torch.zeros_like(p).scatter_(1, tokens.clamp(min=0)[:, None], 1.0)
    size = torch.where(p == 0, 0.0, p * (log_p.abs() + s["entropy"][:, None].abs() + 1))
    return dl * (one - p) - dh * term, dl.abs() * (one + p) + dh.abs() * size


def lora(y, x, a, b, which, scale):
    """y [tokens, out] + scale (x a^T) b^T by each row's adapter (negative: none), float64; and what roundings go by: sum |x a| by rank, and a function of
    errors in v."""
    out, v, size, reach = y.double().clone(), {}, {}, {}
    for i in range(a.shape[0]):
        rows = (which == i).nonzero()[:, 0]
        xa = x[rows].double()
        v[i] = xa @ a[i].double().t()
        size[i] = xa.abs() @ a[i].double().abs().t()
        out[rows] += scale[i].double() * (v[i] @ b[i].double().t())
        reach[i] = rows
    return out, v, size, reach
