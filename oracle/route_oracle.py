"""Routing to experts in 64 bits, token by token and expert by expert (plain Python and torch on the CPU)."""

from __future__ import annotations

import math

import torch


def scores(logits: torch.Tensor, gating: str) -> torch.Tensor:
    """float64 scores; a row of minus infinities has scores of zero."""
    l = logits.double()
    if gating == "sigmoid":
        return 1 / (1 + torch.exp(-l))
    top = l.amax(-1, keepdim=True)
    e = torch.where(l == -math.inf, 0.0, torch.exp(l - top))
    total = e.sum(-1, keepdim=True)
    return torch.where(total == 0, 0.0, e / total)


def route(logits, top_k, gating="softmax", bias=None, groups=1, groups_kept=1, normalize=False, scale=1.0):
    """``(weights float64, indices, counts)``."""
    tokens, experts = logits.shape
    s = scores(logits, gating)
    c = s if bias is None else s + bias.double()
    c = torch.where(torch.isnan(c), -math.inf, c)
    indices = torch.zeros(tokens, top_k, dtype=torch.long)
    size = experts // groups
    for t in range(tokens):
        row = c[t].tolist()
        # what cannot be told apart by its score goes by the logit (the softmax and the sigmoid are increasing)
        tie = logits[t].double().tolist() if bias is None and groups == 1 else [0.0] * experts
        tie = [-math.inf if v != v else v for v in tie]
        allowed = list(range(experts))
        if groups > 1 and groups_kept < groups:
            best = []
            for g in range(groups):
                two = sorted(row[g * size:(g + 1) * size], reverse=True)[:2]
                best.append(sum(two))
            order = sorted(range(groups), key=lambda g: (-best[g], g))[:groups_kept]
            allowed = [e for e in allowed if e // size in order]
        allowed.sort(key=lambda e: (-row[e], -tie[e], e))
        indices[t] = torch.tensor(allowed[:top_k])
    chosen = s.gather(1, indices)
    weights = chosen * scale
    if normalize:
        total = chosen.sum(-1, keepdim=True)
        weights = torch.where(total == 0, 0.0, weights / total)
    return weights, indices, torch.bincount(indices.flatten(), minlength=experts)


def grad(logits, indices, g, gating="softmax", normalize=False, scale=1.0):
    """The logits' gradient by autograd in float64 through the weights of the chosen experts."""
    l = logits.detach().double().requires_grad_(True)
    s = torch.softmax(l, -1) if gating == "softmax" else torch.sigmoid(l)
    w = s.gather(1, indices) * scale
    if normalize:
        w = w / s.gather(1, indices).sum(-1, keepdim=True)
    (out,) = torch.autograd.grad(w, l, g.double())
    return out
