"""Draws from given numbers, row by row from the definition, in 64 bits (CPU)."""

from __future__ import annotations

import torch


def weights(row, T):
    """Weights of a row of logits; NaN counts as -inf, below 2^-44 as 0."""
    x = torch.where(torch.isnan(row), torch.full_like(row, float("-inf")), row).double()
    top = x.max()
    w = torch.where(x == top, torch.ones_like(x), torch.exp((x - top) / T))
    w = torch.nan_to_num(w, nan=0.0)
    w[w < 2.0 ** -44] = 0
    return x, w


def penalised(row, penalty, history):
    row = row.clone()
    if history is not None and len(history):
        at = torch.as_tensor(history)
        v = row[at]
        row[at] = torch.where(v > 0, v / penalty, v * penalty)
    return row


def kept(row, T, top_k, top_p, min_p):
    """(weights of what is kept and 0 elsewhere, all weights)"""
    x, w = weights(row, T)
    order = torch.sort(x, descending=True, stable=True).indices
    n = len(x)
    if 0 < top_k < n:
        order = order[:top_k]
    if top_p < 1:
        mass = torch.cumsum(w[order], 0)
        limit = max(top_p, 0.0) * mass[-1]
        order = order[:1 + int((mass[:-1] <= limit).sum())]
    out = torch.zeros_like(w)
    out[order] = w[order]
    if min_p > 0:
        out[w < min(min_p, 1.0)] = 0
    return out, w


def draw(row, u, T, top_k, top_p, min_p):
    """Returns (tokens, probabilities) for the numbers `u`, and how near a number came to a border."""
    row = row.float()
    x = torch.where(torch.isnan(row), torch.full_like(row, float("-inf")), row)
    if x.max() == float("-inf"):
        return torch.zeros(len(u), dtype=torch.int32), torch.zeros(len(u))
    if not T > 0:
        return torch.full((len(u),), int(torch.nonzero(x == x.max())[0]), dtype=torch.int32), torch.ones(len(u))
    w, _ = kept(x, T, top_k, top_p, min_p)
    cdf = torch.cumsum(w, 0)
    at = torch.searchsorted(cdf, u.double().clamp(min=0) * cdf[-1], right=True)
    at = at.clamp(max=int(torch.nonzero(w)[-1]))
    return at.int(), (w[at] / cdf[-1]).float()
