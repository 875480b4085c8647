"""The choice of a token under a temperature, top-k, min-p and top-p in plain torch, 64 bits, row by row."""

from __future__ import annotations

import torch


def kept_of(logits, temperature, top_k=0, top_p=1.0, min_p=0.0):
    """(tokens that stay, in the order of the vocabulary, and their weights) of one row; how near the limits' borders lie to a weight, as a
    share of the whole: a choice nearer than rounding says nothing."""
    x = logits.double()
    x = torch.where(torch.isnan(x), torch.full_like(x, -torch.inf), x) + 0.0
    best = x.max()
    weight = torch.exp((x - best) / temperature)
    weight = torch.where(x == best, torch.ones_like(x), torch.where(torch.isnan(weight) | (x == -torch.inf), torch.zeros_like(x), weight))
    down = torch.argsort(x, descending=True, stable=True)
    count = len(x)
    if top_p <= 0:
        top_k, top_p = 1, 1.0
    if top_k > 0:
        count = min(count, top_k)
    near = float("inf")
    if min_p > 0:
        near = float((weight - min(min_p, 1.0)).abs()[weight != min(min_p, 1.0)].min()) if bool((weight != min(min_p, 1.0)).any()) else near
        count = min(count, int((weight >= min(min_p, 1.0)).sum()))
    if top_p < 1:
        sums = torch.cumsum(weight[down[:count]], 0)
        target = top_p * float(sums[-1])
        near = min(near, float((sums - target).abs().min()))
        count = min(count, 1 + int((sums < target).sum()))
    kept = torch.sort(down[:count]).values
    return kept, weight[kept], near


def chosen(logits, u, temperature, top_k=0, top_p=1.0, min_p=0.0):
    """(the token, how near the draw came to another one as a share of the whole)."""
    x = torch.where(torch.isnan(logits), torch.full_like(logits, -torch.inf), logits).double() + 0.0
    if bool((x == -torch.inf).all()):
        return 0, float("inf")
    if not temperature > 0:
        return int((x == x.max()).nonzero()[0]), float("inf")
    kept, weight, near = kept_of(logits, temperature, top_k, top_p, min_p)
    kept, weight = kept[weight > 0], weight[weight > 0]
    sums = torch.cumsum(weight, 0)
    target = u * float(sums[-1])
    near = min(near / float(sums[-1]), float((sums - target).abs().min()) / float(sums[-1]) if target > 0 else float("inf"))
    return int(kept[min(int((sums <= target).sum()), len(kept) - 1)]), near
