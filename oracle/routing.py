"""Plain restatement in 64 bits of the routing operators and of gradient clipping.
TEST INFRASTRUCTURE ONLY (results are checked against it; never shipped).

Row by row from the definitions: scores, the order of the experts, groups, the
weights and the gradient of the logits; the stable expert order; the weighted
sum of expert rows and its gradients; the global norm and the clipping factor.
"""
from __future__ import annotations

import math

import numpy as np
import torch

NINF = -math.inf


def _rank_key(value):
    """Sort key of an order value: NaN first, then descending."""
    return (0, 0.0) if math.isnan(value) else (1, -value)


def _best(values, n):
    """Indices of the n best of {index: value} that can be taken, in order."""
    there = [i for i, v in values.items() if v != NINF]
    return sorted(there, key=lambda i: _rank_key(values[i]) + (i,))[:n]


def scores_of(l, score):
    with np.errstate(all="ignore"):
        if score == "softmax":
            p = np.exp(l - l.max())
            return p / p.sum()
        return 1.0 / (1.0 + np.exp(-l))


def route_row(l, k, score, bias, groups, top_groups, group_best):
    """The chosen experts of one row of logits (float64), in order."""
    E = l.shape[0]
    s = scores_of(l, score)
    order = l if bias is None else s + bias
    values = {e: NINF if l[e] == NINF else float(order[e]) for e in range(E)}
    if groups > 1:
        size, of_group = E // groups, {}
        for g in range(groups):
            two = _best({e: values[e] for e in range(g * size, (g + 1) * size)}, 2)
            if not two:
                of_group[g] = NINF
            elif group_best == 1:
                of_group[g] = values[two[0]]
            else:
                of_group[g] = float(sum(s[e] + (0.0 if bias is None else bias[e]) for e in two))
        kept = _best(of_group, top_groups)
        values = {e: v for e, v in values.items() if e // size in kept}
    return _best(values, k)


def shares(l, chosen, score, renorm):
    """Weights of the chosen experts before the scale."""
    with np.errstate(all="ignore"):
        if not renorm:
            return scores_of(l, score)[chosen]
        x = l[chosen]
        if score == "softmax":
            q = np.exp(x - x.max())
        else:  # sigmoid(x) / exp(largest of min(x, 0)): the largest cannot vanish
            low = np.where(x > 0, 0.0, x)
            q = np.exp(low - low.max()) / (1.0 + np.exp(-np.abs(x)))
        return q / q.sum()


def route(logits, k, *, score="softmax", bias=None, mask=None, groups=1, top_groups=None, group_best=1,
          renormalize=True, scale=1.0):
    """(weights float64 [T, k], selected int64 [T, k])."""
    low = logits.detach().cpu().double().numpy()
    b = None if bias is None else bias.detach().cpu().double().numpy()
    T = low.shape[0]
    weights, selected = np.zeros((T, k)), np.full((T, k), -1, dtype=np.int64)
    for t in range(T):
        if mask is not None and not bool(mask[t]):
            continue
        chosen = route_row(low[t], k, score, b, groups, groups if top_groups is None else top_groups, group_best)
        if chosen:
            selected[t, :len(chosen)] = chosen
            weights[t, :len(chosen)] = scale * shares(low[t], chosen, score, renormalize)
    return torch.from_numpy(weights), torch.from_numpy(selected)


def route_grad(logits, selected, dweights, *, score="softmax", renormalize=True, scale=1.0):
    """(dlogits float64 [T, E], size [T, E]): the gradient, and the sum of the
    absolute values of the products it is made of."""
    low = logits.detach().cpu().double().numpy()
    T, E = low.shape
    out, size = np.zeros((T, E)), np.zeros((T, E))
    sel, dw = selected.cpu().numpy(), dweights.detach().cpu().double().numpy()
    for t in range(T):
        n = int((sel[t] >= 0).sum())
        if n == 0:
            continue
        c, g = sel[t, :n], scale * dw[t, :n]
        w = shares(low[t], list(c), score, renormalize)
        with np.errstate(all="ignore"):
            away = 1.0 / (1.0 + np.exp(low[t, c]))  # 1 - sigmoid
            if renormalize:
                f = w * (away if score == "sigmoid" else 1.0)
                out[t, c] = f * (g - (g * w).sum())
                size[t, c] = f * (abs(g) + abs(g * w).sum())
            elif score == "sigmoid":
                out[t, c] = g * w * away
                size[t, c] = abs(out[t, c])
            else:
                p = scores_of(low[t], score)
                out[t] = -p * (g * w).sum()
                size[t] = p * abs(g * w).sum()
                out[t, c] += g * w
                size[t, c] += abs(g * w)
    return torch.from_numpy(out), torch.from_numpy(size)


def expert_order(selected, num_experts):
    """(token_index, inverse_permutation, offsets) of the slots in stable order."""
    k = selected.shape[1]
    flat = [int(e) if 0 <= int(e) < num_experts else num_experts for e in selected.reshape(-1).tolist()]
    order = sorted(range(len(flat)), key=lambda i: flat[i])
    inverse = [-1] * len(flat)
    for row, slot in enumerate(order):
        if flat[slot] < num_experts:
            inverse[slot] = row
    ends = np.cumsum(np.bincount(flat, minlength=num_experts + 1)[:num_experts]) if flat else [0] * num_experts
    return (torch.tensor([i // k for i in order], dtype=torch.int64), torch.tensor(inverse, dtype=torch.int64),
            torch.tensor(np.asarray(ends), dtype=torch.int32))


def combine(rows, weights, inverse):
    """(out [T, D], the sum of the absolute products) in float64."""
    r, w = rows.detach().cpu().double(), weights.detach().cpu().double()
    T, k = w.shape
    out = torch.zeros(T, r.shape[1], dtype=torch.float64)
    size = torch.zeros_like(out)
    for t, j in zip(*(i.tolist() for i in (inverse.view(T, k) >= 0).nonzero(as_tuple=True))):
        x = w[t, j] * r[int(inverse[t * k + j])]
        out[t] += x
        size[t] += x.abs()
    return out, size


def combine_grad(dout, rows, weights, inverse):
    """(drows, dweights, the sum of the absolute products of dweights) in float64."""
    g, r, w = (x.detach().cpu().double() for x in (dout, rows, weights))
    T, k = w.shape
    drows, dw, size = torch.zeros_like(r), torch.zeros_like(w), torch.zeros_like(w)
    for t, j in zip(*(i.tolist() for i in (inverse.view(T, k) >= 0).nonzero(as_tuple=True))):
        row = int(inverse[t * k + j])
        drows[row] = w[t, j] * g[t]
        dw[t, j] = (g[t] * r[row]).sum()
        size[t, j] = (g[t] * r[row]).abs().sum()
    return drows, dw, size


def clip(grads, max_norm):
    """(norm, factor) in float64."""
    norm = math.sqrt(sum(float(g.detach().cpu().double().square().sum()) for g in grads))
    factor = max_norm / (norm + 1e-6)
    return norm, factor if math.isnan(factor) else min(1.0, factor)
