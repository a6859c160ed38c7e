"""The routing operators' definitions (include/cusort_b200.h) in 64 bits over whole batches, for sizes at which the
loops of routing_reference.py would take too long; test_routing_batched.py holds the two against each other."""
from __future__ import annotations

import torch

INF = float("inf")


def scores(x, bias, score):
    """(available, score) of every logit; x: float64 [T, E], bias: float64 [E] or None."""
    ok = x > -INF
    if bias is not None:
        ok = ok & (bias > -INF)
    x = torch.where(ok, x, -INF)
    if score == "sigmoid":
        return ok, torch.where(ok, 1 / (1 + torch.exp(-x)), 0.0)
    return ok, _softmax(x, ok)


def _softmax(x, ok):
    top = torch.where(ok, x, -INF).amax(1, keepdim=True)
    e = torch.where(ok, torch.exp(torch.where(x == top, 0.0, x - top)), 0.0)
    total = e.sum(1, keepdim=True)
    return torch.where(total > 0, e / total, 0.0)


def _taken(values, ids, fill=0.0):
    return torch.where(ids >= 0, values.gather(1, ids.clamp(min=0)), fill)


def _near(a, b, relative):
    """Different values that 32-bit rounding may put in the other order."""
    off = (a - b).abs()
    size = torch.maximum(a.abs(), b.abs()) if relative else 1.0
    return torch.isfinite(a) & torch.isfinite(b) & (off > 0) & (off < 1e-5 * size)


def route(x, k, bias=None, score="softmax", groups=1, groups_kept=None, group_score="max", renormalize=False,
          scale=1.0):
    """(weights, experts, sure), as routing_reference.route."""
    ok, s = scores(x, bias, score)
    order = torch.where(ok, x + 0.0 if bias is None else s + (0.0 if bias is None else bias), -INF)
    sure = torch.ones(len(x), dtype=torch.bool, device=x.device)
    groups_kept = groups if groups_kept is None else groups_kept
    if groups_kept < groups:
        value = torch.where(ok, s, -INF) if group_score == "top2" and bias is None else order
        members = value.view(len(x), groups, -1).sort(2, descending=True).values
        mark = members[..., 0]
        if group_score == "top2" and members.shape[2] > 1:
            mark = mark + torch.where(members[..., 1] > -INF, members[..., 1], 0.0)
        by = mark.sort(dim=1, descending=True, stable=True)
        if group_score == "top2" or bias is not None:
            sure &= ~_near(by.values[:, groups_kept - 1], by.values[:, groups_kept], bias is None)
        keep = torch.zeros_like(mark, dtype=torch.bool).scatter(1, by.indices[:, :groups_kept], True)
        order = torch.where(keep.repeat_interleave(members.shape[2], 1), order, -INF)
    best = order.sort(dim=1, descending=True, stable=True)
    if bias is not None:
        sure &= ~_near(best.values[:, :k + 1][:, :-1], best.values[:, 1:k + 1], False).any(1)
    ids = torch.where(best.values > -INF, best.indices, -1)[:, :k]
    return weights_of(x, s, ids, score, renormalize, scale), ids, sure


def weights_of(x, s, ids, score, renormalize, scale):
    w = _taken(s, ids)
    if renormalize and score == "softmax":
        w = _softmax(_taken(x, ids, -INF), ids >= 0)
    elif renormalize:
        total = w.sum(1, keepdim=True)
        w = torch.where(total > 0, w / total, 0.0)
    return w * scale


def route_backward(grad, x, ids, bias=None, score="softmax", renormalize=False, scale=1.0):
    """For distinct experts in a token."""
    _, s = scores(x, bias, score)
    there = ids >= 0
    grad = torch.where(there, grad, 0.0)
    w = weights_of(x, s, ids, score, renormalize, 1.0)
    used = (grad * w).sum(1, keepdim=True)
    if score == "softmax":
        at = scale * w * (grad - used if renormalize else grad)
    else:
        e = torch.exp(-_taken(x, ids).abs())
        slope = e / (1 + e) ** 2
        total = _taken(s, ids).sum(1, keepdim=True)
        at = scale * slope * (torch.where(total > 0, (grad - used) / total, 0.0) if renormalize else grad)
    out = torch.zeros(len(x), x.shape[1] + 1, dtype=x.dtype, device=x.device)  # the last column takes what has no expert
    out.scatter_(1, torch.where(there, ids, x.shape[1]), torch.where(there, at, 0.0))
    out = out[:, :-1]
    return out - scale * s * used if score == "softmax" and not renormalize else out


def plan(flat, num_experts, align, capacity):
    """(counts, offsets, sources, positions) of int64 experts, on any device."""
    key = torch.where((flat >= 0) & (flat < num_experts), flat, num_experts)
    ordered, order = key.sort(stable=True)
    counts = torch.bincount(key, minlength=num_experts + 1)[:num_experts]
    offsets = torch.zeros(num_experts + 1, dtype=torch.int64, device=flat.device)
    offsets[1:] = ((counts + align - 1) // align * align).cumsum(0)
    begin = counts.cumsum(0) - counts
    on = ordered < num_experts
    pair, expert = order[on], ordered[on]
    row = offsets[expert] + torch.arange(len(pair), device=flat.device) - begin[expert]
    sources = torch.full((capacity,), -1, dtype=torch.int64, device=flat.device)
    positions = torch.full_like(flat, -1)
    sources[row] = pair
    positions[pair] = row
    return counts, offsets, sources, positions
