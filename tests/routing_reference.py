"""Plain 64-bit implementations of the routing and placement operators, for the tests: loops over numpy arrays,
written from the definitions in include/cusort_b200.h."""
from __future__ import annotations

import numpy as np


def order_values(logits, bias, score):
    """(available, score, order value) of every logit, in 64 bits."""
    x = np.asarray(logits, np.float64)
    ok = x > -np.inf
    if bias is not None:
        ok = ok & (np.asarray(bias, np.float64) > -np.inf)
    s = np.zeros_like(x)
    for t in range(x.shape[0]):
        on = ok[t]
        if not on.any():
            continue
        v = x[t, on]
        if score == "sigmoid":
            with np.errstate(over="ignore"):
                s[t, on] = 1 / (1 + np.exp(-v))
        else:
            top = v.max()
            e = np.ones_like(v)
            e[v != top] = np.exp(v[v != top] - top)
            s[t, on] = e / e.sum()
    order = np.where(ok, x if bias is None else s + np.asarray(bias, np.float64), -np.inf)
    return ok, s, order


def route(logits, k, bias=None, score="softmax", groups=1, groups_kept=None, group_score="max", renormalize=False,
          scale=1.0):
    """(weights, experts, sure): `sure` is false for rows where two different values that decide lie within 1e-5
    of each other, so that 32-bit rounding may decide otherwise."""
    ok, s, order = order_values(logits, bias, score)
    T, E = order.shape
    groups_kept = groups if groups_kept is None else groups_kept
    experts, weights, sure = np.full((T, k), -1), np.zeros((T, k)), np.ones(T, bool)
    for t in range(T):
        c = order[t].copy()
        if groups_kept < groups:
            per = E // groups
            value = s[t] if group_score == "top2" and bias is None else c
            marks = []
            for g in range(groups):
                members = sorted((value[e] for e in range(g * per, (g + 1) * per) if ok[t, e]), reverse=True)
                members = members[:2 if group_score == "top2" else 1]
                marks.append(sum(members) if members else -np.inf)
            by = sorted(range(groups), key=lambda g: (-marks[g], g))
            if group_score == "top2" or bias is not None:
                a, b = marks[by[groups_kept - 1]], marks[by[groups_kept]]
                sure[t] &= not (np.isfinite(a) and np.isfinite(b) and 0 < abs(a - b) < 1e-5)
            for g in by[groups_kept:]:
                c[g * per:(g + 1) * per] = -np.inf
        best = sorted((e for e in range(E) if c[e] > -np.inf), key=lambda e: (-c[e], e))
        if bias is not None:
            near = [0 < abs(c[a] - c[b]) < 1e-5 for a, b in zip(best[:k], best[1:k + 1])]
            sure[t] &= not any(near)
        best = best[:k]
        experts[t, :len(best)] = best
        weights[t] = weights_of(logits[t], s[t], experts[t], score, renormalize, scale)
    return weights, experts, sure


def weights_of(x, s, ids, score, renormalize, scale):
    on = ids >= 0
    w = np.zeros(len(ids))
    if not on.any():
        return w
    w[on] = s[ids[on]]
    if renormalize and score == "softmax":
        v = np.asarray(x, np.float64)[ids[on]]
        e = np.ones_like(v)
        e[v != v.max()] = np.exp(v[v != v.max()] - v.max())
        w[on] = e / e.sum()
    elif renormalize:
        w = w / w.sum() if w.sum() > 0 else np.zeros_like(w)
    return w * scale


def route_backward(grad, logits, ids, bias=None, score="softmax", renormalize=False, scale=1.0):
    ok, s, _ = order_values(logits, bias, score)
    out = np.zeros(ok.shape)
    for t in range(ok.shape[0]):
        on = [j for j in range(ids.shape[1]) if 0 <= ids[t, j] < ok.shape[1] and ok[t, ids[t, j]]]
        if not on:
            continue
        e, g = ids[t, on], np.asarray(grad, np.float64)[t, on]
        w = weights_of(logits[t], s[t], e, score, renormalize, 1.0)
        used = (g * w).sum()
        if score == "softmax":
            if renormalize:
                out[t, e] = scale * w * (g - used)
            else:
                out[t] = -scale * s[t] * used
                out[t, e] += scale * w * g
        else:
            x = np.asarray(logits, np.float64)[t, e]
            slope = np.exp(-np.abs(x)) / (1 + np.exp(-np.abs(x))) ** 2
            total = s[t, e].sum()
            if renormalize:
                out[t, e] = scale * (g - used) / total * slope if total > 0 else 0.0
            else:
                out[t, e] = scale * g * slope
    return out


def plan(experts, num_experts, align, capacity):
    flat = np.asarray(experts).reshape(-1)
    rows = [[i for i, e in enumerate(flat) if e == f] for f in range(num_experts)]
    offsets = np.concatenate([[0], np.cumsum([-(-len(r) // align) * align for r in rows])])
    sources, positions = np.full(capacity, -1), np.full(flat.shape, -1)
    for f, members in enumerate(rows):
        for n, i in enumerate(members):
            sources[offsets[f] + n] = i
            positions[i] = offsets[f] + n
    return np.array([len(r) for r in rows]), offsets, sources, positions.reshape(np.shape(experts))


def page_plan(cached, new, tables, block, tokens, free=None, left=0):
    """(slots, positions, starts, served, left); writes into tables."""
    left = 0 if free is None else min(max(left, 0), len(free))
    slots, positions, starts, served, taken, short = [], [], [0], [], 0, False
    for r, (c, n) in enumerate(zip(cached, new)):
        c, n = max(int(c), 0), max(int(n), 0)
        held, end = -(-c // block), -(-(c + n) // block)
        fits = c + n < 2 ** 31 and end <= tables.shape[1]
        need = end - held if fits and free is not None else 0
        short |= need > left - taken
        ok = fits and (need == 0 or not short)
        if ok and need:
            tables[r, held:end] = free[left - taken - need:left - taken][::-1]
            taken += need
        for q in range(n):
            if len(slots) == tokens:
                break
            page, at = divmod(c + q, block)
            there = ok and tables[r, page] >= 0
            slots.append(int(tables[r, page]) * block + at if there else -1)
            positions.append(min(c + q, 2 ** 31 - 1))
        starts.append(min(starts[-1] + n, 2 ** 31 - 1))
        served.append(ok)
    slots += [-1] * (tokens - len(slots))
    positions += [-1] * (tokens - len(positions))
    return np.array(slots, np.int64), np.array(positions), np.array(starts), np.array(served, bool), left - taken
