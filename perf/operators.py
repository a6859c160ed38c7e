"""Cases of the token-routing and cache-placement operators: routing to experts, grouping by expert, moving the
rows there and back, and building block tables and slot maps.  Each operator is given twice: in plain torch
operations, and (where ``own`` is true) through ``libcusort_b200``."""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
INF = math.inf


# --------------------------------------------------------------------------------------------------------- cases

def _route(name, tokens, experts, k, dtype, score, **more):
    return {"name": name, "op": "route", "tokens": tokens, "experts": experts, "k": k, "dtype": dtype, "score": score,
            "groups": 1, "kept": 1, "group_score": "max", "bias": False, "renormalize": False, "scale": 1.0,
            "masked": 0.0, "train": False, **more}


def _plan(name, tokens, experts, k, align, dropped=0.0):
    return {"name": name, "op": "plan", "tokens": tokens, "experts": experts, "k": k, "align": align,
            "dropped": dropped}


def _move(name, tokens, experts, k, hidden, dtype, align, dropped=0.0, residual=False, train=False):
    return {"name": name, "op": "move", "tokens": tokens, "experts": experts, "k": k, "hidden": hidden,
            "dtype": dtype, "align": align, "dropped": dropped, "residual": residual, "train": train}


def _page(name, requests, prefills, chunk, context, block, short=False):
    return {"name": name, "op": "page", "requests": requests, "prefills": prefills, "chunk": chunk,
            "context": context, "block": block, "short": short}


def listed():
    return [
        # one decode step of a small batch: latency alone
        _route("route_decode", 16, 64, 6, "bf16", "softmax"),
        # a prefill batch with the balanced, group-limited sigmoid router; router logits kept in 32 bits
        _route("route_prefill_grouped", 8192, 256, 8, "f32", "sigmoid", groups=8, kept=4, group_score="top2",
               bias=True, renormalize=True, scale=2.5),
        # training, renormalised softmax: the gradient touches the chosen experts alone
        _route("route_train_renorm", 32768, 128, 4, "bf16", "softmax", renormalize=True, train=True),
        # training, plain softmax over an expert count that is no power of two, some experts and rows masked: a
        # dense gradient
        _route("route_train_dense", 16383, 60, 4, "f16", "softmax", masked=0.05, train=True),
        # grouping of a decode batch, segments aligned for a small product tile
        _plan("plan_decode", 64, 256, 8, 16),
        # grouping of a training batch, segments aligned for a 128-row product tile, some pairs dropped
        _plan("plan_train", 32768, 128, 8, 128, dropped=0.02),
        # rows of a decode batch to the experts and back, added to the residual
        _move("move_decode", 32, 64, 8, 2048, "bf16", 1, residual=True),
        # rows of a prefill batch, larger than the cache
        _move("move_prefill", 8192, 128, 8, 4096, "bf16", 1, dropped=0.02),
        # forward and all gradients of a training batch of odd sizes
        _move("move_train", 4099, 60, 6, 2056, "f16", 16, dropped=0.02, train=True),
        # a decode step: one new token for every request
        _page("page_decode", 256, 0, 1, 8192, 16),
        # a serving step: decoding requests and chunks of prompts
        _page("page_mixed", 96, 32, 2048, 16384, 64),
        # an offline batch: many prompts at once
        _page("page_offline", 4096, 4096, 512, 4096, 32),
    ]


def _log(rng, low, high):
    """A whole number between low and high, spread over its logarithm; odd ones and powers of two among them."""
    v = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    if rng.random() < 0.3:
        v = 1 << (v.bit_length() - 1)
    return min(high, max(low, v if v != 3072 else v + 1))


def draw(rng):
    op = rng.choice(["route", "route", "plan", "move", "move", "page"])
    if op == "page":
        requests = _log(rng, 1, 4096)
        return _drop_name(_page("", requests, rng.randint(0, requests), _log(rng, 1, min(2048, (1 << 21) // requests)),
                                _log(rng, 16, 16384 if requests < 512 else 4096), rng.choice([1, 16, 32, 48, 64, 128]),
                                rng.random() < 0.25))
    experts = _log(rng, 8, 512)
    k = rng.randint(1, min(8, experts))
    if op == "plan":
        return _drop_name(_plan("", _log(rng, 1, 32768), experts, k, rng.choice([1, 8, 16, 128]),
                                rng.choice([0.0, 0.02, 0.3])))
    if op == "move":
        hidden = _log(rng, 128, 4096)
        train = rng.random() < 0.4
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
        most = 1_000_000_000 // (hidden * TYPES[dtype].itemsize * (5 * k + 4 if train else 2 * k + 3))
        return _drop_name(_move("", _log(rng, 1, max(1, min(32768, most))), experts, k, hidden, dtype,
                                rng.choice([1, 1, 8, 16]), rng.choice([0.0, 0.02]), rng.random() < 0.5, train))
    # a bias goes with sigmoid scores here: which of two experts with nearly the same softmax score plus bias is
    # the larger one hangs on the order in which the softmax's sum was taken
    score = rng.choice(["softmax", "sigmoid"])
    groups, kept = 1, 1
    if experts >= 32 and rng.random() < 0.5:
        groups = rng.choice([4, 8])
        kept = rng.randint(groups // 4, groups // 2)
        experts = -(-experts // groups) * groups
        k = min(k, kept * (experts // groups))
    if experts == 3072 // groups * groups:
        experts += groups
    return _drop_name(_route("", _log(rng, 1, min(32768, (1 << 22) // experts)), experts, k,
                             rng.choice(["bf16", "f16", "f32"]), score, groups=groups, kept=kept,
                             group_score=rng.choice(["max", "top2"]), bias=score == "sigmoid" and rng.random() < 0.5,
                             renormalize=rng.random() < 0.5, scale=rng.choice([1.0, 2.5]),
                             masked=rng.choice([0.0, 0.0, 0.05]), train=rng.random() < 0.5))


def _drop_name(case):
    del case["name"]
    return case


# -------------------------------------------------------------------------------------------------------- inputs

def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    return {"route": _prepare_route, "plan": _prepare_plan, "move": _prepare_move, "page": _prepare_page}[
        case["op"]](case, gen)


def _normal(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda")


def _chance(gen, *shape):
    return torch.rand(*shape, generator=gen, device="cuda")


def _prepare_route(case, gen):
    T, E = case["tokens"], case["experts"]
    logits = _normal(gen, T, E) * 1.5 + _normal(gen, E) * 0.7  # some experts are liked better than others
    if case["masked"]:
        logits[_chance(gen, T, E) < case["masked"]] = -INF
        logits[_chance(gen, T) < case["masked"] / 5] = -INF  # padding tokens: nothing is left
    return {"case": case, "logits": logits.to(TYPES[case["dtype"]]),
            "bias": _normal(gen, E) * 0.1 if case["bias"] else None,
            "grad": _normal(gen, T, case["k"]) if case["train"] else None}


def _chosen(case, gen):
    """[T, k] expert ids as a router gives them: distinct within a token, some experts liked better."""
    T, E = case["tokens"], case["experts"]
    scores = _normal(gen, T, E) + _normal(gen, E) * 0.7
    ids = scores.topk(case["k"], dim=1).indices.int()
    if case["dropped"]:
        ids[_chance(gen, T, case["k"]) < case["dropped"]] = -1
    return ids


def _capacity(case):
    pairs = case["tokens"] * case["k"]
    return pairs + min(case["experts"], pairs) * (case["align"] - 1)


def _prepare_plan(case, gen):
    return {"case": case, "ids": _chosen(case, gen)}


def _prepare_move(case, gen):
    T, k, H, dtype = case["tokens"], case["k"], case["hidden"], TYPES[case["dtype"]]
    ids = _chosen(case, gen)
    _, _, sources, positions = _plan_plain(ids, case["experts"], case["align"])
    state = {"case": case, "sources": sources, "positions": positions, "x": _normal(gen, T, H).to(dtype),
             "weights": _normal(gen, T, k).softmax(1), "y": _normal(gen, _capacity(case), H).to(dtype),
             "residual": _normal(gen, T, H).to(dtype) if case["residual"] else None}
    if case["train"]:
        state["grad_out"] = _normal(gen, T, H).to(dtype)
        state["grad_rows"] = _normal(gen, _capacity(case), H).to(dtype)
    return state


def _lengths(case, gen):
    R = case["requests"]
    cached = torch.exp(_chance(gen, R) * math.log(case["context"])).int()
    new = torch.ones(R, dtype=torch.int32, device="cuda")
    new[:case["prefills"]] = torch.tensor(_chunks(case), dtype=torch.int32, device="cuda")
    return cached, new[torch.randperm(R, generator=gen, device="cuda")]


def _chunks(case):
    """The lengths of the prompts' chunks, spread from one token to the longest."""
    return [1 + i * case["chunk"] // case["prefills"] for i in range(case["prefills"])]


def _tokens(case):
    """Room for the step's new tokens, as a server rounds it up for its buffers: the last few may hold none."""
    return -(-(case["requests"] - case["prefills"] + sum(_chunks(case))) // 8) * 8


def _width(case):
    return -(-(case["context"] + case["chunk"]) // case["block"]) + 1


def _prepare_page(case, gen):
    R, B, width = case["requests"], case["block"], _width(case)
    cached, new = _lengths(case, gen)
    pool = torch.randperm(R * width, generator=gen, device="cuda").int().view(R, width)
    used = (torch.arange(width, device="cuda") < ((cached + B - 1) // B)[:, None])
    need = (cached + new + B - 1) // B - (cached + B - 1) // B
    free = pool[~used]
    total = int(need.sum())
    left = total // 2 if case["short"] else min(free.numel(), total + 64)
    return {"case": case, "cached": cached, "new": new, "tables": torch.where(used, pool, -1), "free": free,
            "left": torch.tensor([left], dtype=torch.int32, device="cuda"), "tokens": _tokens(case)}


# ---------------------------------------------------------------------------------------------------- plain forms

def _available(logits, bias):
    x = logits.float() + 0.0  # -0 and +0 are the same logit
    ok = x > -INF
    if bias is not None:
        ok = ok & (bias > -INF)
    return torch.where(ok, x, -INF), ok


def _scores(x, ok, score):
    """Unnormalised scores and what divides them (None: nothing does)."""
    if score == "sigmoid":
        return torch.where(ok, 1.0 / (1.0 + torch.exp(-x)), 0.0), None
    top = x.amax(1, keepdim=True)
    e = torch.where(ok, torch.exp(torch.where(x == top, 0.0, x - top)), 0.0)
    return e, e.sum(1, keepdim=True)


def _take(values, ids):
    """values[t, ids[t, j]], and nothing where the id is -1."""
    return torch.where(ids >= 0, values.gather(1, ids.clamp(min=0).long()), 0.0)


def _route_plain(logits, bias, case):
    x, ok = _available(logits, bias)
    e, total = _scores(x, ok, case["score"])
    s = e if total is None else torch.where(ok, e / total, 0.0)
    order = x if bias is None else torch.where(ok, s + bias, -INF)
    if case["kept"] < case["groups"]:
        value = e if bias is None and case["group_score"] == "top2" else order
        best = torch.where(ok, value, -INF).view(len(x), case["groups"], -1).sort(2, descending=True).values
        group = best[..., 0]
        if case["group_score"] == "top2" and best.shape[2] > 1:
            group = group + torch.where(best[..., 1] > -INF, best[..., 1], 0.0)
        ranks = group.sort(dim=1, descending=True, stable=True).indices[:, :case["kept"]]
        keep = torch.zeros_like(group, dtype=torch.bool).scatter(1, ranks, True)
        order = torch.where(keep.repeat_interleave(best.shape[2], 1, output_size=x.shape[1]), order, -INF)
    value, ids = order.sort(dim=1, descending=True, stable=True)
    ids = torch.where(value > -INF, ids, -1)[:, :case["k"]].int()
    return _weights(x, s, ids, case), ids


def _weights(x, s, ids, case):
    chosen = ids >= 0
    if not case["renormalize"]:
        return _take(s, ids) * case["scale"]
    if case["score"] == "softmax":
        xc = torch.where(chosen, _take(x, ids), -INF)
        top = xc.amax(1, keepdim=True)
        w = torch.where(chosen, torch.exp(torch.where(xc == top, 0.0, xc - top)), 0.0)
    else:
        w = _take(s, ids)
    total = w.sum(1, keepdim=True)
    return torch.where(total > 0, w / total, 0.0) * case["scale"]


def _route_backward_plain(grad, logits, bias, ids, case):
    x, ok = _available(logits, bias)
    e, total = _scores(x, ok, case["score"])
    s = e if total is None else torch.where(ok, e / total, 0.0)
    scale, chosen = case["scale"], ids >= 0
    grad = torch.where(chosen, grad, 0.0)
    weights = _weights(x, s, ids, case)
    used = (grad * weights).sum(1, keepdim=True)
    if case["score"] == "sigmoid":
        sc = _take(s, ids)
        both = sc.sum(1, keepdim=True)
        slope = torch.where(both > 0, (scale * grad - used) / both, 0.0) if case["renormalize"] else scale * grad
        at = slope * sc * (1.0 - sc)
    else:
        at = weights * (grad - used / scale) if case["renormalize"] else weights * grad
    out = torch.zeros(len(x), x.shape[1] + 1, device=x.device)  # the last column takes what has no expert
    out.scatter_(1, torch.where(chosen, ids, x.shape[1]).long(), torch.where(chosen, at, 0.0))
    out = out[:, :-1]
    if case["score"] == "softmax" and not case["renormalize"]:
        out = out - s * used
    return out.to(logits.dtype)


def _plan_plain(ids, experts, align):
    flat = ids.reshape(-1).long()
    pairs, cap = flat.numel(), flat.numel() + min(experts, flat.numel()) * (align - 1)
    key = torch.where((flat >= 0) & (flat < experts), flat, experts)
    key, order = key.sort(stable=True)
    first = torch.searchsorted(key, torch.arange(experts + 1, device=key.device))
    counts = first[1:] - first[:-1]
    offsets = torch.zeros(experts + 1, dtype=torch.long, device=key.device)
    offsets[1:] = ((counts + align - 1) // align * align).cumsum(0)
    place = torch.arange(pairs, device=key.device) - first[key] + offsets[key]
    place = torch.where(key < experts, place, cap)
    sources = torch.full((cap + 1,), -1, dtype=torch.int32, device=key.device)
    sources[place] = torch.where(key < experts, order, -1).int()
    positions = torch.empty_like(place)
    positions[order] = torch.where(key < experts, place, -1)
    return counts.int(), offsets.int(), sources[:cap], positions.view(ids.shape).int()


def _dispatch_plain(x, sources, k):
    rows = x[sources.clamp(min=0).long() // k]
    return torch.where((sources >= 0)[:, None], rows, 0)


def _combine_plain(rows, weights, positions, residual):
    at = rows.float()[positions.clamp(min=0).long()]
    if weights is not None:
        at = at * weights[..., None]
    out = torch.where((positions >= 0)[..., None], at, 0.0).sum(1)
    return (out if residual is None else out + residual.float()).to(rows.dtype)


def _combine_backward_plain(grad, rows, weights, sources, positions):
    g = grad.float()
    there, src = (sources >= 0)[:, None], sources.clamp(min=0).long()
    grad_rows = torch.where(there, g[src // positions.shape[1]] * weights.reshape(-1)[src][:, None], 0.0)
    products = (rows.float()[positions.clamp(min=0).long()] * g[:, None, :]).sum(2)
    return grad_rows.to(rows.dtype), torch.where(positions >= 0, products, 0.0)


def _page_plain(cached, new, tables, block, tokens, free, left):
    starts = torch.zeros(len(new) + 1, dtype=torch.long, device=new.device)
    starts[1:] = new.long().cumsum(0)
    old, end = (cached + block - 1) // block, (cached + new + block - 1) // block
    fits = end <= tables.shape[1]
    need = torch.where(fits, end - old, 0)
    taken = need.long().cumsum(0)
    served = fits & ((need == 0) | (taken <= left))
    column = torch.arange(tables.shape[1], device=new.device)
    fresh = served[:, None] & (column >= old[:, None]) & (column < end[:, None])
    rank = left - 1 - ((taken - need)[:, None] + column - old[:, None])
    tables.copy_(torch.where(fresh, free[rank.clamp(0, len(free) - 1)], tables))
    token = torch.arange(tokens, device=new.device)
    there = token < starts[-1]
    request = torch.searchsorted(starts[1:], token, right=True).clamp(max=len(new) - 1)
    place = cached[request] + token - starts[request]
    page = tables[request, (place // block).clamp(max=tables.shape[1] - 1)].long()
    slots = torch.where(there & served[request] & (page >= 0), page * block + place % block, -1)
    remain = left - torch.where(taken <= left, taken, 0).amax().int()
    return {"slots": slots, "positions": torch.where(there, place, -1).int(), "starts": starts.int(), "served": served, "left": remain,
            "tables": tables}


# ------------------------------------------------------------------------------------------------------------ run

def run(state):
    return {"route": _run_route, "plan": _run_plan, "move": _run_move, "page": _run_page}[state["case"]["op"]](state)


def _run_route(state):
    case, logits, bias, grad = state["case"], state["logits"], state["bias"], state["grad"]
    if own:
        from libcusort_b200 import routing
        weights, ids = routing.route(
            logits, case["k"], bias=bias, score=case["score"], groups=case["groups"], groups_kept=case["kept"],
            group_score=case["group_score"], renormalize=case["renormalize"], scale=case["scale"])
        if grad is None:
            return weights, ids
        return weights, ids, routing.route_backward(grad, logits, ids, bias=bias, score=case["score"],
                                                    renormalize=case["renormalize"], scale=case["scale"])
    weights, ids = _route_plain(logits, bias, case)
    if grad is None:
        return weights, ids
    return weights, ids, _route_backward_plain(grad, logits, bias, ids, case)


def _run_plan(state):
    case = state["case"]
    if own:
        from libcusort_b200 import routing
        return tuple(routing.plan_dispatch(state["ids"], case["experts"], align=case["align"]))
    return _plan_plain(state["ids"], case["experts"], case["align"])


def _run_move(state):
    case, sources, positions, weights = state["case"], state["sources"], state["positions"], state["weights"]
    if own:
        from libcusort_b200 import routing
        out = {"rows": routing.dispatch(state["x"], sources, positions),
               "out": routing.combine(state["y"], weights, positions, residual=state["residual"])}
        if case["train"]:
            out["grad_y"], out["grad_weights"] = routing.combine_backward(state["grad_out"], state["y"], weights,
                                                                          sources, positions)
            out["grad_x"] = routing.dispatch_backward(state["grad_rows"], positions)
        return out
    out = {"rows": _dispatch_plain(state["x"], sources, case["k"]),
           "out": _combine_plain(state["y"], weights, positions, state["residual"])}
    if case["train"]:
        out["grad_y"], out["grad_weights"] = _combine_backward_plain(state["grad_out"], state["y"], weights, sources,
                                                                     positions)
        out["grad_x"] = _combine_plain(state["grad_rows"], None, positions, None)
    return out


def _run_page(state):
    if own:
        from libcusort_b200 import paging
        plan = paging.page_plan(state["cached"], state["new"], state["tables"], state["case"]["block"],
                                state["tokens"], free_blocks=state["free"], num_free=state["left"])
        return {"slots": plan.slots, "positions": plan.positions, "starts": plan.starts, "served": plan.served,
                "left": plan.num_free, "tables": state["tables"]}
    return _page_plain(state["cached"], state["new"], state["tables"], state["case"]["block"], state["tokens"],
                       state["free"], state["left"])


# ----------------------------------------------------------------------------------------------------------- work

def work(case):
    if case["op"] == "page":
        requests = case["requests"]
        tokens = _tokens(case)
        blocks = tokens // case["block"] + requests  # entries read or written
        return {"bytes": 17 * requests + 12 * tokens + 12 * blocks, "flops": 4 * tokens}
    pairs = case["tokens"] * case["k"]
    if case["op"] == "plan":
        return {"bytes": 8 * pairs + 4 * _capacity(case) + 8 * case["experts"], "flops": 4 * pairs}
    if case["op"] == "route":
        logits = case["tokens"] * case["experts"]
        size = TYPES[case["dtype"]].itemsize
        nbytes = logits * size + 8 * pairs
        if case["train"]:
            dense = case["score"] == "softmax" and not case["renormalize"]
            read = logits if dense else pairs
            nbytes += (logits + read) * size + 8 * pairs
        return {"bytes": nbytes, "flops": (16 if case["train"] else 8) * logits}
    size, tokens, cap = TYPES[case["dtype"]].itemsize, case["tokens"], _capacity(case)
    row = case["hidden"] * size
    nbytes = row * (2 * tokens + cap + pairs) + 12 * pairs + 4 * cap + (row * tokens if case["residual"] else 0)
    if case["train"]:
        nbytes += row * (2 * tokens + cap + 2 * pairs) + 12 * pairs
    return {"bytes": nbytes, "flops": (6 if case["train"] else 2) * pairs * case["hidden"]}


# ---------------------------------------------------------------------------------------------- 64-bit definitions

def exact(case, seed):
    """What run() returns, from the definitions in 64 bits; nothing where the outputs are whole numbers alone."""
    state = prepare(case, seed)
    if case["op"] == "route":
        return _exact_route(state)
    if case["op"] == "move":
        return _exact_move(state)
    return None


def _exact_route(state):
    case, bias = state["case"], state["bias"]
    x = state["logits"].double().requires_grad_()
    live = torch.isfinite(x) if bias is None else torch.isfinite(x) & torch.isfinite(bias)
    s = torch.sigmoid(x) if case["score"] == "sigmoid" else \
        torch.softmax(x.masked_fill(~live, -1e300), 1)
    s = s.masked_fill(~live, 0.0)
    with torch.no_grad():
        c = (x if bias is None else s + bias.double()).masked_fill(~live, -INF)
        if case["kept"] < case["groups"]:
            value = s.masked_fill(~live, -INF) if bias is None and case["group_score"] == "top2" else c
            members = value.view(-1, case["groups"], value.shape[1] // case["groups"])
            two = members.topk(min(2 if case["group_score"] == "top2" else 1, members.shape[2]), 2).values
            group = torch.where(two > -INF, two, 0.0).sum(2).masked_fill(two[..., 0] == -INF, -INF)
            below = (-group).argsort(dim=1, stable=True).argsort(1) >= case["kept"]
            c = c.masked_fill(below[..., None].expand_as(members).reshape(c.shape), -INF)
        ids = (-c).argsort(dim=1, stable=True)[:, :case["k"]]
        there = c.gather(1, ids) > -INF
    if case["renormalize"] and case["score"] == "softmax":
        w = torch.softmax(x.gather(1, ids).masked_fill(~there, -1e300), 1)
    else:
        w = s.gather(1, ids)
        if case["renormalize"]:
            total = w.masked_fill(~there, 0.0).sum(1, keepdim=True)
            w = w / total.masked_fill(total == 0, 1.0)
    w = (w * case["scale"]).masked_fill(~there, 0.0)
    if state["grad"] is None:
        return w.detach(), None
    (w * state["grad"].double()).sum().backward()
    return w.detach(), None, x.grad


def _exact_move(state):
    case, k = state["case"], state["case"]["k"]
    T, H = case["tokens"], case["hidden"]
    placed = (state["sources"] >= 0).nonzero()[:, 0]
    pair = state["sources"][placed].long()
    token, weight = pair // k, state["weights"].double().reshape(-1)[pair][:, None]
    rows = torch.zeros(_capacity(case), H, dtype=torch.float64, device="cuda")
    rows[placed] = state["x"].double()[token]
    total = torch.zeros(T, H, dtype=torch.float64, device="cuda") if state["residual"] is None else \
        state["residual"].double()
    y = state["y"].double()[placed]
    out = {"rows": rows, "out": total.index_add(0, token, y * weight)}
    if case["train"]:
        g = state["grad_out"].double()[token]
        out["grad_y"] = torch.zeros_like(rows).index_copy(0, placed, g * weight)
        out["grad_weights"] = torch.zeros(T * k, dtype=torch.float64, device="cuda").index_copy(
            0, pair, (g * y).sum(1)).view(T, k)
        out["grad_x"] = torch.zeros(T, H, dtype=torch.float64, device="cuda").index_add(
            0, token, state["grad_rows"].double()[placed])
    return out
