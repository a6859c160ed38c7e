"""Cases of the experts' matrix products (with gradients) and of the life of a paged cache's blocks: forking requests,
freeing, copying and compacting.  Each operator is given twice: in plain torch operations, and (where ``own`` is true)
through ``libcusort_b200``."""
import math

import torch

own = False

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


# --------------------------------------------------------------------------------------------------------- cases

def _product(name, tokens, experts, k, rows_in, out, dtype="bf16", align=1, order="in_out", dropped=0.0, train=False):
    return {"name": name, "op": "product", "tokens": tokens, "experts": experts, "k": k, "in": rows_in, "out": out,
            "dtype": dtype, "align": align, "order": order, "dropped": dropped, "train": train}


def _fork(name, groups, beams, context, grown, block, caches, row):
    return {"name": name, "op": "fork", "groups": groups, "beams": beams, "context": context, "grown": grown,
            "block": block, "caches": caches, "row": row}


def _free(name, groups, beams, context, grown, block, done):
    return {"name": name, "op": "free", "groups": groups, "beams": beams, "context": context, "grown": grown,
            "block": block, "done": done}


def _compact(name, groups, beams, context, grown, block, spread, caches, row):
    return {"name": name, "op": "compact", "groups": groups, "beams": beams, "context": context, "grown": grown,
            "block": block, "spread": spread, "caches": caches, "row": row}


def listed():
    return [
        # one token of one request: six experts' weights for a row each; latency
        _product("products_one_token", 1, 64, 6, 2048, 1024),
        # a decode step: nearly every expert has a few rows, the weights' bytes count
        _product("products_decode", 64, 128, 8, 2048, 1536),
        # a prefill batch; weights stored as linear layers keep them, the contracted width contiguous
        _product("products_prefill", 8192, 64, 6, 4096, 2048, order="out_in", dropped=0.02),
        # a training batch with every gradient
        _product("products_train", 8192, 32, 4, 2048, 4096, align=16, train=True),
        # training with odd token and expert counts, segments aligned to 16 rows, some pairs dropped
        _product("products_train_ragged", 4099, 60, 6, 2056, 1400, "f16", 16, dropped=0.02, train=True),
        # widths that are no multiple of 16 bytes, few experts
        _product("products_train_odd", 1000, 16, 2, 771, 1285, "f16", order="out_in", train=True),
        # beam search on a small server: eight prompts of four beams, a step's reordering and its copies
        _fork("fork_beams", 8, 4, 2048, 128, 16, 8, 1024),
        # beam search over an offline batch
        _fork("fork_offline", 512, 4, 1024, 256, 16, 4, 512),
        # after a decode step: some requests are done, drafted tokens of others were refused
        _free("free_step", 256, 1, 8192, 512, 16, 0.05),
        # an offline batch of samples with common prompts comes to its end
        _free("free_offline", 1024, 4, 4096, 512, 32, 0.5),
        # a small pool closes its holes
        _compact("compact_small", 16, 2, 2048, 128, 16, 1.5, 4, 1024),
        # a large pool shrinks by a third: blocks move in every layer
        _compact("compact_large", 256, 4, 8192, 512, 32, 1.5, 4, 512),
    ]


def _log(rng, low, high):
    """A whole number between low and high, spread over its logarithm; odd ones and powers of two among them."""
    v = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    if rng.random() < 0.3:
        v = 1 << (v.bit_length() - 1)
    return min(high, max(low, v))


def _width_of(rng):
    """A layer's width: mostly a multiple of 8 or 64, sometimes any number."""
    v = _log(rng, 64, 4096)
    step = rng.choice([64, 64, 8, 8, 1])
    return max(64, v // step * step)


def draw(rng):
    op = rng.choice(["product", "product", "product", "fork", "free", "compact"])
    if op == "product":
        experts = _log(rng, 4, 256)
        k = rng.randint(1, min(8, experts))
        rows_in, out = _width_of(rng), _width_of(rng)
        experts = max(4, min(experts, (1 << 28) // (rows_in * out)))
        k = min(k, experts)
        train = rng.random() < 0.5
        most = int(1.6e12 / (2 * k * rows_in * out * (3 if train else 1)))
        return _drop_name(_product("", _log(rng, 1, max(1, min(16384, most))), experts, k, rows_in, out,
                                   rng.choice(["bf16", "bf16", "f16"]), rng.choice([1, 1, 8, 16, 128]),
                                   rng.choice(["in_out", "out_in"]), rng.choice([0.0, 0.02, 0.3]), train))
    beams = rng.choice([1, 2, 4, 4, 8])
    groups = _log(rng, 1, 4096 // beams)
    block = rng.choice([1, 16, 16, 32, 48, 64, 128])
    # the tokens of all requests together stay within 2^21, their blocks within 2^18
    most = min(1 << 21, block << 18) // (groups * beams)
    context = _log(rng, 16, max(16, min(8192, most // 2)))
    grown = _log(rng, 1, max(1, min(512, most // 2)))
    if op == "free":
        return _drop_name(_free("", groups, beams, context, grown, block, rng.choice([0.0, 0.05, 0.5, 1.0])))
    caches = rng.randint(1, 8)
    blocks = groups * (-(-(context + beams * grown) // block) + 2 * beams)
    row = _log(rng, 16, max(16, min(1024, (1 << 28) // (blocks * block * caches))))
    if op == "fork":
        return _drop_name(_fork("", groups, beams, context, grown, block, caches, row))
    return _drop_name(_compact("", groups, beams, context, grown, block, rng.choice([1.1, 1.5, 4.0]), caches, row))


def _drop_name(case):
    del case["name"]
    return case


# -------------------------------------------------------------------------------------------------------- inputs

def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    return _prepare_product(case, gen) if case["op"] == "product" else _prepare_pages(case, gen)


def _normal(gen, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=gen, device="cuda", dtype=dtype)


def _chance(gen, *shape):
    return torch.rand(*shape, generator=gen, device="cuda")


def _below(gen, high, *shape):
    return torch.randint(0, high, shape, generator=gen, device="cuda")


def _capacity(case):
    pairs = case["tokens"] * case["k"]
    return pairs + min(case["experts"], pairs) * (case["align"] - 1)


def _prepare_product(case, gen):
    T, E, k, align, dtype = case["tokens"], case["experts"], case["k"], case["align"], TYPES[case["dtype"]]
    # distinct experts for each token, some liked better than others; some pairs dropped
    ids = (_normal(gen, T, E) + _normal(gen, E) * 0.7).topk(k, dim=1).indices
    ids = torch.where(_chance(gen, T, k) < case["dropped"], E, ids).reshape(-1)
    counts = torch.zeros(E + 1, dtype=torch.long, device="cuda").index_add(0, ids, torch.ones_like(ids))[:E]
    offsets = torch.zeros(E + 1, dtype=torch.long, device="cuda")
    offsets[1:] = ((counts + align - 1) // align * align).cumsum(0)
    row = torch.arange(_capacity(case), device="cuda")
    expert = torch.searchsorted(offsets[1:].contiguous(), row, right=True).clamp(max=E - 1)
    there = row < (offsets[:-1] + counts)[expert]

    def rows(width):  # as dispatch, and the gradient of combine, leave them: zeros where there is no pair
        return _normal(gen, _capacity(case), width, dtype=dtype).masked_fill_(~there[:, None], 0.0)

    shape = (E, case["in"], case["out"]) if case["order"] == "in_out" else (E, case["out"], case["in"])
    weights = _normal(gen, *shape, dtype=dtype).mul_(case["in"] ** -0.5)
    return {"case": case, "rows": rows(case["in"]),
            "weights": weights if case["order"] == "in_out" else weights.transpose(1, 2),
            "counts": counts.int(), "offsets": offsets.int(), "grad": rows(case["out"]) if case["train"] else None,
            # where the segments are, on the host: the plain form's loop goes over them
            "segments": list(zip(offsets.tolist(), counts.tolist()))}


def _prompts(case):
    """The prompts' lengths, even in their logarithm."""
    G = case["groups"]
    return [max(1, int(math.exp(math.log(case["context"]) * (i + 0.5) / G))) for i in range(G)]


def _needed(case):
    """Blocks that the requests hold together: those of the prompts, those of their own on average."""
    B, R = case["block"], case["groups"] * case["beams"]
    return sum(n // B for n in _prompts(case)) + int(R * (case["grown"] / (2 * B) + (1 - 1 / B)))


def _blocks(case):
    """The pool: what the requests may hold at most, and room beside it."""
    B, R = case["block"], case["groups"] * case["beams"]
    most = sum(n // B for n in _prompts(case)) + R * (-(-(B - 1 + case["grown"]) // B))
    return max(most, int(_needed(case) * case.get("spread", 1.25))) + R + 8


def _prepare_pages(case, gen):
    """Requests in groups of beams with a common prompt, whose full blocks they share; the rest of each is its own."""
    G, beams, B = case["groups"], case["beams"], case["block"]
    R = G * beams
    prompt = torch.tensor(_prompts(case), dtype=torch.int32, device="cuda")
    prompt = prompt[torch.randperm(G, generator=gen, device="cuda")]
    lens = prompt.repeat_interleave(beams) + _below(gen, case["grown"] + 1, R).int()
    common = (prompt // B).repeat_interleave(beams)
    held = (lens + B - 1) // B
    width = -(-(case["context"] + case["grown"]) // B) + 1
    total = int((prompt // B).sum() + (held - common).sum())
    blocks = _blocks(case)
    pool = torch.randperm(blocks, generator=gen, device="cuda").int()
    column = torch.arange(width, device="cuda")
    first = (prompt // B).cumsum(0) - prompt // B
    own_first = (prompt // B).sum() + (held - common).cumsum(0) - (held - common)
    place = torch.where(column < common[:, None], first.repeat_interleave(beams)[:, None] + column,
                        own_first[:, None] + column - common[:, None])
    there = column < held[:, None]
    tables = torch.where(there, pool[place.clamp(0, blocks - 1)], -1)
    shares = torch.full((blocks + 1,), -1, dtype=torch.int32, device="cuda")
    shares = shares.index_add(0, torch.where(there, tables, blocks).reshape(-1).long(),
                              torch.ones(R * width, dtype=torch.int32, device="cuda"))[:blocks].clamp(min=0)
    free = torch.cat([pool[total:], torch.full((total,), -1, dtype=torch.int32, device="cuda")])
    state = {"case": case, "tables": tables, "lens": lens, "shares": shares, "free": free,
             "left": torch.tensor([blocks - total], dtype=torch.int32, device="cuda")}
    if case["op"] == "free":
        refused = torch.where(_chance(gen, R) < 0.3, _below(gen, 6, R).int(), 0)
        state["keep"] = torch.where(_chance(gen, R) < case["done"], 0, (lens - refused).clamp(min=0))
    else:
        state["caches"] = [_normal(gen, blocks, B, case["row"], dtype=torch.bfloat16) for _ in range(case["caches"])]
    if case["op"] == "fork":
        # each beam goes on from any beam of its group; a few groups are done
        parents = _below(gen, beams, R) + torch.arange(R, device="cuda") // beams * beams
        done = (_chance(gen, G) < 0.05).repeat_interleave(beams)
        state["parents"] = torch.where(done, -1, parents).int()
    return state


# ---------------------------------------------------------------------------------------------------- plain forms

def _products_plain(rows, weights, segments):
    out = torch.zeros(rows.shape[0], weights.shape[2], dtype=rows.dtype, device=rows.device)
    for e, (first, count) in enumerate(segments):
        if count:
            out[first:first + count] = (rows[first:first + count].float() @ weights[e].float()).to(rows.dtype)
    return out


def _products_backward_plain(grad, rows, weights, segments):
    grad_rows = torch.zeros_like(rows)
    grad_weights = torch.zeros_like(weights)
    for e, (first, count) in enumerate(segments):
        if count:
            x, g = rows[first:first + count].float(), grad[first:first + count].float()
            grad_rows[first:first + count] = (g @ weights[e].float().t()).to(rows.dtype)
            grad_weights[e] = (x.t() @ g).to(weights.dtype)
    return grad_rows, grad_weights


def _held(tables, lens, block):
    """How many entries each request holds, and which of the table's they are."""
    held = ((lens.clamp(min=0) + block - 1) // block).clamp(max=tables.shape[1])
    return held, torch.arange(tables.shape[1], device=tables.device) < held[:, None]


def _add(values, at, there, amounts):
    """values[at] += amounts where there; the last, added entry takes the rest."""
    values = torch.cat([values, values.new_zeros(1)])
    at = torch.where(there, at, len(values) - 1).reshape(-1).long()
    return values.index_add(0, at, amounts.expand(there.shape).reshape(-1).int())[:-1]


def _returned(shares, free, left):
    """Blocks that nothing holds any more, ascending, behind the first ``left`` free ones; -1 behind them."""
    gone = shares < 0
    rank = gone.cumsum(0) - 1
    number = torch.arange(len(free), device=free.device)
    out = torch.cat([torch.where(number < left, free, -1), free.new_zeros(1)])
    out = out.index_copy(0, torch.where(gone, left + rank, len(free)), number.int())[:-1]
    return shares.clamp(min=0), out, (left + gone.sum()).int()


def _fork_plain(tables, lens, parents, block, free, left, shares):
    R, width = tables.shape
    N, blocks = len(parents), len(shares)
    valid = (parents >= 0) & (parents < R)
    p = torch.where(valid, parents, 0).long()
    length = torch.where(valid, lens[p], 0)
    held = (length + block - 1) // block
    last = tables[p, (held - 1).clamp(0, width - 1).long()].long()
    part = (length % block != 0) & (held <= width)
    order = torch.arange(N, device=p.device)
    first = torch.full((R,), N, device=p.device).scatter_reduce(0, p, torch.where(valid, order, N), "amin")
    keeps = (first[p] == order) & (shares[last.clamp(0, blocks - 1)] == 0)
    need = valid & part & ~keeps
    rank = need.cumsum(0) - 1
    served = ~need | (rank < left)
    taken = (need & served).sum().int()
    fresh = free[(left - 1 - rank).clamp(0, len(free) - 1)]
    copied = need & served
    ok = valid & served
    column = torch.arange(width, device=p.device)
    mine = ok[:, None] & (column < held[:, None])
    final = copied[:, None] & (column == (held - 1)[:, None])
    out = torch.where(mine, torch.where(final, fresh[:, None], tables[p]), -1)
    _, old = _held(tables, lens, block)
    shares = _add(shares, out, mine & ~final, shares.new_ones(1))
    shares = _add(shares, tables, old, -shares.new_ones(1))
    shares, free, left = _returned(shares, free, left - taken)
    return {"tables": out, "lens": torch.where(ok, length, 0), "sources": torch.where(copied, last, -1).int(),
            "destinations": torch.where(copied, fresh, -1), "served": served, "shares": shares, "free": free,
            "left": left}


def _free_plain(tables, lens, keep, block, free, left, shares):
    _, old = _held(tables, lens, block)
    _, kept = _held(tables, torch.minimum(keep, lens), block)
    shares = _add(shares, tables, old & ~kept, -shares.new_ones(1))
    shares, free, left = _returned(shares, free, left)
    return {"shares": shares, "free": free, "left": left}


def _compact_plain(tables, lens, block, blocks):
    _, there = _held(tables, lens, block)
    shares = _add(torch.full((blocks,), -1, dtype=torch.int32, device=tables.device), tables, there,
                  tables.new_ones(1))
    used = shares >= 0
    before = used.cumsum(0) - used.int()  # used blocks below each
    number = torch.arange(blocks, device=tables.device)
    total = used.sum(0, keepdim=True)
    below = number < total
    half = blocks // 2
    inside = (used & below).sum()
    sources = torch.full((half + 1,), -1, device=tables.device).index_copy(
        0, torch.where(used & ~below, before - inside, half), number)[:-1]
    holes = torch.full((half + 1,), -1, device=tables.device).index_copy(
        0, torch.where(~used & below, number - before, half), number)[:-1]
    moved = torch.where(used & ~below, holes[(before - inside).clamp(0, max(half - 1, 0))], number)
    out = torch.where(there, moved[tables.clamp(min=0).long()].int(), -1)
    new_shares = torch.zeros(blocks + 1, dtype=torch.int32, device=tables.device).index_copy(
        0, torch.where(used, moved, blocks), shares)[:-1]
    free = torch.where(number < blocks - total, blocks - 1 - number, -1).int()
    return {"tables": out, "sources": sources.int(), "destinations": holes.int(), "shares": new_shares, "free": free,
            "left": (blocks - total).int()}


def _copy_plain(caches, sources, destinations):
    there = (sources >= 0) & (destinations >= 0)
    # pairs that are none repeat one that is; where there is none at all, block 0 goes to itself
    one = there.int().argmax()
    s = torch.where(there, sources, sources[one]).clamp(min=0).long()
    d = torch.where(there, destinations, destinations[one]).clamp(min=0).long()
    for cache in caches:
        cache[d] = cache[s]


# ------------------------------------------------------------------------------------------------------------ run

def run(state):
    return {"product": _run_product, "fork": _run_fork, "free": _run_free, "compact": _run_compact}[
        state["case"]["op"]](state)


def _run_product(state):
    rows, weights, grad = state["rows"], state["weights"], state["grad"]
    if own:
        from libcusort_b200 import experts
        out = experts.expert_products(rows, weights, state["counts"], state["offsets"])
        if grad is None:
            return out
        return (out, *experts.expert_products_backward(grad, rows, weights, state["counts"], state["offsets"]))
    out = _products_plain(rows, weights, state["segments"])
    if grad is None:
        return out
    return (out, *_products_backward_plain(grad, rows, weights, state["segments"]))


def _run_fork(state):
    block = state["case"]["block"]
    if own:
        from libcusort_b200 import paging
        fork = paging.page_fork(state["tables"], state["lens"], state["parents"], block, free_blocks=state["free"],
                                num_free=state["left"], shares=state["shares"])
        paging.page_copy(state["caches"], fork.sources, fork.destinations)
        return {"tables": fork.block_tables, "lens": fork.lens, "sources": fork.sources,
                "destinations": fork.destinations, "served": fork.served, "shares": fork.shares,
                "free": fork.free_blocks, "left": fork.num_free, "caches": state["caches"]}
    out = _fork_plain(state["tables"], state["lens"], state["parents"], block, state["free"], state["left"],
                      state["shares"])
    _copy_plain(state["caches"], out["sources"], out["destinations"])
    return {**out, "caches": state["caches"]}


def _run_free(state):
    block = state["case"]["block"]
    if own:
        from libcusort_b200 import paging
        out = paging.page_free(state["tables"], state["lens"], state["keep"], block, free_blocks=state["free"],
                               num_free=state["left"], shares=state["shares"])
        return {"shares": out.shares, "free": out.free_blocks, "left": out.num_free}
    return _free_plain(state["tables"], state["lens"], state["keep"], block, state["free"], state["left"],
                       state["shares"])


def _run_compact(state):
    block, blocks = state["case"]["block"], len(state["shares"])
    if own:
        from libcusort_b200 import paging
        out = paging.page_compact(state["tables"], state["lens"], block, blocks)
        paging.page_copy(state["caches"], out.sources, out.destinations)
        return {"tables": out.block_tables, "sources": out.sources, "destinations": out.destinations,
                "shares": out.shares, "free": out.free_blocks, "left": out.num_free, "caches": state["caches"]}
    out = _compact_plain(state["tables"], state["lens"], block, blocks)
    _copy_plain(state["caches"], out["sources"], out["destinations"])
    return {**out, "caches": state["caches"]}


# ----------------------------------------------------------------------------------------------------------- work

def work(case):
    if case["op"] == "product":
        T, E, k, fin, fout = (case[n] for n in ("tokens", "experts", "k", "in", "out"))
        pairs = T * k * (1.0 - case["dropped"])
        active = E * (1.0 - (1.0 - k / E) ** T)  # experts that a row comes to
        capacity = _capacity(case)
        nbytes = 2 * (pairs * fin + active * fin * fout + capacity * fout)
        if case["train"]:  # the rows and weights are read above
            nbytes += 2 * (pairs * fout + capacity * fin + E * fin * fout)
        return {"bytes": int(nbytes), "flops": int((6 if case["train"] else 2) * pairs * fin * fout)}
    G, beams, B = case["groups"], case["beams"], case["block"]
    R = G * beams
    width = -(-(case["context"] + case["grown"]) // B) + 1
    blocks, needed = _blocks(case), _needed(case)
    held = needed + (beams - 1) * sum(n // B for n in _prompts(case))  # entries of all tables
    if case["op"] == "free":
        return {"bytes": int(4 * held * case["done"] + 16 * blocks + 8 * R), "flops": int(held)}
    nbytes = 4 * (held + R * width) + (16 if case["op"] == "fork" else 8) * blocks + 24 * R
    if case["op"] == "fork":  # a beam in (beams - 1) / beams is not the first of its parent, about; full blocks stay
        copies = 0.95 * R * (1 - 1 / beams) ** beams * (1 - 1 / B)
    else:  # what lies above the count of used blocks moves
        copies = needed * max(0.0, 1 - needed / blocks)
    return {"bytes": int(nbytes + copies * case["caches"] * B * case["row"] * 4), "flops": int(held)}


# ---------------------------------------------------------------------------------------------- 64-bit definitions

def exact(case, seed):
    """What run() returns, from the definitions in 64 bits; nothing where the outputs are whole numbers and copies."""
    if case["op"] != "product":
        return None
    state = prepare(case, seed)
    x = state["rows"].double()
    E, first = case["experts"], state["offsets"].long()
    row = torch.arange(len(x), device=x.device)
    outs, grads, marks = [], [], []
    for e in range(E):
        at = row[(row >= first[e]) & (row < first[e] + state["counts"][e])]
        w = state["weights"][e].double().requires_grad_(case["train"])
        xe = x[at].requires_grad_(case["train"])
        y = torch.einsum("ri,io->ro", xe, w)
        marks.append(at)
        outs.append(y.detach())
        if case["train"]:
            grads.append(torch.autograd.grad((y * state["grad"][at].double()).sum(), [xe, w]))
    at = torch.cat(marks)
    out = torch.zeros(len(x), case["out"], dtype=torch.float64, device=x.device).index_copy(0, at, torch.cat(outs))
    if not case["train"]:
        return out
    grad_rows = torch.zeros_like(x).index_copy(0, at, torch.cat([g for g, _ in grads]))
    return out, grad_rows, torch.stack([g for _, g in grads])
