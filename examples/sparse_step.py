"""A small sparse (mixture-of-experts) layer on the routing operators, in training and in serving.

    python examples/sparse_step.py

Training: router logits -> route -> plan_dispatch -> dispatch -> the experts' products -> combine, with gradients by
autograd.  Serving: page_plan places each step's new tokens in a paged cache, then the same layer runs on them.
Sampling: page_fork goes on from a prompt with several samples that share its blocks, page_free gives back those of
samples that are dropped, page_compact moves what is left together, page_copy copies the blocks.  Nothing in a step
copies to the host.
"""
from __future__ import annotations

import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

import libcusort_b200.ops  # noqa: E402,F401  (registers torch.ops.cusort)
from libcusort_b200.paging import page_compact, page_copy, page_fork, page_free, page_plan  # noqa: E402

cusort = torch.ops.cusort


class SparseLayer(torch.nn.Module):
    """x + the weighted sum of each token's k experts' two-layer networks."""

    ALIGN = 16  # every expert's rows begin at a multiple of it

    def __init__(self, hidden: int, inner: int, experts: int, k: int, **how):
        super().__init__()
        self.router = torch.nn.Parameter(torch.randn(hidden, experts, **how) / hidden ** 0.5)
        self.up = torch.nn.Parameter(torch.randn(experts, hidden, inner, **how) / hidden ** 0.5)
        self.down = torch.nn.Parameter(torch.randn(experts, inner, hidden, **how) / inner ** 0.5)
        self.k = k

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        weights, experts = cusort.route(x @ self.router, self.k, renormalize=True)
        counts, offsets, sources, positions = cusort.plan_dispatch(experts, self.router.shape[1], self.ALIGN)
        rows = cusort.dispatch(x, sources, positions)
        inner = torch.relu(cusort.expert_products(rows, self.up, counts, offsets))
        y = cusort.expert_products(inner, self.down, counts, offsets)
        return cusort.combine(y, weights, sources, positions, x)

    def dense(self, x: torch.Tensor) -> torch.Tensor:
        """The same by every expert on every token."""
        top = (x @ self.router).float().softmax(1).topk(self.k, dim=1)  # as the layer's router: of the rounded logits
        weights = torch.zeros(x.shape[0], self.router.shape[1], device=x.device).scatter(
            1, top.indices, top.values / top.values.sum(1, keepdim=True))
        y = torch.relu(torch.einsum("th,ehf->etf", x, self.up)) @ self.down
        return x + torch.einsum("te,eth->th", weights.to(y.dtype), y)


def train(tokens: int = 300, hidden: int = 64, inner: int = 96, experts: int = 12, k: int = 3,
          dtype: torch.dtype = torch.float32) -> dict[str, float]:
    """Loss and gradients of the layer against the dense form; the largest differences over the largest values."""
    torch.manual_seed(1)
    layer = SparseLayer(hidden, inner, experts, k, device="cuda", dtype=torch.float32).to(dtype)
    x = torch.randn(tokens, hidden, device="cuda").to(dtype).requires_grad_()
    target = torch.randn(tokens, hidden, device="cuda").to(dtype)

    def gradients(f):
        loss = (f(x) - target).square().mean()
        return dict(zip(("x", "router", "up", "down"),
                        torch.autograd.grad(loss, [x, layer.router, layer.up, layer.down]))) | {"loss": loss.detach()}

    ours, dense = gradients(layer), gradients(layer.dense)
    return {n: float((ours[n] - dense[n]).abs().max() / dense[n].abs().max()) for n in ours}


def serve(steps: int = 4, hidden: int = 64, block: int = 16, blocks: int = 64) -> dict[str, int]:
    """A few serving steps: prompts, then a token a step; every token's row is found again at its place."""
    torch.manual_seed(2)
    layer = SparseLayer(hidden, 96, 12, 3, device="cuda", dtype=torch.float32)
    prompts = torch.tensor([37, 1, 16, 100], dtype=torch.int32, device="cuda")
    cached = torch.zeros_like(prompts)
    tables = torch.full((len(prompts), 16), -1, dtype=torch.int32, device="cuda")
    free = torch.randperm(blocks, device="cuda").int()
    num_free = torch.tensor([blocks], dtype=torch.int32, device="cuda")
    cache = torch.zeros(blocks * block + 1, hidden, device="cuda")  # the last row takes what has no slot
    rows = []
    with torch.no_grad():
        for step in range(steps):
            new = prompts if step == 0 else torch.ones_like(prompts)
            tokens = 160 if step == 0 else 8  # as a server rounds its buffers up
            plan = page_plan(cached, new, tables, block, tokens, free_blocks=free, num_free=num_free)
            x = layer(torch.randn(tokens, hidden, device="cuda"))
            cache[torch.where(plan.slots >= 0, plan.slots, blocks * block)] = x
            rows.append((plan, x))
            cached, num_free = cached + new, plan.num_free
    found = 0
    for plan, x in rows:
        for request in range(len(prompts)):
            for i in range(int(plan.starts[request]), int(plan.starts[request + 1])):
                at = int(plan.positions[i])
                found += torch.equal(cache[int(tables[request, at // block]) * block + at % block], x[i])
    return {"tokens": int(cached.sum()), "found": int(found), "blocks_left": int(num_free)}


def sample(samples: int = 4, steps: int = 24, hidden: int = 64, block: int = 16, blocks: int = 128) -> dict[str, int]:
    """Several samples from each prompt; half of them are replaced by the others' copies on the way, all but one of
    each prompt are dropped at the end, and the pool is compacted.  Every token's row is found again at its place."""
    torch.manual_seed(3)
    layer = SparseLayer(hidden, 96, 12, 3, device="cuda", dtype=torch.float32).bfloat16()
    prompts = torch.tensor([37, 5, 50], dtype=torch.int32, device="cuda")
    requests = len(prompts) * samples
    lens, free = torch.zeros_like(prompts), torch.arange(blocks, dtype=torch.int32, device="cuda")
    left = torch.tensor([blocks], dtype=torch.int32, device="cuda")
    shares = torch.zeros(blocks, dtype=torch.int32, device="cuda")
    tables = torch.full((len(prompts), 8), -1, dtype=torch.int32, device="cuda")
    # the last block takes what has no slot
    cache = torch.zeros(blocks + 1, block, hidden, device="cuda", dtype=torch.bfloat16)
    caches = [cache[:blocks]]
    rows = torch.zeros(len(prompts), 8 * block, hidden, device="cuda", dtype=torch.bfloat16)  # what should be found

    def step(new: torch.Tensor, tokens: int):
        nonlocal lens, left
        plan = page_plan(lens, new, tables, block, tokens, free_blocks=free, num_free=left)
        with torch.no_grad():
            x = layer(torch.randn(tokens, hidden, device="cuda").bfloat16())
        cache.view(-1, hidden)[torch.where(plan.slots >= 0, plan.slots, blocks * block)] = x
        token = torch.arange(tokens, device="cuda", dtype=torch.int32)
        request = torch.searchsorted(plan.starts[1:], token, right=True)
        there = request < len(lens)
        rows[request[there], plan.positions[there].long()] = x[there]
        lens, left = lens + new, plan.num_free

    def fork(parents: torch.Tensor):
        nonlocal tables, lens, free, left, shares, rows
        got = page_fork(tables, lens, parents, block, free_blocks=free, num_free=left, shares=shares)
        page_copy(caches, got.sources, got.destinations)
        tables, lens, free, left, shares = got.block_tables, got.lens, got.free_blocks, got.num_free, got.shares
        rows = rows[parents.long()]

    step(prompts, 96)
    fork(torch.arange(requests, dtype=torch.int32, device="cuda") // samples)
    for i in range(steps):
        step(torch.ones_like(lens), 16)
        if i == steps // 2:  # the second half of each prompt's samples go on from the first half
            at = torch.arange(requests, dtype=torch.int32, device="cuda")
            fork(at - at % samples // (samples // 2) * (samples // 2))
    used = blocks - int(left)
    keep = torch.where(torch.arange(requests, device="cuda") % samples == 0, lens, 0)
    rest = page_free(tables, lens, keep, block, free_blocks=free, num_free=left, shares=shares)
    moved = page_compact(tables, keep, block, blocks)
    page_copy(caches, moved.sources, moved.destinations)
    found = 0
    for r in range(0, requests, samples):
        for i in range(int(keep[r])):
            at = int(moved.block_tables[r, i // block])
            found += at < blocks - int(moved.num_free) and torch.equal(cache[at, i % block], rows[r, i])
    return {"tokens": int(keep.sum()), "found": found, "used": used, "blocks_left": int(rest.num_free),
            "after_compacting": int(moved.num_free)}


if __name__ == "__main__":
    print("training, against the dense form:", train())
    print("training in 16 bits:", train(dtype=torch.bfloat16))
    print("serving:", serve())
    print("sampling:", sample())
