"""A small sparse (mixture-of-experts) layer on the routing operators, in training and in serving.

    python examples/sparse_step.py

Training: router logits -> route -> plan_dispatch -> dispatch -> the experts' products -> combine, with gradients by
autograd.  Serving: page_plan places each step's new tokens in a paged cache, then the same layer runs on them.
Nothing in a step copies to the host.
"""
from __future__ import annotations

import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

import libcusort_b200.ops  # noqa: E402,F401  (registers torch.ops.cusort)
from libcusort_b200.paging import page_plan  # noqa: E402

cusort = torch.ops.cusort


class SparseLayer(torch.nn.Module):
    """x + the weighted sum of each token's k experts' two-layer networks."""

    ALIGN = 16  # rows to a product tile: no tile holds two experts' rows

    def __init__(self, hidden: int, inner: int, experts: int, k: int, **how):
        super().__init__()
        self.router = torch.nn.Parameter(torch.randn(hidden, experts, **how) / hidden ** 0.5)
        self.up = torch.nn.Parameter(torch.randn(experts, hidden, inner, **how) / hidden ** 0.5)
        self.down = torch.nn.Parameter(torch.randn(experts, inner, hidden, **how) / inner ** 0.5)
        self.k = k

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        weights, experts = cusort.route(x @ self.router, self.k, renormalize=True)
        _, offsets, sources, positions = cusort.plan_dispatch(experts, self.router.shape[1], self.ALIGN)
        rows = cusort.dispatch(x, sources, positions)
        # the rows in tiles, each with its expert's matrices; rows that hold no pair are zeros, and so are their products
        tiles = -(-rows.shape[0] // self.ALIGN)
        rows = torch.nn.functional.pad(rows, (0, 0, 0, tiles * self.ALIGN - rows.shape[0]))
        first = torch.arange(tiles, device=x.device, dtype=torch.int32) * self.ALIGN
        expert = torch.searchsorted(offsets[1:], first, right=True).clamp(max=self.router.shape[1] - 1)
        inner = torch.relu(rows.view(tiles, self.ALIGN, -1) @ self.up[expert])
        y = (inner @ self.down[expert]).view(tiles * self.ALIGN, -1)[:sources.shape[0]]
        return cusort.combine(y.contiguous(), weights, sources, positions, x)

    def dense(self, x: torch.Tensor) -> torch.Tensor:
        """The same by every expert on every token."""
        top = (x @ self.router).float().softmax(1).topk(self.k, dim=1)
        weights = torch.zeros(x.shape[0], self.router.shape[1], device=x.device).scatter(
            1, top.indices, top.values / top.values.sum(1, keepdim=True))
        y = torch.relu(torch.einsum("th,ehf->etf", x, self.up)) @ self.down
        return x + torch.einsum("te,eth->th", weights, y)


def train(tokens: int = 300, hidden: int = 64, inner: int = 96, experts: int = 12, k: int = 3) -> dict[str, float]:
    """Loss and gradients of the layer against the dense form; the largest differences over the largest values."""
    torch.manual_seed(1)
    layer = SparseLayer(hidden, inner, experts, k, device="cuda", dtype=torch.float32)
    x = torch.randn(tokens, hidden, device="cuda", requires_grad=True)
    target = torch.randn(tokens, hidden, device="cuda")

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


if __name__ == "__main__":
    print("training, against the dense form:", train())
    print("serving:", serve())
