"""The example's layer in 16 bits where every value on the way can be held in 16 bits: results and gradients are those
of the formula in 64 bits."""
from __future__ import annotations

import importlib.util
from pathlib import Path

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


def _example():
    path = Path(__file__).resolve().parents[1] / "examples" / "sparse_step.py"
    spec = importlib.util.spec_from_file_location("sparse_step", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    return example


def _sparse(gen, each, *shape):
    """Numbers of -1, 0 and 1, `each` that are not 0 in a row."""
    at = torch.rand(*shape, generator=gen).argsort(-1)[..., :each]
    sign = torch.randint(0, 2, at.shape, generator=gen) * 2 - 1
    return torch.zeros(*shape).scatter(-1, at, sign.float())


def _values(tokens=70, hidden=64, inner=96, experts=12):
    """A token has the value 4 at two of the first 12 places, which the router makes the logits of: its two experts,
    with half the weight each."""
    gen = torch.Generator().manual_seed(6)
    x = _sparse(gen, 6, tokens, hidden)
    x[:, :experts] = 0
    chosen = torch.rand(tokens, experts, generator=gen).argsort(1)[:, :2]
    x.scatter_(1, chosen, 4.0)
    router = torch.zeros(hidden, experts)
    router[:experts] = torch.eye(experts)
    return (x, router, _sparse(gen, 3, experts, hidden, inner), _sparse(gen, 2, experts, inner, hidden),
            _sparse(gen, 8, tokens, hidden))


def _formula(x, router, up, down):
    """x + the weighted sum of the two experts' networks."""
    logits = x @ router
    chosen = torch.zeros_like(logits).scatter(1, logits.topk(2, dim=1).indices, 1.0)
    weights = (logits - logits.amax(1, keepdim=True)).exp() * chosen
    weights = weights / weights.sum(1, keepdim=True)
    y = torch.relu(torch.einsum("th,ehf->etf", x, up)) @ down
    return x + torch.einsum("te,eth->th", weights, y)


def test_the_example_in_16_bits():
    """To the bit, but for what the router's gradient goes into: a logit's is worked out in 32 bits from values up to
    12, in 8 operations at most (8 * 12 * 2^-24), and the router's adds up those of 70 tokens times 4 (below 2^-9
    together); what is off so before it is rounded may be rounded the other way (2^-8 of it)."""
    *values, g = _values()
    wide = [v.cuda().double().requires_grad_() for v in values]
    want = _formula(*wide)
    grads = torch.autograd.grad(want, wide, g.cuda().double())
    for v in (want, *grads):  # what is compared can be held in 16 bits, and there is something to compare
        assert torch.equal(v, v.bfloat16().double()) and v.abs().amax() > 1
    layer = _example().SparseLayer(64, 96, 12, 2, device="cuda", dtype=torch.bfloat16)
    with torch.no_grad():
        for p, v in zip((layer.router, layer.up, layer.down), values[1:]):
            p.copy_(v)
    x = values[0].cuda().bfloat16().requires_grad_()
    out = layer(x)
    assert out.dtype == torch.bfloat16 and torch.equal(out.double(), want)
    got = torch.autograd.grad(out, [x, layer.router, layer.up, layer.down], g.cuda().bfloat16())
    for a, b in zip(got[2:], grads[2:]):
        assert torch.equal(a.double(), b)
    for a, b in zip(got[:2], grads[:2]):
        assert ((a.double() - b).abs() <= 2.0 ** -8 * b.abs() + 2.0 ** -9).all()
