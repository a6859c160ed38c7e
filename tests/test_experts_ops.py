"""torch.ops.cusort.expert_products and the page operators: gradients through autograd and by differences, tracing,
CUDA graphs, and the example that runs them with routing and placement."""
from __future__ import annotations

import importlib.util
from pathlib import Path

import pytest

torch = pytest.importorskip("torch")

import libcusort_b200.ops  # noqa: E402,F401  (registers the operators)
from libcusort_b200 import experts as X, paging  # noqa: E402

pytestmark = pytest.mark.gpu
ops = torch.ops.cusort


def ints(*values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def whole(gen, low, high, *shape):
    """Small whole numbers, exact in 16 bits, and so are their products' sums here (below 256)."""
    return torch.randint(low, high + 1, shape, generator=gen, device="cuda").bfloat16()


@pytest.mark.parametrize("order", ["in_out", "out_in"])
def test_gradients_by_differences(order):
    """The product is linear in each operand: with whole numbers differences are exact, and so have to be the
    gradients."""
    gen = torch.Generator(device="cuda").manual_seed(0)
    counts, offsets, capacity, E, fin, fout = ints(17, 0, 40, 3), ints(0, 24, 24, 64, 68), 75, 4, 24, 40
    shape = (E, fin, fout) if order == "in_out" else (E, fout, fin)

    def weights():
        w = whole(gen, -2, 2, *shape)
        return w if order == "in_out" else w.transpose(1, 2)
    x, dx, w, dw = whole(gen, -2, 2, capacity, fin), whole(gen, -1, 1, capacity, fin), weights(), weights()
    g = whole(gen, -1, 1, capacity, fout)
    xg, wg = x.clone().requires_grad_(), w.clone().requires_grad_()
    assert wg.stride() == w.stride()
    grad_x, grad_w = torch.autograd.grad(ops.expert_products(xg, wg, counts, offsets), [xg, wg], g)
    assert grad_w.stride() == w.stride()

    def loss(x, w):
        return (ops.expert_products(x, w, counts, offsets).double() * g.double()).sum()
    assert loss(x + dx, w) - loss(x, w) == (grad_x.double() * dx.double()).sum()
    assert loss(x, w + dw) - loss(x, w) == (grad_w.double() * dw.double()).sum()


def test_gradients_are_those_of_the_functions():
    gen = torch.Generator(device="cuda").manual_seed(1)
    counts, offsets = ints(30, 100, 0), ints(0, 32, 132, 132)
    x = torch.randn(140, 72, generator=gen, device="cuda").half().requires_grad_()
    w = torch.randn(3, 72, 136, generator=gen, device="cuda").half().requires_grad_()
    out = ops.expert_products(x, w, counts, offsets)
    # an expanded gradient, as that of a sum
    gx, gw = torch.autograd.grad(out.sum(), [x, w], retain_graph=True)
    ones = torch.ones_like(out)
    rx, rw = X.expert_products_backward(ones, x.detach(), w.detach(), counts, offsets)
    assert torch.equal(gx, rx) and torch.equal(gw, rw)
    only, = torch.autograd.grad(out, [w], ones, retain_graph=True)
    assert torch.equal(only, rw)
    t = torch.randn(136, 140, generator=gen, device="cuda").half()
    gx, gw = torch.autograd.grad(out, [x, w], t.t())  # rows that are not contiguous in themselves
    rx, rw = X.expert_products_backward(t.t().contiguous(), x.detach(), w.detach(), counts, offsets)
    assert torch.equal(gx, rx) and torch.equal(gw, rw)


def _layer(x, router, up, down, k=2):
    weights, experts = ops.route(x @ router, k, renormalize=True)
    counts, offsets, sources, positions = ops.plan_dispatch(experts, router.shape[1], 8)
    rows = ops.dispatch(x, sources, positions)
    y = ops.expert_products(torch.relu(ops.expert_products(rows, up, counts, offsets)), down, counts, offsets)
    return ops.combine(y, weights, sources, positions, x)


def _inputs(tokens, seed=2):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return [torch.randn(*s, generator=gen, device="cuda").mul_(s[-2] ** -0.5 if len(s) == 3 else 1).bfloat16()
            for s in ((tokens, 64), (64, 8), (8, 64, 96), (8, 96, 64))]


def test_a_layer_compiles_and_is_captured():
    inputs = _inputs(50)
    f = torch.compile(_layer, backend="eager", fullgraph=True)
    assert torch.equal(f(*inputs), _layer(*inputs))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _layer(*inputs)
    for seed in (3, 4):
        for a, b in zip(inputs, _inputs(50, seed)):
            a.copy_(b)
        graph.replay()
        assert torch.equal(out, _layer(*inputs))


def test_a_training_step_captured():
    """Forward and backward in one graph, replayed on other inputs."""
    inputs = [t.requires_grad_() for t in _inputs(40)]

    def step():
        return torch.autograd.grad(_layer(*inputs).float().square().sum(), inputs)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            captured = step()
    torch.cuda.synchronize()
    with torch.no_grad():
        for a, b in zip(inputs, _inputs(40, 7)):
            a.copy_(b)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(captured, step()))


def test_page_operators():
    tables, lens, parents = ints(3, 5, -1, 1, 5, -1).view(2, 3), ints(20, 30), ints(1, 1, 7)
    free, left, shares = ints(0, 2, 4, 6, -1, -1, -1), ints(4), ints(0, 0, 0, 0, 0, 1, 0)
    pool = dict(free_blocks=free, num_free=left, shares=shares)
    got = ops.page_fork(tables, lens, parents, 16, free, left, shares)
    assert all(torch.equal(a, b) for a, b in zip(got, paging.page_fork(tables, lens, parents, 16, **pool)))
    got = ops.page_free(tables, lens, ints(0, 16), 16, free, left, shares)
    assert all(torch.equal(a, b) for a, b in zip(got, paging.page_free(tables, lens, ints(0, 16), 16, **pool)))
    got = ops.page_compact(tables, lens, 16, 7)
    assert all(torch.equal(a, b) for a, b in zip(got, paging.page_compact(tables, lens, 16, 7)))
    # blocks 1, 3 and 5 are held: 3 and 5 move to 0 and 2
    assert got[1].tolist() == [3, 5, -1] and got[2].tolist() == [0, 2, -1]
    cache = torch.arange(14, device="cuda").view(7, 2)
    version = cache._version
    ops.page_copy([cache], got[1], got[2])
    assert cache.tolist()[:3] == [[6, 7], [2, 3], [10, 11]]
    assert cache._version > version
    f = torch.compile(lambda c, s, d: (ops.page_copy([c], s, d), c + 1)[1], backend="eager", fullgraph=True)
    assert torch.equal(f(cache.clone(), got[1], got[2]), cache + 1)


def _example():
    path = Path(__file__).resolve().parents[1] / "examples" / "sparse_step.py"
    spec = importlib.util.spec_from_file_location("sparse_step", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    return example


def test_example_samples():
    got = _example().sample()
    assert got["found"] == got["tokens"] == 37 + 5 + 50 + 3 * 24
    held = sum(-(-(n + 24) // 16) for n in (37, 5, 50))
    assert got["blocks_left"] == got["after_compacting"] == 128 - held and got["used"] > held


def test_example_in_16_bits():
    """Its gradients exist and are finite; how near they are to the dense form's hangs on which experts tie."""
    off = _example().train(dtype=torch.bfloat16)
    assert set(off) == {"x", "router", "up", "down", "loss"} and all(v == v for v in off.values())
