"""torch.ops.cusort.route / plan_dispatch / dispatch / combine / page_plan: registration and fake shapes on CPU; on the
GPU their gradients through autograd, tracing under torch.compile, and the example that runs them together."""
from __future__ import annotations

import importlib.util
from pathlib import Path

import pytest

torch = pytest.importorskip("torch")

import libcusort_b200.ops  # noqa: E402,F401  (registers the operators)
from libcusort_b200 import paging, routing  # noqa: E402

gpu = pytest.mark.skipif(not torch.cuda.is_available(), reason="no CUDA device")
ops = torch.ops.cusort


def test_fake_shapes():
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        logits = torch.empty(30, 16, dtype=torch.bfloat16, device="cuda")
        w, ids = ops.route(logits, 4)
        assert w.shape == ids.shape == (30, 4) and w.dtype == torch.float32 and ids.dtype == torch.int32
        assert ops.route_backward(w, logits, ids).dtype == torch.bfloat16
        counts, offsets, sources, positions = ops.plan_dispatch(ids, 16, 8)
        assert counts.shape == (16,) and offsets.shape == (17,) and positions.shape == (30, 4)
        assert sources.shape == (routing.dispatch_capacity(120, 16, 8),)
        x = torch.empty(30, 50, dtype=torch.float16, device="cuda")
        rows = ops.dispatch(x, sources, positions)
        assert rows.shape == (sources.shape[0], 50) and rows.dtype == x.dtype
        assert ops.dispatch_backward(rows, positions).shape == x.shape
        assert ops.combine(rows, w, sources, positions, x).shape == x.shape
        gy, gw = ops.combine_backward(x, rows, w, sources, positions)
        assert gy.shape == rows.shape and gw.shape == w.shape
        lens = torch.empty(5, dtype=torch.int32, device="cuda")
        slots, places, starts, served, left = ops.page_plan(lens, lens, torch.empty(5, 7, dtype=torch.int32,
                                                                                    device="cuda"), 16, 40, lens, lens)
        assert slots.shape == places.shape == (40,) and slots.dtype == torch.int64 and starts.shape == (6,)
        assert served.dtype == torch.bool and left.shape == (1,)


def test_cpu_tensors_are_rejected():
    with pytest.raises(ValueError, match="CUDA"):
        ops.route(torch.zeros(4, 8), 2)
    with pytest.raises(ValueError, match="CUDA"):
        ops.plan_dispatch(torch.zeros(4, 2, dtype=torch.int32), 8)


def _layer(x, logits, y, residual, k):
    w, ids = ops.route(logits, k, renormalize=True, scale=1.5)
    _, _, sources, positions = ops.plan_dispatch(ids, logits.shape[1], 4)
    rows = ops.dispatch(x, sources, positions)
    return ops.combine(rows * y, w, sources, positions, residual)


def _plain(x, logits, y, residual, k):
    top = logits.topk(k, dim=1)
    w = top.values.softmax(1) * 1.5
    plan = routing.plan_dispatch(top.indices, logits.shape[1], align=4)
    rows = x[plan.sources.clamp(min=0).long() // k] * y
    return residual + (rows[plan.positions.long()] * w[..., None]).sum(1)


def _inputs(T, E, H, k):
    torch.manual_seed(3)
    cap = routing.dispatch_capacity(T * k, E, 4)
    return [t.cuda().requires_grad_() for t in (torch.randn(T, H), torch.randn(T, E), torch.randn(cap, H),
                                                torch.randn(T, H))]


@pytest.mark.gpu
@gpu
def test_gradients_through_autograd():
    """All gradients of route -> dispatch -> combine against the plain form's, in 32 bits: sums of up to 40 products,
    each within a few roundings of 2^-24 of the largest values met (below 30)."""
    inputs = _inputs(50, 12, 40, 3)
    target = torch.randn(50, 40, device="cuda")
    ours, plain = (torch.autograd.grad(((f(*inputs, 3) - target) ** 2).sum(), inputs) for f in (_layer, _plain))
    for a, b in zip(ours, plain):
        assert (a - b).abs().max() <= 1e-5 * b.abs().max()


@pytest.mark.gpu
@gpu
def test_expanded_gradient_and_unused_outputs():
    x, logits, y, residual = _inputs(20, 8, 16, 2)
    out = _layer(x, logits, y, residual, 2)
    gx, = torch.autograd.grad(out.sum(), [x], retain_graph=True)  # the gradient comes expanded from one number
    ref, = torch.autograd.grad(out, [x], torch.ones_like(out))
    assert torch.equal(gx, ref)
    w, ids = ops.route(logits, 2)
    assert not ids.requires_grad
    g, = torch.autograd.grad(w[:, 0].sum(), [logits])
    assert torch.isfinite(g).all()


@pytest.mark.gpu
@gpu
def test_compile_keeps_the_operators_whole():
    inputs = [t.detach() for t in _inputs(33, 8, 24, 2)]
    f = torch.compile(lambda *a: _layer(*a, 2), backend="eager", fullgraph=True)
    assert torch.equal(f(*inputs), _layer(*inputs, 2))


@pytest.mark.gpu
@gpu
def test_graph_capture():
    """The operators in a CUDA graph, replayed on other inputs."""
    x, logits, y, residual = (t.detach() for t in _inputs(33, 8, 24, 2))
    _layer(x, logits, y, residual, 2)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _layer(x, logits, y, residual, 2)
    for _ in range(2):
        logits.normal_()
        x.normal_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, _layer(x, logits, y, residual, 2))


@pytest.mark.gpu
@gpu
def test_page_plan_writes_the_tables():
    lens = torch.tensor([3, 16], dtype=torch.int32, device="cuda")
    new = torch.tensor([20, 1], dtype=torch.int32, device="cuda")
    free, left = torch.arange(9, dtype=torch.int32, device="cuda"), torch.tensor([9], dtype=torch.int32, device="cuda")
    a = torch.full((2, 4), 7, dtype=torch.int32, device="cuda")
    b = a.clone()
    got = ops.page_plan(lens, new, a, 16, 24, free, left)
    ref = paging.page_plan(lens, new, b, 16, 24, free_blocks=free, num_free=left)
    assert torch.equal(a, b) and a.tolist() == [[7, 8, 7, 7], [7, 7, 7, 7]]
    assert all(torch.equal(p, q) for p, q in zip(got, ref))


@pytest.mark.gpu
@gpu
def test_example():
    path = Path(__file__).resolve().parents[1] / "examples" / "sparse_step.py"
    spec = importlib.util.spec_from_file_location("sparse_step", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    off = example.train()
    assert all(v < 2e-3 for v in off.values()), off  # the products may run in tf32: 2^-11 each
    served = example.serve()
    assert served["tokens"] == served["found"] == 37 + 1 + 16 + 100 + 3 * 4
    assert served["blocks_left"] == 64 - (3 + 1 + 2 + 7)
