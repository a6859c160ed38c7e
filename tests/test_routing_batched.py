"""The routing and placement kernels at the sizes where other variants of them run than in a small batch: several
tokens to a warp, several vectors to a lane, several steps to a tile, several tokens to a thread."""
from __future__ import annotations

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from libcusort_b200 import routing  # noqa: E402
from tests import routing_reference as R  # noqa: E402
from tests import routing_reference_batched as B  # noqa: E402
from tests.test_paging_gpu import _run as page_step, _step as page_inputs  # noqa: E402
from tests.test_routing_gpu import ATOL, RTOL, TYPES, _logits, _wide  # noqa: E402
from tests.test_routing_gpu import test_rows_there_and_back as rows_there_and_back  # noqa: E402

FORMS = [("softmax", False, "max", False), ("softmax", False, "top2", True), ("softmax", True, "top2", False),
         ("softmax", True, "max", True), ("sigmoid", False, "max", True), ("sigmoid", False, "top2", False),
         ("sigmoid", True, "top2", True), ("sigmoid", True, "max", False)]


def _rng(*key):
    return np.random.default_rng([ord(c) for c in repr(key)])


# ------------------------------------------------------------------------------- the batched reference itself (CPU)

@pytest.mark.parametrize("score,with_bias,group_score,renormalize", FORMS)
@pytest.mark.parametrize("T,E,k,groups,kept", [(40, 12, 3, 4, 2), (30, 9, 9, 1, 1), (25, 24, 4, 24, 7)])
def test_batched_reference(T, E, k, groups, kept, score, with_bias, group_score, renormalize):
    rng = _rng(T, E, score, with_bias, group_score, renormalize)
    x = rng.normal(size=(T, E)) * 2
    x[rng.random((T, E)) < 0.2] = -np.inf
    x[rng.random((T, E)) < 0.05] = np.inf
    x[rng.random((T, E)) < 0.05] = np.nan
    x[rng.random((T, E)) < 0.1] = 0.0
    x[rng.random(T) < 0.1] = -np.inf
    bias = rng.normal(size=E) if with_bias else None
    if with_bias:
        bias[1], bias[4] = -np.inf, np.nan
    how = dict(score=score, groups=groups, groups_kept=kept, group_score=group_score, renormalize=renormalize, scale=1.5)
    w, ids, sure = R.route(x, k, bias, **how)
    b = None if bias is None else torch.from_numpy(bias)
    bw, bids, bsure = B.route(torch.from_numpy(x), k, b, **how)
    both = sure & bsure.numpy()
    assert both.mean() > 0.8
    np.testing.assert_array_equal(bids.numpy()[both], ids[both])
    np.testing.assert_allclose(bw.numpy()[both], w[both], rtol=1e-12, atol=1e-300)
    grad = rng.normal(size=(T, k))
    back = dict(score=score, renormalize=renormalize, scale=1.5)
    np.testing.assert_allclose(B.route_backward(torch.from_numpy(grad), torch.from_numpy(x), bids, b, **back).numpy(),
                               R.route_backward(grad, x, bids.numpy(), bias, **back), rtol=1e-9, atol=1e-12)


@pytest.mark.parametrize("n,E,align", [(0, 3, 4), (57, 5, 1), (400, 60, 16)])
def test_batched_plan_reference(n, E, align):
    ids = _rng(n, E).integers(-2, E + 2, n)
    cap = routing.dispatch_capacity(n, E, align)
    for got, ref in zip(B.plan(torch.from_numpy(ids), E, align, cap), R.plan(ids, E, align, cap)):
        np.testing.assert_array_equal(got.numpy(), ref)


# --------------------------------------------------------------------------------------------------------- kernels

# Tokens to a warp: 2 from 7104 tokens on, 4 from 14208, 8 from 28416 and so on, up to 32 / (k as a power of two).
BATCHES = [(7105, 64, 8, 8, 3), (8191, 256, 8, 8, 4), (14213, 60, 5, 4, 2), (28419, 36, 3, 12, 5),
           (32771, 128, 4, 1, 1), (56837, 24, 2, 1, 1), (113667, 16, 1, 4, 1), (7109, 520, 12, 8, 3),
           (14211, 300, 6, 1, 1)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("score,with_bias,group_score,renormalize", FORMS)
@pytest.mark.parametrize("shape", BATCHES, ids=str)
def test_route_batches(shape, score, with_bias, group_score, renormalize, dtype):
    """As test_route of a small batch, with its bounds: the kernels' arithmetic is the same for any batch."""
    T, E, k, groups, kept = shape
    rng = _rng(shape, score, with_bias, group_score, renormalize, dtype)
    logits, _ = _logits(rng, T, E, dtype)
    x = logits.double()
    bias = torch.from_numpy(rng.normal(size=E).astype(np.float32)).cuda() if with_bias else None
    if with_bias:
        bias[1], bias[5] = -float("inf"), float("nan")
    b = None if bias is None else bias.double()
    how = dict(score=score, groups=groups, groups_kept=kept, group_score=group_score, renormalize=renormalize,
               scale=1.75)
    grad = torch.from_numpy(rng.normal(size=(T, k)).astype(np.float32)).cuda()
    back = dict(score=score, renormalize=renormalize, scale=1.75)
    rw, rids, sure = B.route(x, k, b, **how)
    assert 2 * int(sure.sum()) >= T
    for rows in (logits, _wide(logits)):  # rows as whole vectors where E allows it, and one by one
        w, ids = routing.route(rows, k, bias=bias, **how)
        assert torch.equal(ids[sure].long(), rids[sure])
        assert ((w - rw).abs() <= 1e-5 * rw + 1e-37)[sure].all()
        g = routing.route_backward(grad, rows, ids, bias=bias, **back)
        rg = B.route_backward(grad.double(), x, ids.long(), b, **back)
        bound = 4 * RTOL[dtype] * rg.abs() + max(ATOL[dtype], 2e-6 * 1.75 * float(grad.abs().max()))
        assert ((g.double() - rg).abs() <= bound).all()


# 16-byte vectors to a row; a lane takes 4, 4, 3, 2, 3 (two parts of the row), 4 (two parts) and 1 of them.
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vectors,apart", [(128, 0), (125, 8), (90, 0), (61, 8), (180, 0), (250, 8), (129, 0)])
def test_rows_of_several_vectors(vectors, apart, dtype):
    rows_there_and_back((2501, 2, 60, 16, vectors * 16 // TYPES[dtype].itemsize), dtype, apart)


# More than 148 tiles of 4096 pairs: tiles of several steps.
@pytest.mark.gpu
@pytest.mark.parametrize("kind", [torch.int32, torch.int64])
@pytest.mark.parametrize("n,E,align", [(606_209, 128, 8), (700_001, 5, 1), (700_001, 1000, 16), (3_000_001, 300, 128)])
def test_plan_of_several_steps(n, E, align, kind):
    rng = _rng("steps", n, E)
    ids = np.minimum(rng.integers(-1, E + 2, n), rng.integers(0, E + 2, n))
    ids = torch.from_numpy(ids).cuda()
    plan = routing.plan_dispatch(ids.to(kind), E, align=align)
    for name, got, ref in zip(plan._fields, plan, B.plan(ids, E, align, routing.dispatch_capacity(n, E, align))):
        assert torch.equal(got.long(), ref), name


# Four tokens to a thread from 148 * 1024 tokens on; more than 148 * 4096 of them: several rounds of the grid.
@pytest.mark.gpu
@pytest.mark.parametrize("block", [1, 16, 17, 64])
@pytest.mark.parametrize("requests,context,chunk", [(45, 300, 9000), (700, 200, 500)])
def test_page_plan_of_many_tokens(requests, context, chunk, block):
    rng = _rng("page", requests, block)
    cached, new, tables, pool = page_inputs(rng, requests, context, chunk, block)
    new[::3] = 0
    new[1::5] = 1
    new[2] = chunk
    new[4] += max(0, 155_000 - int(new.sum()))
    width = -(-int((cached + new).max()) // block)
    wider = np.full((requests, width), -1)
    wider[:, :tables.shape[1]] = tables[:, :width]
    need = int((-(-(cached + new) // block) - -(-cached // block)).sum())
    pool = np.concatenate([pool, np.arange(need) + requests * tables.shape[1] * 2])
    total = int(new.sum())
    for tokens in (total + 13, 152_001):
        page_step(cached, new, wider, block, tokens, pool, len(pool), apart=3)
    for left in (need // 2, need - 1, need):
        page_step(cached, new, wider, block, total, pool, left)


@pytest.mark.gpu
def test_page_plan_of_many_rounds():
    rng = _rng("rounds")
    cached, new, tables, pool = page_inputs(rng, 3000, 64, 420, 16)
    assert new.sum() > 148 * 4096
    page_step(cached, new, tables, 16, int(new.sum()) + 5, pool, len(pool) // 3)


@pytest.mark.gpu
def test_page_plan_of_many_tokens_other_tables():
    """Tables that are too narrow for some requests, and tables that hold all blocks already."""
    rng = _rng("tables")
    cached, new, tables, pool = page_inputs(rng, 900, 100, 400, 16, width=20)
    cached = np.minimum(cached, 320)
    _, served = page_step(cached, new, tables, 16, int(new.sum()), pool, len(pool))
    assert new.sum() > 148 * 1024 and served.any() and not served.all()
    cached, new, tables, pool = page_inputs(rng, 900, 100, 400, 16)
    tables = rng.permutation(tables.size).reshape(tables.shape)
    tables[3, 2:] = -1
    page_step(cached, new, tables, 16, int(new.sum()) + 1, None, 0)
