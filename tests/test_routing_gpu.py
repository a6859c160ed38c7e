"""Routing operators on the GPU against plain 64-bit implementations (tests/routing_reference.py)."""
from __future__ import annotations

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from libcusort_b200 import routing  # noqa: E402
from tests import routing_reference as R  # noqa: E402

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
# Half a unit in the last place of the output's type (f32: exp within 2 units, two quotients, a product, and a sum of
# up to 1024 terms over a tree: below 2e-6), and the smallest step of the type's subnormals.
RTOL = {"f32": 2e-6, "f16": 2.0 ** -11 + 2e-6, "bf16": 2.0 ** -8 + 2e-6}
ATOL = {"f32": 1e-37, "f16": 2.0 ** -24, "bf16": 1e-37}


def _rng(*key):
    return np.random.default_rng([ord(c) for c in repr(key)])


def _cuda(a, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    return t if dtype is None else t.to(dtype)


def _wide(t, by=5):
    """The same matrix with its rows further apart."""
    out = torch.full((t.shape[0], t.shape[1] + by), float("nan"), dtype=t.dtype, device=t.device)
    out[:, :t.shape[1]] = t
    return out[:, :t.shape[1]]


def _logits(rng, T, E, dtype, masks=True):
    x = rng.normal(size=(T, E)) * 2
    if masks:
        x[rng.random((T, E)) < 0.05] = -np.inf
        x[rng.random((T, E)) < 0.01] = np.nan
        x[rng.random((T, E)) < 0.05] = -0.0
        x[rng.random((T, E)) < 0.05] = 0.0
        x[rng.random(T) < 0.1] = -np.inf
        lowest = torch.finfo(TYPES[dtype]).min
        x[rng.random((T, E)) < 0.02] = lowest
        x[rng.random(T) < 0.05] = lowest
    t = _cuda(x).to(TYPES[dtype])
    return t, t.double().cpu().numpy()


SHAPES = [(1, 1, 1, 1, 1), (3, 7, 7, 1, 1), (5, 32, 2, 4, 2), (97, 60, 4, 1, 1), (33, 64, 6, 8, 3), (41, 96, 5, 12, 5),
          (64, 128, 8, 32, 9), (19, 257, 8, 1, 1), (23, 256, 8, 8, 4), (9, 1000, 32, 8, 2), (6, 1024, 32, 1, 1),
          (21, 36, 3, 12, 2), (17, 24, 6, 6, 6)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("score,with_bias,group_score,renormalize", [
    ("softmax", False, "max", False), ("softmax", False, "top2", True), ("softmax", True, "top2", False),
    ("softmax", True, "max", True), ("sigmoid", False, "max", True), ("sigmoid", False, "top2", False),
    ("sigmoid", True, "top2", True), ("sigmoid", True, "max", False)])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_route(shape, score, with_bias, group_score, renormalize, dtype):
    T, E, k, groups, kept = shape
    rng = _rng(shape, score, with_bias, group_score, renormalize, dtype)
    logits, x = _logits(rng, T, E, dtype)
    bias = rng.normal(size=E).astype(np.float32) if with_bias else None
    if with_bias and E > 8:
        bias[1], bias[5] = -np.inf, np.nan
    b = None if bias is None else _cuda(bias)
    how = dict(score=score, groups=groups, groups_kept=kept, group_score=group_score, renormalize=renormalize,
               scale=1.75)
    w, ids = routing.route(_wide(logits), k, bias=b, **how)
    rw, rids, sure = R.route(x, k, bias, **how)
    assert 2 * sure.sum() >= T  # enough rows are left to be compared
    np.testing.assert_array_equal(ids.cpu().numpy()[sure], rids[sure])
    np.testing.assert_allclose(w.cpu().numpy()[sure], rw[sure], rtol=1e-5, atol=1e-37)

    grad = rng.normal(size=(T, k)).astype(np.float32)
    ids_np = ids.cpu().numpy()
    back = dict(score=score, renormalize=renormalize, scale=1.75)
    g = routing.route_backward(_cuda(grad), _wide(logits), ids, bias=b, **back)
    rg = R.route_backward(grad, x, ids_np, bias, **back)
    assert g.dtype == TYPES[dtype] and g.is_contiguous()
    # the differences g - u cancel: an error of 2e-6 of the largest |scale g| (at most 8 of them are added)
    np.testing.assert_allclose(g.double().cpu().numpy(), rg, rtol=RTOL[dtype] * 4,
                               atol=max(ATOL[dtype], 2e-6 * 1.75 * np.abs(grad).max()))


@pytest.mark.parametrize("score,renormalize", [("softmax", False), ("softmax", True), ("sigmoid", False),
                                               ("sigmoid", True)])
def test_route_infinite_logits(score, renormalize):
    x = np.array([[np.inf, 1, 2, np.inf], [-np.inf] * 4, [np.nan] * 4, [-np.inf, np.inf, np.nan, 0],
                  [3e38, -3e38, 0, -3e38], [-3e38] * 4, [-0.0, 0.0, -0.0, 0.0]], np.float32)
    w, ids = routing.route(_cuda(x), 3, score=score, renormalize=renormalize)
    rw, rids, _ = R.route(x, 3, score=score, renormalize=renormalize)
    np.testing.assert_array_equal(ids.cpu().numpy(), rids)
    np.testing.assert_allclose(w.cpu().numpy(), rw, rtol=1e-6)
    g = routing.route_backward(torch.ones(7, 3, device="cuda"), _cuda(x), ids, score=score, renormalize=renormalize)
    assert torch.isfinite(g).all()


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [False, True])
def test_route_gradient_against_differences(score, renormalize):
    """Central differences of the forward kernel: logits half apart keep their order under a step of 1/64; the third
    derivative of a softmax or sigmoid weight is below 1, so the error is below (1/64)^2 / 6 times the sum of |g|
    (at most 4 x 3), and 1e-6 / (1/64) from rounding."""
    rng = _rng("differences", score, renormalize)
    T, E, k, step = 16, 16, 4, 1 / 64
    x = np.stack([rng.permutation(E) * 0.5 - 4 for _ in range(T)]).astype(np.float32)
    grad = np.clip(rng.normal(size=(T, k)), -3, 3).astype(np.float32)
    how = dict(score=score, renormalize=renormalize)
    _, ids = routing.route(_cuda(x), k, **how)
    got = routing.route_backward(_cuda(grad), _cuda(x), ids, **how).double().cpu().numpy()
    for e in range(E):
        up, down = x.copy(), x.copy()
        up[:, e] += step
        down[:, e] -= step
        wu, iu = routing.route(_cuda(up), k, **how)
        wd, _ = routing.route(_cuda(down), k, **how)
        assert torch.equal(iu, ids)
        slope = ((wu - wd).double().cpu().numpy() * grad).sum(1) / (2 * step)
        np.testing.assert_allclose(got[:, e], slope, atol=12 * step ** 2 / 6 + 1e-4)


@pytest.mark.parametrize("kind", [torch.int32, torch.int64])
@pytest.mark.parametrize("T,k,E,align", [
    (0, 1, 4, 8), (1, 1, 1, 1), (1, 8, 256, 16), (7, 3, 5, 1), (333, 6, 60, 128), (300, 8, 1024, 4), (2049, 1, 3, 7),
    (1024, 2, 64, 1), (1025, 2, 64, 16), (9001, 8, 300, 16), (40000, 8, 1000, 3)])
def test_plan(T, k, E, align, kind):
    rng = _rng("plan", T, k, E, align)
    ids = np.minimum(rng.integers(-1, E + 2, (T, k)), rng.integers(0, E + 2, (T, k)))  # skewed, some outside
    ids[ids == E + 1] = -7 if kind == torch.int32 else 2 ** 33  # outside as 64 bits, expert 0 if cut to 32
    plan = routing.plan_dispatch(_cuda(ids.astype(np.int64)).to(kind), E, align=align)
    cap = routing.dispatch_capacity(T * k, E, align)
    expect = R.plan(ids, E, align, cap)
    for name, got, ref in zip(plan._fields, plan, expect):
        assert got.dtype == torch.int32
        np.testing.assert_array_equal(got.cpu().numpy(), ref, err_msg=name)


def test_plan_one_expert_for_all():
    for n in (1, 31, 2048, 100_003):
        plan = routing.plan_dispatch(torch.full((n, 1), 2, dtype=torch.int32, device="cuda"), 4, align=64)
        assert plan.counts.tolist() == [0, 0, n, 0]
        assert torch.equal(plan.positions[:, 0], torch.arange(n, dtype=torch.int32, device="cuda"))
        assert torch.equal(plan.sources[:n], plan.positions[:, 0]) and (plan.sources[n:] == -1).all()


def test_plan_drops_everything():
    plan = routing.plan_dispatch(torch.full((50, 4), -1, dtype=torch.int32, device="cuda"), 16, align=8)
    assert not plan.counts.any() and not plan.offsets.any()
    assert (plan.sources == -1).all() and (plan.positions == -1).all()


def _planned(rng, T, k, E, align, dropped=0.1):
    ids = rng.integers(0, E, (T, k))
    ids[rng.random((T, k)) < dropped] = -1
    plan = routing.plan_dispatch(_cuda(ids.astype(np.int32)), E, align=align)
    return plan, plan.sources.cpu().numpy(), plan.positions.cpu().numpy()


MOVES = [(1, 1, 1, 1, 1), (1, 8, 16, 4, 4096), (5, 3, 4, 1, 7), (33, 8, 60, 16, 130), (64, 2, 8, 1, 264),
         (129, 6, 30, 8, 1021), (17, 32, 64, 1, 96), (3, 4, 8, 1, 2056), (50, 5, 8, 1, 100)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", MOVES, ids=str)
@pytest.mark.parametrize("apart", [0, 3, 8])
def test_rows_there_and_back(shape, dtype, apart):
    T, k, E, align, H = shape
    rng = _rng("move", shape, dtype, apart)
    plan, sources, positions = _planned(rng, T, k, E, align)
    cap = len(sources)
    spread = (lambda t: _wide(t, apart)) if apart else (lambda t: t)

    def matrix(n):
        t = _cuda(rng.normal(size=(n, H))).to(TYPES[dtype])
        return spread(t), t.double().cpu().numpy()

    x, xr = matrix(T)
    res, resr = matrix(T)
    gout, goutr = matrix(T)
    y, yr = matrix(cap)
    y = y.contiguous()
    w = rng.random((T, k)).astype(np.float32)
    wt = _cuda(w)

    rows = routing.dispatch(x, plan.sources, plan.positions)
    expect = np.where(sources[:, None] >= 0, xr[np.maximum(sources, 0) // k], 0)
    np.testing.assert_array_equal(rows.double().cpu().numpy(), expect)

    there = (positions >= 0)[..., None]
    picked = np.where(there, yr[np.maximum(positions, 0)] if cap else 0, 0)
    for residual, base in ((None, 0), (res, resr)):
        out = routing.combine(y, wt, plan.positions, residual=residual)
        assert out.dtype == TYPES[dtype]
        size = (np.abs(picked) * w[..., None]).sum(1) + np.abs(base)  # a sum's error goes by its terms' sizes
        off = np.abs(out.double().cpu().numpy() - ((picked * w[..., None]).sum(1) + base))
        half = {"f32": 0, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}[dtype]
        assert (off <= (half + (k + 2) * 2.0 ** -24) * size + ATOL[dtype]).all()

    back = routing.dispatch_backward(y, plan.positions)
    size = np.abs(picked).sum(1)
    off = np.abs(back.double().cpu().numpy() - picked.sum(1))
    assert (off <= (half + (k + 2) * 2.0 ** -24) * size + ATOL[dtype]).all()

    grad_rows, grad_w = routing.combine_backward(gout, y, wt, plan.sources, plan.positions)
    expect = np.where(sources[:, None] >= 0,
                      goutr[np.maximum(sources, 0) // k] * w.reshape(-1)[np.maximum(sources, 0)][:, None], 0)
    np.testing.assert_allclose(grad_rows.double().cpu().numpy(), expect, rtol=half + 2.0 ** -23, atol=ATOL[dtype])
    size = (np.abs(picked) * np.abs(goutr)[:, None]).sum(2)
    off = np.abs(grad_w.double().cpu().numpy() - (picked * goutr[:, None]).sum(2))
    assert (off <= (H / 32 + 8) * 2.0 ** -24 * size + 1e-37).all()


def test_rows_of_other_types():
    rng = _rng("types")
    plan, sources, _ = _planned(rng, 37, 4, 8, 8)
    for dtype, width in ((torch.uint8, 33), (torch.int64, 5), (torch.float64, 3), (torch.int16, 48), (torch.uint8, 0)):
        x = _cuda(rng.integers(0, 100, (37, width))).to(dtype)
        rows = routing.dispatch(x, plan.sources, plan.positions).cpu().numpy()
        np.testing.assert_array_equal(rows, np.where(sources[:, None] >= 0, x.cpu().numpy()[np.maximum(sources, 0) // 4], 0))


def test_rows_unaligned_base():
    """A base address that is no multiple of 16 bytes."""
    rng = _rng("base")
    plan, sources, positions = _planned(rng, 40, 4, 8, 1)
    flat = torch.randn(len(sources) * 64 + 3, device="cuda").to(torch.bfloat16)
    for skip in (1, 2, 3):
        y = flat[skip:skip + len(sources) * 64].view(len(sources), 64)
        w = torch.ones(40, 4, device="cuda")
        assert torch.equal(routing.combine(y, w, plan.positions), routing.combine(y.clone(), w, plan.positions))
        x = flat[skip:skip + 40 * 64].view(40, 64)
        assert torch.equal(routing.dispatch(x, plan.sources, plan.positions),
                           routing.dispatch(x.clone(), plan.sources, plan.positions))
        (ga, wa), (gb, wb) = (routing.combine_backward(*t, w, plan.sources, plan.positions)
                              for t in ((x, y), (x.clone(), y.clone())))
        assert torch.equal(ga, gb)
        # the dot products are added up in another order: 64 terms, each side within (64 / 32 + 8) roundings
        size = (x.float().abs()[:, None] * y.float().abs()[plan.positions.clamp(min=0).long()]).sum(2)
        assert ((wa - wb).abs() <= 2 * 10 * 2.0 ** -24 * size).all()


def test_unwritten_rows_do_not_matter():
    """Rows that hold no pair take part in nothing, whatever is in them."""
    rng = _rng("nan")
    plan, sources, _ = _planned(rng, 40, 4, 8, 16)
    y = torch.randn(len(sources), 64, device="cuda")
    y[plan.sources < 0] = float("nan")
    w = torch.rand(40, 4, device="cuda")
    assert torch.isfinite(routing.combine(y, w, plan.positions)).all()
    gy, gw = routing.combine_backward(torch.randn(40, 64, device="cuda"), y, w, plan.sources, plan.positions)
    assert torch.isfinite(gy).all() and torch.isfinite(gw).all()
    assert (gy[plan.sources < 0] == 0).all()


def test_combine_gradient_against_differences():
    """combine is linear in its rows and in its weights, so differences are exact up to rounding."""
    rng = _rng("linear")
    plan, sources, _ = _planned(rng, 9, 3, 4, 4)
    T, k, H = 9, 3, 16
    y = torch.randn(len(sources), H, device="cuda")
    w, g = torch.rand(T, k, device="cuda"), torch.randn(T, H, device="cuda")
    gy, gw = routing.combine_backward(g, y, w, plan.sources, plan.positions)
    dy, dw = torch.randn_like(y), torch.randn_like(w)
    dot = lambda a, b: float((a.double() * b.double()).sum())  # noqa: E731
    slope_y = dot(routing.combine(dy, w, plan.positions), g)
    slope_w = dot(routing.combine(y, dw, plan.positions), g)
    assert abs(slope_y - dot(gy, dy)) < 1e-4 and abs(slope_w - dot(gw, dw)) < 1e-4
    x, gr = torch.randn(T, H, device="cuda"), torch.randn_like(y)
    assert abs(dot(routing.dispatch(x, plan.sources, plan.positions), gr)
               - dot(x, routing.dispatch_backward(gr, plan.positions))) < 1e-4


def test_rows_beyond_32_bits():
    """More than 2^31 elements in the grouped rows."""
    T, k, E, H = (1 << 18) + 3, 8, 64, 1032
    ids = (torch.arange(T * k, device="cuda", dtype=torch.int32) * 7 % E).view(T, k)
    plan = routing.plan_dispatch(ids, E)
    x = torch.randn(T, H, device="cuda").to(torch.bfloat16)
    rows = routing.dispatch(x, plan.sources, plan.positions)
    assert rows.numel() > 1 << 31
    for at in (0, rows.shape[0] // 2, rows.shape[0] - 5000):
        assert torch.equal(rows[at:at + 5000], x[plan.sources[at:at + 5000].long() // k])
    w = torch.full((T, k), 0.125, device="cuda")
    assert torch.equal(routing.combine(rows, w, plan.positions), x)  # eight eighths of the same row, exactly
    gy, gw = routing.combine_backward(x, rows, w, plan.sources, plan.positions)
    assert torch.equal(gy[-5000:], (x[plan.sources[-5000:].long() // k].float() * 0.125).to(torch.bfloat16))
    ref = (x[-100:].double() ** 2).sum(1)
    np.testing.assert_allclose(gw[-100:].double().cpu().numpy(), ref[:, None].expand(100, k).cpu().numpy(), rtol=1e-5)


def test_other_stream():
    rng = _rng("stream")
    logits, x = _logits(rng, 500, 64, "bf16")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        w, ids = routing.route(logits, 4, renormalize=True)
        plan = routing.plan_dispatch(ids, 64, align=8)
        rows = routing.dispatch(logits, plan.sources, plan.positions)
        out = routing.combine(rows, w, plan.positions)
    side.synchronize()
    rw, rids, _ = R.route(x, 4, renormalize=True)
    np.testing.assert_array_equal(ids.cpu().numpy(), rids)
    on = (rids >= 0).any(1)
    got, ref = out.double().cpu().numpy()[on], x[on]
    np.testing.assert_allclose(got[np.isfinite(ref)], ref[np.isfinite(ref)], rtol=2.0 ** -7)


def test_same_inputs_same_bits():
    rng = _rng("again")
    logits, _ = _logits(rng, 2000, 96, "f32")
    w, ids = routing.route(logits, 6)
    g = torch.randn(2000, 6, device="cuda")
    first = routing.route_backward(g, logits, ids)
    plan = routing.plan_dispatch(ids, 96, align=4)
    y = torch.randn(plan.sources.numel(), 333, device="cuda")
    gout = torch.randn(2000, 333, device="cuda")
    a = (w, first, routing.combine(y, w, plan.positions),
         *routing.combine_backward(gout, y, w, plan.sources, plan.positions))
    for _ in range(3):
        b = (routing.route(logits, 6)[0], routing.route_backward(g, logits, ids), routing.combine(y, w, plan.positions),
             *routing.combine_backward(gout, y, w, plan.sources, plan.positions))
        assert all(torch.equal(p, q) for p, q in zip(a, b))


@pytest.mark.parametrize("separate", [False, True])
def test_plan_tensors_do_not_overlap(separate):
    for T, k, E, align in ((0, 2, 3, 1), (5, 3, 7, 4), (2000, 5, 33, 16)):
        ids = torch.randint(0, E, (T, k), device="cuda", dtype=torch.int32)
        plan = routing.plan_dispatch(ids, E, align=align, separate=separate)
        expect = R.plan(ids.cpu().numpy(), E, align, plan.sources.numel())
        spans = sorted((t.data_ptr(), t.data_ptr() + t.numel() * 4) for t in plan if t.numel())
        assert all(a[1] <= b[0] for a, b in zip(spans, spans[1:]))
        assert all(t.data_ptr() % 16 == 0 and t.is_contiguous() for t in plan)
        assert len({t.untyped_storage().data_ptr() for t in plan if t.numel()}) == (len(spans) if separate else 1)
        for t in plan:  # each can be written without the others' noticing
            kept = [u.clone() for u in plan]
            t.fill_(77)
            for u, was in zip(plan, kept):
                assert u is t or torch.equal(u, was)
            t.copy_(kept[[u is t for u in plan].index(True)])
        for got, ref in zip(plan, expect):
            np.testing.assert_array_equal(got.cpu().numpy(), ref)


@pytest.mark.parametrize("score,renormalize", [("softmax", False), ("sigmoid", False)])
def test_route_gradient_adds_up_repeated_experts(score, renormalize):
    """Experts that a caller repeats within a token: their parts add up."""
    rng = _rng("repeated", score)
    logits, x = _logits(rng, 70, 24, "f32", masks=False)
    ids = rng.integers(0, 24, (70, 6))
    ids[:, 3] = ids[:, 0]
    ids[::2, 4] = ids[::2, 0]
    grad = rng.normal(size=(70, 6)).astype(np.float32)
    g = routing.route_backward(_cuda(grad), logits, _cuda(ids.astype(np.int32)), score=score, renormalize=renormalize)
    # the reference adds each pair's part by itself
    ref = np.zeros((70, 24))
    for j in range(6):
        ref += R.route_backward(grad[:, j:j + 1], x, ids[:, j:j + 1], None, score, renormalize)
    np.testing.assert_allclose(g.double().cpu().numpy(), ref, rtol=1e-5, atol=2e-6 * np.abs(grad).max())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("score,renormalize", [("softmax", False), ("softmax", True), ("sigmoid", False),
                                               ("sigmoid", True)])
@pytest.mark.parametrize("shape", [(40, 8, 3, 1, 1), (40, 60, 4, 1, 1), (40, 64, 6, 8, 3), (40, 128, 4, 1, 1),
                                   (40, 256, 8, 8, 4), (40, 512, 8, 1, 1), (40, 1000, 5, 4, 2), (7105, 64, 4, 1, 1)],
                         ids=str)
def test_route_infinite_logits_of_all_types(shape, score, renormalize, dtype):
    """Positive infinity is the best logit there is, for any type (f16 logits reach it from 65520 on)."""
    T, E, k, groups, kept = shape
    rng = _rng("infinite", shape, score, renormalize, dtype)
    x = rng.normal(size=(T, E))
    x[rng.random((T, E)) < 1.5 / E] = np.inf
    x[rng.random((T, E)) < 0.1] = -np.inf
    x[rng.random((T, E)) < 0.1] = np.nan
    x[rng.random((T, E)) < 0.1] = torch.finfo(TYPES[dtype]).max
    logits = _cuda(x).to(TYPES[dtype])
    x = logits.double().cpu().numpy()
    how = dict(score=score, groups=groups, groups_kept=kept, renormalize=renormalize)
    w, ids = routing.route(logits, k, **how)
    rw, rids, _ = R.route(x, k, **how)  # logits alone decide: no rounding takes part
    np.testing.assert_array_equal(ids.cpu().numpy(), rids)
    np.testing.assert_allclose(w.cpu().numpy(), rw, rtol=1e-5, atol=1e-37)
    grad = rng.normal(size=(T, k)).astype(np.float32)
    g = routing.route_backward(_cuda(grad), logits, ids, score=score, renormalize=renormalize)
    rg = R.route_backward(grad, x, rids, None, score, renormalize)
    np.testing.assert_allclose(g.double().cpu().numpy(), rg, rtol=RTOL[dtype] * 4,
                               atol=max(ATOL[dtype], 2e-6 * np.abs(grad).max()))


def test_route_gradient_of_tiny_scores():
    """Renormalised sigmoids that are subnormal in 32 bits: their quotient by their sum is an ordinary number, and so is
    the gradient, w (1 - s) (g - u).  The scores are multiples of 2^-149 above 3e-39, off by 3e-7 of themselves and by
    expf's 2 units, 2.4e-7; their quotients and differences of those, g = +-20, add up to less than 3e-6 of 20."""
    x = np.array([[-88.5, -88.5], [-88.0, -88.25], [-87.5, -88.5], [-88.6, -30.0]], np.float32)
    grad = np.array([[20, -20]] * 4, np.float32)
    w, ids = routing.route(_cuda(x), 2, score="sigmoid", renormalize=True)
    rw, rids, _ = R.route(x, 2, score="sigmoid", renormalize=True)
    np.testing.assert_array_equal(ids.cpu().numpy(), rids)
    np.testing.assert_allclose(w.cpu().numpy(), rw, rtol=3e-6, atol=1e-37)
    g = routing.route_backward(_cuda(grad), _cuda(x), ids, score="sigmoid", renormalize=True)
    rg = R.route_backward(grad, x, rids, None, "sigmoid", True)
    np.testing.assert_allclose(g.cpu().numpy(), rg, rtol=3e-6, atol=20 * 3e-6)
