"""Calls of the experts' products that their documentation allows and a plan of plan_dispatch does not make, against a
plain implementation in 64 bits."""
from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

from libcusort_b200 import experts as X  # noqa: E402
from tests.test_experts_gpu import TYPES, close, matrix, weights_of  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def no_wait_ran_out():
    yield
    assert X.product_status() == 0


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def check(first, count, capacity, fin, fout, dtype, order="in_out"):
    """Products and gradients of segments [first, first + count) that do not overlap, as they are meant."""
    dtype = TYPES[dtype]
    c, o = ints(count), ints(list(first) + [capacity])
    there = torch.zeros(capacity, dtype=torch.bool, device="cuda")
    spans = [(max(f, 0), max(max(f, 0), min(f + max(n, 0), capacity))) for f, n in zip(first, count)]
    for begin, end in spans:
        there[begin:end] = True
    x, g = matrix(capacity, fin, dtype, there), matrix(capacity, fout, dtype, there, seed=2)
    w = weights_of(len(count), fin, fout, dtype, order)
    out = X.expert_products(x, w, c, o)
    grad_rows, grad_weights = X.expert_products_backward(g, x, w, c, o)
    assert not out[~there].any() and not grad_rows[~there].any()
    for e, (begin, end) in enumerate(spans):
        at = slice(begin, end)
        xe, ge, we = x[at].double(), g[at].double(), w[e].double()
        close(out[at], xe @ we, xe.abs() @ we.abs(), fin)
        close(grad_rows[at], ge @ we.T, ge.abs() @ we.T.abs(), fout)
        close(grad_weights[e], xe.T @ ge, xe.T.abs() @ ge.abs(), max(end - begin, 1))


ORDERS = [
    # the later expert's rows first
    ([20, 0], [10, 20], 30),
    # gaps of all sizes, empty experts that begin at 0, in the middle of a segment and behind the rows
    ([0, 60, 5, 0, 10, 70, 200], [0, 30, 5, 0, 40, 0, 0], 100),
    # nothing but gaps before, between and behind
    ([150, 0, 90, 400], [100, 0, 1, 33], 1000),
    # the fewest rows
    ([9, 0, 3], [5, 2, 4], 16),
    # many rows an expert
    ([700, 0, 300, 1300], [600, 290, 400, 130], 1500),
]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("order", ["in_out", "out_in"])
@pytest.mark.parametrize("first,count,capacity", ORDERS, ids=lambda v: str(v)[:24])
def test_segments_in_any_order(first, count, capacity, order, dtype):
    check(first, count, capacity, 72, 136, dtype, order)
    check(first, count, capacity, 33, 7, "f16" if dtype == "bf16" else dtype, order)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_segments_that_begin_before_the_rows(dtype):
    """Only the rows that there are: of ten from -4 on the first six."""
    check([-4, 6, -30, 90], [10, 20, 25, 1 << 30], 100, 72, 136, dtype)
    check([-2 ** 31, -1], [2 ** 31 - 1, 8], 300, 72, 40, dtype)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("most", [3, 40])
def test_many_experts_in_any_order(most, dtype):
    gen = torch.Generator().manual_seed(most)
    order, at = torch.randperm(1024, generator=gen).tolist(), 5
    first, count = [0] * 1024, torch.randint(0, most + 1, (1024,), generator=gen).tolist()
    for e in order:
        first[e] = at
        at += count[e] + int(torch.randint(0, 4, (1,), generator=gen))
    check(first, count, at, 24, 40, dtype)
