"""Waits inside the experts' products that run out: what they cost is NaN in the results, never a sum that is not
whole or what lay in memory before; all else is as it should be."""
from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

from libcusort_b200 import _capi, experts as X  # noqa: E402
from tests.test_experts_gpu import matrix, plan, weights_of  # noqa: E402

pytestmark = pytest.mark.gpu


def _products(counts, fin, fout, order="in_out", align=1):
    c, o, capacity, there = plan(counts, align, 3)
    x, w = matrix(capacity, fin, torch.bfloat16, there), weights_of(len(counts), fin, fout, torch.bfloat16, order)
    mask = there[:, None].expand(capacity, fout)
    return lambda: X.expert_products(x, w, c, o), mask, fin


def _gradient(counts, fin, fout):
    c, o, capacity, there = plan(counts, 8, 3)
    x, g = matrix(capacity, fin, torch.float16, there), matrix(capacity, fout, torch.float16, there, seed=2)
    mask = torch.tensor([n > 0 for n in counts], device="cuda")[:, None, None].expand(len(counts), fin, fout)
    return lambda: X.expert_products_grad_weights(g, x, c, o), mask, max(counts)


CASES = {
    "fewest rows, 64 columns": lambda: _products([3, 0, 5], 1024, 520),
    "fewest rows": lambda: _products([4, 2, 7], 1024, 14344, "out_in"),
    "few rows": lambda: _products([70, 0, 1, 30, 9], 1024, 4104),
    "few rows, widths off 16 bytes": lambda: _products([40, 3, 20], 771, 4099),
    "many rows": lambda: _products([600, 0, 300, 1300, 1], 1024, 4104, "out_in", 8),
    "gradient": lambda: _gradient([640, 0, 300, 1301, 1], 520, 4104),
    "gradient, widths off 16 bytes": lambda: _gradient([100, 77, 0, 300], 257, 2051),
}


@pytest.mark.parametrize("skip", [0, 1, 3, 13, 40])
@pytest.mark.parametrize("name", CASES)
def test_what_is_lost_is_nan(name, skip):
    """Step `skip` of every CTA never comes: the sums that it belongs to, and the later ones of the CTA, are lost."""
    call, mask, contracted = CASES[name]()
    assert X.product_status() == 0
    lib, right = _capi.load(), call()
    assert torch.isfinite(right).all()
    poison = torch.full_like(right, 12345.0)  # what lies in memory that the results may get
    del poison
    before = lib.cusort_set_wait_limit_ns(1_000_000)
    lib.cusort_debug_set_skip_tile(skip)
    try:
        got = call()
    finally:
        lib.cusort_debug_set_skip_tile(-1)
        lib.cusort_set_wait_limit_ns(before)
    told, nan = X.product_status(), torch.isnan(got)
    assert (nan | (got == right)).all()
    assert told == int(nan.any())
    assert not nan[~mask].any()
    if skip == 0:  # in every CTA with a tile
        assert nan[mask].all() or "gradient" in name
    if skip <= 3:
        assert told == 1
    assert torch.equal(call(), right) and X.product_status() == 0


@pytest.mark.parametrize("limit", [1, 2000, 20000])
@pytest.mark.parametrize("name", CASES)
def test_waits_that_get_hardly_any_time(name, limit):
    """Any wait may run out here, in any role: every result is right or NaN, and NaN is told."""
    call, mask, _ = CASES[name]()
    assert X.product_status() == 0
    lib, right = _capi.load(), call()
    for _ in range(5):
        before = lib.cusort_set_wait_limit_ns(limit)
        try:
            got = call()
        finally:
            lib.cusort_set_wait_limit_ns(before)
        told, nan = X.product_status(), torch.isnan(got)
        assert (nan | (got == right)).all()
        assert told == 1 or not nan.any()
        assert not nan[~mask].any()
    assert torch.equal(call(), right) and X.product_status() == 0


def test_a_status_set_while_it_is_read_is_told():
    """One CTA gives up in each call while another stream's status is read without a pause: every call is told by a read
    that began before the next call, whichever."""
    c, o, capacity, there = plan([4])
    x, w = matrix(capacity, 64, torch.bfloat16, there), weights_of(1, 64, 64, torch.bfloat16, "in_out")
    lib, stream, reader = _capi.load(), torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    assert X.product_status() == 0
    before, missed = lib.cusort_set_wait_limit_ns(1000), 0
    lib.cusort_debug_set_skip_tile(0)
    try:
        for _ in range(300):
            with torch.cuda.stream(stream):
                X.expert_products(x, w, c, o)
                done = stream.record_event()
            told, over = 0, False
            while not over:
                over = done.query()
                with torch.cuda.stream(reader):
                    told += X.product_status()
            missed += told != 1
    finally:
        lib.cusort_debug_set_skip_tile(-1)
        lib.cusort_set_wait_limit_ns(before)
    assert missed == 0
