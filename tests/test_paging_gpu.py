"""page_plan on the GPU against a plain implementation (tests/routing_reference.py)."""
from __future__ import annotations

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from libcusort_b200 import paging  # noqa: E402
from tests import routing_reference as R  # noqa: E402

pytestmark = pytest.mark.gpu


def _cuda(a, dtype=torch.int32):
    return torch.from_numpy(np.ascontiguousarray(a)).to(dtype).cuda()


def _step(rng, requests, context, chunk, block, width=None, apart=0):
    cached, new = rng.integers(0, context + 1, requests), rng.integers(0, chunk + 1, requests)
    width = -(-(context + chunk) // block) if width is None else width
    pool = rng.permutation(requests * width * 2)
    tables = np.full((requests, width), -1)
    for r in range(requests):
        held = min(width, -(-cached[r] // block))
        tables[r, :held], pool = pool[:held], pool[held:]
    return cached, new, tables, pool


def _run(cached, new, tables, block, tokens, free, left, apart=0):
    wide = np.full((tables.shape[0], tables.shape[1] + apart), -9)
    wide[:, :tables.shape[1]] = tables
    t = _cuda(wide)
    how = {} if free is None else dict(free_blocks=_cuda(free), num_free=_cuda([left]))
    plan = paging.page_plan(_cuda(cached), _cuda(new), t[:, :tables.shape[1]], block, tokens, **how)
    ref_tables = tables.copy()
    slots, positions, starts, served, rest = R.page_plan(cached, new, ref_tables, block, tokens, free, left)
    np.testing.assert_array_equal(plan.starts.cpu().numpy(), starts)
    np.testing.assert_array_equal(plan.served.cpu().numpy(), served)
    np.testing.assert_array_equal(plan.positions.cpu().numpy(), positions)
    np.testing.assert_array_equal(plan.slots.cpu().numpy(), slots)
    np.testing.assert_array_equal(t[:, :tables.shape[1]].cpu().numpy(), ref_tables)
    assert (t[:, tables.shape[1]:] == -9).all()
    assert plan.num_free is None if free is None else plan.num_free.tolist() == [rest]
    return plan, served


@pytest.mark.parametrize("block", [1, 16, 17, 64])
@pytest.mark.parametrize("requests,context,chunk", [(1, 0, 1), (1, 100, 1), (1, 0, 5000), (7, 33, 0), (64, 200, 1),
                                                    (255, 40, 9), (256, 64, 64), (300, 10, 3), (1025, 20, 2)])
def test_step(requests, context, chunk, block):
    rng = np.random.default_rng([requests, context, chunk, block])
    cached, new, tables, pool = _step(rng, requests, context, chunk, block)
    total = int(new.sum())
    for tokens in {total, total + 13, max(0, total - 3), 0}:
        _run(cached, new, tables, block, tokens, pool, len(pool), apart=3)
    need = int((-(-(cached + new) // block) - -(-cached // block)).sum())
    for left in {0, 1, need // 2, max(0, need - 1), need}:  # too few free blocks, and just enough
        _run(cached, new, tables, block, total, pool, left)


def test_tables_that_hold_all_blocks():
    rng = np.random.default_rng(5)
    cached, new, tables, pool = _step(rng, 50, 100, 20, 16)
    tables = rng.permutation(tables.size).reshape(tables.shape)
    tables[3, :] = -1  # nothing there: no slots
    _run(cached, new, tables, 16, int(new.sum()) + 1, None, 0)


def test_narrow_table():
    """A request that outgrows its table is not served, takes no block, and holds up nobody."""
    rng = np.random.default_rng(6)
    cached, new, tables, pool = _step(rng, 40, 100, 30, 16, width=6)
    cached = np.minimum(cached, 96)
    _, served = _run(cached, new, tables, 16, int(new.sum()), pool, len(pool))
    assert served.any() and not served.all()


def test_lengths_out_of_the_ordinary():
    big = 2 ** 31 - 1
    cached = np.array([5, -3, big, 0, big - 7, 12, 0])
    new = np.array([0, 4, 1, -2, 7, 3, 40])
    tables = np.full((7, 4), -1)
    tables[0, 0], tables[5, 0] = 11, 12
    _run(cached, new, tables, 16, 60, np.arange(100, 120), 20)
    # 2^31 tokens and more: the sum stops there
    cached, new = np.zeros(3, int), np.array([3, big, big])
    plan, _ = _run(cached, new, np.full((3, 2), -1), 16, 10, np.arange(9), 9)
    assert plan.starts.tolist() == [0, 3, big, big]


def test_slots_beyond_32_bits():
    cached, new = np.array([2 ** 20 * 2 + 5, 7]), np.array([3, 2])
    tables = np.array([[2 ** 30 - 1, 2 ** 30 - 2, 2 ** 30 - 3], [2 ** 30 - 4, -1, -1]])
    plan, _ = _run(cached, new, tables, 2 ** 20, 5, np.array([8]), 1)
    assert int(plan.slots[0]) == (2 ** 30 - 3) * 2 ** 20 + 5


def test_no_requests_and_empty_free_list():
    empty = np.zeros(0, int)
    _run(empty, empty, np.zeros((0, 4), int), 16, 5, np.arange(3), 3)
    _run(np.array([3, 16]), np.array([2, 1]), np.array([[4], [5]]), 16, 3, empty, 0)
    _run(np.array([3]), np.array([2]), np.zeros((1, 0), int), 16, 3, np.arange(3), 3)
    _run(np.array([0]), np.array([20]), np.full((1, 4), -1), 16, 20, np.arange(3), 99)  # more than the list holds
    _run(np.array([0]), np.array([20]), np.full((1, 4), -1), 16, 20, np.arange(3), -2)


@pytest.mark.parametrize("requests", [5000, 16384])
def test_many_requests(requests):
    rng = np.random.default_rng(requests)
    cached, new, tables, pool = _step(rng, requests, 40, 2, 8)
    _run(cached, new, tables, 8, int(new.sum()) + 1, pool, len(pool) // 3)


def test_planned_again():
    """The free list is only read: the same step gives the same plan."""
    rng = np.random.default_rng(9)
    cached, new, tables, pool = _step(rng, 30, 50, 10, 16)
    t, f, n = _cuda(tables), _cuda(pool), _cuda([len(pool)])
    a = paging.page_plan(_cuda(cached), _cuda(new), t, 16, int(new.sum()), free_blocks=f, num_free=n)
    was = t.clone()
    b = paging.page_plan(_cuda(cached), _cuda(new), t, 16, int(new.sum()), free_blocks=f, num_free=n)
    assert torch.equal(t, was) and all(torch.equal(p, q) for p, q in zip(a, b))


def test_c_abi_from_two_threads():
    """Steps of different numbers of requests, planned from two host threads at once: the C ABI is called without the
    interpreter's lock.  Each thread has tensors and a stream of its own."""
    import threading

    from libcusort_b200 import _capi
    lib = _capi.load()
    refused = []

    def plan(requests, stream):
        with torch.cuda.stream(stream):
            lens, new = torch.zeros(requests, dtype=torch.int32, device="cuda"), _cuda(np.ones(requests))
            tables, free = torch.zeros(requests, 1, dtype=torch.int32, device="cuda"), _cuda(np.arange(requests))
            left, rest = _cuda([requests]), _cuda([0])
            slots = torch.zeros(requests, dtype=torch.int64, device="cuda")
            positions, starts = torch.zeros_like(lens), torch.zeros(requests + 1, dtype=torch.int32, device="cuda")
            served = torch.zeros(requests, dtype=torch.uint8, device="cuda")
            stream.synchronize()
            args = (lens.data_ptr(), new.data_ptr(), requests, 16, tables.data_ptr(), 1, 1, free.data_ptr(), requests,
                    left.data_ptr(), requests, slots.data_ptr(), positions.data_ptr(), starts.data_ptr(),
                    served.data_ptr(), rest.data_ptr(), stream.cuda_stream)
            refused.extend(rc for rc in (lib.cusort_page_plan(*args) for _ in range(4000)) if rc != 0)
            stream.synchronize()
            assert bool(served.all()) and int(rest) == 0 and int(starts[-1]) == requests

    threads = [threading.Thread(target=plan, args=(n, torch.cuda.Stream())) for n in (16384, 7000)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not refused, f"{len(refused)} calls refused, with {set(refused)}"
