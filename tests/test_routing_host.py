"""Host-side refusals of the routing and placement operators (no GPU): the Python checks on meta tensors, the C ABI's
argument checks, which come before any CUDA call."""
from __future__ import annotations

import ctypes as C

import pytest

torch = pytest.importorskip("torch")

from libcusort_b200 import _capi, paging, routing  # noqa: E402

INVALID = _capi.CUDA_ERROR_INVALID_VALUE
M = "meta"


def _t(*shape, dtype=torch.float32):
    return torch.empty(*shape, dtype=dtype, device=M)


def _i(*shape):
    return _t(*shape, dtype=torch.int32)


@pytest.mark.parametrize("call,match", [
    (lambda: routing.route(_t(4, 8), 2), "CUDA"),
    (lambda: routing.route(torch.zeros(4, 8), 2), "CUDA"),
    (lambda: routing.route(_t(8), 2), "2-D"),
    (lambda: routing.route(_t(8, 4).t(), 2), "rows are contiguous"),
    (lambda: routing.route(_t(4, 8), 0), "k must be"),
    (lambda: routing.route(_t(4, 8), 9), "k must be"),
    (lambda: routing.route(_t(4, 64), 33), "k must be"),
    (lambda: routing.route(_t(4, 0), 1), "experts are supported"),
    (lambda: routing.route(_t(4, 1025), 1), "experts are supported"),
    (lambda: routing.route(_t(4, 8), 2, score="tanh"), "score must be"),
    (lambda: routing.route(_t(4, 8), 2, group_score="mean"), "group_score must be"),
    (lambda: routing.route(_t(4, 8), 2, groups=3), "groups must divide"),
    (lambda: routing.route(_t(4, 64), 2, groups=64), "at most 32"),
    (lambda: routing.route(_t(4, 8), 3, groups=4, groups_kept=1), "leave at least"),
    (lambda: routing.route(_t(4, 8), 2, groups=4, groups_kept=5), "groups_kept"),
    (lambda: routing.route(_t(4, 8), 2, bias=_t(7)), "bias"),
    (lambda: routing.route(_t(4, 8), 2, bias=_t(8, dtype=torch.bfloat16)), "bias"),
    (lambda: routing.route(_t(4, 8), 2, bias=torch.zeros(8)), "bias"),
    (lambda: routing.route_backward(_t(4, 2), _t(4, 8), _i(3, 2)), "experts"),
    (lambda: routing.route_backward(_t(4, 3), _t(4, 8), _i(4, 2)), "grad_weights"),
    (lambda: routing.route_backward(_t(4, 2), _t(4, 8), _i(8)), "experts"),
    (lambda: routing.plan_dispatch(_i(4, 2), 8), "CUDA"),
    (lambda: routing.plan_dispatch(_t(4, 2), 8), "int32 or int64"),
    (lambda: routing.plan_dispatch(_i(4, 2).t(), 8), "contiguous"),
    (lambda: routing.plan_dispatch(_i(4, 2), 0), "experts are supported"),
    (lambda: routing.plan_dispatch(_i(4, 2), 1025), "experts are supported"),
    (lambda: routing.plan_dispatch(_i(4, 2), 8, align=0), "align"),
    (lambda: routing.plan_dispatch(_i((1 << 29) + 1000, 2), 1024, align=1 << 20), "2\\^31 rows"),
    (lambda: routing.dispatch(_t(4, 16), _i(8), _i(4, 2)), "CUDA"),
    (lambda: routing.dispatch(_t(5, 16), _i(8), _i(4, 2)), "rows"),
    (lambda: routing.dispatch(_t(4, 16), _i(8), _i(8)), "positions"),
    (lambda: routing.dispatch(_t(4, 66), _i(8), _i(4, 33)), "k must be"),
    (lambda: routing.dispatch(_t(4, 16), _t(8), _i(4, 2)), "sources"),
    (lambda: routing.dispatch(_t(16, 4).t(), _i(8), _i(4, 2)), "rows are contiguous"),
    (lambda: routing.dispatch_backward(_t(8, 16, dtype=torch.float64), _i(4, 2)), "float32, float16 or bfloat16"),
    (lambda: routing.combine(_t(8, 16), _t(4, 2), _i(4, 2)), "CUDA"),
    (lambda: routing.combine(_t(8, 16), None, _i(4, 2)), "weights"),
    (lambda: routing.combine(_t(8, 16), _t(4, 3), _i(4, 2)), "weights"),
    (lambda: routing.combine(_t(16, 8).t(), _t(4, 2), _i(4, 2)), "contiguous"),
    (lambda: routing.combine(_t(8, 16), _t(4, 2), _i(4, 2), residual=_t(4, 15)), "residual"),
    (lambda: routing.combine(_t(8, 16), _t(4, 2), _i(4, 2), residual=_t(4, 16, dtype=torch.float16)), "residual"),
    (lambda: routing.combine_backward(_t(4, 16), _t(8, 16), _t(4, 2), _i(9), _i(4, 2)), "sources"),
    (lambda: routing.combine_backward(_t(3, 16), _t(8, 16), _t(4, 2), _i(8), _i(4, 2)), "grad_out"),
    (lambda: paging.page_plan(_i(3), _i(3), _i(3, 4), 16, 9), "CUDA"),
    (lambda: paging.page_plan(_i(3), _i(2), _i(3, 4), 16, 9), "new_lens"),
    (lambda: paging.page_plan(_t(3), _i(3), _i(3, 4), 16, 9), "cached_lens"),
    (lambda: paging.page_plan(_i(16385), _i(16385), _i(16385, 4), 16, 9), "at most 16384"),
    (lambda: paging.page_plan(_i(3), _i(3), _i(2, 4), 16, 9), "block_tables"),
    (lambda: paging.page_plan(_i(3), _i(3), _i(1, 4).expand(3, 4), 16, 9), "overlap"),
    (lambda: paging.page_plan(_i(3), _i(3), _i(3, 4), 0, 9), "block_size"),
    (lambda: paging.page_plan(_i(3), _i(3), _i(3, 4), 16, -1), "num_tokens"),
    (lambda: paging.page_plan(_i(3), _i(3), _i(3, 4), 16, 9, free_blocks=_i(5)), "go together"),
    (lambda: paging.page_plan(_i(3), _i(3), _i(3, 4), 16, 9, free_blocks=_i(5), num_free=_i(2)), "num_free"),
    (lambda: paging.page_plan(_i(3), _i(3), _i(3, 4), 16, 9, free_blocks=_t(5), num_free=_i(1)), "free_blocks"),
])
def test_refused_with_a_reason(call, match):
    with pytest.raises((ValueError, TypeError), match=match):
        call()


def test_unsupported_logit_type():
    with pytest.raises(TypeError, match="float32, float16 or bfloat16"):
        routing.route(_t(4, 8, dtype=torch.float64), 2)


P = C.c_void_p(0x10000)  # never dereferenced: every call below is refused first


def _route(kind=0, logits=P, stride=8, weights=P, experts=P, T=4, E=8, k=2, groups=1, kept=1, score=0, group=0):
    return _capi.load().cusort_route(kind, logits, stride, None, weights, experts, T, E, k, groups, kept, score, group,
                                     0, 1.0, None)


@pytest.mark.parametrize("bad", [
    dict(kind=3), dict(kind=-1), dict(logits=None), dict(stride=-1), dict(weights=None), dict(experts=None),
    dict(T=-1), dict(E=0), dict(E=1025), dict(k=0), dict(k=9), dict(E=64, k=33), dict(groups=0), dict(groups=3),
    dict(E=64, groups=64, kept=64), dict(groups=4, kept=0), dict(groups=4, kept=5), dict(groups=8, kept=1),
    dict(score=2), dict(group=-1), dict(T=1 << 40)], ids=str)
def test_route_arguments(bad):
    assert _route(**bad) == INVALID


def test_nothing_to_do_makes_no_cuda_call():
    lib = _capi.load()
    assert _route(T=0, logits=None, weights=None, experts=None) == 0
    assert lib.cusort_route_backward(0, None, None, 8, None, None, None, 0, 8, 2, 0, 0, 1.0, None) == 0
    assert lib.cusort_dispatch_rows(None, 0, 16, None, None, None, 0, 2, 0, None) == 0
    assert lib.cusort_combine_rows(0, None, None, None, None, 0, None, 0, 2, 0, 16, None) == 0
    assert lib.cusort_combine_rows_backward(0, None, 0, None, None, None, None, None, None, 0, 2, 0, 16, None) == 0


def test_route_backward_arguments():
    def call(kind=0, grad=P, logits=P, experts=P, out=P, T=4, E=8, k=2, score=0, stride=8):
        return _capi.load().cusort_route_backward(kind, grad, logits, stride, None, experts, out, T, E, k, score, 0,
                                                  1.0, None)
    for bad in (dict(kind=7), dict(grad=None), dict(logits=None), dict(experts=None), dict(out=None), dict(T=-1),
                dict(E=1025), dict(k=0), dict(k=9), dict(score=5), dict(stride=-4)):
        assert call(**bad) == INVALID, bad


def _plan(temp=P, room=1 << 20, size=4, experts=P, n=100, E=8, align=1, cap=100, counts=P, offsets=P, sources=P,
          positions=P):
    nb = C.c_size_t(room)
    rc = _capi.load().cusort_plan_dispatch(temp, C.byref(nb), size, experts, n, E, align, cap, counts, offsets,
                                           sources, positions, None)
    return rc, nb.value


def test_plan_arguments():
    for bad in (dict(size=2), dict(n=-1), dict(E=0), dict(E=1025), dict(align=0), dict(align=(1 << 20) + 1),
                dict(cap=99), dict(align=2, cap=107), dict(n=1 << 31, cap=1 << 31), dict(cap=1 << 31),
                dict(experts=None), dict(counts=None), dict(offsets=None), dict(sources=None), dict(positions=None),
                dict(temp=C.c_void_p(0x10008)), dict(n=100_000, cap=100_000, room=8)):
        assert _plan(**bad)[0] == INVALID, bad
    assert _capi.load().cusort_plan_dispatch(None, None, 4, P, 100, 8, 1, 100, P, P, P, P, None) == INVALID


def test_plan_size_query():
    rc, small = _plan(temp=None, experts=None, counts=None, offsets=None, sources=None, positions=None)
    assert rc == 0 and small >= 1
    rc, large = _plan(temp=None, n=1 << 20, cap=1 << 20)
    assert rc == 0 and large > small


def test_rows_arguments():
    lib = _capi.load()

    def dispatch(x=P, stride=16, width=16, sources=P, positions=P, rows=P, T=4, k=2, cap=8):
        return lib.cusort_dispatch_rows(x, stride, width, sources, positions, rows, T, k, cap, None)
    for bad in (dict(x=None), dict(stride=-16), dict(width=1 << 31), dict(sources=None), dict(positions=None),
                dict(rows=None), dict(T=-1), dict(k=0), dict(k=33), dict(cap=-1), dict(cap=1 << 31),
                dict(T=1 << 30, k=2)):
        assert dispatch(**bad) == INVALID, bad

    def combine(kind=0, rows=P, positions=P, residual=None, stride=0, out=P, T=4, k=2, cap=8, hidden=16):
        return lib.cusort_combine_rows(kind, rows, P, positions, residual, stride, out, T, k, cap, hidden, None)
    for bad in (dict(kind=3), dict(rows=None), dict(positions=None), dict(out=None), dict(T=-1), dict(k=0),
                dict(k=33), dict(cap=-1), dict(hidden=-1), dict(hidden=1 << 31), dict(residual=P, stride=-1)):
        assert combine(**bad) == INVALID, bad

    def backward(kind=0, grad=P, stride=16, rows=P, weights=P, sources=P, positions=P, gr=P, gw=P, T=4, k=2, cap=8,
                 hidden=16):
        return lib.cusort_combine_rows_backward(kind, grad, stride, rows, weights, sources, positions, gr, gw, T, k,
                                                cap, hidden, None)
    for bad in (dict(kind=3), dict(grad=None), dict(stride=-1), dict(rows=None), dict(weights=None),
                dict(sources=None), dict(positions=None), dict(gr=None), dict(gw=None), dict(T=-1), dict(k=0),
                dict(k=33), dict(cap=-1), dict(hidden=-1)):
        assert backward(**bad) == INVALID, bad


def test_page_arguments():
    def call(cached=P, new=P, R=4, block=16, tables=P, stride=8, width=8, free=P, blocks=32, left=P, tokens=9,
             slots=P, positions=P, starts=P, served=P, rest=P):
        return _capi.load().cusort_page_plan(cached, new, R, block, tables, stride, width, free, blocks, left, tokens,
                                             slots, positions, starts, served, rest, None)
    for bad in (dict(cached=None), dict(new=None), dict(R=-1), dict(R=16385), dict(block=0), dict(block=(1 << 20) + 1),
                dict(tables=None), dict(stride=7), dict(width=-1), dict(free=None), dict(blocks=-1),
                dict(blocks=(1 << 30) + 1), dict(left=None), dict(tokens=-1), dict(tokens=1 << 31), dict(slots=None),
                dict(positions=None), dict(starts=None), dict(served=None), dict(rest=None)):
        assert call(**bad) == INVALID, bad


def test_page_plan_counts_apart():
    """The count of free blocks may not be updated in place: it is read by every CTA, and written by one."""
    lens, starts = C.c_void_p(0x20000), C.c_void_p(0x30000)
    rc = _capi.load().cusort_page_plan(lens, lens, 4, 16, P, 8, 8, P, 32, C.c_void_p(0x40000), 9, P, P, starts, P,
                                       C.c_void_p(0x40000), None)
    assert rc == INVALID


@pytest.mark.parametrize("call", [
    lambda: routing.dispatch(_t(4, 16, dtype=torch.complex64).conj(), _i(8), _i(4, 2)),
    lambda: routing.dispatch(torch._neg_view(_t(4, 16)), _i(8), _i(4, 2)),
    lambda: routing.route(torch._neg_view(_t(4, 8)), 2),
    lambda: routing.route(_t(4, 8), 2, bias=torch._neg_view(_t(8))),
    lambda: routing.combine(torch._neg_view(_t(8, 16)), _t(4, 2), _i(4, 2)),
    lambda: routing.combine(_t(8, 16), torch._neg_view(_t(4, 2)), _i(4, 2)),
    lambda: routing.combine(_t(8, 16), torch._efficientzerotensor((4, 2), device=M), _i(4, 2)),
    lambda: paging.page_plan(torch._neg_view(_i(3)), _i(3), _i(3, 4), 16, 9),
])
def test_lazy_views_are_refused(call):
    """Tensors whose memory does not hold their values yet."""
    with pytest.raises(ValueError, match="resolve"):
        call()
