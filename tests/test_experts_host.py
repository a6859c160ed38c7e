"""Host-side refusals of the experts' products and of the page operators (no GPU): the checks of the PyTorch functions
on meta tensors, the C ABI's argument checks and size queries, which come before any CUDA call."""
from __future__ import annotations

import ctypes as C

import pytest

torch = pytest.importorskip("torch")

import libcusort_b200.ops  # noqa: E402,F401  (registers the operators)
from libcusort_b200 import _capi, experts, paging  # noqa: E402

INVALID = _capi.CUDA_ERROR_INVALID_VALUE
ops = torch.ops.cusort


def _t(*shape, dtype=torch.bfloat16):
    return torch.empty(*shape, dtype=dtype, device="meta")


def _i(*shape):
    return _t(*shape, dtype=torch.int32)


def _products(rows=None, weights=None, counts=None, offsets=None):
    return experts.expert_products(_t(20, 16) if rows is None else rows, _t(3, 16, 24) if weights is None else weights,
                                   _i(3) if counts is None else counts, _i(4) if offsets is None else offsets)


def _pool(blocks=9, **other):
    return dict(free_blocks=_i(blocks), num_free=_i(1), shares=_i(blocks)) | other


@pytest.mark.parametrize("call,match", [
    (lambda: _products(), "CUDA"),
    (lambda: _products(rows=_t(20, 16, dtype=torch.float32)), "weights"),
    (lambda: _products(rows=_t(20, 16, dtype=torch.float64)), "float32, float16 or bfloat16"),
    (lambda: _products(rows=_t(20, 16, dtype=torch.float16)), "weights"),
    (lambda: _products(rows=_t(16, 20).t()), "rows are contiguous"),
    (lambda: _products(rows=_t(20)), "2-D"),
    (lambda: _products(rows=_t(20, 17)), "weights"),
    (lambda: _products(weights=_t(4, 16, 24)), "weights"),
    (lambda: _products(weights=_t(3, 16)), "weights"),
    (lambda: _products(weights=_t(3, 16, 24, 2)[..., 0]), "contiguous along one"),
    (lambda: _products(weights=_t(3, 16, 0)), "1 to 1048576"),
    (lambda: _products(rows=_t(20, 0), weights=_t(3, 0, 24)), "1 to 1048576"),
    (lambda: _products(counts=_i(3, 1)), "counts"),
    (lambda: _products(counts=_t(3, dtype=torch.int64)), "counts"),
    (lambda: _products(counts=_i(0), offsets=_i(1), weights=_t(0, 16, 24)), "1 to 1024"),
    (lambda: _products(counts=_i(1025), offsets=_i(1026), weights=_t(1025, 16, 24)), "1 to 1024"),
    (lambda: _products(offsets=_i(3)), "offsets"),
    (lambda: _products(offsets=torch.zeros(4, dtype=torch.int32)), "offsets"),
    (lambda: _products(rows=torch._neg_view(_t(20, 16))), "resolve"),
    (lambda: experts.expert_products_grad_rows(_t(20, 16), _t(3, 16, 24), _i(3), _i(4)), "weights"),
    (lambda: experts.expert_products_grad_rows(_t(20, 24), _t(3, 16, 24), _i(3), _i(4)), "CUDA"),
    (lambda: experts.expert_products_grad_weights(_t(20, 24), _t(20, 16), _i(3), _i(4)), "CUDA"),
    (lambda: experts.expert_products_grad_weights(_t(19, 24), _t(20, 16), _i(3), _i(4)), "grad_out"),
    (lambda: experts.expert_products_grad_weights(_t(20), _t(20, 16), _i(3), _i(4)), "grad_out"),
    (lambda: experts.expert_products_grad_weights(_t(20, 24, dtype=torch.float16), _t(20, 16), _i(3), _i(4)),
     "grad_out"),
    (lambda: experts.expert_products_backward(_t(20, 24), _t(20, 16), _t(3, 16, 24, 2)[..., 0], _i(3), _i(4)),
     "contiguous along one"),
    (lambda: paging.page_fork(_i(3, 4), _i(3), _i(5), 16, **_pool()), "CUDA"),
    (lambda: paging.page_fork(_i(3, 4), _i(3), _t(5), 16, **_pool()), "parents"),
    (lambda: paging.page_fork(_i(3, 4), _i(3), _i(5, 1), 16, **_pool()), "parents"),
    (lambda: paging.page_fork(_i(3, 4), _i(3), _i(16385), 16, **_pool()), "at most 16384"),
    (lambda: paging.page_fork(_i(16385, 4), _i(16385), _i(5), 16, **_pool()), "at most 16384"),
    (lambda: paging.page_fork(_i(2, 4), _i(3), _i(5), 16, **_pool()), "block_tables"),
    (lambda: paging.page_fork(_t(3, 4), _i(3), _i(5), 16, **_pool()), "block_tables"),
    (lambda: paging.page_fork(_i(1, 4).expand(3, 4), _i(3), _i(5), 16, **_pool()), "overlap"),
    (lambda: paging.page_fork(_i(3, 4), _t(3), _i(5), 16, **_pool()), "lens"),
    (lambda: paging.page_fork(_i(3, 4), _i(3), _i(5), 0, **_pool()), "block_size"),
    (lambda: paging.page_fork(_i(3, 4), _i(3), _i(5), 16, **_pool(free_blocks=_i(8))), "free_blocks"),
    (lambda: paging.page_fork(_i(3, 4), _i(3), _i(5), 16, **_pool(num_free=_i(2))), "num_free"),
    (lambda: paging.page_fork(_i(3, 4), _i(3), _i(5), 16, **_pool(shares=_i(3, 3))), "shares"),
    (lambda: paging.page_fork(_i(3, 4), _i(3), _i(5), 16, **_pool(shares=_t(9))), "shares"),
    (lambda: paging.page_free(_i(3, 4), _i(3), _i(3), 16, **_pool()), "CUDA"),
    (lambda: paging.page_free(_i(3, 4), _i(3), _i(2), 16, **_pool()), "keep_lens"),
    (lambda: paging.page_free(_i(3, 4), _i(3), _i(3), (1 << 20) + 1, **_pool()), "block_size"),
    (lambda: paging.page_compact(_i(3, 4), _i(3), 16, 9), "CUDA"),
    (lambda: paging.page_compact(_i(3, 4), _i(3), 16, -1), "num_blocks"),
    (lambda: paging.page_compact(_i(3, 4), _i(3), 16, (1 << 30) + 1), "num_blocks"),
    (lambda: paging.page_compact(_i(4, 3).t(), _i(3), 16, 9), "rows are contiguous"),
    (lambda: paging.page_copy([_t(9, 2)], _i(3), _i(3)), "CUDA"),
    (lambda: paging.page_copy(_t(9, 2), _i(3), _i(3)), "list or tuple"),
    (lambda: paging.page_copy([3], _i(3), _i(3)), "tensor"),
    (lambda: paging.page_copy([_t(9, 2)], _t(3), _i(3)), "sources"),
    (lambda: paging.page_copy([_t(9, 2)], _i(3), _i(4)), "destinations"),
    (lambda: paging.page_copy([_t(9, 2), _t(8, 2)], _i(3), _i(3)), "with 9 blocks"),
    (lambda: paging.page_copy([_t(9, 2, 3).transpose(1, 2)], _i(3), _i(3)), "contiguous in itself"),
    (lambda: paging.page_copy([_t(1, 2).expand(9, 2)], _i(3), _i(3)), "overlap"),
    (lambda: paging.page_copy([torch.zeros(9, 2)], _i(3), _i(3)), "every cache"),
    (lambda: paging.page_copy([torch._neg_view(_t(9, 2))], _i(3), _i(3)), "resolve"),
])
def test_refused_with_a_reason(call, match):
    with pytest.raises((ValueError, TypeError), match=match):
        call()


def test_fake_shapes():
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        def ints(*shape):
            return torch.empty(*shape, dtype=torch.int32, device="cuda")
        rows = torch.empty(20, 16, dtype=torch.bfloat16, device="cuda")
        for w in (rows.new_empty(3, 16, 24), rows.new_empty(3, 24, 16).transpose(1, 2)):
            out = ops.expert_products(rows, w, ints(3), ints(4))
            assert out.shape == (20, 24) and out.dtype == rows.dtype
            assert ops.expert_products_grad_rows(out, w, ints(3), ints(4)).shape == rows.shape
            for order in (False, True):
                assert ops.expert_products_grad_weights(out, rows, ints(3), ints(4), order).shape == w.shape
        fork = ops.page_fork(ints(3, 4), ints(3), ints(5), 16, ints(9), ints(1), ints(9))
        assert [tuple(t.shape) for t in fork] == [(5, 4), (5,), (5,), (5,), (5,), (9,), (9,), (1,)]
        assert fork[4].dtype == torch.bool
        assert [tuple(t.shape) for t in ops.page_free(ints(3, 4), ints(3), ints(3), 16, ints(9), ints(1),
                                                      ints(9))] == [(9,), (9,), (1,)]
        assert [tuple(t.shape) for t in ops.page_compact(ints(3, 4), ints(3), 16, 9)] == [(3, 4), (4,), (4,), (9,),
                                                                                         (9,), (1,)]
        assert ops.page_copy([rows], ints(3), ints(3)) is None


P = C.c_void_p(0x10000)  # never dereferenced: every call below is refused first, or asks for a size


def _call(temp=P, room=1 << 40, kind=2, rows=P, row_stride=64, weights=P, expert=64 * 72, fin=72, fout=1, counts=P,
          offsets=P, out=P, capacity=10, width=64, result=72, num=3):
    nb = C.c_size_t(room)
    rc = _capi.load().cusort_expert_products(temp, C.byref(nb), kind, rows, row_stride, weights, expert, fin, fout,
                                             counts, offsets, out, capacity, width, result, num, None)
    return rc, nb.value


def test_products_arguments():
    for bad in (dict(kind=-1), dict(kind=3), dict(capacity=-1), dict(capacity=1 << 31), dict(capacity=(1 << 31) - 1024), dict(width=0),
                dict(width=(1 << 20) + 1), dict(result=0), dict(result=(1 << 20) + 1), dict(num=0), dict(num=1025),
                dict(row_stride=-1), dict(expert=-8), dict(fin=-1), dict(fin=3, fout=2), dict(rows=None),
                dict(weights=None), dict(counts=None), dict(offsets=None), dict(out=None),
                dict(out=C.c_void_p(0x10002)), dict(row_stride=65, room=16), dict(row_stride=65, temp=C.c_void_p(8)),
                dict(capacity=(1 << 31) - 2000, result=1 << 20, num=1024)):
        assert _call(**bad)[0] == INVALID, bad
    assert _call(capacity=0, rows=None, weights=None, counts=None, offsets=None, out=None)[0] == 0
    assert _capi.load().cusort_expert_products(P, None, 2, P, 64, P, 64, 72, 1, P, P, P, 10, 64, 72, 3, None) == INVALID


def test_products_size_query():
    """A workspace where an operand's address or stride is no multiple of 16 bytes."""
    assert _call(temp=None) == (0, 1)
    assert _call(temp=None, capacity=0, row_stride=65) == (0, 1)
    rows = _call(temp=None, row_stride=65)[1]
    assert rows >= 10 * 64 * 2
    assert _call(temp=None, rows=C.c_void_p(0x10002))[1] == rows
    weights = _call(temp=None, fin=73, expert=64 * 73)[1]
    assert weights >= 3 * 64 * 72 * 2
    assert _call(temp=None, row_stride=65, fin=73, expert=64 * 73)[1] == rows + weights
    assert _call(temp=None, fin=1, fout=64)[1] == 1  # the other order
    assert _call(temp=None, kind=0, row_stride=65, rows=C.c_void_p(0x10004))[1] == 1  # 32 bits: wherever they are


def test_products_gradient_arguments():
    def call(temp=P, room=1 << 40, kind=1, rows=P, row_stride=64, grad=P, grad_stride=72, counts=P, offsets=P, out=P,
             order=0, capacity=10, fin=64, fout=72, num=3):
        nb = C.c_size_t(room)
        return _capi.load().cusort_expert_products_grad_weights(temp, C.byref(nb), kind, rows, row_stride, grad,
                                                                grad_stride, counts, offsets, out, order, capacity,
                                                                fin, fout, num, None), nb.value
    for bad in (dict(kind=3), dict(capacity=-1), dict(fin=0), dict(fout=0), dict(num=0), dict(num=1025),
                dict(row_stride=-1), dict(grad_stride=-1), dict(rows=None), dict(grad=None), dict(counts=None),
                dict(offsets=None), dict(out=None), dict(out=C.c_void_p(0x10008)), dict(grad_stride=73, room=1)):
        assert call(**bad)[0] == INVALID, bad
    assert call(temp=None) == (0, 1)
    assert call(temp=None, row_stride=66)[1] >= 10 * 64 * 2


def test_pages_arguments():
    lib = _capi.load()
    a, b, c, d = (C.c_void_p(0x10000 * i) for i in range(2, 6))

    def fork(temp=P, room=1 << 20, tables=P, stride=4, width=4, lens=P, R=3, parents=P, N=5, block=16, free=a, left=b,
             shares=c, blocks=9, tables_out=d, lens_out=d, sources=d, destinations=d, served=d, shares_out=d,
             free_out=d, left_out=d):
        nb = C.c_size_t(room)
        return lib.cusort_page_fork(temp, C.byref(nb), tables, stride, width, lens, R, parents, N, block, free, left,
                                    shares, blocks, tables_out, lens_out, sources, destinations, served, shares_out,
                                    free_out, left_out, None)
    for bad in (dict(room=4), dict(temp=C.c_void_p(0x10004)), dict(tables=None), dict(stride=3), dict(width=-1),
                dict(lens=None), dict(R=-1), dict(R=16385), dict(parents=None), dict(N=-1), dict(N=16385),
                dict(block=0), dict(free=None), dict(left=None), dict(shares=None), dict(blocks=-1),
                dict(blocks=(1 << 30) + 1), dict(tables_out=None), dict(lens_out=None), dict(sources=None),
                dict(destinations=None), dict(served=None), dict(shares_out=None), dict(free_out=None),
                dict(left_out=None), dict(left_out=b), dict(free_out=a), dict(shares_out=c), dict(tables_out=P),
                dict(lens_out=P)):
        assert fork(**bad) == INVALID, bad

    def free(temp=P, tables=P, stride=4, width=4, lens=P, keep=P, R=3, block=16, free=a, left=b, shares=c, blocks=9,
             shares_out=d, free_out=d, left_out=d):
        nb = C.c_size_t(1 << 20)
        return lib.cusort_page_free(temp, C.byref(nb), tables, stride, width, lens, keep, R, block, free, left, shares,
                                    blocks, shares_out, free_out, left_out, None)
    for bad in (dict(tables=None), dict(stride=3), dict(lens=None), dict(keep=None), dict(R=16385), dict(block=0),
                dict(free=None), dict(left=None), dict(shares=None), dict(shares_out=None), dict(free_out=None),
                dict(left_out=None), dict(left_out=b), dict(free_out=a), dict(shares_out=c)):
        assert free(**bad) == INVALID, bad

    def compact(temp=P, room=1 << 20, tables=P, stride=4, width=4, lens=P, R=3, block=16, blocks=9, tables_out=d,
                sources=d, destinations=d, shares=d, free_out=d, left=d):
        nb = C.c_size_t(room)
        return lib.cusort_page_compact(temp, C.byref(nb), tables, stride, width, lens, R, block, blocks, tables_out,
                                       sources, destinations, shares, free_out, left, None)
    for bad in (dict(room=4), dict(tables=None), dict(stride=3), dict(lens=None), dict(R=16385), dict(block=0),
                dict(blocks=-1), dict(tables_out=None), dict(tables_out=P), dict(sources=None),
                dict(destinations=None), dict(shares=None), dict(free_out=None), dict(left=None)):
        assert compact(**bad) == INVALID, bad
    for query in (lambda n: lib.cusort_page_fork(None, n, *[P, 4, 4, P, 3, P, 5, 16] + [P] * 3 + [9] + [P] * 8, None),
                  lambda n: lib.cusort_page_compact(None, n, P, 4, 4, P, 3, 16, 1 << 20, *[P] * 6, None)):
        nb = C.c_size_t(0)
        assert query(C.byref(nb)) == 0 and nb.value > 0
        assert query(None) == INVALID


def test_copy_arguments():
    lib = _capi.load()

    def call(data=(0x10000,), strides=(64,), sizes=(64,), count=1, blocks=9, sources=P, destinations=P, n=3):
        return lib.cusort_page_copy((C.c_void_p * 1)(*data), (C.c_int64 * 1)(*strides), (C.c_size_t * 1)(*sizes), count,
                                    blocks, sources, destinations, n, None)
    for bad in (dict(data=(None,)), dict(strides=(63,)), dict(count=-1), dict(blocks=-1), dict(sources=None),
                dict(destinations=None), dict(n=-1), dict(n=1 << 31), dict(sizes=((1 << 40) + 1,), strides=(1 << 41,))):
        assert call(**bad) == INVALID, bad
    assert lib.cusort_page_copy(None, None, None, 1, 9, P, P, 3, None) == INVALID
    assert call(n=0) == 0 and call(blocks=1) == 0 and call(sizes=(0,), data=(None,)) == 0
    assert lib.cusort_page_copy(None, None, None, 0, 9, P, P, 3, None) == 0
