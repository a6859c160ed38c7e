"""Refusals of the page operators at the edge of what they take (no GPU): meta tensors for the PyTorch functions, the C
ABI's argument checks, which come before any CUDA call."""
from __future__ import annotations

import ctypes as C

import pytest

torch = pytest.importorskip("torch")

from libcusort_b200 import _capi, paging  # noqa: E402

P = C.c_void_p(0x10000)  # never dereferenced: every call below is refused, or asks for a size
MOST = 1 << 30  # entries of a table; the kernels number them, and some more, in 32 bits


def _i(*shape):
    return torch.empty(*shape, dtype=torch.int32, device="meta")


@pytest.mark.parametrize("width,match", [(MOST + 1, "2\\^30"), (2 ** 31 - 1, "2\\^30"), (2 ** 31, "2\\^30"),
                                         (MOST, "CUDA")])
def test_width_of_tables(width, match):
    pool = dict(free_blocks=_i(9), num_free=_i(1), shares=_i(9))
    for call in (lambda t: paging.page_fork(t, _i(1), _i(2), 16, **pool),
                 lambda t: paging.page_free(t, _i(1), _i(1), 16, **pool),
                 lambda t: paging.page_compact(t, _i(1), 16, 9)):
        with pytest.raises(ValueError, match=match):
            call(_i(1, width))


def test_width_of_tables_from_c():
    lib, room = _capi.load(), C.c_size_t(0)
    calls = (lambda w: lib.cusort_page_fork(None, C.byref(room), P, w, w, P, 1, P, 2, 16, *[P] * 3, 9, *[P] * 8, None),
             lambda w: lib.cusort_page_free(None, C.byref(room), P, w, w, P, P, 1, 16, *[P] * 3, 9, *[P] * 3, None),
             lambda w: lib.cusort_page_compact(None, C.byref(room), P, w, w, P, 1, 16, 9, *[P] * 6, None))
    for call in calls:
        assert call(MOST) == 0
        for width in (MOST + 1, 2 ** 31 - 128, 2 ** 31 - 1):
            assert call(width) == _capi.CUDA_ERROR_INVALID_VALUE
