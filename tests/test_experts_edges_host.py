"""Operands of the experts' products that no kernel can load (no GPU): the C ABI refuses them before any CUDA call."""
from __future__ import annotations

import ctypes as C

import pytest

from libcusort_b200 import _capi

P, BIG = C.c_void_p(0x10000), 1 << 40  # never dereferenced
F32, F16, BF16 = 0, 1, 2


def _products(kind, rows=P, weights=P, temp=None):
    room = C.c_size_t(BIG)
    return _capi.load().cusort_expert_products(temp, C.byref(room), kind, rows, 64, weights, 64 * 72, 72, 1, P, P, P,
                                               10, 64, 72, 3, None)


def _gradient(kind, rows=P, grad=P, temp=None):
    room = C.c_size_t(BIG)
    return _capi.load().cusort_expert_products_grad_weights(temp, C.byref(room), kind, rows, 64, grad, 72, P, P, P, 0,
                                                            10, 64, 72, 3, None)


@pytest.mark.parametrize("call", [_products, _gradient])
@pytest.mark.parametrize("kind,size", [(F32, 4), (F16, 2), (BF16, 2)])
def test_operands_between_elements(call, kind, size):
    """An address that is no multiple of the element's size, in the call and in its size query."""
    for off in range(1, 8):
        at = C.c_void_p(0x10000 + off)
        # whole elements are asked for their workspace only: the call itself would go to the GPU
        expected = 0 if off % size == 0 else _capi.CUDA_ERROR_INVALID_VALUE
        assert call(kind, at) == expected and call(kind, P, at) == expected
        if expected:
            assert call(kind, at, temp=P) == expected and call(kind, P, at, temp=P) == expected
