"""The experts' matrix products over the C ABI (zero-copy on CUDA tensors):
what stands between ``routing.dispatch`` and ``routing.combine``.

``expert_products`` multiplies every row of a plan by its expert's weights;
``expert_products_grad_rows`` and ``expert_products_grad_weights`` (both:
``expert_products_backward``) are its gradients as functions of their own, and
``torch.ops.cusort.expert_products`` (``libcusort_b200.ops``) ties them to
autograd.

    plan = plan_dispatch(experts, num_experts)
    rows = dispatch(x, plan.sources, plan.positions)
    inner = torch.relu(expert_products(rows, up, plan.counts, plan.offsets))
    y = expert_products(inner, down, plan.counts, plan.offsets)
    out = combine(y, weights, plan.positions, residual=x)

The work runs on torch's current stream and nothing synchronises it; the
segments' sizes stay on the device.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _capi

MAX_WIDTH = 1 << 20


def expert_products(rows: torch.Tensor, weights: torch.Tensor, counts: torch.Tensor,
                    offsets: torch.Tensor) -> torch.Tensor:
    """out[r] = rows[r] @ weights[e] for the rows r of expert e's segment, ``offsets[e] <= r <
    offsets[e] + counts[e]`` (int32, as ``plan_dispatch`` gives them; the segments may come in any order, but
    must not overlap), zeros for all others.

    ``rows`` [capacity, in] (rows any distance apart) and ``weights`` [experts, in, out] (contiguous
    along either of the last two dimensions, so that linear layers' [experts, out, in] go in as
    ``w.transpose(1, 2)``) are bfloat16, float16 or float32; sums are held in 32 bits and rounded once.
    What lies in ``rows`` outside the segments has no influence, whatever it is.  16-bit rows or
    weights whose addresses and strides are no multiples of 16 bytes are copied to a workspace first;
    32-bit ones are multiplied as they are, without the tensor cores, which would round them."""
    return _capi.native().expert_products(rows, weights, counts, offsets, False, "rows")


def expert_products_grad_rows(grad_out: torch.Tensor, weights: torch.Tensor, counts: torch.Tensor,
                              offsets: torch.Tensor) -> torch.Tensor:
    """Gradient of ``expert_products``' rows: grad_out[r] @ weights[e] transposed, zeros outside the segments."""
    return _capi.native().expert_products(grad_out, weights, counts, offsets, True, "grad_out")


def expert_products_grad_weights(grad_out: torch.Tensor, rows: torch.Tensor, counts: torch.Tensor,
                                 offsets: torch.Tensor, *, in_contiguous: bool = False) -> torch.Tensor:
    """Gradient of ``expert_products``' weights [experts, in, out]: the sum of rows[r] transposed @
    grad_out[r] over each segment, zeros for experts without rows.  ``in_contiguous``: it lies as
    [experts, out, in] does, transposed."""
    return _capi.native().expert_products_grad_weights(grad_out, rows, counts, offsets, in_contiguous)


def expert_products_backward(grad_out: torch.Tensor, rows: torch.Tensor, weights: torch.Tensor, counts: torch.Tensor,
                             offsets: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Gradients of ``expert_products``' rows and weights (these in the weights' order) from that of its result."""
    return (expert_products_grad_rows(grad_out, weights, counts, offsets),
            expert_products_grad_weights(grad_out, rows, counts, offsets,
                                         in_contiguous=_capi.native().weights_in_contiguous(weights)))


def product_status(device: torch.device | int | None = None) -> int:
    """1 if a bounded wait inside one of these products ran out on the device since the last call, else 0.
    What such a wait has cost is NaN in the results; nothing else says so before this call, which
    synchronises the current stream.  The bound (``cusort_set_wait_limit_ns``, 2 s where nothing is set)
    is the calling host thread's, and autograd computes gradients in threads of its own."""
    status = C.c_uint32()
    with torch.cuda.device(device):
        _capi.check(_capi.load().cusort_read_product_status(
            C.byref(status), C.c_void_p(torch.cuda.current_stream().cuda_stream)), "cusort_read_product_status")
    return int(status.value)
