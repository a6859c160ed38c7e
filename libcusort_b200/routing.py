"""Token routing over the C ABI (zero-copy on CUDA tensors): which experts a
token goes to, its rows grouped by expert, and back.

``route`` chooses the k best experts of every token and their weights;
``plan_dispatch`` groups the (token, expert) pairs by expert, stably;
``dispatch`` copies the tokens' rows into that order and ``combine`` adds the
experts' rows up again.  Each has its gradient as a function of its own
(``route_backward``, ``dispatch_backward``, ``combine_backward``);
``torch.ops.cusort.route / dispatch / combine`` (``libcusort_b200.ops``) tie
them to autograd.

    weights, experts = route(logits, k, renormalize=True)
    plan = plan_dispatch(experts, num_experts)
    rows = dispatch(x, plan.sources, plan.positions)      # expert e: rows[offsets[e] : offsets[e] + counts[e]]
    y = ...                                               # the experts' products on their rows
    out = combine(y, weights, plan.positions, residual=x)

The work runs on torch's current stream and nothing synchronises it; row
counts stay on the device, so outputs have the size of the worst case.
"""
from __future__ import annotations

import ctypes as C
from typing import NamedTuple

import torch

from . import _capi

MAX_EXPERTS = 1024
MAX_CHOSEN = 32
MAX_GROUPS = 32

_FLOATS = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_SCORES = {"softmax": 0, "sigmoid": 1}
_GROUP_SCORES = {"max": 0, "top2": 1}


class DispatchPlan(NamedTuple):
    """What ``plan_dispatch`` returns (int32 tensors on the experts' device)."""
    counts: torch.Tensor     # [num_experts] pairs of each expert
    offsets: torch.Tensor    # [num_experts + 1] first row of each expert's segment, and the end of the last
    sources: torch.Tensor    # [capacity] the pair (token * k + j) at each row, -1 where there is none
    positions: torch.Tensor  # as the experts: the row of each pair, -1 where it has none


def _float_type(name: str, t: torch.Tensor) -> int:
    try:
        return _FLOATS[t.dtype]
    except KeyError:
        raise TypeError(f"{name} must be float32, float16 or bfloat16 (got {t.dtype})") from None


def _check_rows(name: str, t: torch.Tensor) -> None:
    """A matrix whose rows may lie any distance apart, each contiguous in itself."""
    if t.dim() != 2 or (t.shape[1] > 1 and t.stride(1) != 1 and t.numel()):
        raise ValueError(f"{name} must be a 2-D tensor whose rows are contiguous "
                         f"(got shape {tuple(t.shape)}, strides {t.stride()})")


def _check(name: str, t: torch.Tensor, dtype: torch.dtype, device: torch.device, shape: tuple) -> None:
    if t.dtype != dtype or t.device != device or t.shape != shape or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dtype} tensor of shape {tuple(shape)} on {device} "
                         f"(got {t.dtype}, {tuple(t.shape)}, {t.device})")


def _check_cuda(name: str, t: torch.Tensor) -> None:
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor (this path has no CPU implementation)")


def _stream(device: torch.device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


def _call(what: str, device: torch.device, *args) -> None:
    """Calls the C entry point with the device current and its current stream last."""
    fn = getattr(_capi.load(), what)
    if device.index == torch.cuda.current_device():
        rc = fn(*args, _stream(device))
    else:
        with torch.cuda.device(device):
            rc = fn(*args, _stream(device))
    _capi.check(rc, what)


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def _choice(name: str, value: str, table: dict) -> int:
    try:
        return table[value]
    except KeyError:
        raise ValueError(f"{name} must be one of {', '.join(table)} (got {value!r})") from None


def _check_route(logits: torch.Tensor, k: int, bias: torch.Tensor | None, score: str) -> tuple[int, int]:
    """Checks what route and route_backward share; the type and score codes.  No CUDA call."""
    kind = _float_type("logits", logits)
    _check_rows("logits", logits)
    experts = logits.shape[1]
    if not 1 <= experts <= MAX_EXPERTS:
        raise ValueError(f"1 to {MAX_EXPERTS} experts are supported (got {experts})")
    if not 1 <= k <= min(MAX_CHOSEN, experts):
        raise ValueError(f"k must be between 1 and {min(MAX_CHOSEN, experts)} (got {k})")
    if bias is not None:
        _check("bias", bias, torch.float32, logits.device, (experts,))
    return kind, _choice("score", score, _SCORES)


def _check_groups(experts: int, k: int, groups: int, groups_kept: int) -> None:
    if not 1 <= groups <= MAX_GROUPS or experts % groups:
        raise ValueError(f"groups must divide the {experts} experts and be at most {MAX_GROUPS} (got {groups})")
    if not 1 <= groups_kept <= groups or k > groups_kept * (experts // groups):
        raise ValueError(f"groups_kept must be between 1 and groups={groups} and leave at least k={k} experts "
                         f"(got {groups_kept})")


def route(logits: torch.Tensor, k: int, *, bias: torch.Tensor | None = None, score: str = "softmax", groups: int = 1,
          groups_kept: int | None = None, group_score: str = "max", renormalize: bool = False,
          scale: float = 1.0) -> tuple[torch.Tensor, torch.Tensor]:
    """The k best experts of every row of ``logits`` [tokens, experts] (float32, float16 or
    bfloat16; rows any distance apart).  Returns (weights float32 [tokens, k], experts int32
    [tokens, k]), best first.

    The score is the ``"softmax"`` over the row or the ``"sigmoid"``; ``bias`` (float32 [experts])
    is added to it for the choice alone.  Of ``groups`` equal contiguous groups the best
    ``groups_kept`` stay, by their best expert (``group_score="max"``) or the sum of their two best
    (``"top2"``).  ``renormalize`` divides the weights by their sum; ``scale`` multiplies them.
    Equal experts go to the lower index.  A logit or bias of -inf or NaN takes its expert out; where
    fewer than k are left, expert -1 and weight 0 fill up."""
    kind, score_id = _check_route(logits, k, bias, score)
    tokens, experts = logits.shape
    groups_kept = groups if groups_kept is None else groups_kept
    _check_groups(experts, k, groups, groups_kept)
    group_id = _choice("group_score", group_score, _GROUP_SCORES)
    _check_cuda("logits", logits)
    weights = torch.empty((tokens, k), dtype=torch.float32, device=logits.device)
    chosen = torch.empty((tokens, k), dtype=torch.int32, device=logits.device)
    _call("cusort_route", logits.device, kind, logits.data_ptr(), logits.stride(0), _ptr(bias), weights.data_ptr(),
          chosen.data_ptr(), tokens, experts, k, groups, groups_kept, score_id, group_id, int(renormalize), scale)
    return weights, chosen


def route_backward(grad_weights: torch.Tensor, logits: torch.Tensor, experts: torch.Tensor, *,
                   bias: torch.Tensor | None = None, score: str = "softmax", renormalize: bool = False,
                   scale: float = 1.0) -> torch.Tensor:
    """Gradient of ``route``'s logits (their type, contiguous) from that of its weights
    (float32 [tokens, k]), with the experts it chose and the same arguments."""
    if experts.dim() != 2:
        raise ValueError(f"experts must be [tokens, k] (got shape {tuple(experts.shape)})")
    k = experts.shape[1]
    kind, score_id = _check_route(logits, k, bias, score)
    tokens, num = logits.shape
    _check("experts", experts, torch.int32, logits.device, (tokens, k))
    _check("grad_weights", grad_weights, torch.float32, logits.device, (tokens, k))
    _check_cuda("logits", logits)
    grad = torch.empty((tokens, num), dtype=logits.dtype, device=logits.device)
    _call("cusort_route_backward", logits.device, kind, grad_weights.data_ptr(), logits.data_ptr(), logits.stride(0),
          _ptr(bias), experts.data_ptr(), grad.data_ptr(), tokens, num, k, score_id, int(renormalize), scale)
    return grad


def dispatch_capacity(num_pairs: int, num_experts: int, align: int = 1) -> int:
    """Rows that ``num_pairs`` pairs may need at most: every segment starts at a multiple of ``align``."""
    return num_pairs + min(num_experts, num_pairs) * (align - 1)


def plan_dispatch(experts: torch.Tensor, num_experts: int, *, align: int = 1) -> DispatchPlan:
    """Groups (token, expert) pairs by expert, stably.  ``experts``: contiguous int32 or int64,
    [tokens, k] or of any shape; values outside [0, num_experts) (such as -1) are dropped.  Every
    expert's segment starts at a multiple of ``align`` rows; rows between hold no pair."""
    if experts.dtype not in (torch.int32, torch.int64) or not experts.is_contiguous():
        raise ValueError(f"experts must be a contiguous int32 or int64 tensor (got {experts.dtype}, strides "
                         f"{experts.stride()})")
    if not 1 <= num_experts <= MAX_EXPERTS:
        raise ValueError(f"1 to {MAX_EXPERTS} experts are supported (got {num_experts})")
    if not 1 <= align <= 1 << 20:
        raise ValueError(f"align must be between 1 and 2^20 (got {align})")
    pairs = experts.numel()
    capacity = dispatch_capacity(pairs, num_experts, align)
    if capacity >= 1 << 31:
        raise ValueError(f"{pairs} pairs over {num_experts} segments aligned to {align} rows need more than 2^31 rows")
    _check_cuda("experts", experts)
    device, size = experts.device, experts.element_size()
    nbytes = C.c_size_t(0)
    _capi.check(_capi.load().cusort_plan_dispatch(None, C.byref(nbytes), size, None, pairs, num_experts, align,
                                                  capacity, None, None, None, None, None), "plan size query")
    temp = torch.empty(nbytes.value, dtype=torch.uint8, device=device)
    counts = torch.empty(num_experts, dtype=torch.int32, device=device)
    offsets = torch.empty(num_experts + 1, dtype=torch.int32, device=device)
    sources = torch.empty(capacity, dtype=torch.int32, device=device)
    positions = torch.empty(experts.shape, dtype=torch.int32, device=device)
    _call("cusort_plan_dispatch", device, temp.data_ptr(), C.byref(nbytes), size, experts.data_ptr(), pairs,
          num_experts, align, capacity, counts.data_ptr(), offsets.data_ptr(), sources.data_ptr(),
          positions.data_ptr())
    return DispatchPlan(counts, offsets, sources, positions)


def _check_plan(positions: torch.Tensor, sources: torch.Tensor | None, device: torch.device) -> tuple[int, int]:
    """Shape checks of a plan's tensors; (tokens, k).  No CUDA call."""
    if positions.dim() != 2:
        raise ValueError(f"positions must be [tokens, k] (got shape {tuple(positions.shape)})")
    tokens, k = positions.shape
    if not 1 <= k <= MAX_CHOSEN:
        raise ValueError(f"k must be between 1 and {MAX_CHOSEN} (got {k})")
    _check("positions", positions, torch.int32, device, (tokens, k))
    if sources is not None:
        _check("sources", sources, torch.int32, device, (sources.numel(),))
    return tokens, k


def dispatch(x: torch.Tensor, sources: torch.Tensor, positions: torch.Tensor) -> torch.Tensor:
    """rows[r] = x[sources[r] // k], zeros where sources[r] is -1: the tokens' rows ([tokens, hidden]
    of any type, rows any distance apart) in the order of a plan."""
    _check_rows("x", x)
    tokens, k = _check_plan(positions, sources, x.device)
    if x.shape[0] != tokens:
        raise ValueError(f"x has {x.shape[0]} rows, positions {tokens}")
    _check_cuda("x", x)
    rows = torch.empty((sources.numel(), x.shape[1]), dtype=x.dtype, device=x.device)
    size = x.element_size()
    _call("cusort_dispatch_rows", x.device, x.data_ptr(), x.stride(0) * size, x.shape[1] * size, sources.data_ptr(),
          positions.data_ptr(), rows.data_ptr(), tokens, k, sources.numel())
    return rows


def dispatch_backward(grad_rows: torch.Tensor, positions: torch.Tensor) -> torch.Tensor:
    """Gradient of ``dispatch``'s x: every token's rows added up."""
    return _combine(grad_rows, None, positions, None, "grad_rows")


def combine(rows: torch.Tensor, weights: torch.Tensor, positions: torch.Tensor, *,
            residual: torch.Tensor | None = None) -> torch.Tensor:
    """out[t] = residual[t] + sum over j of weights[t, j] * rows[positions[t, j]], in 32 bits and
    rounded once to the rows' type (float32, float16 or bfloat16).  ``rows``: contiguous [capacity,
    hidden]; weights float32; a position of -1 adds nothing."""
    if weights is None:
        raise ValueError("weights must be a float32 tensor of the positions' shape")
    return _combine(rows, weights, positions, residual, "rows")


def _combine(rows, weights, positions, residual, name) -> torch.Tensor:
    kind = _float_type(name, rows)
    if rows.dim() != 2 or not rows.is_contiguous():
        raise ValueError(f"{name} must be a contiguous 2-D tensor (got shape {tuple(rows.shape)})")
    tokens, k = _check_plan(positions, None, rows.device)
    capacity, hidden = rows.shape
    if weights is not None:
        _check("weights", weights, torch.float32, rows.device, (tokens, k))
    if residual is not None:
        _check_rows("residual", residual)
        if residual.dtype != rows.dtype or residual.device != rows.device or residual.shape != (tokens, hidden):
            raise ValueError(f"residual must be {rows.dtype} of shape {(tokens, hidden)} on {rows.device} "
                             f"(got {residual.dtype}, {tuple(residual.shape)}, {residual.device})")
    _check_cuda(name, rows)
    out = torch.empty((tokens, hidden), dtype=rows.dtype, device=rows.device)
    _call("cusort_combine_rows", rows.device, kind, rows.data_ptr(), _ptr(weights), positions.data_ptr(),
          _ptr(residual), 0 if residual is None else residual.stride(0), out.data_ptr(), tokens, k, capacity, hidden)
    return out


def combine_backward(grad_out: torch.Tensor, rows: torch.Tensor, weights: torch.Tensor, sources: torch.Tensor,
                     positions: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Gradients of ``combine``'s rows and weights from that of its result (which is the residual's
    gradient itself)."""
    kind = _float_type("rows", rows)
    if rows.dim() != 2 or not rows.is_contiguous():
        raise ValueError(f"rows must be a contiguous 2-D tensor (got shape {tuple(rows.shape)})")
    capacity, hidden = rows.shape
    tokens, k = _check_plan(positions, sources, rows.device)
    if sources.numel() != capacity:
        raise ValueError(f"rows has {capacity} rows, sources {sources.numel()}")
    _check("weights", weights, torch.float32, rows.device, (tokens, k))
    _check_rows("grad_out", grad_out)
    if grad_out.dtype != rows.dtype or grad_out.device != rows.device or grad_out.shape != (tokens, hidden):
        raise ValueError(f"grad_out must be {rows.dtype} of shape {(tokens, hidden)} on {rows.device} "
                         f"(got {grad_out.dtype}, {tuple(grad_out.shape)}, {grad_out.device})")
    _check_cuda("rows", rows)
    grad_rows = torch.empty_like(rows)
    grad_weights = torch.empty((tokens, k), dtype=torch.float32, device=rows.device)
    _call("cusort_combine_rows_backward", rows.device, kind, grad_out.data_ptr(), grad_out.stride(0), rows.data_ptr(),
          weights.data_ptr(), sources.data_ptr(), positions.data_ptr(), grad_rows.data_ptr(),
          grad_weights.data_ptr(), tokens, k, capacity, hidden)
    return grad_rows, grad_weights
