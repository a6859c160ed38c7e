"""Token routing over the C ABI (zero-copy on CUDA tensors): which experts a
token goes to, its rows grouped by expert, and back.

``route`` chooses the k best experts of every token and their weights;
``plan_dispatch`` groups the (token, expert) pairs by expert, stably;
``dispatch`` copies the tokens' rows into that order and ``combine`` adds the
experts' rows up again.  Each has its gradient as a function of its own
(``route_backward``, ``dispatch_backward``, ``combine_backward``);
``torch.ops.cusort.route / dispatch / combine`` (``libcusort_b200.ops``) tie
them to autograd; the functions here take tensors that require a gradient and
return ones that do not.

    weights, experts = route(logits, k, renormalize=True)
    plan = plan_dispatch(experts, num_experts)
    rows = dispatch(x, plan.sources, plan.positions)      # expert e: rows[offsets[e] : offsets[e] + counts[e]]
    y = ...                                               # the experts' products on their rows
    out = combine(y, weights, plan.positions, residual=x)

The work runs on torch's current stream and nothing synchronises it; row
counts stay on the device, so outputs have the size of the worst case.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _capi

MAX_EXPERTS = 1024
MAX_CHOSEN = 32
MAX_GROUPS = 32

_SCORES = {"softmax": 0, "sigmoid": 1}
_GROUP_SCORES = {"max": 0, "top2": 1}


class DispatchPlan(NamedTuple):
    """What ``plan_dispatch`` returns (int32 tensors on the experts' device)."""
    counts: torch.Tensor     # [num_experts] pairs of each expert
    offsets: torch.Tensor    # [num_experts + 1] first row of each expert's segment, and the end of the last
    sources: torch.Tensor    # [capacity] the pair (token * k + j) at each row, -1 where there is none
    positions: torch.Tensor  # as the experts: the row of each pair, -1 where it has none


def _choice(name: str, value: str, table: dict) -> int:
    try:
        return table[value]
    except (KeyError, TypeError):
        raise ValueError(f"{name} must be one of {', '.join(table)} (got {value!r})") from None


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
    return _capi.native().route(logits, k, bias, _choice("score", score, _SCORES), groups, groups_kept,
                                _choice("group_score", group_score, _GROUP_SCORES), renormalize, scale)


def route_backward(grad_weights: torch.Tensor, logits: torch.Tensor, experts: torch.Tensor, *,
                   bias: torch.Tensor | None = None, score: str = "softmax", renormalize: bool = False,
                   scale: float = 1.0) -> torch.Tensor:
    """Gradient of ``route``'s logits (their type, contiguous) from that of its weights
    (float32 [tokens, k]), with the experts it chose and the same arguments.  Where a caller repeats
    an expert in a token, its parts are added up in no fixed order."""
    return _capi.native().route_backward(grad_weights, logits, experts, bias, _choice("score", score, _SCORES),
                                         renormalize, scale)


def dispatch_capacity(num_pairs: int, num_experts: int, align: int = 1) -> int:
    """Rows that ``num_pairs`` pairs may need at most: every segment starts at a multiple of ``align``."""
    return num_pairs + min(num_experts, num_pairs) * (align - 1)


def plan_dispatch(experts: torch.Tensor, num_experts: int, *, align: int = 1,
                  separate: bool = False) -> DispatchPlan:
    """Groups (token, expert) pairs by expert, stably.  ``experts``: contiguous int32 or int64,
    [tokens, k] or of any shape; values outside [0, num_experts) (such as -1) are dropped.  Every
    expert's segment starts at a multiple of ``align`` rows; rows between hold no pair.  The plan's
    tensors are parts of one allocation, unless ``separate``."""
    return DispatchPlan._make(_capi.native().plan_dispatch(experts, num_experts, align, separate))


def dispatch(x: torch.Tensor, sources: torch.Tensor, positions: torch.Tensor) -> torch.Tensor:
    """rows[r] = x[sources[r] // k], zeros where sources[r] is -1: the tokens' rows ([tokens, hidden]
    of any type, rows any distance apart) in the order of a plan.  Its gradient is there for
    float32, float16 and bfloat16 rows."""
    return _capi.native().dispatch(x, sources, positions)


def dispatch_backward(grad_rows: torch.Tensor, positions: torch.Tensor) -> torch.Tensor:
    """Gradient of ``dispatch``'s x: every token's rows added up."""
    return _capi.native().combine(grad_rows, None, positions, None, "grad_rows")


def combine(rows: torch.Tensor, weights: torch.Tensor, positions: torch.Tensor, *,
            residual: torch.Tensor | None = None) -> torch.Tensor:
    """out[t] = residual[t] + sum over j of weights[t, j] * rows[positions[t, j]], in 32 bits and
    rounded once to the rows' type (float32, float16 or bfloat16).  ``rows``: contiguous [capacity,
    hidden]; weights float32; a position of -1 adds nothing."""
    if weights is None:
        raise ValueError("weights must be a float32 tensor of the positions' shape")
    return _capi.native().combine(rows, weights, positions, residual, "rows")


def combine_backward(grad_out: torch.Tensor, rows: torch.Tensor, weights: torch.Tensor, sources: torch.Tensor,
                     positions: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Gradients of ``combine``'s rows and weights from that of its result (which is the residual's
    gradient itself)."""
    return _capi.native().combine_backward(grad_out, rows, weights, sources, positions)
