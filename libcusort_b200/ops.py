"""PyTorch operators over the C ABI: ``torch.ops.cusort.*``.

Importing this module registers, in the ``cusort`` namespace:

* ``sort_keys(Tensor keys, bool descending=False, int begin_bit=0, int end_bit=-1) -> Tensor``
* ``sort_pairs(Tensor keys, Tensor values, bool descending=False, int begin_bit=0, int end_bit=-1)
  -> (Tensor, Tensor)``
* ``argsort(Tensor keys, bool descending=False) -> Tensor`` (int64 indices)
* ``segmented_sort_keys(Tensor keys, Tensor begin_offsets, Tensor end_offsets, bool descending=False,
  int begin_bit=0, int end_bit=-1) -> Tensor``
* ``segmented_sort_pairs(Tensor keys, Tensor values, Tensor begin_offsets, Tensor end_offsets,
  bool descending=False, int begin_bit=0, int end_bit=-1) -> (Tensor, Tensor)``

* ``route(Tensor logits, int k, Tensor? bias=None, str score="softmax", int groups=1, int groups_kept=0,
  str group_score="max", bool renormalize=False, float scale=1.0) -> (Tensor weights, Tensor experts)``
  (``groups_kept=0``: all of them)
* ``plan_dispatch(Tensor experts, int num_experts, int align=1) -> (Tensor counts, Tensor offsets,
  Tensor sources, Tensor positions)``
* ``dispatch(Tensor x, Tensor sources, Tensor positions) -> Tensor``
* ``combine(Tensor rows, Tensor weights, Tensor sources, Tensor positions, Tensor? residual=None) -> Tensor``
* ``expert_products(Tensor rows, Tensor weights, Tensor counts, Tensor offsets) -> Tensor``
* ``page_plan(Tensor cached_lens, Tensor new_lens, Tensor(a!) block_tables, int block_size, int num_tokens,
  Tensor free_blocks, Tensor num_free) -> (Tensor slots, Tensor positions, Tensor starts, Tensor served,
  Tensor num_free)``
* ``page_fork(Tensor block_tables, Tensor lens, Tensor parents, int block_size, Tensor free_blocks, Tensor num_free,
  Tensor shares) -> (Tensor block_tables, Tensor lens, Tensor sources, Tensor destinations, Tensor served,
  Tensor shares, Tensor free_blocks, Tensor num_free)``
* ``page_free(Tensor block_tables, Tensor lens, Tensor keep_lens, int block_size, Tensor free_blocks, Tensor num_free,
  Tensor shares) -> (Tensor shares, Tensor free_blocks, Tensor num_free)``
* ``page_compact(Tensor block_tables, Tensor lens, int block_size, int num_blocks) -> (Tensor block_tables,
  Tensor sources, Tensor destinations, Tensor shares, Tensor free_blocks, Tensor num_free)``
* ``page_copy(Tensor(a!)[] caches, Tensor sources, Tensor destinations) -> ()``

``sort_pairs`` takes payload rows of any width (rows of 1, 2, 4, 8 or 16 bytes move with the keys,
others are gathered by the sorted permutation).  The segmented operators sort every segment
[begin_offsets[s], end_offsets[s]) (int64 offsets, non-overlapping) independently; positions
outside every segment keep their input.

The routing operators are those of ``libcusort_b200.routing`` (its docstrings have the details), with
gradients through autograd: ``route`` to the logits, ``dispatch`` to the rows (float32, float16 or bfloat16
ones), ``combine`` to the rows, the weights and the residual.  ``expert_products`` is that of
``libcusort_b200.experts``, with gradients to the rows and the weights.  ``page_plan`` (with a free list) and the
other page operators are those of ``libcusort_b200.paging``.

All of them are stable, allocate fresh outputs (the inputs are never written, except ``page_plan``'s block tables and
``page_copy``'s caches), run on torch's current CUDA stream through the C ABI (``cusort_sort_keys``, ``cusort_sort_pairs``, ``cusort_route`` and so on) and have
fake (meta) implementations, so they trace under ``torch.compile`` / ``torch.export`` as opaque
calls.  ``end_bit = -1`` means all key bits.  There is no CPU implementation: a CPU tensor raises.
Floating-point keys follow the radix (IEEE total) order of the reference: -0.0 sorts before +0.0
and NaNs by sign and payload, where ``torch.sort`` treats the zeros as equal.
"""
from __future__ import annotations

import torch

from . import experts as _experts, paging, routing
from .torch_sort import radix_sort, segmented_sort


def _end(keys: torch.Tensor, end_bit: int) -> int:
    return 8 * keys.element_size() if end_bit < 0 else end_bit


@torch.library.custom_op("cusort::sort_keys", mutates_args=())
def sort_keys(keys: torch.Tensor, descending: bool = False, begin_bit: int = 0, end_bit: int = -1) -> torch.Tensor:
    k, _ = radix_sort(keys, None, descending=descending, begin_bit=begin_bit, end_bit=_end(keys, end_bit))
    return k


@sort_keys.register_fake
def _(keys, descending=False, begin_bit=0, end_bit=-1):
    return torch.empty_like(keys)


@torch.library.custom_op("cusort::sort_pairs", mutates_args=())
def sort_pairs(keys: torch.Tensor, values: torch.Tensor, descending: bool = False, begin_bit: int = 0,
               end_bit: int = -1) -> tuple[torch.Tensor, torch.Tensor]:
    k, v = radix_sort(keys, values, descending=descending, begin_bit=begin_bit, end_bit=_end(keys, end_bit))
    return k, v


@sort_pairs.register_fake
def _(keys, values, descending=False, begin_bit=0, end_bit=-1):
    return torch.empty_like(keys), torch.empty_like(values)


@torch.library.custom_op("cusort::argsort", mutates_args=())
def argsort(keys: torch.Tensor, descending: bool = False) -> torch.Tensor:
    idx = torch.arange(keys.numel(), device=keys.device, dtype=torch.int64)
    _, perm = radix_sort(keys, idx, descending=descending)
    return perm


@argsort.register_fake
def _(keys, descending=False):
    return torch.empty(keys.shape, dtype=torch.int64, device=keys.device)


@torch.library.custom_op("cusort::segmented_sort_keys", mutates_args=())
def segmented_sort_keys(keys: torch.Tensor, begin_offsets: torch.Tensor, end_offsets: torch.Tensor,
                        descending: bool = False, begin_bit: int = 0, end_bit: int = -1) -> torch.Tensor:
    k, _ = segmented_sort(keys, begin_offsets, end_offsets, None, descending=descending, begin_bit=begin_bit,
                          end_bit=_end(keys, end_bit))
    return k


@segmented_sort_keys.register_fake
def _(keys, begin_offsets, end_offsets, descending=False, begin_bit=0, end_bit=-1):
    return torch.empty_like(keys)


@torch.library.custom_op("cusort::segmented_sort_pairs", mutates_args=())
def segmented_sort_pairs(keys: torch.Tensor, values: torch.Tensor, begin_offsets: torch.Tensor,
                         end_offsets: torch.Tensor, descending: bool = False, begin_bit: int = 0,
                         end_bit: int = -1) -> tuple[torch.Tensor, torch.Tensor]:
    k, v = segmented_sort(keys, begin_offsets, end_offsets, values, descending=descending, begin_bit=begin_bit,
                          end_bit=_end(keys, end_bit))
    return k, v


@segmented_sort_pairs.register_fake
def _(keys, values, begin_offsets, end_offsets, descending=False, begin_bit=0, end_bit=-1):
    return torch.empty_like(keys), torch.empty_like(values)


@torch.library.custom_op("cusort::route", mutates_args=())
def route(logits: torch.Tensor, k: int, bias: torch.Tensor | None = None, score: str = "softmax", groups: int = 1,
          groups_kept: int = 0, group_score: str = "max", renormalize: bool = False,
          scale: float = 1.0) -> tuple[torch.Tensor, torch.Tensor]:
    return routing.route(logits, k, bias=bias, score=score, groups=groups, groups_kept=groups_kept or groups,
                         group_score=group_score, renormalize=renormalize, scale=scale)


@route.register_fake
def _(logits, k, bias=None, score="softmax", groups=1, groups_kept=0, group_score="max", renormalize=False, scale=1.0):
    shape = (logits.shape[0], k)
    return logits.new_empty(shape, dtype=torch.float32), logits.new_empty(shape, dtype=torch.int32)


@torch.library.custom_op("cusort::route_backward", mutates_args=())
def route_backward(grad_weights: torch.Tensor, logits: torch.Tensor, experts: torch.Tensor,
                   bias: torch.Tensor | None = None, score: str = "softmax", renormalize: bool = False,
                   scale: float = 1.0) -> torch.Tensor:
    return routing.route_backward(grad_weights.contiguous(), logits, experts, bias=bias, score=score,
                                  renormalize=renormalize, scale=scale)


@route_backward.register_fake
def _(grad_weights, logits, experts, bias=None, score="softmax", renormalize=False, scale=1.0):
    return logits.new_empty(logits.shape)


def _route_setup(ctx, inputs, output):
    logits, _, bias, ctx.score, _, _, _, ctx.renormalize, ctx.scale = inputs
    ctx.mark_non_differentiable(output[1])
    ctx.save_for_backward(logits, bias, output[1])


def _route_grad(ctx, grad_weights, _):
    logits, bias, experts = ctx.saved_tensors
    grad = torch.ops.cusort.route_backward(grad_weights, logits, experts, bias, ctx.score, ctx.renormalize, ctx.scale)
    return (grad,) + (None,) * 8


route.register_autograd(_route_grad, setup_context=_route_setup)


@torch.library.custom_op("cusort::plan_dispatch", mutates_args=())
def plan_dispatch(experts: torch.Tensor, num_experts: int,
                  align: int = 1) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    return tuple(routing.plan_dispatch(experts, num_experts, align=align, separate=True))


@plan_dispatch.register_fake
def _(experts, num_experts, align=1):
    pairs = experts.numel()
    # min() of a traced size and a number would fix which is less
    rows = pairs + torch.sym_min(num_experts, pairs) * (align - 1)
    return tuple(experts.new_empty(s, dtype=torch.int32) for s in ((num_experts,), (num_experts + 1,), (rows,),
                                                                   experts.shape))


def _rowwise(t: torch.Tensor) -> torch.Tensor:
    """Gradients may come expanded or transposed; the kernels want rows that are contiguous in themselves."""
    return t if t.dim() == 2 and t.stride(1) == 1 else t.contiguous()


@torch.library.custom_op("cusort::dispatch", mutates_args=())
def dispatch(x: torch.Tensor, sources: torch.Tensor, positions: torch.Tensor) -> torch.Tensor:
    return routing.dispatch(x, sources, positions)


@dispatch.register_fake
def _(x, sources, positions):
    return x.new_empty((sources.shape[0], x.shape[1]))


@torch.library.custom_op("cusort::dispatch_backward", mutates_args=())
def dispatch_backward(grad_rows: torch.Tensor, positions: torch.Tensor) -> torch.Tensor:
    return routing.dispatch_backward(grad_rows.contiguous(), positions)


@dispatch_backward.register_fake
def _(grad_rows, positions):
    return grad_rows.new_empty((positions.shape[0], grad_rows.shape[1]))


def _dispatch_setup(ctx, inputs, output):
    ctx.save_for_backward(inputs[2])


def _dispatch_grad(ctx, grad_rows):
    return torch.ops.cusort.dispatch_backward(grad_rows, *ctx.saved_tensors), None, None


dispatch.register_autograd(_dispatch_grad, setup_context=_dispatch_setup)


@torch.library.custom_op("cusort::combine", mutates_args=())
def combine(rows: torch.Tensor, weights: torch.Tensor, sources: torch.Tensor, positions: torch.Tensor,
            residual: torch.Tensor | None = None) -> torch.Tensor:
    return routing.combine(rows, weights, positions, residual=residual)


@combine.register_fake
def _(rows, weights, sources, positions, residual=None):
    return rows.new_empty((positions.shape[0], rows.shape[1]))


@torch.library.custom_op("cusort::combine_backward", mutates_args=())
def combine_backward(grad_out: torch.Tensor, rows: torch.Tensor, weights: torch.Tensor, sources: torch.Tensor,
                     positions: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    return routing.combine_backward(_rowwise(grad_out), rows, weights, sources, positions)


@combine_backward.register_fake
def _(grad_out, rows, weights, sources, positions):
    return rows.new_empty(rows.shape), weights.new_empty(weights.shape)


def _combine_setup(ctx, inputs, output):
    ctx.save_for_backward(*inputs[:4])
    ctx.has_residual = inputs[4] is not None


def _combine_grad(ctx, grad_out):
    grad_rows, grad_weights = torch.ops.cusort.combine_backward(grad_out, *ctx.saved_tensors)
    return grad_rows, grad_weights, None, None, (grad_out if ctx.has_residual else None)


combine.register_autograd(_combine_grad, setup_context=_combine_setup)


@torch.library.custom_op("cusort::expert_products", mutates_args=())
def expert_products(rows: torch.Tensor, weights: torch.Tensor, counts: torch.Tensor,
                    offsets: torch.Tensor) -> torch.Tensor:
    return _experts.expert_products(rows, weights, counts, offsets)


@expert_products.register_fake
def _(rows, weights, counts, offsets):
    return rows.new_empty((rows.shape[0], weights.shape[2]))


@torch.library.custom_op("cusort::expert_products_grad_rows", mutates_args=())
def expert_products_grad_rows(grad_out: torch.Tensor, weights: torch.Tensor, counts: torch.Tensor,
                              offsets: torch.Tensor) -> torch.Tensor:
    return _experts.expert_products_grad_rows(_rowwise(grad_out), weights, counts, offsets)


@expert_products_grad_rows.register_fake
def _(grad_out, weights, counts, offsets):
    return grad_out.new_empty((grad_out.shape[0], weights.shape[1]))


@torch.library.custom_op("cusort::expert_products_grad_weights", mutates_args=())
def expert_products_grad_weights(grad_out: torch.Tensor, rows: torch.Tensor, counts: torch.Tensor,
                                 offsets: torch.Tensor, in_contiguous: bool = False) -> torch.Tensor:
    return _experts.expert_products_grad_weights(_rowwise(grad_out), rows, counts, offsets, in_contiguous=in_contiguous)


@expert_products_grad_weights.register_fake
def _(grad_out, rows, counts, offsets, in_contiguous=False):
    shape = counts.shape[0], rows.shape[1], grad_out.shape[1]
    return rows.new_empty((shape[0], shape[2], shape[1])).transpose(1, 2) if in_contiguous else rows.new_empty(shape)


def _products_setup(ctx, inputs, output):
    ctx.save_for_backward(*inputs)


def _products_grad(ctx, grad_out):
    rows, weights, counts, offsets = ctx.saved_tensors
    grad_rows = grad_weights = None
    if ctx.needs_input_grad[0]:
        grad_rows = torch.ops.cusort.expert_products_grad_rows(grad_out, weights, counts, offsets)
    if ctx.needs_input_grad[1]:
        # in the weights' order: their contiguous dimension is that of the gradient
        in_contiguous = weights.stride(2) != 1 and weights.shape[2] != 1
        grad_weights = torch.ops.cusort.expert_products_grad_weights(grad_out, rows, counts, offsets, in_contiguous)
    return grad_rows, grad_weights, None, None


expert_products.register_autograd(_products_grad, setup_context=_products_setup)


@torch.library.custom_op("cusort::page_plan", mutates_args=("block_tables",))
def page_plan(cached_lens: torch.Tensor, new_lens: torch.Tensor, block_tables: torch.Tensor, block_size: int,
              num_tokens: int, free_blocks: torch.Tensor, num_free: torch.Tensor
              ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    return tuple(paging.page_plan(cached_lens, new_lens, block_tables, block_size, num_tokens,
                                  free_blocks=free_blocks, num_free=num_free, separate=True))


@page_plan.register_fake
def _(cached_lens, new_lens, block_tables, block_size, num_tokens, free_blocks, num_free):
    requests = cached_lens.shape[0]
    new = cached_lens.new_empty
    return (new(num_tokens, dtype=torch.int64), new(num_tokens), new(requests + 1), new(requests, dtype=torch.bool),
            new(1))


@torch.library.custom_op("cusort::page_fork", mutates_args=())
def page_fork(block_tables: torch.Tensor, lens: torch.Tensor, parents: torch.Tensor, block_size: int,
              free_blocks: torch.Tensor, num_free: torch.Tensor, shares: torch.Tensor
              ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor,
                         torch.Tensor, torch.Tensor]:
    return tuple(paging.page_fork(block_tables, lens, parents, block_size, free_blocks=free_blocks, num_free=num_free,
                                  shares=shares, separate=True))


@page_fork.register_fake
def _(block_tables, lens, parents, block_size, free_blocks, num_free, shares):
    new, children, blocks = lens.new_empty, parents.shape[0], shares.shape[0]
    return (new((children, block_tables.shape[1])), new(children), new(children), new(children),
            new(children, dtype=torch.bool), new(blocks), new(blocks), new(1))


@torch.library.custom_op("cusort::page_free", mutates_args=())
def page_free(block_tables: torch.Tensor, lens: torch.Tensor, keep_lens: torch.Tensor, block_size: int,
              free_blocks: torch.Tensor, num_free: torch.Tensor, shares: torch.Tensor
              ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    return tuple(paging.page_free(block_tables, lens, keep_lens, block_size, free_blocks=free_blocks,
                                  num_free=num_free, shares=shares, separate=True))


@page_free.register_fake
def _(block_tables, lens, keep_lens, block_size, free_blocks, num_free, shares):
    blocks = shares.shape[0]
    return lens.new_empty(blocks), lens.new_empty(blocks), lens.new_empty(1)


@torch.library.custom_op("cusort::page_compact", mutates_args=())
def page_compact(block_tables: torch.Tensor, lens: torch.Tensor, block_size: int, num_blocks: int
                 ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    return tuple(paging.page_compact(block_tables, lens, block_size, num_blocks, separate=True))


@page_compact.register_fake
def _(block_tables, lens, block_size, num_blocks):
    new, half = lens.new_empty, num_blocks // 2
    return new(block_tables.shape), new(half), new(half), new(num_blocks), new(num_blocks), new(1)


@torch.library.custom_op("cusort::page_copy", mutates_args=("caches",))
def page_copy(caches: list[torch.Tensor], sources: torch.Tensor, destinations: torch.Tensor) -> None:
    paging.page_copy(list(caches), sources, destinations)


@page_copy.register_fake
def _(caches, sources, destinations):
    return None
