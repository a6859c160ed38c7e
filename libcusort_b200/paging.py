"""Placement of a serving step in a paged cache, over the C ABI.

``page_plan`` takes the requests' lengths and gives, in one launch and without
a host copy, the blocks that the step's new tokens need (from a free list on
the device, into the requests' block tables) and a cache slot and position for
every new token.  It runs on torch's current stream.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from .routing import _call, _check, _check_cuda, _check_rows, _ptr

MAX_REQUESTS = 16384


class PagePlan(NamedTuple):
    """What ``page_plan`` returns."""
    slots: torch.Tensor            # int64 [num_tokens]: block * block_size + position % block_size, -1 for none
    positions: torch.Tensor        # int32 [num_tokens]: position in the request, -1 beyond the last token
    starts: torch.Tensor           # int32 [requests + 1]: the first new token of each request, and their number
    served: torch.Tensor           # bool [requests]: whether the request got its blocks
    num_free: torch.Tensor | None  # int32 [1]: free blocks that are left (None without a free list)


def _check_page(cached_lens, new_lens, block_tables, block_size, num_tokens, free_blocks, num_free) -> int:
    """Argument checks of page_plan; the number of requests.  No CUDA call."""
    device = cached_lens.device
    if cached_lens.dim() != 1 or cached_lens.numel() > MAX_REQUESTS:
        raise ValueError(f"cached_lens must be 1-D with at most {MAX_REQUESTS} requests "
                         f"(got shape {tuple(cached_lens.shape)})")
    requests = cached_lens.numel()
    _check("cached_lens", cached_lens, torch.int32, device, (requests,))
    _check("new_lens", new_lens, torch.int32, device, (requests,))
    _check_rows("block_tables", block_tables)
    if block_tables.dtype != torch.int32 or block_tables.device != device or block_tables.shape[0] != requests:
        raise ValueError(f"block_tables must be int32 with {requests} rows on {device} (got {block_tables.dtype}, "
                         f"{tuple(block_tables.shape)}, {block_tables.device})")
    if requests > 1 and block_tables.numel() and block_tables.stride(0) < block_tables.shape[1]:
        raise ValueError(f"block_tables' rows must not overlap (strides {block_tables.stride()})")
    if not 1 <= block_size <= 1 << 20:
        raise ValueError(f"block_size must be between 1 and 2^20 (got {block_size})")
    if not 0 <= num_tokens < 1 << 31:
        raise ValueError(f"num_tokens must be between 0 and 2^31 - 1 (got {num_tokens})")
    if (free_blocks is None) != (num_free is None):
        raise ValueError("free_blocks and num_free go together")
    if free_blocks is not None:
        if free_blocks.dim() != 1 or free_blocks.numel() > 1 << 30:
            raise ValueError(f"free_blocks must be 1-D with at most 2^30 blocks (got shape {tuple(free_blocks.shape)})")
        _check("free_blocks", free_blocks, torch.int32, device, (free_blocks.numel(),))
        _check("num_free", num_free, torch.int32, device, (1,))
    return requests


def page_plan(cached_lens: torch.Tensor, new_lens: torch.Tensor, block_tables: torch.Tensor, block_size: int,
              num_tokens: int, *, free_blocks: torch.Tensor | None = None,
              num_free: torch.Tensor | None = None) -> PagePlan:
    """Request r has ``cached_lens[r]`` tokens in the cache and brings ``new_lens[r]``; row r of
    ``block_tables`` (int32 [requests, width], written in place) names its blocks of ``block_size``
    tokens.  New blocks come from the end of ``free_blocks[:num_free]`` in the requests' order; a
    request that does not get all of its blocks, or whose table is too narrow, is not served: its
    slots are -1 and its table stays.  ``free_blocks`` and ``num_free`` are only read, so a step can
    be planned again; its caller goes on with the returned ``num_free``.  Without a free list the
    tables hold all blocks already.  ``num_tokens``: the length of the slot map, which may be more
    or less than there are new tokens."""
    requests = _check_page(cached_lens, new_lens, block_tables, block_size, num_tokens, free_blocks, num_free)
    _check_cuda("cached_lens", cached_lens)
    device, width = cached_lens.device, block_tables.shape[1]
    slots = torch.empty(num_tokens, dtype=torch.int64, device=device)
    positions = torch.empty(num_tokens, dtype=torch.int32, device=device)
    starts = torch.empty(requests + 1, dtype=torch.int32, device=device)
    served = torch.empty(requests, dtype=torch.bool, device=device)
    left = None if num_free is None else torch.empty(1, dtype=torch.int32, device=device)
    _call("cusort_page_plan", device, cached_lens.data_ptr(), new_lens.data_ptr(), requests, block_size,
          block_tables.data_ptr(), max(block_tables.stride(0), width), width, _ptr(free_blocks),
          0 if free_blocks is None else free_blocks.numel(), _ptr(num_free), num_tokens, slots.data_ptr(),
          positions.data_ptr(), starts.data_ptr(), served.data_ptr(), _ptr(left))
    return PagePlan(slots, positions, starts, served, left)
