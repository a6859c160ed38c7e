"""Placement of a serving step in a paged cache, over the C ABI.

``page_plan`` takes the requests' lengths and gives, in one launch and without
a host copy, the blocks that the step's new tokens need (from a free list on
the device, into the requests' block tables) and a cache slot and position for
every new token.  It runs on torch's current stream.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _capi

MAX_REQUESTS = 16384


class PagePlan(NamedTuple):
    """What ``page_plan`` returns."""
    slots: torch.Tensor            # int64 [num_tokens]: block * block_size + position % block_size, -1 for none
    positions: torch.Tensor        # int32 [num_tokens]: position in the request, -1 beyond the last token
    starts: torch.Tensor           # int32 [requests + 1]: the first new token of each request, and their number
    served: torch.Tensor           # bool [requests]: whether the request got its blocks
    num_free: torch.Tensor | None  # int32 [1]: free blocks that are left (None without a free list)


def page_plan(cached_lens: torch.Tensor, new_lens: torch.Tensor, block_tables: torch.Tensor, block_size: int,
              num_tokens: int, *, free_blocks: torch.Tensor | None = None,
              num_free: torch.Tensor | None = None, separate: bool = False) -> PagePlan:
    """Request r has ``cached_lens[r]`` tokens in the cache and brings ``new_lens[r]``; row r of
    ``block_tables`` (int32 [requests, width], written in place) names its blocks of ``block_size``
    tokens.  New blocks come from the end of ``free_blocks[:num_free]`` in the requests' order; a
    request that does not get all of its blocks, or whose table is too narrow, is not served: its
    slots are -1 and its table stays.  ``free_blocks`` and ``num_free`` are only read, so a step can
    be planned again; its caller goes on with the returned ``num_free``.  Without a free list the
    tables hold all blocks already.  ``num_tokens``: the length of the slot map, which may be more
    or less than there are new tokens; blocks that begin beyond it are written one after the other,
    so a map that leaves out most of a long prompt makes the call slow.  The plan's tensors are parts of one allocation, unless
    ``separate``."""
    return PagePlan._make(_capi.native().page_plan(cached_lens, new_lens, block_tables, block_size, num_tokens,
                                                   free_blocks, num_free, separate))
