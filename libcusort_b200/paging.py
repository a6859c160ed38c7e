"""Blocks of a paged cache, over the C ABI: where a serving step's tokens go, and what becomes of the blocks.

``page_plan`` takes the requests' lengths and gives, in one launch and without
a host copy, the blocks that the step's new tokens need (from a free list on
the device, into the requests' block tables) and a cache slot and position for
every new token.

``page_fork`` lets requests go on from others' (parallel samples, beams) with
their whole blocks shared, ``page_free`` gives blocks back, ``page_compact``
moves the used ones together and ``page_copy`` copies blocks as they say:

    shares = torch.zeros(num_blocks, dtype=torch.int32, device="cuda")   # tables beyond the first, of each block
    fork = page_fork(tables, lens, parents, block_size, free_blocks=free, num_free=left, shares=shares)
    page_copy(caches, fork.sources, fork.destinations)
    tables, lens, shares, free, left = fork.block_tables, fork.lens, fork.shares, fork.free_blocks, fork.num_free

A request holds the first ceil(len / block_size) blocks of its table.  All of
it runs on torch's current stream, without a host copy.  Except for
``page_plan``'s tables and ``page_copy``'s caches nothing is written in place:
a step can be planned again, and its caller goes on with the results.
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
    so a map that leaves out most of a long prompt makes the call slow.  The plan's tensors are parts
    of one allocation, unless ``separate``."""
    return PagePlan._make(_capi.native().page_plan(cached_lens, new_lens, block_tables, block_size, num_tokens,
                                                   free_blocks, num_free, separate))


class PageFork(NamedTuple):
    """What ``page_fork`` returns (int32 unless said otherwise)."""
    block_tables: torch.Tensor  # [children, width], -1 behind what is held
    lens: torch.Tensor          # [children]: the parent's, 0 for none
    sources: torch.Tensor       # [children]: the block to be copied for the child, -1 for none
    destinations: torch.Tensor  # [children]: where to, -1 for none
    served: torch.Tensor        # bool [children]: whether it got the block that it needed
    shares: torch.Tensor        # [num_blocks]
    free_blocks: torch.Tensor   # [num_blocks], -1 behind the free ones
    num_free: torch.Tensor      # [1]


class PageFree(NamedTuple):
    """What ``page_free`` returns (int32)."""
    shares: torch.Tensor       # [num_blocks]
    free_blocks: torch.Tensor  # [num_blocks], -1 behind the free ones
    num_free: torch.Tensor     # [1]


class PageCompact(NamedTuple):
    """What ``page_compact`` returns (int32)."""
    block_tables: torch.Tensor  # [requests, width], -1 behind what is held
    sources: torch.Tensor       # [num_blocks // 2]: the blocks that move, ascending, -1 behind the last
    destinations: torch.Tensor  # [num_blocks // 2]: where to, ascending
    shares: torch.Tensor        # [num_blocks]
    free_blocks: torch.Tensor   # [num_blocks]: the highest first, -1 behind the free ones
    num_free: torch.Tensor      # [1]


def page_fork(block_tables: torch.Tensor, lens: torch.Tensor, parents: torch.Tensor, block_size: int, *,
              free_blocks: torch.Tensor, num_free: torch.Tensor, shares: torch.Tensor,
              separate: bool = False) -> PageFork:
    """Child r goes on from request ``parents[r]`` (int32; outside [0, requests) it is empty), with its
    length.  All requests' tables are given up for the children's: a request that is not among the
    parents is over, ``parents = arange(requests)`` changes nothing but shared last blocks.

    Whole blocks are shared.  A part-filled last block goes to the request's first child if no other
    table holds it; every other child gets one from the end of ``free_blocks[:num_free]`` and a pair
    of ``sources`` and ``destinations`` for ``page_copy``.  A child for which there is none is not
    served, and empty.  ``shares`` (int32 [num_blocks]) is the number of tables that hold each
    block beyond the first, zeros at the start.  Blocks that no table holds any more join the free
    list, ascending; the copy may read from one of them, so it comes before the next step's writes.
    ``free_blocks`` is as long as ``shares``; tables are at most 2^30 blocks wide.  The results are
    parts of one allocation, unless ``separate``."""
    return PageFork._make(_capi.native().page_fork(block_tables, lens, parents, block_size, free_blocks, num_free,
                                                   shares, separate))


def page_free(block_tables: torch.Tensor, lens: torch.Tensor, keep_lens: torch.Tensor, block_size: int, *,
              free_blocks: torch.Tensor, num_free: torch.Tensor, shares: torch.Tensor,
              separate: bool = False) -> PageFree:
    """Request r keeps the first ``keep_lens[r]`` of its ``lens[r]`` tokens (0: it is done) and gives
    up the blocks behind; those that no table holds any more join the free list, ascending.  The
    tables are only read: go on with ``keep_lens`` as the lengths.  Where a request keeps part of a
    block that others hold too, ``page_fork`` (each its own parent) gives it its own before it writes
    there.  The rest as in ``page_fork``."""
    return PageFree._make(_capi.native().page_free(block_tables, lens, keep_lens, block_size, free_blocks, num_free,
                                                   shares, separate))


def page_compact(block_tables: torch.Tensor, lens: torch.Tensor, block_size: int, num_blocks: int, *,
                 separate: bool = False) -> PageCompact:
    """Moves the U blocks that the tables hold to the numbers 0 to U - 1: those numbered U and more, ascending,
    to the unused ones below, ascending (``page_copy`` does it in the caches).  Tables, shares (counted
    from the tables, which have to be all there are) and the free list follow the new numbers."""
    return PageCompact._make(_capi.native().page_compact(block_tables, lens, block_size, num_blocks, separate))


def page_copy(caches: list[torch.Tensor] | tuple[torch.Tensor, ...], sources: torch.Tensor,
              destinations: torch.Tensor) -> None:
    """cache[destinations[i]] = cache[sources[i]] in each of ``caches`` ([blocks, ...] of any type, each
    block contiguous in itself), in place; pairs with a negative number or one beyond the blocks are left
    out.  No block may be in two pairs unless it is a source in both.  64 caches to a launch."""
    _capi.native().page_copy(caches, sources, destinations)
