"""Compacting and copying where another answer than the defined one is near."""
from __future__ import annotations

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from libcusort_b200 import paging  # noqa: E402
from tests import pages_reference as ref  # noqa: E402
from tests.test_pages_gpu import dev, same  # noqa: E402

pytestmark = pytest.mark.gpu


def test_ascending_blocks_go_to_ascending_holes():
    """Of blocks 0, 3, 5 and 7 the last two move, 5 to 1 and 7 to 2, whichever table comes first."""
    tables = np.array([[5, -3, 99, 2 ** 31 - 1], [-1, 7, 0, 3]])
    for order in ([0, 1], [1, 0]):
        got = paging.page_compact(dev(tables[order]), dev(np.array([64, 60])), 16, 8)
        want = np.array([[1, -3, 99, 2 ** 31 - 1], [-1, 2, 0, 3]])[order]
        assert got.block_tables.tolist() == want.tolist()
        assert got.sources.tolist() == [5, 7, -1, -1] and got.destinations.tolist() == [1, 2, -1, -1]
        assert got.shares.tolist() == [0] * 8 and got.num_free.tolist() == [4]
        assert got.free_blocks.tolist() == [7, 6, 5, 4, -1, -1, -1, -1]


@pytest.mark.parametrize("blocks", [64, 30_000])  # in one CTA, and by a launch for each phase
def test_every_used_block_moves(blocks):
    """The upper half of a pool is used, in descending order of the tables' entries."""
    tables = np.arange(blocks - 1, blocks // 2 - 1, -1).reshape(8, -1)
    lens = np.full(8, tables.shape[1] * 4)
    got = paging.page_compact(dev(tables), dev(lens), 4, blocks)
    same(got, ref.compact(tables, lens, 4, blocks))
    assert got.sources.tolist() == list(range(blocks // 2, blocks))
    assert got.destinations.tolist() == list(range(blocks // 2))


def test_copying_the_moves_of_a_pool():
    """What compacting says is copied: every request finds its blocks' values at the new numbers."""
    rng = np.random.default_rng(8)
    blocks = 900
    tables = rng.permutation(blocks)[:400].reshape(20, 20)
    lens = rng.integers(0, 20 * 16 + 1, 20)
    cache = torch.arange(blocks, device="cuda").float()[:, None].expand(blocks, 48).contiguous()
    got = paging.page_compact(dev(tables), dev(lens), 16, blocks)
    paging.page_copy([cache], got.sources, got.destinations)
    for old, new, length in zip(tables, got.block_tables.tolist(), lens):
        n = len(ref.held(old, length, 16))
        assert (cache[new[:n]] == torch.tensor(old[:n], device="cuda")[:, None]).all() and new[n:] == [-1] * (20 - n)
