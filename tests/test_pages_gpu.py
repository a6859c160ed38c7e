"""Forking, freeing, compacting and copying blocks of a paged cache against a plain implementation, block by block."""
from __future__ import annotations

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from libcusort_b200 import paging  # noqa: E402
from tests import pages_reference as ref  # noqa: E402

pytestmark = pytest.mark.gpu


def scene(requests, width, block_size, blocks=None, seed=0, group=3, spare=0.0, stale=True):
    """Requests in groups that share the whole blocks of a common beginning: tables, lens, free list, left, shares."""
    rng = np.random.default_rng(seed)
    lens = rng.integers(0, width * block_size + 1, requests)
    lens[rng.random(requests) < 0.1] = 0
    lens[rng.random(requests) < 0.1] = width * block_size
    pages = [[] for _ in range(requests)]
    count, common = 0, []
    for r in range(requests):
        n = -(-int(lens[r]) // block_size)
        if r % group == 0:
            common = []
        same = min(len(common), int(lens[r]) // block_size)
        pages[r] = common[:same] + list(range(count, count + n - same))
        count += n - same
        if r % group == 0:
            common = pages[r][:int(lens[r]) // block_size]
    blocks = max(blocks or 0, count + int(count * spare) + 4)
    name = rng.permutation(blocks)
    tables = np.full((requests, width), -7 if stale else -1)  # what lies behind the held entries is anything
    shares = np.full(blocks, -1)
    for r in range(requests):
        mine = name[pages[r]] if pages[r] else []
        tables[r, :len(mine)] = mine
        shares[mine] += 1
    free = np.concatenate([name[count:], np.full(count, -1)])
    return tables, lens, free, blocks - count, np.maximum(shares, 0)


def dev(x, pad=0):
    t = torch.from_numpy(np.ascontiguousarray(x)).int().cuda()
    if pad:
        t = torch.nn.functional.pad(t, (0, pad), value=12345)[:, :x.shape[1]]
    return t


def same(got, want):
    for name, value in want.items():
        mine = getattr(got, name).cpu().numpy()
        value = np.asarray(value).reshape(mine.shape)
        assert np.array_equal(mine, value), (name, np.argwhere(mine != value)[:5], mine[mine != value][:5],
                                             value[mine != value][:5])


def pool(free, left, shares):
    return dict(free_blocks=dev(free), num_free=dev(np.array([left])), shares=dev(shares))


# the last two pools are of the form with a launch for each phase
SIZES = [(1, 1, 1), (3, 2, 16), (32, 137, 16), (100, 5, 1), (257, 33, 64), (1500, 9, 3), (2048, 80, 16), (16384, 3, 2)]


@pytest.mark.parametrize("requests,width,block_size", SIZES)
@pytest.mark.parametrize("short", [False, True])
def test_fork(requests, width, block_size, short):
    tables, lens, free, left, shares = scene(requests, width, block_size, seed=requests, spare=0.5)
    rng = np.random.default_rng(1)
    if short:
        left = min(left, requests // 4)
    parents = rng.integers(0, requests, requests)
    parents[rng.random(requests) < 0.1] = -1
    inputs = [t.clone() for t in pool(free, left, shares).values()]
    given = pool(free, left, shares)
    got = paging.page_fork(dev(tables, pad=5), dev(lens), dev(parents), block_size, **given)
    same(got, ref.fork(tables, lens, parents, block_size, free, left, shares))
    assert all(torch.equal(a, b) for a, b in zip(inputs, given.values()))  # nothing is written in place


@pytest.mark.parametrize("children", [0, 1, 7, 400])
def test_fork_to_another_number_of_requests(children):
    tables, lens, free, left, shares = scene(50, 12, 16, seed=3, spare=3.0)
    parents = np.random.default_rng(2).integers(-3, 55, children)
    parents[:3] = [2 ** 31 - 1, -2 ** 31, 0][:children]
    got = paging.page_fork(dev(tables), dev(lens), dev(parents), 16, **pool(free, left, shares))
    same(got, ref.fork(tables, lens, parents, 16, free, left, shares))


def test_fork_of_nothing():
    empty = torch.empty(0, dtype=torch.int32, device="cuda")
    none = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = paging.page_fork(empty.view(0, 4), empty, dev(np.array([0, -1])), 16, free_blocks=empty, num_free=none,
                           shares=empty)
    assert got.block_tables.tolist() == [[-1] * 4] * 2 and got.lens.tolist() == [0, 0] and got.served.all()
    assert got.num_free.tolist() == [0]


def test_a_truncated_request_gets_its_own_last_block():
    """Two requests share whole blocks; one is cut back into a shared one and forked from itself."""
    tables, lens = np.array([[3, 1, -1], [3, 1, 5]]), np.array([32, 40])
    free, shares = np.array([0, 2, 4, 6, 7, -1, -1, -1]), np.array([0, 1, 0, 1, 0, 0, 0, 0])
    cut = np.array([20, 40])
    got = paging.page_fork(dev(tables), dev(cut), dev(np.array([0, 1])), 16, **pool(free, 5, shares))
    assert got.block_tables.tolist() == [[3, 7, -1], [3, 1, 5]]
    assert got.sources.tolist() == [1, -1] and got.destinations.tolist() == [7, -1]
    assert got.shares.tolist() == [0, 0, 0, 1, 0, 0, 0, 0] and got.num_free.tolist() == [4]


@pytest.mark.parametrize("requests,width,block_size", SIZES)
@pytest.mark.parametrize("done", [0.0, 0.3, 1.0])
def test_free(requests, width, block_size, done):
    tables, lens, free, left, shares = scene(requests, width, block_size, seed=requests + 1)
    rng = np.random.default_rng(4)
    keep = np.where(rng.random(requests) < 0.5, lens - rng.integers(-2, 2 * block_size + 2, requests), lens)
    keep[rng.random(requests) < done] = 0
    got = paging.page_free(dev(tables, pad=1), dev(lens), dev(keep), block_size, **pool(free, left, shares))
    same(got, ref.free(tables, lens, keep, block_size, free, left, shares))


@pytest.mark.parametrize("requests,width,block_size", SIZES)
@pytest.mark.parametrize("spare", [0.0, 0.6, 5.0])
def test_compact(requests, width, block_size, spare):
    tables, lens, _, _, shares = scene(requests, width, block_size, seed=requests + 2, spare=spare)
    got = paging.page_compact(dev(tables, pad=3), dev(lens), block_size, len(shares))
    same(got, ref.compact(tables, lens, block_size, len(shares)))


def test_compact_large_pool_and_none():
    tables, lens, _, _, shares = scene(40, 50, 16, blocks=700_001, seed=5)
    same(paging.page_compact(dev(tables), dev(lens), 16, 700_001), ref.compact(tables, lens, 16, 700_001))
    empty = torch.empty(0, dtype=torch.int32, device="cuda")
    got = paging.page_compact(empty.view(0, 3), empty, 16, 1)
    assert got.free_blocks.tolist() == [0] and got.num_free.tolist() == [1] and got.sources.numel() == 0
    assert paging.page_compact(empty.view(0, 3), empty, 16, 0).num_free.tolist() == [0]


def test_lengths_below_zero_and_beyond_the_table():
    tables, lens, free, left, shares = scene(20, 6, 16, seed=7, spare=2.0)
    lens[:5] = [-5, -2 ** 31, 6 * 16 + 1, 2 ** 31 - 1, 0]
    tables[:5] = -1
    full = [b for b in free[:left]][:12]
    left -= 12
    free = np.concatenate([free[12:12 + left], np.full(len(free) - left, -1)])
    tables[2], tables[3] = full[:6], full[6:]
    shares = np.maximum(np.bincount([b for t, n in zip(tables, lens) for b in ref.held(t, n, 16)],
                                    minlength=len(shares)) - 1, 0)
    parents = np.arange(20)[::-1].copy()
    same(paging.page_fork(dev(tables), dev(lens), dev(parents), 16, **pool(free, left, shares)),
         ref.fork(tables, lens, parents, 16, free, left, shares))
    keep = lens // 2
    same(paging.page_free(dev(tables), dev(lens), dev(keep), 16, **pool(free, left, shares)),
         ref.free(tables, lens, keep, 16, free, left, shares))
    same(paging.page_compact(dev(tables), dev(lens), 16, len(shares)), ref.compact(tables, lens, 16, len(shares)))


def test_entries_and_counts_that_are_none_stay_inside():
    """Numbers outside the pool are kept in tables and counted nowhere; a free count beyond the list is cut."""
    tables = np.array([[5, -3, 99, 2 ** 31 - 1], [-1, 7, 0, 3]])
    got = paging.page_fork(dev(tables), dev(np.array([64, 60])), dev(np.array([0, 1, 1])), 16, free_blocks=dev(
        np.arange(8)), num_free=dev(np.array([1000])), shares=dev(np.zeros(8)))
    assert got.block_tables.tolist() == [tables[0].tolist(), tables[1].tolist(), [-1, 7, 0, 7]]
    assert got.shares.tolist() == [1, 0, 0, 0, 0, 0, 0, 1]
    got = paging.page_compact(dev(tables), dev(np.array([64, 60])), 16, 8)
    assert got.num_free.tolist() == [4]
    assert got.block_tables.tolist() == [[2, -3, 99, 2 ** 31 - 1], [-1, 1, 0, 3]] or got.block_tables.tolist() == [
        [1, -3, 99, 2 ** 31 - 1], [-1, 2, 0, 3]]


@pytest.mark.parametrize("shapes,dtype", [
    ([(20, 16, 8, 64)] * 3, torch.bfloat16), ([(20, 3, 5), (20, 7), (20,)], torch.float16),
    ([(20, 4100)], torch.uint8), ([(20, 16, 2, 640)], torch.float32), ([(20, 9001), (20, 3)], torch.int16),
    ([(20, 4)] * 130, torch.float32), ([(20, 0), (20, 8)], torch.float32), ([(20, 6)], torch.float64)],
    ids=lambda v: str(v)[:40])
def test_copy(shapes, dtype):
    caches = [torch.randint(0, 100, s, device="cuda").to(dtype) for s in shapes]
    sources = dev(np.array([3, -1, 5, 3, 20, 7, 9, -2 ** 31, 2 ** 31 - 1, 11]))
    destinations = dev(np.array([1, 2, 0, 19, 4, -1, 9, 6, 8, 12]))
    want = [c.clone() for c in caches]
    for w in want:
        for s, d in ((3, 1), (5, 0), (3, 19), (11, 12)):
            w[d] = w[s]
    paging.page_copy(caches, sources, destinations)
    assert all(torch.equal(a, b) for a, b in zip(caches, want))


def test_copy_of_blocks_apart_and_off_16_bytes():
    whole = torch.randn(12, 3, 70, device="cuda").bfloat16()
    caches = [whole[:, 0, :64], whole[:, 1, 1:65], whole[:, 2, 2:3], whole[:, 2, 6:70]]
    want = whole.clone()
    for part in (want[:, 0, :64], want[:, 1, 1:65], want[:, 2, 2:3], want[:, 2, 6:70]):
        part[4] = part[2]
    paging.page_copy(tuple(caches), dev(np.array([2])), dev(np.array([4])))
    assert torch.equal(whole, want)


def test_many_pairs():
    """More pairs than there are CTAs, nearly all of them none."""
    cache = torch.randn(60_000, 33, device="cuda")
    want = cache.clone()
    sources, destinations = np.full(30_000, -1), np.full(30_000, -1)
    at = np.random.default_rng(0).permutation(30_000)[:5000]
    sources[at], destinations[at] = np.arange(5000), 59_999 - np.arange(5000)
    want[59_999 - torch.arange(5000)] = cache[:5000]
    paging.page_copy([cache], dev(sources), dev(destinations))
    assert torch.equal(cache, want)


def test_copy_beyond_32_bits():
    cache = torch.zeros(70_000, 65_536, dtype=torch.uint8, device="cuda")  # 4.6 GB
    cache[69_998] = 7
    cache[1] = 9
    paging.page_copy([cache], dev(np.array([69_998, 1])), dev(np.array([0, 69_999])))
    assert (cache[0] == 7).all() and (cache[69_999] == 9).all() and not cache[2:69_998:997].any()


def test_a_life_of_blocks():
    """Steps of placing, forking, freeing and compacting, with the tokens' values in two caches: every request finds
    its own tokens again, and no block is lost or held twice by mistake."""
    rng = np.random.default_rng(11)
    R, width, B, blocks = 12, 10, 4, 90
    caches = [torch.full((blocks, B), -1.0, device="cuda") for _ in range(2)]
    tables = torch.full((R, width), -1, dtype=torch.int32, device="cuda")
    lens = torch.zeros(R, dtype=torch.int32, device="cuda")
    free, left = torch.arange(blocks, device="cuda").int(), torch.tensor([blocks], device="cuda").int()
    shares = torch.zeros(blocks, dtype=torch.int32, device="cuda")
    history = [[] for _ in range(R)]
    for step in range(30):
        new = rng.integers(0, 4, R)
        new = np.minimum(new, width * B - np.array([len(h) for h in history]))
        plan = paging.page_plan(lens, dev(new), tables, B, int(new.sum()), free_blocks=free, num_free=left)
        served = plan.served.tolist()
        values = torch.arange(int(new.sum()), device="cuda").float() + 1000 * step
        ok = plan.slots >= 0
        for i, cache in enumerate(caches):
            cache.view(-1)[plan.slots[ok]] = values[ok] + i
        at = 0
        for r in range(R):
            mine = [1000 * step + at + j for j in range(new[r])]
            at += new[r]
            if served[r]:
                history[r] = history[r] + mine
        lens, left = dev(np.array([len(h) for h in history])), plan.num_free
        kind = step % 3
        if kind == 0:
            parents = rng.integers(-1, R, R)
            fork = paging.page_fork(tables, lens, dev(parents), B, free_blocks=free, num_free=left, shares=shares)
            paging.page_copy(caches, fork.sources, fork.destinations)
            tables, lens, shares, free, left = (fork.block_tables.clone(), fork.lens, fork.shares, fork.free_blocks,
                                                fork.num_free)
            history = [list(history[p]) if p >= 0 and ok else [] for p, ok in zip(parents, fork.served.tolist())]
        elif kind == 1:
            keep = np.array([len(h) if rng.random() < 0.7 else rng.integers(0, len(h) + 1) for h in history])
            done = paging.page_free(tables, lens, dev(keep), B, free_blocks=free, num_free=left, shares=shares)
            shares, free, left = done.shares, done.free_blocks, done.num_free
            history = [h[:k] for h, k in zip(history, keep)]
            lens = dev(keep)
            own = paging.page_fork(tables, lens, dev(np.arange(R)), B, free_blocks=free, num_free=left, shares=shares)
            paging.page_copy(caches, own.sources, own.destinations)
            history = [h if ok else [] for h, ok in zip(history, own.served.tolist())]
            tables, lens, shares, free, left = (own.block_tables.clone(), own.lens, own.shares, own.free_blocks,
                                                own.num_free)
        else:
            moved = paging.page_compact(tables, lens, B, blocks)
            paging.page_copy(caches, moved.sources, moved.destinations)
            assert torch.equal(moved.num_free, left)
            tables, shares, free = moved.block_tables.clone(), moved.shares, moved.free_blocks
        for i, cache in enumerate(caches):
            flat = cache.cpu().view(-1)
            for table, h in zip(tables.tolist(), history):
                assert [flat[table[j // B] * B + j % B] for j in range(len(h))] == [v + i for v in h]
        counts = np.bincount([b for t, h in zip(tables.tolist(), history) for b in ref.held(t, len(h), B)],
                             minlength=blocks)
        assert np.array_equal(shares.cpu().numpy(), np.maximum(counts - 1, 0))
        assert sorted(free[:int(left)].tolist()) == [b for b in range(blocks) if counts[b] == 0]


def test_the_same_again_captured_and_on_another_stream():
    tables, lens, free, left, shares = scene(64, 20, 16, seed=9, spare=1.0)
    given = pool(free, left, shares)
    args = dev(tables), dev(lens), dev(np.arange(64)[::-1] // 2), 16
    first = paging.page_fork(*args, **given)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        again = paging.page_fork(*args, separate=True, **given)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            captured = paging.page_fork(*args, **given)
        graph.replay()
        stream.synchronize()
    assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(first, again, captured))
