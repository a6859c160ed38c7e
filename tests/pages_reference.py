"""What forking, freeing and compacting blocks of a paged cache mean, block by block in plain Python."""
from __future__ import annotations

import numpy as np


def held(table, length, block_size):
    """The blocks that a request holds."""
    return list(table[:min(len(table), -(-max(int(length), 0) // block_size))])


def give_back(counts, before, free, left, blocks):
    """The free list with the blocks that were held before and are not any more."""
    out = list(free[:left]) + [b for b in range(blocks) if before[b] > 0 and counts[b] == 0]
    return out + [-1] * (blocks - len(out)), len(out)


def holders(tables, lens, block_size, shares):
    """Tables that hold each block: from these tables and the shares of others."""
    own = np.zeros(len(shares), dtype=int)
    for table, length in zip(tables, lens):
        for b in held(table, length, block_size):
            own[b] += 1
    return np.where(own > 0, shares + 1, 0)


def fork(tables, lens, parents, block_size, free, left, shares):
    R, width, blocks = len(tables), tables.shape[1], len(shares)
    before = holders(tables, lens, block_size, shares)
    counts = before.copy()
    for table, length in zip(tables, lens):
        for b in held(table, length, block_size):
            counts[b] -= 1
    seen, taken = set(), 0
    out = {"block_tables": [], "lens": [], "sources": [], "destinations": [], "served": []}
    wanted = 0
    for p in map(int, parents):
        table, length, pair, served = [], 0, (-1, -1), True
        if 0 <= p < R:
            length = max(int(lens[p]), 0)
            table = held(tables[p], length, block_size)
            part = length % block_size != 0 and -(-length // block_size) <= width
            if part and (p in seen or shares[table[-1]] != 0):
                wanted += 1
                if wanted <= left:
                    pair = (table[-1], free[left - wanted])
                    table[-1] = pair[1]
                    taken += 1
                else:
                    table, length, served = [], 0, False
            seen.add(p)
        for b in table:
            counts[b] += 1
        out["block_tables"].append(table + [-1] * (width - len(table)))
        out["lens"].append(length)
        out["sources"].append(pair[0])
        out["destinations"].append(pair[1])
        out["served"].append(served)
    out["shares"] = np.maximum(counts - 1, 0)
    out["free_blocks"], out["num_free"] = give_back(counts, before, free, left - taken, blocks)
    return out


def free(tables, lens, keep, block_size, free_list, left, shares):
    before = holders(tables, lens, block_size, shares)
    counts = before.copy()
    for table, length, k in zip(tables, lens, keep):
        mine = held(table, length, block_size)
        for b in mine[len(held(table, min(int(k), int(length)), block_size)):]:
            counts[b] -= 1
    out = {"shares": np.maximum(counts - 1, 0)}
    out["free_blocks"], out["num_free"] = give_back(counts, before, free_list, left, len(shares))
    return out


def compact(tables, lens, block_size, blocks):
    counts = holders(tables, lens, block_size, np.zeros(blocks, dtype=int))
    counts[:] = 0
    for table, length in zip(tables, lens):
        for b in held(table, length, block_size):
            counts[b] += 1
    used = int((counts > 0).sum())
    move = [b for b in range(used, blocks) if counts[b] > 0]
    holes = [b for b in range(used) if counts[b] == 0]
    to = dict(zip(move, holes))
    shares = np.zeros(blocks, dtype=int)
    for b in range(blocks):
        if counts[b] > 0:
            shares[to.get(b, b)] = counts[b] - 1
    rest = blocks // 2 - len(move)
    width = tables.shape[1]
    new = []
    for table, length in zip(tables, lens):
        mine = [to.get(int(b), int(b)) for b in held(table, length, block_size)]
        new.append(mine + [-1] * (width - len(mine)))
    return {"block_tables": new, "sources": move + [-1] * rest, "destinations": holes + [-1] * rest, "shares": shares,
            "free_blocks": list(range(blocks - 1, used - 1, -1)) + [-1] * used, "num_free": blocks - used}
