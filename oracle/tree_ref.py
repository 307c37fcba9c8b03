"""Plain 64-bit forms of the drafted-tree operators, one sequence, one row, one node at a time (numpy)."""

from __future__ import annotations

import numpy as np


def index(parents, starts, tables, block_size, max_blocks, words):
    """``(positions, slots, mask)`` of the trees ``parents`` (a list per sequence); mask words as int64."""
    positions, slots, mask = [], [], []
    for tree, start, table in zip(parents, starts, tables):
        for i in range(len(tree)):
            chain, at = [], i
            while at >= 0:
                chain.append(at)
                up = tree[at]
                at = up if 0 <= up < at else -1
            positions.append(start + len(chain) - 1)
            p = start + i
            slots.append(table[p // block_size] * block_size + p % block_size if p // block_size < max_blocks else -1)
            bits = sum(1 << j for j in chain)
            mask.append([(bits >> (64 * w)) & (2**64 - 1) for w in range(words)])
    return (np.array(positions, np.int64), np.array(slots, np.int64),
            np.array(mask, np.uint64).reshape(len(positions), words).view(np.int64))


def sees(mask_row, j: int) -> bool:
    return j // 64 < len(mask_row) and (int(mask_row[j // 64]) >> (j % 64)) & 1 == 1


def attention(q, k_pool, v_pool, tables, starts, counts, mask, block_size, scale, max_blocks=None):
    """Attention of packed nodes in 64 bits, and what an error bound needs.

    Returns ``out``, ``spread`` (the weighted mean of |v|) and ``reach`` (the largest scale * sum |q_d k_d| of a
    row's keys), each of ``[N, Hq, D]`` or ``[N, Hq]``. ``tables`` is a list of block-id lists; an id outside the pool
    hides its keys.
    """
    n, hq, d = q.shape
    group = hq // k_pool.shape[1]
    out, spread, reach = np.zeros((n, hq, d)), np.zeros((n, hq, d)), np.zeros((n, hq))
    r = 0
    for table, start, count in zip(tables, starts, counts):
        end = start + count
        if max_blocks is not None:
            end = min(end, max_blocks * block_size)
        for i in range(count):
            keys = [j for j in range(end) if (j < start or sees(mask[r], j - start))
                    and 0 <= table[j // block_size] < k_pool.shape[0]]
            blk = np.array([table[j // block_size] for j in keys], dtype=np.int64)
            off = np.array([j % block_size for j in keys], dtype=np.int64)
            for h in range(hq if keys else 0):
                k, v = (x[blk, h // group, off].astype(np.float64) for x in (k_pool, v_pool))
                qr = q[r, h].astype(np.float64)
                s = scale * (k @ qr)
                w = np.exp(s - s.max())
                w /= w.sum()
                out[r, h] = w @ v
                spread[r, h] = w @ np.abs(v)
                reach[r, h] = scale * (np.abs(k) @ np.abs(qr)).max()
            r += 1
    return out, spread, reach


def verify(logits, tokens, parents):
    """``(target, paths, next)`` of one batch; ``tokens`` and ``parents`` lists per sequence, logits in packed rows."""
    target = []
    for row in logits:
        nan = np.flatnonzero(np.isnan(row))
        target.append(int(nan[0]) if len(nan) else int(np.flatnonzero(row == row.max())[0]))
    paths, following, at = [], [], 0
    for toks, tree in zip(tokens, parents):
        path = [0] if tree else []
        while path:
            want = target[at + path[-1]]
            child = [i for i in range(path[-1] + 1, len(tree)) if tree[i] == path[-1] and toks[i] == want]
            if not child:
                break
            path.append(child[0])
        paths.append(path)
        following.append(target[at + path[-1]] if path else -1)
        at += len(tree)
    return target, paths, following
