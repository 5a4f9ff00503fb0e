"""CPU oracle for the draft-tree stages — TEST INFRASTRUCTURE ONLY.

Plain numpy loops in 64 bits, from the definitions in include/mvb200.h
(mvb_build_draft_tree, mvb_tree_attention, mvb_accept_draft_tree,
mvb_compact_draft_kv).  The reference project has no counterpart.
"""

from __future__ import annotations

import numpy as np


def _parent(parents: np.ndarray, first: int, i: int) -> int:
    p = int(parents[first + i])
    return p if -1 <= p < i else -1


def ancestors(parents: np.ndarray, first: int, i: int) -> list[int]:
    """Node i of the request whose rows start at ``first``, then its parent,
    and so on up to its root."""

    path = [i]
    while (p := _parent(parents, first, path[-1])) >= 0:
        path.append(p)
    return path


def build_draft_tree(parents, starts, committed, table, block_size, context_start, words):
    """(positions, context_starts, lengths, slots, mask) of one step;
    ``context_start(position)`` is the spec."""

    rows = len(parents)
    positions, begin = np.zeros(rows, np.int64), np.zeros(rows, np.int64)
    slots, mask = np.full(rows, -1, np.int64), np.zeros((rows, words), np.uint64)
    lengths = np.zeros(len(committed), np.int64)
    for r, c in enumerate(committed):
        first, n = int(starts[r]), int(starts[r + 1] - starts[r])
        if first < 0 or n < 0 or first + n > rows or n > 64 * words or c < 0 or c + n > 1 << 30:
            continue
        lengths[r] = c + n
        for i in range(n):
            path = ancestors(parents, first, i)
            positions[first + i] = c + len(path) - 1
            begin[first + i] = context_start(c + len(path) - 1)
            page = (c + i) // block_size
            if page < table.shape[1] and table[r, page] >= 0:
                slots[first + i] = table[r, page] * block_size + (c + i) % block_size
            for j in path:
                if c + len(ancestors(parents, first, j)) - 1 >= begin[first + i]:
                    mask[first + i, j // 64] |= np.uint64(1) << np.uint64(j % 64)
    return positions, begin, lengths, slots, mask.view(np.int64)


def tree_attention(query, cache, begin, starts, lengths, table, mask, scale):
    """(output, weighted |value|, sum of |q||k| of each row's largest key) in
    64 bits.  ``query`` [T, Hq, D], ``cache`` [2, NB, bs, Hkv, D]."""

    rows, q_heads, dim = query.shape
    _, blocks, block_size, kv_heads, _ = cache.shape
    group, words = q_heads // kv_heads, mask.view(np.uint64)
    out, size, reach = np.zeros(query.shape), np.zeros(query.shape), np.zeros((rows, q_heads))
    for r, length in enumerate(lengths):
        first, n = int(starts[r]), int(starts[r + 1] - starts[r])
        if n <= 0 or first < 0 or first + n > rows or n > 64 * words.shape[1] or length < n:
            continue
        c = int(length) - n
        for i in range(n):
            t = first + i
            keys = list(range(max(int(begin[first]), int(begin[t]), 0), c))
            keys += [c + j for j in range(n) if (int(words[t, j // 64]) >> (j % 64)) & 1]
            keys = [p for p in keys if p // block_size < table.shape[1] and 0 <= table[r, p // block_size] < blocks]
            if not keys:
                continue
            at = np.asarray(keys)
            block, offset = table[r, at // block_size], at % block_size
            k = np.repeat(cache[0, block, offset].astype(np.float64), group, axis=1)
            v = np.repeat(cache[1, block, offset].astype(np.float64), group, axis=1)
            q = query[t].astype(np.float64)
            s = np.einsum("hd,khd->hk", q, k) * scale
            p = np.exp(s - s.max(1, keepdims=True))
            p /= p.sum(1, keepdims=True)
            out[t] = np.einsum("hk,khd->hd", p, v)
            size[t] = np.einsum("hk,khd->hd", p, np.abs(v))
            reach[t] = np.einsum("hd,khd->hk", np.abs(q), np.abs(k)).max(1) * scale
    return out, size, reach


def accept_draft_tree(draft, target, parents, starts, committed, max_accepted):
    """(nodes, num_accepted, tokens, new lengths, last rows)."""

    requests = len(committed)
    nodes, tokens = (np.full((requests, max_accepted), -1, np.int64) for _ in range(2))
    count, last = np.zeros(requests, np.int64), np.full(requests, -1, np.int64)
    for r in range(requests):
        first, n = int(starts[r]), int(starts[r + 1] - starts[r])
        if first < 0 or n <= 0 or first + n > len(draft) or n > 1024:
            continue
        p = 0
        while count[r] < max_accepted:
            nodes[r, count[r]], tokens[r, count[r]] = p, target[first + p]
            count[r] += 1
            last[r] = first + p
            heirs = [i for i in range(n) if int(parents[first + i]) == p and i > p and draft[first + i] == target[first + p]]
            if not heirs:
                break
            p = heirs[0]
    return nodes, count, tokens, np.asarray(committed) + count, last


def compact_draft_kv(cache, table, committed, nodes, count):
    """The moved cache (a new array) of one layer, [2, NB, bs, Hkv, D]."""

    out, block_size = cache.copy(), cache.shape[2]
    for r, c in enumerate(committed):
        for k in range(int(count[r])):
            source, goal = int(c + nodes[r, k]), int(c + k)
            out[:, table[r, goal // block_size], goal % block_size] = \
                cache[:, table[r, source // block_size], source % block_size]
    return out
