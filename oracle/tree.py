"""Oracle of drafted token trees and of log probabilities, in 64 bits, row by row, without the
product's code: what a node sees by following its parents, attention over exactly those keys with
a bound on what fp32 arithmetic may be off, the accepted path, the move of its rows, and softmax
with entropy, ranks and order by their definitions.
"""

from __future__ import annotations

import math

import numpy as np


def ancestors(parents: list[int]) -> list[list[int] | None]:
    """Of each node, the nodes that it sees (itself last); None where a parent on the way is not
    before its child."""
    out: list[list[int] | None] = []
    for i, p in enumerate(parents):
        if p == -1:
            out.append([i])
        elif 0 <= p < i and out[p] is not None:
            out.append(out[p] + [i])
        else:
            out.append(None)
    return out


def layout(parents, starts, ctx, num_tokens, max_nodes):
    """(masks uint64 [T, words], positions int64 [T])."""
    words = -(-max_nodes // 64)
    masks, positions = np.zeros((num_tokens, words), np.uint64), np.zeros(num_tokens, np.int64)
    for i, n in enumerate(ctx):
        a, b = starts[i], starts[i + 1]
        if b - a > max_nodes or b - a > n:
            continue
        for t, line in enumerate(ancestors(list(parents[a:b]))):
            if line is None:
                continue
            for j in line:
                masks[a + t, j // 64] |= np.uint64(1 << (j % 64))
            positions[a + t] = n - (b - a) + len(line) - 1
    return masks, positions


def accept(tokens, parents, targets, starts, max_depth):
    """(paths [B, max_depth], counts [B], next tokens [B])."""
    paths, counts, following = [], [], []
    for a, b in zip(starts, starts[1:]):
        path = [0] if b > a else []
        while path and len(path) < max_depth:
            at = path[-1]
            child = next((c for c in range(at + 1, b - a)
                          if parents[a + c] == at and tokens[a + c] == targets[a + at]), None)
            if child is None:
                break
            path.append(child)
        paths.append(path + [-1] * (max_depth - len(path)))
        counts.append(len(path))
        following.append(targets[a + path[-1]] if path else -1)
    return np.array(paths, np.int64).reshape(-1, max_depth), np.array(counts, np.int64), np.array(following, np.int64)


def keep(slots, tables, ctx, starts, paths, bs, num_blocks):
    """Moves rows of `slots` [num_blocks, bs, ...] in place."""
    for i, path in enumerate(paths):
        nodes = int(starts[i + 1] - starts[i])
        first, before = int(ctx[i]) - nodes, -1
        for d, node in enumerate(path):
            if node <= before or node >= nodes:
                break
            before = node
            a, b = first + int(node), first + d
            if a // bs >= tables.shape[1]:
                continue
            x, y = tables[i][a // bs], tables[i][b // bs]
            if 0 <= x < num_blocks and 0 <= y < num_blocks:
                slots[y, b % bs] = slots[x, a % bs]


def attention(q, k, v, tables, ctx, qlens, sees, scale):
    """q [T, H, D], k / v [NB, bs, Hkv, D] float64; sees[t]: the drafted nodes that token t sees.
    Returns (out, size, slack, flat): the exact output; sum of p |v|; the relative error that
    fp32 dot products of any order, exponentials and sums may put on the weights; and sum of |v|."""
    heads, dim = q.shape[1:]
    bs, kv = k.shape[1:3]
    out, size, flat = np.zeros(q.shape), np.zeros(q.shape), np.zeros(q.shape)
    slack = np.zeros(q.shape[:2] + (1,))
    at = 0
    for i, (n, m) in enumerate(zip(ctx, qlens)):
        pos = np.arange(n)
        keys, vals = (x[tables[i][pos // bs], pos % bs].transpose(1, 0, 2) for x in (k, v))
        for t in range(m):
            seen = list(range(n - m)) + [n - m + j for j in sees[at + t] if j < m]
            if not seen:
                continue
            kk, vv = keys[:, seen], vals[:, seen]                       # [Hkv, seen, D]
            qq = q[at + t].reshape(kv, heads // kv, dim).transpose(0, 2, 1)
            with np.errstate(invalid="ignore", over="ignore"):
                s = (kk @ qq * scale).transpose(0, 2, 1)                # [Hkv, group, seen]
                w = np.exp(s - s.max(-1, keepdims=True))
                p = w / w.sum(-1, keepdims=True)
                out[at + t] = (p @ vv).reshape(heads, dim)
                size[at + t] = (p @ np.abs(vv)).reshape(heads, dim)
                flat[at + t] = np.abs(vv).sum(1).repeat(heads // kv, 0)
                # |error of a score| <= (dim + 8) half steps of the sum of its terms' sizes; it
                # enters a weight and the sum of weights.
                reach = (np.abs(kk) @ np.abs(qq)).max(1).reshape(heads, 1) * abs(scale)
                slack[at + t] = 2.0 ** -24 * (2 * (dim + 8) * reach + len(seen) + 8)
        at += m
    return out, size, slack, flat


def logprobs(logits, ids, top):
    """logits float64 [rows, vocab]. (logprobs, ranks, entropy, top_logprobs, top_ids)."""
    rows, vocab = logits.shape
    lp, rank, entropy = np.full(rows, np.nan), np.zeros(rows, np.int64), np.full(rows, np.nan)
    top_lp, top_ids = np.full((rows, top), np.nan), np.full((rows, top), -1, np.int64)
    for r, x in enumerate(logits):
        if np.isnan(x).any() or x.max() in (math.inf, -math.inf):
            continue
        log_p = x - x.max() - math.log(math.fsum(np.exp(x - x.max())))
        p = np.exp(log_p)
        entropy[r] = -math.fsum(p[p > 0] * log_p[p > 0])
        order = np.argsort(-x, kind="stable")[:top]
        top_lp[r], top_ids[r] = log_p[order], order
        if 0 <= ids[r] < vocab:
            lp[r], rank[r] = log_p[ids[r]], 1 + (x > x[ids[r]]).sum()
    return lp, rank, entropy, top_lp, top_ids
