"""Inputs and tolerances shared by the tests of drafted token trees."""

from __future__ import annotations

from types import SimpleNamespace

import numpy as np
import torch

from oracle import tree as oracle

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
HALF_STEP = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}
#: Least step of the type's subnormals.
LEAST = {F32: 2.0 ** -149, F16: 2.0 ** -24, BF16: 2.0 ** -133}
#: What two pieces of the type leave of a weight (fp32 weights are whole).
PIECES = {F32: 0.0, F16: 2.0 ** -22, BF16: 2.0 ** -16}


def random_tree(n, rng, spread=8):
    """Parents of a tree of n nodes, first nodes shallow and later ones anywhere behind."""
    return [-1] + [int(rng.integers(max(0, i - spread), i)) for i in range(1, n)]


def words_of(sees, width):
    """Visibility lists as mask words, int64."""
    masks = np.zeros((len(sees), width), np.uint64)
    for t, nodes in enumerate(sees):
        for j in nodes:
            masks[t, j // 64] |= np.uint64(1 << (j % 64))
    return torch.from_numpy(masks.view(np.int64))


def tree_masks(new, rng, kind="tree"):
    """Of every token, the nodes that it sees: its ancestors, those before it, or any."""
    out = []
    for n in new:
        if kind == "tree":
            out += oracle.ancestors(random_tree(int(n), rng)) if n else []
        elif kind == "chain":
            out += [list(range(t + 1)) for t in range(n)]
        elif kind == "none":
            out += [[] for _ in range(n)]
        else:                                   # any, later nodes and none among them
            out += [sorted(int(j) for j in np.nonzero(rng.random(n) < rng.choice([0.0, 0.2, 0.9]))[0]) for _ in range(n)]
    return out


def batch(lens, *, heads, kv, d, bs, dtype, seed=0, device="cpu", kind="tree", width=None, spare=3, words=None):
    """`lens`: (cached, nodes) of each sequence. Slots past a context, and blocks of no sequence,
    hold any bits (NaN among them)."""
    rng = np.random.default_rng(seed)
    cached, new = np.array(lens, dtype=np.int64).reshape(-1, 2).T
    ctx = cached + new
    need = -(-ctx // bs)
    n_blocks = int(need.sum()) + spare
    ids = rng.permutation(n_blocks)
    width = max(1, int(need.max(initial=0))) if width is None else width
    tables = np.zeros((len(lens), width), dtype=np.int64)
    at = 0
    for i, n in enumerate(need):
        tables[i, :n] = ids[at:at + n]
        at += n
    s = SimpleNamespace(ctx=ctx, new=new, tables=tables, dtype=dtype, scale=d ** -0.5, device=device)

    def pool():
        size = torch.empty(0, dtype=dtype).element_size()
        raw = torch.from_numpy(rng.integers(0, 256, (n_blocks, bs, kv, d * size), dtype=np.uint8)).view(dtype)
        for i, n in enumerate(ctx):
            pos = np.arange(n)
            rows = rng.standard_normal((n, kv, d)) * np.exp(0.5 * rng.standard_normal((n, kv, 1)))
            raw[tables[i, pos // bs], pos % bs] = torch.from_numpy(rows).to(dtype)
        return raw

    s.k, s.v = pool().to(device), pool().to(device)
    s.q = (torch.from_numpy(rng.standard_normal((int(new.sum()), heads, d))) * 1.5).to(dtype).to(device)
    s.sees = tree_masks(new, rng, kind)
    s.masks = words_of(s.sees, max(1, -(-int(new.max(initial=0)) // 64)) if words is None else words).to(device)
    s.args = tuple(torch.from_numpy(x).to(device) for x in (tables, ctx, new))
    s.start = torch.from_numpy(np.concatenate([[0], np.cumsum(new)])).to(device)
    return s


def check(s, out, scale=None):
    """out against the exact attention: one rounding to the type, what pieces of the type leave
    of each weight, and what fp32 leaves. fp16 pieces are off by half a subnormal step, 2^-25, where
    they are small, against sums of at least the largest weight, 1 or more."""
    want, size, slack, flat = oracle.attention(
        s.q.double().cpu().numpy(), s.k.double().cpu().numpy(), s.v.double().cpu().numpy(), s.tables, s.ctx, s.new,
        s.sees, s.scale if scale is None else scale)
    u = HALF_STEP[s.dtype]
    tol = u * np.abs(want) + (1 + u) * (PIECES[s.dtype] + slack) * size + LEAST[s.dtype]
    if s.dtype is F16:
        tol = tol + 2.0 ** -25 * flat
    got = out.double().cpu().numpy()
    assert got.shape == want.shape
    special = ~np.isfinite(want)
    assert np.array_equal(got[special], want[special], equal_nan=True)
    assert np.isfinite(got[~special]).all()
    off = np.abs(got[~special] - want[~special]) - tol[~special]
    assert off.size == 0 or off.max() <= 0, f"off by {off.max():.3g} more than {tol[~special][off.argmax()]:.3g}"
