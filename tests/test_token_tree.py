"""Masks, positions, accepted paths of drafted token trees and the move of their cached rows, on
tensor ops and on the kernels, against the definitions."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from inference_server.config import CONFIG
from inference_server.core.kv8 import Kv8Pool
from inference_server.core.kv_pool import ModelDims, PagedKVPool
from inference_server.core.token_tree import MAX_NODES, accept_tree, tree_layout
from oracle import tree as oracle
from tree_cases import BF16, F16, F32, random_tree

BACKENDS = [pytest.param("gather", id="gather"), pytest.param("hip", id="hip", marks=pytest.mark.gpu)]


@pytest.fixture(params=BACKENDS)
def device(request, monkeypatch):
    monkeypatch.setattr(CONFIG, "attention", request.param)
    return "cuda" if request.param == "hip" else "cpu"


def long(x, device):
    return torch.as_tensor(np.asarray(x), dtype=torch.long).to(device)


def trees(counts, seed=0, spread=8):
    rng = np.random.default_rng(seed)
    parents = [p for n in counts for p in (random_tree(n, rng, spread) if n else [])]
    starts = np.concatenate([[0], np.cumsum(counts)]).astype(np.int64)
    return parents, starts, rng


COUNTS = [[1], [0], [5, 0, 1, 64, 3], [65, 64, 63, 1], [130, 7], [300, 1, 2], [1] * 70, [0, 0], []]


# ------------------------------------------------------------------ layout
@pytest.mark.parametrize("counts", COUNTS, ids=str)
@pytest.mark.parametrize("padding", [0, 1, 200])
@pytest.mark.parametrize("spread", [1, 8, 10 ** 6])
def test_layout_is_the_ancestors(device, counts, padding, spread):
    parents, starts, rng = trees(counts, len(counts), spread)
    parents = parents + [7] * padding                     # rows of no sequence hold anything
    ctx = np.array(counts, dtype=np.int64) + rng.integers(0, 5000, len(counts))
    for most in {max(counts, default=0), max(counts, default=0) + 100}:
        masks, positions = oracle.layout(parents, starts, ctx, len(parents), most)
        got = tree_layout(long(parents, device), long(starts, device), long(ctx, device), most)
        assert got.masks.shape == masks.shape
        assert np.array_equal(got.masks.cpu().numpy().view(np.uint64), masks)
        assert np.array_equal(got.positions.cpu().numpy(), positions)


def test_layout_of_long_chains_and_bushes(device):
    for parents in (list(range(-1, 999)), [-1] + [0] * 999, [-1] * 1000):
        starts, ctx = [0, 1000], [1000]
        masks, positions = oracle.layout(parents, starts, ctx, 1000, 1000)
        got = tree_layout(long(parents, device), long(starts, device), long(ctx, device), 1000)
        assert np.array_equal(got.masks.cpu().numpy().view(np.uint64), masks)
        assert np.array_equal(got.positions.cpu().numpy(), positions)


def test_layout_of_as_many_nodes_as_there_may_be(device):
    n = MAX_NODES
    parents = np.where(np.arange(n) == 0, -1, (np.arange(n) - 1) // 3)
    got = tree_layout(long(parents, device), long([0, n], device), long([n + 5], device), n)
    masks, positions = oracle.layout(parents.tolist(), [0, n], [n + 5], n, n)
    assert np.array_equal(got.masks.cpu().numpy().view(np.uint64), masks)
    assert np.array_equal(got.positions.cpu().numpy(), positions)


def test_layout_gives_impossible_nodes_nothing(device):
    # A parent that is the node itself, behind it, or below -1: it and the nodes below it.
    parents = [-1, 0, 2, 2, 9, 4, -2, 0, 6] + [-1, 0, 1] + [-1, 0]
    starts, ctx = [0, 9, 12, 14], [20, 2, 2]              # the second has more nodes than context
    masks, positions = oracle.layout(parents, starts, ctx, 14, 9)
    assert (masks[:, 0] != 0).tolist() == [True, True, False, False, False, False, False, True, False] + [False] * 3 + [True] * 2
    got = tree_layout(long(parents, device), long(starts, device), long(ctx, device), 9)
    assert np.array_equal(got.masks.cpu().numpy().view(np.uint64), masks)
    assert np.array_equal(got.positions.cpu().numpy(), positions)
    # More nodes than there is room for.
    got = tree_layout(long(parents, device), long(starts, device), long([20, 20, 20], device), 3)
    assert (got.masks[:, 0] != 0).tolist() == [False] * 9 + [True] * 5
    assert got.positions.tolist() == [0] * 9 + [17, 18, 19, 18, 19]
    # A refused step: query starts of 0.
    got = tree_layout(long(parents, device), long([0, 0, 0, 0], device), long(ctx, device), 9)
    assert not got.masks.any() and not got.positions.any()


def test_layout_of_rows_that_no_sequence_has(device):
    # Starts that leave rows before the first sequence, and that end behind the step.
    parents = [0, 3, -1, 0, 1, -1, 0, 0, 1]
    for starts, real in (([2, 5, 7], range(2, 7)), ([2, 5, 12], range(2, 5)), ([9, 9, 9], ()), ([12, 13, 20], ()),
                         ([-3, 2, 5], range(2, 5)), ([0, 0, 5], ())):
        got = tree_layout(long(parents, device), long(starts, device), long([9, 9], device), 4)
        assert [t for t in range(9) if got.masks[t, 0]] == list(real), starts
        assert not got.positions[[t for t in range(9) if t not in real]].any()


@pytest.mark.gpu
def test_a_captured_walk_follows_its_inputs(monkeypatch):
    """Layout, path and the rows' move in one graph, replayed over other trees."""
    monkeypatch.setattr(CONFIG, "attention", "hip")
    counts, bs, depth = [9, 0, 40, 17], 8, 12
    pools = [PagedKVPool(ModelDims(2, 2, 16, F16), num_blocks=40, block_size=bs, device="cuda") for _ in range(2)]

    def case(seed):
        tokens, parents, targets, starts = drafted(counts, seed)
        rng = np.random.default_rng(seed)
        ctx = rng.integers(0, 20, 4) + counts
        return tokens, parents, targets, starts, ctx, rng.permutation(40).reshape(4, 10)

    at = [long(x, "cuda") for x in case(0)]

    def step(pool):
        tokens, parents, targets, starts, ctx, tables = at
        tree = tree_layout(parents, starts, ctx, 64)
        path = accept_tree(tokens, parents, targets, starts, depth)
        pool.keep_paths(tables, ctx, starts, path.paths)
        return (*tree, *path)

    stream, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.stream(stream):
        with pytest.raises(RuntimeError, match="pointer_table"), torch.cuda.graph(torch.cuda.CUDAGraph(), stream=stream):
            at[0] + 1                                     # (a graph of something)
            step(pools[0])
    torch.cuda.synchronize()
    for pool in pools:
        pool.pointer_table()
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=stream):
        outs = step(pools[0])
    for seed in range(1, 6):
        for dst, x in zip(at, case(seed)):
            dst.copy_(long(x, "cuda"))
        for pool in pools:
            fill(pool, seed)
        torch.cuda.synchronize()
        g.replay()
        want = step(pools[1])
        torch.cuda.synchronize()
        for a, b in zip(outs, want):
            assert torch.equal(a, b)
        for a, b in zip(pools[0].k + pools[0].v, pools[1].k + pools[1].v):
            assert np.array_equal(bits(a), bits(b))
        tokens, parents, targets, starts, ctx, tables = case(seed)
        assert np.array_equal(want[2].cpu().numpy(), oracle.accept(tokens, parents, targets, starts, depth)[0])


def test_layout_refusals(device):
    p, s, c = long([-1, 0], device), long([0, 2], device), long([4], device)
    for bad in ((p[None], s, c, 2), (p, s[None], c, 2), (p, s, c[None], 2), (p.int(), s, c, 2), (p, s.int(), c, 2),
                (p, s, c.int(), 2), (p, s, long([4, 4], device), 2), (p, s, c, -1), (p, s, c, MAX_NODES + 1),
                (p, s[:0], c, 2)):
        with pytest.raises(ValueError):
            tree_layout(*bad)


# ------------------------------------------------------------------ accept
def drafted(counts, seed, agree=0.7, vocab=5):
    parents, starts, rng = trees(counts, seed)
    n = len(parents)
    targets, tokens = rng.integers(0, vocab, n), rng.integers(0, vocab, n)
    for a, b in zip(starts, starts[1:]):
        for t in range(a + 1, b):
            if rng.random() < agree:
                tokens[t] = targets[a + parents[t]]
    return tokens, parents, targets, starts


@pytest.mark.parametrize("counts", COUNTS, ids=str)
@pytest.mark.parametrize("depth", [1, 3, 12, 200])
def test_accept_walks_while_tokens_agree(device, counts, depth):
    for seed in range(3):
        tokens, parents, targets, starts = drafted(counts, seed)
        want = oracle.accept(tokens, parents, targets, starts, depth)
        got = accept_tree(*(long(x, device) for x in (tokens, parents, targets, starts)), depth)
        for a, b in zip(got, want):
            assert np.array_equal(a.cpu().numpy(), b)


@pytest.mark.parametrize("n", [2048, 2049, MAX_NODES])
def test_accept_of_chains_that_agree_throughout(device, n):
    parents, tokens = np.arange(-1, n - 1), np.arange(n)
    targets = tokens + 1
    got = accept_tree(*(long(x, device) for x in (tokens, parents, targets, [0, n])), n)
    assert got.paths.tolist() == [list(range(n))] and got.counts.tolist() == [n] and got.next_tokens.tolist() == [n]
    got = accept_tree(*(long(x, device) for x in (tokens, parents, targets, [0, n])), 100)
    assert got.paths.tolist() == [list(range(100))] and got.next_tokens.tolist() == [100]


def test_accept_takes_the_first_of_equal_children(device):
    # 0 -> 1, 2, 3; 1 and 2 carry the same fitting token. 2 has a child that fits, 1 none that does.
    tokens, parents, targets = [9, 5, 5, 6, 7, 8], [-1, 0, 0, 0, 2, 1], [5, 7, 7, 1, 2, 3]
    got = accept_tree(*(long(x, device) for x in (tokens, parents, targets, [0, 6])), 4)
    assert got.paths.tolist() == [[0, 1, -1, -1]] and got.next_tokens.tolist() == [7]


def test_accept_without_nodes_or_with_impossible_ones(device):
    x = long([1, 1, 1, 1], device)
    # Parents that are the node itself, behind it, below -1: no child of anything.
    got = accept_tree(x, long([-1, 1, 3, -5], device), x, long([0, 4, 4], device), 3)
    assert got.paths.tolist() == [[0, -1, -1], [-1, -1, -1]] and got.counts.tolist() == [1, 0]
    assert got.next_tokens.tolist() == [1, -1]
    got = accept_tree(x[:0], x[:0], x[:0], long([0, 0], device), 2)
    assert got.counts.tolist() == [0] and got.next_tokens.tolist() == [-1] and got.paths.tolist() == [[-1, -1]]
    got = accept_tree(x, x, x, long([0, 9], device), 2)           # bounds past the step
    assert got.counts.tolist() == [0]
    with pytest.raises(ValueError):
        accept_tree(x, x, x, long([0, 4], device), 0)
    with pytest.raises(ValueError):
        accept_tree(x, x[:3], x, long([0, 4], device), 2)
    with pytest.raises(ValueError):
        accept_tree(x, x, x.int(), long([0, 4], device), 2)


# ------------------------------------------------------------------ keep
def keep_case(counts, bs, seed, device, depth=12):
    rng = np.random.default_rng(seed)
    new = np.array(counts, dtype=np.int64)
    cached = rng.integers(0, 40, len(counts))
    ctx = cached + new
    need = -(-ctx // bs)
    n_blocks = int(need.sum()) + 2
    ids = rng.permutation(n_blocks)
    tables = np.zeros((len(counts), max(1, int(need.max(initial=0)))), np.int64)
    at = 0
    for i, n in enumerate(need):
        tables[i, :n] = ids[at:at + n]
        at += n
    paths = np.full((len(counts), depth), -1, np.int64)
    for i, n in enumerate(counts):
        m = int(rng.integers(0, min(n, depth) + 1))
        paths[i, :m] = np.sort(rng.choice(n, m, replace=False)) if m else paths[i, :m]
    starts = np.concatenate([[0], np.cumsum(new)])
    return n_blocks, tables, ctx, starts, paths


def fill(pool, seed):
    g = torch.Generator().manual_seed(seed)
    for t in pool.k + pool.v:
        t.copy_(torch.randint(0, 256, t.view(torch.uint8).shape, generator=g, dtype=torch.uint8).view(t.dtype))


def bits(t):
    return t.contiguous().view(torch.uint8).cpu().numpy().copy()


@pytest.mark.parametrize("cls", [PagedKVPool, Kv8Pool])
@pytest.mark.parametrize("dtype,kv,d,bs", [(F32, 2, 64, 16), (F16, 12, 64, 16), (BF16, 8, 128, 16), (F16, 1, 3, 8),
                                           (F16, 3, 10, 5), (F32, 1, 1, 1), (BF16, 2, 40, 64)])
@pytest.mark.parametrize("counts", [[1], [9, 0, 64, 3, 30], [200, 2]], ids=str)
def test_keep_moves_rows(device, cls, dtype, kv, d, bs, counts):
    for depth in (1, 12, 150):
        n_blocks, tables, ctx, starts, paths = keep_case(counts, bs, depth + bs, device, depth)
        pool = cls(ModelDims(3, kv, d, dtype), num_blocks=n_blocks, block_size=bs, device=device)
        fill(pool, depth)
        want = [bits(t) for t in pool._slot_tensors()]
        for w in want:
            oracle.keep(w, tables, ctx, starts, paths, bs, n_blocks)
        pool.keep_paths(*(long(x, device) for x in (tables, ctx, starts, paths)))
        for t, w in zip(pool._slot_tensors(), want):
            assert np.array_equal(bits(t), w)


def test_keep_ends_a_path_that_does_not_ascend_and_skips_bad_blocks(device):
    bs, n_blocks = 4, 10
    tables = np.array([[0, 1, 2], [3, 4, 5], [6, 77, -1], [7, 8, 9]])
    ctx, starts = np.array([10, 12, 12, 6]), np.array([0, 8, 18, 30, 38])     # the last: more nodes than context
    paths = np.array([[0, 3, 3, 5], [1, 2, 99, 3], [0, 2, 6, 9], [0, 1, 2, 4]])
    pool = PagedKVPool(ModelDims(1, 2, 8, F32), num_blocks=n_blocks, block_size=bs, device=device)
    fill(pool, 0)
    before = [bits(t) for t in pool.k + pool.v]
    want = [b.copy() for b in before]
    for w in want:
        oracle.keep(w, tables[:3], ctx[:3], starts[:4], paths[:3], bs, n_blocks)
    pool.keep_paths(*(long(x, device) for x in (tables, ctx, starts, paths)))
    for t, w, b in zip(pool.k + pool.v, want, before):
        assert np.array_equal(bits(t), w) and not np.array_equal(w, b)


def test_keep_refusals(device):
    pool = PagedKVPool(ModelDims(1, 2, 8, F32), num_blocks=4, block_size=4, device=device)
    t, c, s, p = (long(x, device) for x in ([[0, 1]], [6], [0, 4], [[0, 2]]))
    pool.keep_paths(t, c, s, p)
    pool.keep_paths(t[:0], c[:0], s[:1], p[:0])
    pool.keep_paths(t, c, s, p[:, :0])
    for bad in ((t[0], c, s, p), (t, c[:0], s, p), (t, c, s[:1], p), (t, c, s, p[0]), (t, c, s, p.int()),
                (t.int(), c, s, p), (t, c, s.int(), p)):
        with pytest.raises(ValueError):
            pool.keep_paths(*bad)


@pytest.mark.gpu
def test_keep_refuses_more_sequences_than_a_grid_has(monkeypatch):
    monkeypatch.setattr(CONFIG, "attention", "hip")
    pool = PagedKVPool(ModelDims(1, 1, 8, F32), num_blocks=2, block_size=4, device="cuda")
    before = [bits(t) for t in pool.k + pool.v]
    for n in (65535, 65536):
        args = (torch.zeros(n, 1, dtype=torch.long, device="cuda"), torch.full((n,), 4, device="cuda"),
                torch.zeros(n + 1, dtype=torch.long, device="cuda"), torch.zeros(n, 2, dtype=torch.long, device="cuda"))
        if n > 65535:
            with pytest.raises(RuntimeError, match="keep_paths"):
                pool.keep_paths(*args)
        else:
            pool.keep_paths(*args)                        # no nodes: nothing moves
    for t, b in zip(pool.k + pool.v, before):
        assert np.array_equal(bits(t), b)
