"""step_layout against the host's own bookkeeping (BlockTable), on the torch backend (CPU)
and, marked gpu, on the kernel; and what it refuses."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from inference_server.config import CONFIG
from inference_server.core.block_allocator import BlockAllocator
from inference_server.core.block_table import BlockTable
from inference_server.core.step_layout import step_layout

BACKENDS = [pytest.param("cpu", id="torch"), pytest.param("cuda", id="hip", marks=pytest.mark.gpu)]


@pytest.fixture(params=BACKENDS)
def device(request, monkeypatch):
    monkeypatch.setattr(CONFIG, "attention", "hip" if request.param == "cuda" else "gather")
    return request.param


def inputs(cached, new, held, bs, width=None, seed=0, spare=5):
    """Device-independent tensors: tables filled as far as held, and a shuffled free list."""
    cached, new, held = (np.array(x, dtype=np.int64) for x in (cached, new, held))
    ctx = cached + new
    need = np.maximum(-(-ctx // bs), held)
    ids = np.random.default_rng(seed).permutation(int(need.sum()) + spare)
    tables = np.full((len(ctx), int(need.max(initial=0)) + 2 if width is None else width), -7, dtype=np.int64)
    at = 0
    for i, h in enumerate(held):
        tables[i, :h] = ids[at:at + h]
        at += h
    return [torch.from_numpy(x) for x in (tables, held, ctx, new, ids[at:].copy())]


def expected(tables, held, ctx, new, free, bs, tokens):
    """BlockTable's arithmetic, sequence by sequence."""
    tables, held, free = tables.clone(), held.clone(), free.tolist()
    slots, positions, starts, taken = [], [], [0], 0
    for i, (n, m) in enumerate(zip(ctx.tolist(), new.tolist())):
        table = BlockTable(BlockAllocator(1), block_size=bs)
        missing = max(0, table.blocks_for(n) - int(held[i]))
        tables[i, held[i]:held[i] + missing] = torch.tensor(free[taken:taken + missing], dtype=torch.long)
        taken += missing
        held[i] += missing
        table._append(tables[i, :held[i]].tolist())
        slots += table.slot_range(n - m, n).tolist() if m else []
        positions += range(n - m, n)
        starts.append(len(slots))
    pad = tokens - len(slots)
    return (tables, held, torch.tensor(slots + [-1] * pad, dtype=torch.long),
            torch.tensor(positions + [0] * pad, dtype=torch.long), torch.tensor(starts), torch.tensor([taken, taken, 0]))


def run(device, args, bs, tokens):
    args = [a.to(device) for a in args]
    got = step_layout(*args, bs, tokens)
    assert got.block_tables is args[0]
    return got


def same(got, want):
    for name, g, w in zip(got._fields, got, want):
        assert g.dtype is torch.long and torch.equal(g.cpu(), w), name


def many(n, seed, top):
    rng = np.random.default_rng(seed)
    cached, new = rng.integers(0, top, n), rng.integers(0, 9, n)
    return cached, new


@pytest.mark.parametrize("bs", [1, 8, 16, 24, 64])
@pytest.mark.parametrize("cached,new,pad", [
    ([0], [1], 0), ([16], [1], 0), ([15], [1], 3), ([0], [0], 2), ([], [], 4),
    ([0, 5, 0, 31, 32], [17, 0, 0, 1, 100], 0),
    (*many(257, 1, 300), 7), (*many(1024, 2, 90), 0), (*many(1025, 3, 90), 1), (*many(3000, 4, 60), 500),
])
def test_matches_the_hosts_tables(device, bs, cached, new, pad):
    cached, new = np.array(cached, dtype=np.int64), np.array(new, dtype=np.int64)
    for held in (-(-cached // bs), 0 * cached, -(-(cached + new) // bs) + 1):   # as cached; none; more than needed
        args = inputs(cached, new, held, bs)
        tokens = int(new.sum()) + pad
        want = expected(*args, bs, tokens)
        got = run(device, args, bs, tokens)
        same(got, want)
        # Repeated on the same inputs (the tables as the first call left them): the same.
        again = step_layout(got.block_tables, *(a.to(device) for a in args[1:]), bs, tokens)
        same(again, want)


def test_long_prompt_and_wide_table(device):
    args = inputs([0, 70000], [50000, 1], [0, 70000 // 8], 8, width=20000)
    same(run(device, args, 8, 50001), expected(*args, 8, 50001))


def nothing(device, args, bs, tokens, counts):
    before = args[0].clone()
    got = run(device, args, bs, tokens)
    b = args[0].shape[0]
    same(got, (before, args[1], torch.full((tokens,), -1), torch.zeros(tokens, dtype=torch.long),
               torch.zeros(b + 1, dtype=torch.long), torch.tensor(counts)))


@pytest.mark.parametrize("n", [3, 2000])
def test_all_or_nothing(device, n):
    cached, new = many(n, 5, 50)
    new[0] += 1
    args = inputs(cached, new, -(-cached // 8), 8)
    need = int((-(-(cached + new) // 8) - args[1].numpy()).sum())
    exact = [*args[:4], args[4][:need]]
    same(run(device, exact, 8, int(new.sum())), expected(*exact, 8, int(new.sum())))
    args = inputs(cached, new, -(-cached // 8), 8)
    nothing(device, [*args[:4], args[4][:need - 1]], 8, int(new.sum()), [0, need, 0])   # one block short


@pytest.mark.parametrize("change,wrong", [
    (dict(new=[-1, 2]), 1), (dict(new=[3, 400]), 1), (dict(ctx=[10 ** 6, 9]), 1), (dict(ctx=[2 ** 62, 9]), 1),
    (dict(held=[-1, 0]), 1), (dict(held=[0, 100]), 1), (dict(ctx=[-5, -5]), 2), (dict(tokens=4), 1),
])
def test_impossible_lengths_change_nothing(device, change, wrong):
    tables, held, ctx, new, free = inputs([2, 7], [3, 2], [0, 1], 8)
    held, ctx, new = (torch.tensor(change[k]) if k in change else t
                      for k, t in (("held", held), ("ctx", ctx), ("new", new)))
    ok = [i for i in range(2) if 0 <= new[i] <= ctx[i] and 0 <= held[i] <= tables.shape[1]
          and ctx[i] <= 8 * tables.shape[1]]
    need = sum(max(0, -(-int(ctx[i]) // 8) - int(held[i])) for i in ok)
    nothing(device, [tables, held, ctx, new, free], 8, change.get("tokens", 6), [0, need, wrong])


def test_refusals(device):
    t, h, c, n, f = (x.to(device) for x in inputs([2, 7], [3, 2], [0, 1], 8))
    for bad in ([t[0], h, c, n, f], [t, h[:1], c, n, f], [t, h, c[:1], n, f], [t, h, c, n[:, None], f],
                [t, h, c, n, f[None]], [t, h.int(), c, n, f], [t.int(), h, c, n, f]):
        with pytest.raises(ValueError):
            step_layout(*bad, 8, 5)
    with pytest.raises(ValueError):
        step_layout(t, h, c, n, f, 0, 5)
    with pytest.raises(ValueError):
        step_layout(t, h, c, n, f, 8, -1)


def test_hip_needs_a_device(monkeypatch):
    monkeypatch.setattr(CONFIG, "attention", "hip")
    with pytest.raises(NotImplementedError):
        step_layout(*inputs([2], [1], [0], 8), 8, 1)


@pytest.mark.gpu
def test_rows_of_wider_tables_and_refused_ones(monkeypatch):
    monkeypatch.setattr(CONFIG, "attention", "hip")
    args = inputs([2, 30], [3, 20], [0, 1], 8)
    want = expected(*args, 8, 23)
    wide = torch.full((2, args[0].shape[1] + 5), 99, device="cuda")
    part = wide[:, 2:2 + args[0].shape[1]]
    part.copy_(args[0])
    got = step_layout(part, *(a.cuda() for a in args[1:]), 8, 23)
    same(got, want)
    assert (wide[:, :2] == 99).all() and (wide[:, -3:] == 99).all()
    for bad in (part.t().contiguous().t(), part[:1].expand(2, -1)):
        with pytest.raises(ValueError, match="in place"):
            step_layout(bad, *(a.cuda() for a in args[1:]), 8, 23)


@pytest.mark.gpu
def test_in_a_graph(monkeypatch):
    """Captured once, replayed on other lengths and lists, with eager work between."""
    monkeypatch.setattr(CONFIG, "attention", "hip")
    stages = [inputs([3, 40, 0], [m, 1, 2], [1, 5, 0], 8, width=12, seed=m, spare=20 - m) for m in (1, 9, 4)]
    size = min(s[4].numel() for s in stages)
    static = [x.cuda() for x in stages[0][:4]] + [stages[0][4][:size].cuda()]
    step_layout(*static, 8, 16)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step_layout(*static, 8, 16)
    for s in (*stages, stages[1]):
        s = [*s[:4], s[4][:size]]
        for to, x in zip(static, s):
            to.copy_(x)
        graph.replay()
        same(got, expected(*s, 8, 16))
        torch.zeros(1000, device="cuda").sum().item()
