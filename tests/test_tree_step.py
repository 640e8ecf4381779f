"""The operators of a step with drafted trees as they are used together: a small model over the paged
pool decodes greedily token by token, and again by verified trees; both give the same tokens."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from inference_server.config import CONFIG
from inference_server.core.attention import paged_attention
from inference_server.core.attention_hip import attach_host, attach_query_start
from inference_server.core.kv_pool import ModelDims, PagedKVPool
from inference_server.core.sampling import token_logprobs
from inference_server.core.step_layout import step_layout
from inference_server.core.token_tree import accept_tree, paged_tree_attention, tree_layout

BACKENDS = [pytest.param("gather", id="gather"), pytest.param("hip", id="hip", marks=pytest.mark.gpu)]
LAYERS, HEADS, KV, DIM, VOCAB, BS, LONGEST = 2, 4, 2, 32, 61, 16, 400
DEPTH = 6


@pytest.fixture(params=BACKENDS)
def device(request, monkeypatch):
    monkeypatch.setattr(CONFIG, "attention", request.param)
    return "cuda" if request.param == "hip" else "cpu"


class Model:
    """Attention with residuals and learned positions, in fp32."""

    def __init__(self, device):
        g = torch.Generator().manual_seed(3)
        w = lambda *shape: (torch.randn(*shape, generator=g) * shape[0] ** -0.5).to(device)  # noqa: E731
        size = HEADS * DIM
        self.tokens, self.positions = w(VOCAB, size) * 8, w(LONGEST, size) * 8
        self.layers = [(w(size, (HEADS + 2 * KV) * DIM), w(size, size)) for _ in range(LAYERS)]

    def __call__(self, ids, positions, attend):
        x = self.tokens[ids] + self.positions[positions]
        for layer, (qkv, out) in enumerate(self.layers):
            y = x / x.norm(dim=-1, keepdim=True) * HEADS * DIM ** 0.5
            q, k, v = (y @ qkv).view(-1, HEADS + 2 * KV, DIM).split([HEADS, KV, KV], 1)
            x = x + attend(layer, q, k, v).flatten(1) @ out
        return x / x.norm(dim=-1, keepdim=True) @ self.tokens.t() * 4


class Step:
    """Tables, lengths and free blocks of a batch, on the device."""

    def __init__(self, prompts, device):
        self.device, self.model = device, Model(device)
        self.pool = PagedKVPool(ModelDims(LAYERS, KV, DIM, torch.float32), num_blocks=64, block_size=BS, device=device)
        n = len(prompts)
        self.tables = self.long(np.zeros((n, LONGEST // BS)))
        self.held, self.cached, self.free = self.long([0] * n), self.long([0] * n), self.long(np.arange(64)[::-1].copy())
        lens = [len(p) for p in prompts]
        logits = self.forward(self.long(sum(prompts, [])), self.long(lens), None)
        self.cached = self.long(lens)
        self.last = logits[np.cumsum(lens) - 1].argmax(-1)

    def long(self, x):
        return torch.as_tensor(np.asarray(x), dtype=torch.long).to(self.device)

    def forward(self, ids, new, parents, max_nodes=0):
        ctx = self.cached + new
        self.layout = lay = step_layout(self.tables, self.held, ctx, new, self.free, BS, ids.shape[0])
        self.held, self.free = lay.held, self.free[int(lay.counts[0]):]
        tree = tree_layout(parents, lay.query_start, ctx, max_nodes) if parents is not None else None

        def attend(layer, q, k, v):
            self.pool.append(layer, k, v, lay.slots)
            args = (q, self.pool.k[layer], self.pool.v[layer], lay.block_tables, ctx, new)
            if tree is None:
                return paged_attention(*args, DIM ** -0.5)
            return paged_tree_attention(*args, tree.masks, DIM ** -0.5)

        return self.model(ids, lay.positions if tree is None else tree.positions, attend)


def drafts(rng, last, truth, most):
    """A tree below `last`: some of its branches hold what will be decoded, down to some depth."""
    n = int(rng.integers(1, most + 1))
    tokens, parents, depth = [last], [-1], [0]
    for i in range(1, n):
        p = int(rng.integers(max(0, i - 6), i))
        d = depth[p] + 1
        right = d - 1 < len(truth) and rng.random() < 0.8
        tokens.append(truth[d - 1] if right else int(rng.integers(0, VOCAB)))
        parents.append(p)
        depth.append(d)
    return tokens, parents


def test_verified_trees_decode_what_single_tokens_do(device):
    rng = np.random.default_rng(11)
    prompts = [[int(t) for t in rng.integers(0, VOCAB, n)] for n in (1, 17, 40, 100)]
    plain = Step(prompts, device)
    want = [plain.last]
    scores = []
    for _ in range(60):
        logits = plain.forward(plain.last, plain.long([1] * 4), None)
        scores.append(token_logprobs(logits, logits.argmax(-1), 3))
        plain.cached, plain.last = plain.cached + 1, logits.argmax(-1)
        want.append(plain.last)
    want = torch.stack(want, 1).tolist()
    for s in scores:
        assert torch.equal(s.ranks, torch.ones_like(s.ranks)) and (s.logprobs == s.top_logprobs[:, 0]).all()

    tree = Step(prompts, device)
    got = [[t] for t in tree.last.tolist()]
    steps = longest = 0
    while min(len(g) for g in got) < 40:
        made = [drafts(rng, g[-1], w[len(g):], 20) for g, w in zip(got, want)]
        new = [len(t) for t, _ in made]
        tokens = tree.long(sum((t for t, _ in made), []))
        parents = tree.long(sum((p for _, p in made), []))
        logits = tree.forward(tokens, tree.long(new), parents, max(new))
        targets = logits.argmax(-1)
        # Every drafted token's log probability at its parent, as a server reports or samples by it.
        up = torch.where(parents >= 0, parents + tree.layout.query_start[:-1].repeat_interleave(tree.long(new)), 0)
        at_parent = token_logprobs(logits[up], tokens, 2)
        path = accept_tree(tokens, parents, targets, tree.layout.query_start, DEPTH)
        tree.pool.keep_paths(tree.layout.block_tables, tree.cached + tree.long(new), tree.layout.query_start, path.paths)
        tree.cached = tree.cached + path.counts
        first = 0
        for i, nodes in enumerate(path.paths.tolist()):
            kept = [n for n in nodes if n >= 0]
            assert len(kept) == int(path.counts[i]) and kept[0] == 0
            for n in kept[1:]:
                assert int(at_parent.ranks[first + n]) == 1
            got[i] += [made[i][0][n] for n in kept[1:]] + [int(path.next_tokens[i])]
            longest = max(longest, len(kept))
            first += new[i]
        steps += 1
    for g, w in zip(got, want):
        n = min(len(g), len(w))
        assert g[:n] == w[:n]
    assert longest == DEPTH and steps < 39


@pytest.mark.gpu
@pytest.mark.parametrize("starts", ["layout", "host"])
def test_a_step_reads_nothing_back(monkeypatch, starts):
    """With bounds of the lengths on the host and the layout's query starts (or lengths that the host has), no operator waits for
    the device, in its first call or later ones; results are those of a step that reads the lengths back."""
    monkeypatch.setattr(CONFIG, "attention", "hip")
    rng = np.random.default_rng(3)
    dims, new, cached = ModelDims(2, 2, 64, torch.float16), [7, 20, 1, 12], [30, 5, 90, 500]
    pool = PagedKVPool(dims, num_blocks=64, block_size=BS, device="cuda")
    for t in pool.k + pool.v:
        t.normal_()
    tokens, parents = zip(*(drafts(rng, 1, [1] * 9, n + 1) for n in new))
    new = [len(t) for t in tokens]
    total = sum(new)
    cuda = lambda x: torch.as_tensor(x, dtype=torch.long).cuda()  # noqa: E731
    tokens, parents = cuda(sum(tokens, [])), cuda(sum(parents, []))
    held = [-(-c // BS) for c in cached]
    tables = torch.zeros(4, 40, dtype=torch.long)
    for i, h in enumerate(held):
        tables[i, :h] = torch.arange(sum(held[:i]), sum(held[:i]) + h)
    tables, free = tables.cuda(), torch.arange(sum(held), 64).cuda()
    q, logits = torch.randn(total, 8, 64, device="cuda").half(), torch.randn(total, 61, device="cuda")
    lens = [c + n for c, n in zip(cached, new)]
    bounds = ([640] * 4, [total - 3, 1, 1, 1]) if starts == "layout" else (lens, new)

    def step(attached):
        ctx, query_lens = cuda(lens), cuda(new)
        held_d, targets = cuda(held), logits.argmax(-1)
        if attached:
            attach_host(ctx, torch.tensor(bounds[0])), attach_host(query_lens, torch.tensor(bounds[1]))
            torch.cuda.synchronize()
            torch.cuda.set_sync_debug_mode("error")
        try:
            lay = step_layout(tables.clone(), held_d, ctx, query_lens, free, BS, total)
            if attached and starts == "layout":
                attach_query_start(query_lens, lay.query_start)
            tree = tree_layout(parents, lay.query_start, ctx, 32)
            out = [paged_tree_attention(q, k, v, lay.block_tables, ctx, query_lens, tree.masks, 0.125)
                   for k, v in zip(pool.k, pool.v)]
            scores = token_logprobs(logits, tokens, 3)
            path = accept_tree(tokens, parents, targets, lay.query_start, DEPTH)
            pool.keep_paths(lay.block_tables, ctx, lay.query_start, path.paths * 0 - 1)
        finally:
            torch.cuda.set_sync_debug_mode("default")
        return [*tree, *out, *scores, *path]

    pool.pointer_table()
    want = step(False)
    for _ in range(2):
        for a, b in zip(step(True), want):
            if a.dtype is torch.float16:            # contexts may be cut otherwise: one rounding of the output
                assert (a.float() - b.float()).abs().max() <= 2.0 ** -10 * b.float().abs().max()
            else:
                assert torch.equal(a, b)
