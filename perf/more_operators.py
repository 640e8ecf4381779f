"""The operators that verify drafted token trees, and what each costs: a step's visibility masks
and positions built from the nodes' parents, attention of the nodes over the paged cache, log
probabilities of given tokens (with entropy, ranks and the likeliest alternatives), the walk that
accepts a path, and the move of the accepted rows in the cache.

A drafted tree is a sequence's last tokens in the cache: its nodes in an order in which parents
come first, node 0 the token that was sampled before. A node sees the cached tokens, its
ancestors and itself.

Lengths are fixed by the case (so the work is); values, trees and block placement come from the
seed.
"""

from __future__ import annotations

import math
import os
import sys
from pathlib import Path
from types import SimpleNamespace

import numpy as np
import torch

own = False

DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
DEVICE = "cuda"

GPT2 = {"heads": 12, "kv_heads": 12, "head_dim": 64, "block_size": 16}
GQA = {"heads": 32, "kv_heads": 8, "head_dim": 128, "block_size": 16}
GPT2_VOCAB = 50257
MAX_DEPTH = 12          # nodes of a tree's longest path: what a draft model is asked for


# ---------------------------------------------------------------------- cases
def _attend(name, dtype, shape, seqs, nodes, cached):
    return {"name": name, "op": "attend", "dtype": dtype, **shape, "seqs": seqs, "new_min": nodes[0],
            "new_max": nodes[1], "cached_min": cached[0], "cached_max": cached[1]}


def _logprobs(name, dtype, rows, vocab, top):
    return {"name": name, "op": "logprobs", "dtype": dtype, "rows": rows, "vocab": vocab, "top": top}


def _trees_of(name, op, seqs, nodes):
    return {"name": name, "op": op, "seqs": seqs, "new_min": nodes[0], "new_max": nodes[1], "cached_min": 1,
            "cached_max": 4000}


def _keep(name, dtype, shape, layers, seqs, nodes):
    return {"name": name, "op": "keep", "dtype": dtype, "layers": layers, "kv_heads": shape["kv_heads"],
            "head_dim": shape["head_dim"], "block_size": shape["block_size"], "seqs": seqs, "new_min": nodes[0],
            "new_max": nodes[1], "cached_min": 1, "cached_max": 64}


def listed():
    return [
        # Masks and positions of a step at low concurrency: the smallest call.
        _trees_of("layout x8", "layout", 8, (8, 32)),
        # The same of a full batch with wide trees.
        _trees_of("layout x256", "layout", 256, (16, 256)),
        # One layer's attention of a GPT-2 step: a serving batch, each sequence with a tree.
        _attend("attend gpt2 fp16 x32", "fp16", GPT2, 32, (8, 32), (16, 960)),
        # The same at the framework's default dtype.
        _attend("attend gpt2 fp32 x32", "fp32", GPT2, 32, (8, 32), (16, 960)),
        # A full batch of long conversations with large trees.
        _attend("attend gqa bf16 x64", "bf16", GQA, 64, (16, 64), (1024, 8192)),
        # A lone very long conversation.
        _attend("attend gqa bf16 x1 long", "bf16", GQA, 1, (32, 32), (100000, 100000)),
        # Log probabilities and five alternatives for the sampled tokens of a decode step.
        _logprobs("logprobs gpt2 fp16 x8", "fp16", 8, GPT2_VOCAB, 5),
        # Those of every token of long prompts, over a large vocabulary.
        _logprobs("logprobs 128000 bf16 x2048", "bf16", 2048, 128000, 20),
        # The walk over a step's trees, at low concurrency and of a full batch with wide trees.
        _trees_of("accept x8", "accept", 8, (8, 32)),
        _trees_of("accept x256", "accept", 256, (16, 256)),
        # The accepted rows of a GPT-2 step, every layer.
        _keep("keep gpt2 fp16 x32", "fp16", GPT2, 12, 32, (8, 32)),
        # The same of a full batch of a deep model with grouped heads.
        _keep("keep gqa bf16 x64", "bf16", GQA, 32, 64, (16, 64)),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _shape(rng):
    """Head layouts: the two usual ones, or any of the others that caches come in."""
    if rng.random() < 0.5:
        return dict(rng.choice([GPT2, GQA]))
    kv = rng.choice([1, 2, 3, 4, 5, 8, 12])
    return {"heads": kv * rng.choice([1, 2, 3, 4, 6, 8]), "kv_heads": kv,
            "head_dim": rng.choice([32, 48, 64, 80, 96, 112, 128]), "block_size": rng.choice([8, 16, 32, 64])}


def draw(rng):
    kind = rng.choice(["layout", "attend", "attend", "attend", "attend long", "logprobs", "logprobs", "accept", "keep"])
    if kind in ("layout", "accept"):
        hi = _log(rng, 1, 256)
        c = _trees_of("", kind, _log(rng, 1, 256), (rng.randint(1, hi), hi))
    elif kind == "logprobs":
        vocab = rng.choice([GPT2_VOCAB, _log(rng, 1000, 160000)])
        dtype = rng.choice(["fp32", "fp16", "bf16"])
        most = 260_000_000 // vocab // (2 if dtype == "fp32" else 1)
        c = _logprobs("", dtype, _log(rng, 1, min(2048, most)), vocab, rng.choice([0, 1, 5, 20, rng.randint(2, 64)]))
    elif kind == "keep":
        shape, layers, hi = _shape(rng), _log(rng, 2, 32), _log(rng, 1, 64)
        most = 64 * 32 * GQA["kv_heads"] * GQA["head_dim"] // (layers * shape["kv_heads"] * shape["head_dim"])
        dtype = rng.choice(["fp32", "fp16", "bf16"])
        c = _keep("", dtype, shape, layers, _log(rng, 1, max(1, min(64, most // 2))), (rng.randint(1, hi), hi))
    else:
        shape, dtype = _shape(rng), rng.choice(["fp16", "bf16", "bf16", "fp32"])
        hi = _log(rng, 1, 256 if dtype != "fp32" else 64)
        if kind == "attend":
            lo = _log(rng, 1, 1024)
            cached = (lo, _log(rng, lo, 8192))
        else:
            n = _log(rng, 8192, 100000)
            cached = (n // 2, n)
        # Flops and bytes of the longest contexts stay below those of the largest listed case.
        node = 4 * (cached[1] + hi) * shape["heads"] * shape["head_dim"] * (8 if dtype == "fp32" else 1)
        hi = min(hi, 150_000_000_000 // node)
        each = hi * node
        size = 2 * (cached[1] + hi) * shape["kv_heads"] * shape["head_dim"] * (4 if dtype == "fp32" else 2)
        most = max(1, min(64 if kind == "attend" else 4, 150_000_000_000 // each, 1_000_000_000 // size))
        c = _attend("", dtype, shape, _log(rng, 1, most), (rng.randint(1, hi), hi), cached)
    c.pop("name", None)
    return c


# ---------------------------------------------------------------------- inputs
def _lengths(c):
    """(cached tokens, nodes) per sequence, the same for every seed."""
    rng = np.random.default_rng(1337)
    new = rng.integers(c["new_min"], c["new_max"] + 1, c["seqs"])
    cached = rng.integers(c["cached_min"], c["cached_max"] + 1, c["seqs"])
    return cached.astype(np.int64), new.astype(np.int64)


def _kept(c):
    """Nodes of each accepted path in the `keep` cases, the same for every seed."""
    _, new = _lengths(c)
    return np.minimum(np.random.default_rng(7).integers(1, 8, c["seqs"]), (new + 1) // 2)


def _parents(new, host):
    """A tree for each sequence: node i hangs below one of the nodes before it, at most
    MAX_DEPTH nodes deep."""
    most = int(new.max())
    parents = np.full((len(new), most), -1, dtype=np.int64)
    depth = np.zeros((len(new), most), dtype=np.int64)
    rows = np.arange(len(new))
    for i in range(1, most):
        p = host.integers(max(0, i - 24), i, len(new))
        deep = depth[rows, p] >= MAX_DEPTH - 1
        p = np.where(deep, parents[rows, p], p)
        parents[:, i], depth[:, i] = p, depth[rows, p] + 1
    return parents


def _packed(dense, new):
    return torch.from_numpy(np.concatenate([row[:n] for row, n in zip(dense, new)])).to(DEVICE)


def _tables(c, host, need):
    num_blocks = int(need.sum()) * 5 // 4 + 1
    ids = host.permutation(num_blocks)
    tables = np.zeros((len(need), max(1, int(need.max()))), dtype=np.int64)
    at = 0
    for i, n in enumerate(need):
        tables[i, :n] = ids[at:at + n]
        at += n
    return num_blocks, torch.from_numpy(tables).to(DEVICE)


def prepare(case, seed):
    c = case
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    host = np.random.default_rng(seed)
    s = SimpleNamespace(case=c)
    if c["op"] == "logprobs":
        n, v = c["rows"], c["vocab"]
        x = torch.empty(n, v, device=DEVICE).normal_(0.0, 2.5, generator=g)
        # Trained models put most of a row's weight on a few tokens; every eighth row is of a
        # decode with a grammar, which leaves the lower half of the vocabulary.
        half = v // 2
        peaks = torch.from_numpy(host.integers(0, half, (n, 8))).to(DEVICE)
        x.scatter_add_(1, peaks, torch.empty(n, 8, device=DEVICE).uniform_(3.0, 12.0, generator=g))
        x[::8, half:] = -math.inf
        s.logits = x.to(DTYPES[c["dtype"]])
        ids = host.integers(0, half, n)
        s.ids = torch.where(torch.from_numpy(host.random(n) < 0.7).to(DEVICE), peaks[:, 0],
                            torch.from_numpy(ids).to(DEVICE))
        return s
    cached, new = _lengths(c)
    s.tokens, s.max_new = int(new.sum()), int(new.max())
    s.ctx_host, s.new_host = torch.from_numpy(cached + new), torch.from_numpy(new)
    s.ctx, s.new = s.ctx_host.to(DEVICE), s.new_host.to(DEVICE)
    s.start = torch.cat([s.new.new_zeros(1), s.new.cumsum(0)])
    dense = _parents(new, host)
    s.parents = _packed(dense, new)
    if c["op"] == "layout":
        return s
    if c["op"] == "accept":
        # The drafted tokens, and the target's token after each node: along one path of a tree
        # they agree down to some depth, elsewhere by chance only.
        target = host.integers(0, GPT2_VOCAB, dense.shape)
        token = host.integers(0, GPT2_VOCAB, dense.shape)
        for i, n in enumerate(new):
            path, at = [], int(host.integers(0, n))
            while at > 0:
                path.append(at)
                at = int(dense[i, at])
            for node in path[::-1][:int(host.integers(0, MAX_DEPTH))]:
                token[i, node] = target[i, dense[i, node]]
        s.token, s.target = _packed(token, new), _packed(target, new)
        return s
    need = -(-(cached + new) // c["block_size"])
    num_blocks, s.tables = _tables(c, host, need)
    dt, kv, d = DTYPES[c["dtype"]], c["kv_heads"], c["head_dim"]
    shape = (num_blocks, c["block_size"], kv, d)
    if c["op"] == "attend":
        # Keys and values whose size varies by row; queries a little larger than unit, so that
        # scores spread over several units, as in trained heads.
        def rows():
            x = torch.empty(shape, device=DEVICE).normal_(generator=g)
            return x.mul_(torch.empty(*shape[:3], 1, device=DEVICE).normal_(0.0, 0.5, generator=g).exp_()).to(dt)

        s.k, s.v = rows(), rows()
        s.q = torch.empty(s.tokens, c["heads"], d, device=DEVICE).normal_(0.0, 1.5, generator=g).to(dt)
        s.scale = d ** -0.5
        # From `layout` before the first layer.
        s.masks, _ = _plain_layout(s.parents, s.start, s.new, s.ctx, s.max_new)
        s.dense_parents = dense
        return s
    # keep: accepted paths whose moved nodes lie behind the places that they move to, so that a
    # pass can be repeated.
    kept = _kept(c)
    paths = np.full((c["seqs"], int(kept.max())), -1, dtype=np.int64)
    for i, (n, m) in enumerate(zip(new, kept)):
        paths[i, 0] = 0
        paths[i, 1:m] = np.sort(host.choice(np.arange(m, n), m - 1, replace=False))
    s.paths = torch.from_numpy(paths).to(DEVICE)
    if own:
        s.pool = _framework().PagedKVPool(_framework().ModelDims(c["layers"], kv, d, dt), num_blocks, c["block_size"],
                                          DEVICE)
        s.k, s.v = s.pool.k, s.pool.v
    else:
        s.k, s.v = ([torch.empty(shape, dtype=dt, device=DEVICE) for _ in range(c["layers"])] for _ in range(2))
    for t in s.k + s.v:
        t.normal_(generator=g)
    return s


# ---------------------------------------------------------------------- run
def run(state):
    s, c = state, state.case
    if c["op"] == "logprobs":
        if own:
            got = _framework().token_logprobs(s.logits, s.ids, top=c["top"])
            return {"logprobs": got.logprobs, "ranks": got.ranks, "entropy": got.entropy,
                    "top_logprobs": got.top_logprobs, "top_ids": got.top_ids}
        return _plain_logprobs(s.logits, s.ids, c["top"])
    if c["op"] == "layout":
        if own:
            masks, positions = _framework().tree_layout(s.parents, s.start, s.ctx, s.max_new)
        else:
            masks, positions = _plain_layout(s.parents, s.start, s.new, s.ctx, s.max_new)
        return {"masks": masks, "positions": positions}
    if c["op"] == "accept":
        if own:
            got = _framework().accept_tree(s.token, s.parents, s.target, s.start, MAX_DEPTH)
            return {"paths": got.paths, "counts": got.counts, "next": got.next_tokens}
        return _plain_accept(s.token, s.parents, s.target, s.start, s.new, s.max_new)
    if c["op"] == "keep":
        if own:
            s.pool.keep_paths(s.tables, s.ctx, s.start, s.paths)
        else:
            _plain_keep(s.k, s.v, s.tables, s.ctx - s.new, s.paths, c["block_size"])
        return {"k": s.k, "v": s.v}
    if own:
        f = _framework()
        ctx, new = f.attach_host(s.ctx, s.ctx_host), f.attach_host(s.new, s.new_host)
        return {"out": f.paged_tree_attention(s.q, s.k, s.v, s.tables, ctx, new, s.masks, s.scale)}
    return {"out": _plain_attention(s.q, s.k, s.v, s.tables, s.ctx, s.new, s.start, s.masks, s.scale,
                                    int(s.ctx_host.max()), s.max_new)}


_imported = None


def _framework():
    """The entry points that a user calls, on the library's kernels."""
    global _imported
    if _imported is None:
        os.environ["ATTENTION"] = "hip"
        sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "llm-inference-server_amd"))
        from inference_server.core.attention_hip import attach_host
        from inference_server.core.kv_pool import ModelDims, PagedKVPool
        from inference_server.core.sampling import token_logprobs
        from inference_server.core.token_tree import accept_tree, paged_tree_attention, tree_layout

        _imported = SimpleNamespace(attach_host=attach_host, ModelDims=ModelDims, PagedKVPool=PagedKVPool,
                                    token_logprobs=token_logprobs, accept_tree=accept_tree,
                                    paged_tree_attention=paged_tree_attention, tree_layout=tree_layout)
    return _imported


# ---------------------------------------------------------------------- plain forms
def _rows(start, new, most):
    """Row of node t of each sequence [seqs, most], and whether there is one."""
    t = torch.arange(most, device=start.device)
    live = t < new[:, None]
    return torch.where(live, start[:-1, None] + t, 0), live


def _plain_layout(parents, start, new, ctx, most):
    rows, live = _rows(start, new, most)
    t = torch.arange(most, device=start.device)
    up = torch.where(live, parents[rows], -1)
    seen = (t == t[:, None]).expand(len(new), most, most) & live[..., None]
    # Each round doubles the ancestors that a node knows of.
    for _ in range(max(1, (most - 1).bit_length())):
        at = up.clamp(min=0)
        seen = seen | torch.where((up >= 0)[..., None], seen.gather(1, at[..., None].expand_as(seen)), False)
        up = torch.where(up >= 0, up.gather(1, at), -1)
    words = -(-most // 64)
    bits = torch.zeros(len(new), most, words * 64, dtype=torch.long, device=start.device)
    bits[..., :most] = seen
    masks = (bits.view(len(new), most, words, 64) << torch.arange(64, device=start.device)).sum(-1)
    positions = (ctx - new)[:, None] + seen.sum(-1) - 1
    return masks[live], positions[live]


def _plain_attention(q, k, v, tables, ctx, new, start, masks, scale, max_ctx, most):
    tokens, heads, dim = q.shape
    bs, kv = k.shape[1:3]
    seqs = ctx.shape[0]
    wide = tables[:, :-(-max_ctx // bs)]
    keys = k[wide].float().flatten(1, 2).transpose(1, 2)                      # [seqs, kv, keys, dim]
    vals = v[wide].float().flatten(1, 2).transpose(1, 2)
    rows, live = _rows(start, new, most)
    qs = q[rows].float().view(seqs, most, kv, heads // kv, dim).permute(0, 2, 3, 1, 4)
    score = torch.matmul(qs.reshape(seqs, kv, -1, dim), keys.transpose(-1, -2)) * scale
    score = score.view(seqs, kv, heads // kv, most, -1)
    node = torch.arange(score.shape[-1], device=q.device) - (ctx - new)[:, None]          # [seqs, keys]
    at = node.clamp(0, masks.shape[1] * 64 - 1)
    words = masks[rows].gather(2, (at // 64)[:, None].expand(-1, most, -1))   # [seqs, nodes, keys]
    seen = (node < 0)[:, None] | (((words >> (at % 64)[:, None]) & 1) > 0) & (node < new[:, None])[:, None]
    score = score.masked_fill(~seen[:, None, None], -math.inf)
    w = torch.exp(score - score.amax(-1, keepdim=True))
    total = w.sum(-1, keepdim=True)
    out = torch.matmul(w.flatten(2, 3), vals).view(seqs, kv, heads // kv, most, dim) / total
    return out.permute(0, 3, 1, 2, 4).reshape(seqs, most, heads, dim)[live].to(q.dtype)


def _plain_logprobs(logits, ids, top):
    x = logits.float()
    own_x = x.gather(1, ids[:, None])
    m = x.amax(1, keepdim=True)
    d = x - m
    e = torch.exp(d)
    z = e.sum(1, keepdim=True)
    log_z = torch.log(z)
    entropy = log_z - torch.where(e > 0, e * d, 0.0).sum(1, keepdim=True) / z
    del d, e
    ranks = (x > own_x).sum(1) + 1
    values, order = torch.sort(x, dim=1, descending=True, stable=True)
    return {"logprobs": (own_x - m - log_z)[:, 0], "ranks": ranks, "entropy": entropy[:, 0],
            "top_logprobs": values[:, :top] - m - log_z, "top_ids": order[:, :top].clone()}


def _plain_accept(token, parents, target, start, new, most):
    rows, live = _rows(start, new, most)
    token, parents = token[rows], torch.where(live, parents[rows], -2)
    target = target[rows]
    t = torch.arange(most, device=start.device)
    at = torch.zeros_like(new)
    going = new > 0
    counts = going.long()
    paths = torch.full((len(new), MAX_DEPTH), -1, dtype=torch.long, device=start.device)
    paths[:, 0] = torch.where(going, 0, -1)
    for d in range(1, MAX_DEPTH):
        fits = (parents == at[:, None]) & (token == target.gather(1, at[:, None])) & going[:, None]
        first = torch.where(fits, t, most).amin(1)
        going = first < most
        at = torch.where(going, first, at)
        paths[:, d] = torch.where(going, first, -1)
        counts = counts + going
    return {"paths": paths, "counts": counts, "next": target.gather(1, at[:, None])[:, 0]}


def _plain_keep(k, v, tables, cached, paths, bs):
    d = torch.arange(paths.shape[1], device=tables.device)
    to = cached[:, None] + torch.where(paths < 0, 0, d)
    source = cached[:, None] + paths.clamp(min=0)                             # past a path's end: node 0 to itself
    slot = lambda pos: (tables.gather(1, pos // bs) * bs + pos % bs).flatten()  # noqa: E731
    to, source = slot(to), slot(source)
    for t in k + v:
        rows = t.view(-1, *t.shape[2:])
        rows[to] = rows[source]


# ---------------------------------------------------------------------- work
def work(case):
    c = case
    size = {"fp32": 4}.get(c.get("dtype"), 2)
    if c["op"] == "logprobs":
        n = c["rows"] * c["vocab"]
        return {"bytes": n * size + c["rows"] * (8 + 16 + 12 * c["top"]), "flops": 4 * n}
    cached, new = _lengths(c)
    tokens = int(new.sum())
    if c["op"] == "layout":
        return {"bytes": 8 * (tokens * (2 + -(-int(new.max()) // 64)) + 2 * c["seqs"]), "flops": 0}
    if c["op"] == "accept":
        return {"bytes": 8 * (3 * tokens + (MAX_DEPTH + 3) * c["seqs"]), "flops": 0}
    if c["op"] == "keep":
        rows = int((_kept(c) - 1).sum())
        return {"bytes": 2 * c["layers"] * 2 * rows * c["kv_heads"] * c["head_dim"] * size
                + 8 * int((_kept(c) + 4).sum()), "flops": 0}
    row = c["heads"] * c["head_dim"]
    # A node sees the cached tokens and itself at least.
    return {"bytes": 2 * int((cached + new).sum()) * c["kv_heads"] * c["head_dim"] * size + 2 * tokens * row * size,
            "flops": 4 * int((new * (cached + 1)).sum()) * row}


# ---------------------------------------------------------------------- exact
def exact(case, seed):
    """The definitions in 64 bits, sequences and rows one by one, trees from their parents."""
    c = case
    s = prepare(case, seed)
    if c["op"] == "logprobs":
        return _exact_logprobs(s, c)
    new, ctx = s.new_host.tolist(), s.ctx_host.tolist()
    long = lambda x: torch.tensor(x, dtype=torch.long)  # noqa: E731
    if c["op"] == "keep":
        k, v = [t.cpu() for t in s.k], [t.cpu() for t in s.v]
        tables, paths, bs = s.tables.tolist(), s.paths.tolist(), c["block_size"]
        for i, path in enumerate(paths):
            first = ctx[i] - new[i]
            for d, node in enumerate(path):
                if node < 0:
                    break
                a, b = first + node, first + d
                for t in k + v:
                    t[tables[i][b // bs], b % bs] = t[tables[i][a // bs], a % bs]
        return {"k": k, "v": v}
    parents, starts = s.parents.tolist(), s.start.tolist()
    if c["op"] == "accept":
        token, target = s.token.tolist(), s.target.tolist()
        paths, counts, following = [], [], []
        for at, n in zip(starts, new):
            path, going = [0], True
            while going and len(path) < MAX_DEPTH:
                going = False
                for child in range(path[-1] + 1, n):
                    if parents[at + child] == path[-1] and token[at + child] == target[at + path[-1]]:
                        path.append(child)
                        going = True
                        break
            counts.append(len(path))
            following.append(target[at + path[-1]])
            paths.append(path + [-1] * (MAX_DEPTH - len(path)))
        return {"paths": long(paths), "counts": long(counts), "next": long(following)}
    # Ancestors of each node, itself among them.
    lines = []
    for at, n in zip(starts, new):
        for node in range(n):
            up = parents[at + node]
            lines.append((lines[at + up] if up >= 0 else []) + [node])
    if c["op"] == "layout":
        words = -(-max(new) // 64)
        masks = np.zeros((len(lines), words), dtype=np.uint64)
        for t, line in enumerate(lines):
            for node in line:
                masks[t, node // 64] |= np.uint64(1) << np.uint64(node % 64)
        first = [n - m for n, m in zip(ctx, new) for _ in range(m)]
        return {"masks": torch.from_numpy(masks.view(np.int64)),
                "positions": long([f + len(line) - 1 for f, line in zip(first, lines)])}
    group, bs = c["heads"] // c["kv_heads"], c["block_size"]
    out = torch.empty(s.q.shape, dtype=torch.float64, device=DEVICE)
    for i, (at, m, n) in enumerate(zip(starts, new, ctx)):
        ids = s.tables[i, :-(-n // bs)]
        k, v = (x[ids].double().reshape(-1, c["kv_heads"], c["head_dim"])[:n].transpose(0, 1).contiguous()
                for x in (s.k, s.v))
        hidden = torch.zeros(m, n, dtype=torch.bool)
        hidden[:, n - m:] = True
        for node in range(m):
            hidden[node, [n - m + j for j in lines[at + node]]] = False
        hidden = hidden.to(DEVICE)
        for h in range(c["heads"]):
            score = s.q[at:at + m, h].double() @ k[h // group].t().contiguous() * s.scale
            out[at:at + m, h] = score.masked_fill(hidden, -math.inf).softmax(-1) @ v[h // group]
    return {"out": out}


def _exact_logprobs(s, c):
    n, top = c["rows"], c["top"]
    out = {"logprobs": torch.empty(n, dtype=torch.float64), "ranks": torch.empty(n, dtype=torch.long),
           "entropy": torch.empty(n, dtype=torch.float64), "top_logprobs": torch.empty(n, top, dtype=torch.float64),
           "top_ids": torch.empty(n, top, dtype=torch.long)}
    for i in range(n):
        x = s.logits[i].double()
        logp = torch.log_softmax(x, 0)
        p = logp.exp()
        out["logprobs"][i] = logp[s.ids[i]]
        out["ranks"][i] = (x > x[s.ids[i]]).sum() + 1
        out["entropy"][i] = -(p[p > 0] * logp[p > 0]).sum()
        if top:
            # Everything at least as large as the k-th, in the order of index, then by value.
            least = x.topk(top).values[-1]
            at = torch.nonzero(x >= least)[:, 0]
            order = at[torch.argsort(x[at], descending=True, stable=True)][:top]
            out["top_ids"][i], out["top_logprobs"][i] = order.cpu(), logp[order].cpu()
    return out
