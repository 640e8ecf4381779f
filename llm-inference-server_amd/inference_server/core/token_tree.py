"""Steps that verify drafted token trees: masks and positions of the nodes, their attention over
the paged cache, and the path that the target model accepts.

A sequence's new tokens of such a step are the nodes of a tree of continuations, in an order in
which parents come first; node 0 is the token that was sampled before. In the cache they take the
sequence's last positions, in that order (step_layout's slots), while a node's position for
the model is the cached tokens plus its depth. A step is

    layout = step_layout(...)                                   # slots, query starts
    attach_host(context_lens, bounds), attach_host(query_lens, more_bounds)
    attach_query_start(query_lens, layout.query_start)
    tree = tree_layout(parents, layout.query_start, context_lens, max_nodes)
    # per layer: append K/V to layout.slots, then
    paged_tree_attention(q, k, v, layout.block_tables, context_lens, query_lens, tree.masks, scale)
    # logits of all nodes: targets = their argmax, or samples; token_logprobs(logits, ...)
    path = accept_tree(tokens, parents, targets, layout.query_start, max_depth)
    pool.keep_paths(layout.block_tables, context_lens, layout.query_start, path.paths)

after which a sequence has its cached tokens and path.counts more, and path.next_tokens is
sampled. The reference has no such steps; the contract of the attention is core/attention.py's.

These operators leave their results on the device and read nothing back but the lengths, which the
attention checks on the host: without the attached copies it reads both from the device in every call, every
layer's. path.counts, and so the next step's lengths, only the device knows: the copies may be bounds (attach_host says
which), and the layout's query starts are then what the kernels go by. Outside these operators, PagedKVPool.append reads
its slots back unless it is given host_slots.

Who computes follows CONFIG, as for the operators beside these: tensor ops on any device, or,
with ATTENTION=hip, libpagedkv's kernels, never falling back.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from inference_server import native
from inference_server.config import CONFIG
from inference_server.core.attention import check_contract
from inference_server.core.attention_hip import (_ALONE, _WORKSPACES, _attached_start, _on_device, _query_start,
                                                 _step_facts)

#: Most nodes of a sequence that the layout and the walk take.
MAX_NODES = 8192


class TreeLayout(NamedTuple):
    """int64 tensors on the parents' device."""

    masks: torch.Tensor       # [T, ceil(max_nodes / 64)]: bit j % 64 of word j / 64: sees node j
    positions: torch.Tensor   # [T]: cached tokens + depth


class TreePath(NamedTuple):
    """int64 tensors on the tokens' device."""

    paths: torch.Tensor         # [B, max_depth]: accepted nodes, -1 past the last
    counts: torch.Tensor        # [B]: how many
    next_tokens: torch.Tensor   # [B]: the target's token at the last one


def _check_rows(inputs, query_start: torch.Tensor) -> tuple[int, int]:
    """(tokens, sequences) of int64 rows [T] and query starts [B + 1], on one device."""
    name0, first = inputs[0]
    rows, starts, dev = first.shape, query_start.shape, first.get_device()
    if len(rows) != 1:
        raise ValueError(f"{name0} must be one row of tokens, got {tuple(rows)}")
    if len(starts) != 1 or starts[0] < 1:
        raise ValueError(f"query_start must be [batch + 1], got {tuple(starts)}")
    for name, t in inputs:
        if t.dtype is not torch.long:
            raise ValueError(f"{name} must be int64, got {t.dtype}")
        if t is not first:
            if t.get_device() != dev:
                raise ValueError(f"{name} is on {t.device}, {name0} on {first.device}")
            if t.shape != rows:
                raise ValueError(f"{name} must be [{rows[0]}] to match {name0}, got {tuple(t.shape)}")
    if query_start.dtype is not torch.long:
        raise ValueError(f"query_start must be int64, got {query_start.dtype}")
    if query_start.get_device() != dev:
        raise ValueError(f"query_start is on {query_start.device}, {name0} on {first.device}")
    return rows[0], starts[0] - 1


def _dense(t: torch.Tensor) -> torch.Tensor:
    return t if t.is_contiguous() else t.contiguous()


# ----------------------------------------------------------------------- layout
def tree_layout(parents: torch.Tensor, query_start: torch.Tensor, context_lens: torch.Tensor,
                max_nodes: int) -> TreeLayout:
    """What each node sees, itself and its ancestors, and its position.

    parents [T]: a node's parent as its number in the sequence, -1 for a root; query_start
    [B + 1]: the sequences' first rows (step_layout's); context_lens [B]: tokens cached after the
    step, the nodes among them. max_nodes: the most nodes of a sequence, 8,192 at most. All int64.

    Masks of 0 and position 0 for rows of no sequence, for a node whose parent is not
    before it and the nodes below that one, and for sequences with more nodes than max_nodes or
    than their context, or rows past the last token: the host does not read the lengths back to refuse them."""
    tokens, batch = _check_rows((("parents", parents),), query_start)
    if context_lens.dim() != 1 or context_lens.shape[0] != batch:
        raise ValueError(f"context_lens must be [{batch}] to match query_start, got {tuple(context_lens.shape)}")
    if context_lens.dtype is not torch.long:
        raise ValueError(f"context_lens must be int64, got {context_lens.dtype}")
    if context_lens.get_device() != parents.get_device():
        raise ValueError(f"context_lens is on {context_lens.device}, parents on {parents.device}")
    if not 0 <= max_nodes <= MAX_NODES:
        raise ValueError(f"max_nodes must be between 0 and {MAX_NODES}, got {max_nodes}")
    words = -(-max_nodes // 64)
    if CONFIG.kv_backend != "hip":
        return _layout_torch(parents, query_start, context_lens, max_nodes, words)
    native.require_gpu(parents, "tree_layout")
    dev = parents.device
    with native.on_device(dev):
        parents, query_start, context_lens = _dense(parents), _dense(query_start), _dense(context_lens)
        # One allocation, and the views that cost least: the call is bound by its host time.
        buf = torch.empty(tokens * (words + 1), dtype=torch.long, device=dev)
        masks = buf.as_strided((tokens, words), (words, 1))
        positions = buf.as_strided((tokens,), (1,), tokens * words)
        rc = native.lib().pkv_tree_layout(
            parents.data_ptr(), query_start.data_ptr(), context_lens.data_ptr(), batch, tokens, max_nodes,
            masks.data_ptr(), positions.data_ptr(), native.stream_handle(dev))
        native.check(rc, "pkv_tree_layout")
    return TreeLayout(masks, positions)


def _nodes(starts: torch.Tensor, tokens: int, most: int):
    """Of each row: its sequence, its number there, and whether the sequence's bounds are possible;
    of each sequence: its nodes, 0 where they are not."""
    begin, end = starts[:-1], starts[1:]
    counts = torch.where((begin >= 0) & (begin <= end) & (end <= tokens) & (end - begin <= most), end - begin, 0)
    t = torch.arange(tokens, device=starts.device)
    seq = torch.searchsorted(end.contiguous(), t, right=True).clamp(max=max(0, len(begin) - 1))
    node = t - begin[seq]
    return seq, node, (node >= 0) & (node < counts[seq]), counts


def _layout_torch(parents, starts, ctx, max_nodes, words) -> TreeLayout:
    tokens, dev = parents.shape[0], parents.device
    masks, positions = torch.zeros(tokens, words, dtype=torch.long, device=dev), torch.zeros_like(parents)
    if tokens == 0 or starts.shape[0] == 1 or max_nodes == 0:
        return TreeLayout(masks, positions)
    seq, node, real, counts = _nodes(starts, tokens, max_nodes)
    cached = ctx - counts
    good = real & (cached[seq] >= 0) & (parents >= -1) & (parents < node)
    # Each round doubles the ancestors that a node knows of.
    up = torch.where(good & (parents >= 0), starts[seq] + parents, -1)
    seen = torch.zeros(tokens, words * 64, dtype=torch.bool, device=dev)
    seen.scatter_(1, torch.where(real, node, 0)[:, None], True)
    for _ in range(max(1, (max_nodes - 1).bit_length())):
        at, has = up.clamp(min=0), up >= 0
        seen = seen | (seen[at] & has[:, None])
        good = good & (good[at] | ~has)
        up = torch.where(has, up[at], -1)
    seen = seen & good[:, None]
    bits = seen.view(tokens, words, 64).long() << torch.arange(64, device=dev)
    return TreeLayout(bits.sum(-1), torch.where(good, cached[seq] + seen.sum(-1) - 1, 0))


# ----------------------------------------------------------------------- accept
def accept_tree(tokens: torch.Tensor, parents: torch.Tensor, targets: torch.Tensor, query_start: torch.Tensor,
                max_depth: int) -> TreePath:
    """The path of each tree that the target model agrees with: from node 0, on to the first
    child whose token is the target's token at the node, until there is none. Where a node's children have
    tokens of their own, as a draft's likeliest ones have, that is the longest such path; of children with one token
    the walk takes the first, also where only another goes on.

    tokens, parents, targets [T]: the nodes' tokens, their parents' numbers, and the target's token
    after each node (its argmax, or a sample); query_start [B + 1]; all int64. At most
    max_depth nodes are accepted. A sequence without nodes, or with more than 8,192, has count 0 and next
    token -1."""
    n_tok, batch = _check_rows((("tokens", tokens), ("parents", parents), ("targets", targets)), query_start)
    if not 1 <= max_depth <= MAX_NODES:
        raise ValueError(f"max_depth must be between 1 and {MAX_NODES}, got {max_depth}")
    if CONFIG.kv_backend != "hip":
        return _accept_torch(tokens, parents, targets, query_start, max_depth)
    native.require_gpu(tokens, "accept_tree")
    dev = tokens.device
    with native.on_device(dev):
        tokens, parents, targets, query_start = _dense(tokens), _dense(parents), _dense(targets), _dense(query_start)
        buf = torch.empty(batch * (max_depth + 2), dtype=torch.long, device=dev)
        paths = buf.as_strided((batch, max_depth), (max_depth, 1))
        counts = buf.as_strided((batch,), (1,), batch * max_depth)
        following = buf.as_strided((batch,), (1,), batch * (max_depth + 1))
        rc = native.lib().pkv_tree_accept(
            tokens.data_ptr(), parents.data_ptr(), targets.data_ptr(), query_start.data_ptr(), batch, n_tok, max_depth,
            paths.data_ptr(), counts.data_ptr(), following.data_ptr(), native.stream_handle(dev))
        native.check(rc, "pkv_tree_accept")
    return TreePath(paths, counts, following)


def _accept_torch(tokens, parents, targets, starts, max_depth) -> TreePath:
    n_tok, batch, dev = tokens.shape[0], starts.shape[0] - 1, tokens.device
    paths = torch.full((batch, max_depth), -1, dtype=torch.long, device=dev)
    if batch == 0 or n_tok == 0:
        return TreePath(paths, paths.new_zeros(batch), paths.new_full((batch,), -1))
    seq, node, real, nodes = _nodes(starts, n_tok, MAX_NODES)
    up = torch.where(real & (parents >= 0) & (parents < node), starts[seq] + parents, -1)
    fits = (up >= 0) & (tokens == targets[up.clamp(min=0)])
    first = torch.full((n_tok,), MAX_NODES, dtype=torch.long, device=dev)
    first.scatter_reduce_(0, up.clamp(min=0), torch.where(fits, node, MAX_NODES), "amin")
    base = torch.where(nodes > 0, starts[:-1], 0)
    at, last, counts = torch.where(nodes > 0, 0, -1), torch.full_like(nodes, -1), torch.zeros_like(nodes)
    for d in range(max_depth):
        paths[:, d] = at
        going = at >= 0
        counts += going
        last = torch.where(going, at, last)
        following = first[base + at.clamp(min=0)]
        at = torch.where(going & (following < MAX_NODES), following, -1)
        if not bool((at >= 0).any()):
            break
    return TreePath(paths, counts, torch.where(last >= 0, targets[base + last.clamp(min=0)], -1))


# ----------------------------------------------------------------------- attention
def paged_tree_attention(query: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor, block_tables: torch.Tensor,
                         context_lens: torch.Tensor, query_lens: torch.Tensor, masks: torch.Tensor,
                         scale: float) -> torch.Tensor:
    """`core.attention.paged_attention` for drafted trees: a sequence's query_lens[i] new tokens, its
    context's last, see the cached tokens before them, all of these, and of the new ones those
    whose bits are set in the token's row of masks (int64 [T, W], 64 W at least the longest
    query length): tree_layout's, or any others. Everything else is as there: query [T, heads,
    head_dim] in the pools' dtype (fp32, fp16, bf16), block_tables [B, W], context_lens and
    query_lens [B], the same checks and messages; returns [T, heads, head_dim].

    Softmax and sums are in fp32 and the output is rounded once. (ATTENTION=hip: weights meet 16-bit V as two
    pieces of its type, which leave at most 2^-16 of a bf16 weight, and of an fp16 one 2^-22, or 2^-38 of the row's
    largest where that is more; values of 2^100 and more in size, or scores of 2^126, in fp16 2^26, may leave
    the range.) The 8-bit cache has no such attention. A key that a token does
    not see does not reach it, whatever its K and V hold (NaN and infinities among it); a token that
    sees none gets zeros. Lengths with host copies attached (attach_host) are checked without a
    device round trip."""
    backend = CONFIG.attention
    if backend == "hip":
        return _attention_hip(query, k_pool, v_pool, block_tables, context_lens, query_lens, masks, scale)
    if backend == "gather":
        return _attention_gather(query, k_pool, v_pool, block_tables, context_lens, query_lens, masks, scale)
    if backend == "triton":
        raise NotImplementedError("ATTENTION=triton: this MI355X build ships no Triton kernel; use ATTENTION=hip "
                                  "(libpagedkv CDNA4 kernels) or ATTENTION=gather")
    raise ValueError(f"unknown ATTENTION={backend!r}; expected 'gather', 'triton' or 'hip'")


def _check_operands(query, k_pool, v_pool, tables, masks) -> None:
    if tables.dim() != 2:
        raise ValueError(f"block_tables must be [batch, width], got {tuple(tables.shape)}")
    if k_pool.shape != v_pool.shape:
        raise ValueError(f"k_pool {tuple(k_pool.shape)} and v_pool {tuple(v_pool.shape)} differ")
    dev, dtype = query.get_device(), query.dtype
    for name, t in (("k_pool", k_pool), ("v_pool", v_pool)):
        if t.get_device() != dev:
            raise ValueError(f"{name} is on {t.device}, query is on {query.device}")
        if t.dtype is not dtype:
            raise ValueError(f"{name} dtype {t.dtype} differs from query dtype {dtype}")
    heads, dim = query.shape[1:]
    kv, pool_dim = k_pool.shape[2:]
    if dim != pool_dim:
        raise ValueError(f"query head_dim {dim} != pool head_dim {pool_dim}")
    if heads % kv:
        raise ValueError(f"{heads} query heads not divisible by {kv} kv heads")
    if masks.dim() != 2 or masks.shape[0] != query.shape[0]:
        raise ValueError(f"masks must be [{query.shape[0]}, words], got {tuple(masks.shape)}")
    if masks.dtype is not torch.long:
        raise ValueError(f"masks must be int64, got {masks.dtype}")
    if masks.get_device() != dev:
        raise ValueError(f"masks is on {masks.device}, query is on {query.device}")


def _check_lengths(negative: bool, max_q: int, masks) -> None:
    if negative:
        raise ValueError("query_lens must not be negative")
    if max_q > 64 * masks.shape[1]:
        raise ValueError(f"masks of {masks.shape[1]} words hold fewer nodes than the {max_q} of a sequence")


def _attention_gather(query, k_pool, v_pool, tables, ctx, qlens, masks, scale):
    bs = k_pool.shape[1] if k_pool.dim() == 4 else 1
    width = tables.shape[1] if tables.dim() == 2 else 0
    check_contract(query.dim(), tuple(query.shape), k_pool.dim(), tuple(k_pool.shape), tables.shape, ctx.shape,
                   qlens.shape, lambda: (int(qlens.sum()), bool((qlens > ctx).any()),
                                         bool(((-(-ctx // bs)) > width).any())))
    _check_operands(query, k_pool, v_pool, tables, masks)
    _check_lengths(bool((qlens < 0).any()), int(qlens.max()) if qlens.numel() else 0, masks)
    group, dev = query.shape[1] // k_pool.shape[2], query.device
    out = torch.empty_like(query)
    start = 0
    for i, (n, m) in enumerate(zip(ctx.tolist(), qlens.tolist())):
        if m == 0:
            continue
        blocks = tables[i, :-(-n // bs)].to(dev, torch.long)
        keys, vals = (p[blocks].flatten(0, 1)[:n].float().transpose(0, 1).repeat_interleave(group, 0)
                      for p in (k_pool, v_pool))                              # [H, ctx, D]
        node = torch.arange(m, device=dev)
        seen = torch.ones(m, n, dtype=torch.bool, device=dev)
        seen[:, n - m:] = (masks[start:start + m][:, node // 64] >> (node % 64)) & 1 != 0
        q = query[start:start + m].float().transpose(0, 1).contiguous()
        scores = torch.matmul(q, keys.transpose(-1, -2).contiguous()) * scale
        scores = scores.masked_fill(~seen, float("-inf"))
        top = scores.amax(-1, keepdim=True)
        w = torch.exp(scores - torch.where(top == float("-inf"), 0.0, top))   # amax keeps NaN
        total = w.sum(-1, keepdim=True)
        finite = torch.isfinite(vals)
        o = torch.matmul(w / torch.where(total == 0, 1.0, total), torch.where(finite, vals, 0.0))
        if not bool(finite.all()):
            # Values that are not finite reach the tokens that see them alone.
            sees = seen.float().expand(vals.shape[0], m, n)
            for what, value in ((vals == float("inf"), float("inf")), (vals == float("-inf"), float("-inf")),
                                (torch.isnan(vals), float("nan"))):
                o = torch.where(torch.matmul(sees, what.float()) > 0, o + value, o)
        out[start:start + m] = o.transpose(0, 1).to(query.dtype)
        start += m
    return out


def _attention_hip(query, k_pool, v_pool, tables, context_lens, query_lens, masks, scale):
    native.require_gpu(query, "paged_tree_attention")
    q_shape, p_shape, t_shape = query.shape, k_pool.shape, tables.shape
    bs = p_shape[1] if len(p_shape) == 4 else 1
    width = t_shape[1] if len(t_shape) == 2 else 0
    facts: dict | None = None

    def values():
        nonlocal facts
        facts = _step_facts(context_lens, query_lens, bs, width)
        if "negative" not in facts:
            facts["negative"] = bool((facts["hql"] < 0).any())
        return facts["total"], facts["q_gt_c"], facts["too_few_blocks"]

    check_contract(len(q_shape), q_shape, len(p_shape), p_shape, t_shape, context_lens.shape, query_lens.shape, values)
    _check_operands(query, k_pool, v_pool, tables, masks)
    _check_lengths(facts["negative"], facts["max_q"], masks)
    dev, (n_tok, n_heads, head_dim) = query.device, q_shape
    dt = native.dtype_code(query.dtype)
    n_blocks, block_size, n_kv, _ = p_shape
    n_seqs = t_shape[0]
    with native.on_device(dev):
        out = torch.empty(q_shape, dtype=query.dtype, device=dev)
        if n_tok == 0 or n_seqs == 0:
            return out
        q_st = query.stride()
        if q_st[2] != 1:
            query = query.contiguous()
            q_st = query.stride()
        k_st = k_pool.stride()
        if k_st[3] != 1 or v_pool.stride() != k_st:
            k_pool, v_pool = k_pool.contiguous(), v_pool.contiguous()
            k_st = k_pool.stride()
        tables = _on_device(tables, dev)
        t_st = tables.stride()
        if t_st[1] != 1:
            tables = tables.contiguous()
            t_st = tables.stride()
        m_st, words = masks.stride(), masks.shape[1]
        if (words > 1 and m_st[1] != 1) or (n_tok > 1 and m_st[0] < words):
            masks = masks.contiguous()
            m_st = masks.stride()
        # (A lone row is contiguous whatever its stride.)
        mask_stride = m_st[0] if n_tok > 1 else words
        ctx_dev = _on_device(context_lens, dev).contiguous()
        stream = native.stream_handle(dev)
        qsl = _attached_start(query_lens, dev)
        if qsl is None:
            qsl = _query_start(facts, context_lens, dev, stream)
        lib = native.lib()
        max_q = facts["max_q"]
        lens = (facts["hctx"].data_ptr(), facts["hql"].data_ptr())
        # Workspace for contexts that are cut, sized by a step's first layer.
        key = ("tree", n_heads, n_kv, head_dim, n_tok, dt)
        ws_bytes = facts["split_ws"].get(key)
        if ws_bytes is None:
            ws_bytes = facts["split_ws"][key] = lib.pkv_tree_attention_workspace_bytes(
                n_seqs, n_heads, n_kv, head_dim, n_tok, max_q, dt, *lens)
        ws_ptr, ws_size = None, 0
        with _WORKSPACES.turn(dev, stream) if ws_bytes else _ALONE:
            if ws_bytes:
                # A capture's calls have one of their own: replays of graphs that were captured on
                # one stream may overlap.
                capturing = torch.cuda.is_current_stream_capturing()
                ws = (_WORKSPACES.of_capture if capturing else _WORKSPACES.partials)(dev, stream, ws_bytes)
                ws_ptr, ws_size = ws.data_ptr(), ws_bytes
            rc = lib.pkv_tree_attention(
                out.data_ptr(), n_heads * head_dim, head_dim, query.data_ptr(), q_st[0], q_st[1],
                k_pool.data_ptr(), v_pool.data_ptr(), k_st[0], k_st[1], k_st[2], n_blocks, block_size, n_kv, head_dim,
                tables.data_ptr(), t_st[0], width, ctx_dev.data_ptr(), qsl.data_ptr(),
                masks.data_ptr(), mask_stride, words, n_seqs, n_heads, n_tok, max_q, *lens,
                float(scale), dt, ws_ptr, ws_size, stream)
        native.check(rc, "pkv_tree_attention")
        return out
