"""Block tables and slot maps of a step, from request lengths, on the device.

`BlockTable` (core/block_table.py) and `PagedExecutor._host_step` lay a step out on the
host, sequence by sequence, and upload the result. `step_layout` does it for a batch whose
tables, lengths and free list live on the device (reference: core/block_table.py:70-108,
137-159 for the arithmetic, core/paged_executor.py:211-263 for the packing), so that a step
can be prepared, or replayed from a graph, without the host reading a length.

Who does it depends on CONFIG.kv_backend, as for the pool's byte movers: "torch" runs tensor
ops on any device, "hip" one launch of libpagedkv (`pkv_step_layout`).
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from inference_server import native
from inference_server.config import CONFIG


class StepLayout(NamedTuple):
    """int64 tensors on the tables' device."""

    block_tables: torch.Tensor   # [B, W]: the argument, its new blocks written in place
    held: torch.Tensor           # [B]: blocks held now
    slots: torch.Tensor          # [T]: flat pool slot of each new token, -1 past the last one
    positions: torch.Tensor      # [T]: its position in its sequence, 0 past the last one
    query_start: torch.Tensor    # [B + 1]: first new token of each sequence
    counts: torch.Tensor         # [3]: blocks taken, blocks needed, impossible lengths


def step_layout(block_tables: torch.Tensor, held: torch.Tensor, context_lens: torch.Tensor, query_lens: torch.Tensor,
                free_blocks: torch.Tensor, block_size: int, num_tokens: int) -> StepLayout:
    """Give every sequence the blocks that its context needs and every new token its slot.

    block_tables [B, W]: row i holds held[i] blocks; context_lens [B]: tokens cached after
    the step; query_lens [B]: the new ones among them, the context's last; free_blocks [F]:
    ids that may be taken, from the front, in sequence order (the caller drops
    counts[0] of them afterwards). num_tokens: rows of the packed step, at least the sum of
    query_lens; the rest is padding. All int64.

    All or nothing, as BlockTable.ensure_capacity: if the free list is short (counts[1] >
    F) or a length is impossible (counts[2] > 0: a query length below 0 or above its
    context, a context wider than the table, held outside it, more new tokens than
    num_tokens), nothing is taken or written, every slot is -1 and query_start is all 0.
    `held` is not changed: the call can be repeated."""
    inputs = (("block_tables", block_tables), ("held", held), ("context_lens", context_lens),
              ("query_lens", query_lens), ("free_blocks", free_blocks))
    if block_tables.dim() != 2:
        raise ValueError(f"block_tables must be [batch, width], got {tuple(block_tables.shape)}")
    batch, width = block_tables.shape
    for name, t in inputs[1:4]:
        if t.dim() != 1 or t.shape[0] != batch:
            raise ValueError(f"{name} must be [{batch}] to match block_tables, got {tuple(t.shape)}")
    if free_blocks.dim() != 1:
        raise ValueError(f"free_blocks must be one row of block ids, got {tuple(free_blocks.shape)}")
    if block_size < 1 or num_tokens < 0:
        raise ValueError(f"block_size must be positive and num_tokens not negative, got {block_size}, {num_tokens}")
    where = block_tables.get_device()
    for name, t in inputs:
        if t.dtype is not torch.long:
            raise ValueError(f"{name} must be int64, got {t.dtype}")
        if t.get_device() != where:
            raise ValueError(f"{name} is on {t.device}, block_tables on {block_tables.device}")
    if CONFIG.kv_backend != "hip":
        return _layout_torch(block_tables, held, context_lens, query_lens, free_blocks, block_size, num_tokens)
    native.require_gpu(block_tables, "step_layout")
    stride = block_tables.stride()
    if batch and (width > 1 and stride[1] != 1 or batch > 1 and stride[0] < width):
        raise ValueError(f"block_tables are written in place: rows must be contiguous and distinct, "
                         f"got strides {stride}")
    held, context_lens = held.contiguous(), context_lens.contiguous()
    query_lens, free_blocks = query_lens.contiguous(), free_blocks.contiguous()
    dev = block_tables.device
    with native.on_device(dev):
        # One allocation: held | query_start | counts | slots | positions.
        buf = torch.empty(2 * batch + 4 + 2 * num_tokens, dtype=torch.long, device=dev)
        new_held, starts, counts, slots, positions = buf.split_with_sizes(
            (batch, batch + 1, 3, num_tokens, num_tokens))
        rc = native.lib().pkv_step_layout(
            block_tables.data_ptr(), stride[0], width, held.data_ptr(), context_lens.data_ptr(),
            query_lens.data_ptr(), batch, free_blocks.data_ptr(), free_blocks.shape[0], block_size, num_tokens,
            new_held.data_ptr(), slots.data_ptr(), positions.data_ptr(), starts.data_ptr(), counts.data_ptr(),
            native.stream_handle(dev))
        native.check(rc, "pkv_step_layout")
    return StepLayout(block_tables, new_held, slots, positions, starts, counts)


def _layout_torch(tables, held, ctx, new, free, bs, tokens) -> StepLayout:
    batch, width = tables.shape
    need = torch.where(ctx > 0, (ctx - 1).div(bs, rounding_mode="floor") + 1, 0)
    bad = (new < 0) | (new > ctx) | (held < 0) | (held > width) | (need > width)
    q = torch.where(bad, 0, new)
    fresh = torch.where(bad, 0, need - held).clamp(min=0)
    start = torch.cat([q.new_zeros(1), q.cumsum(0)])
    wanted, wrong = fresh.sum(), bad.sum() + (start[-1] > tokens)
    ok = (wrong == 0) & (wanted <= free.shape[0])
    counts = torch.stack([torch.where(ok, wanted, 0), wanted, wrong])
    slots, positions = tables.new_full((tokens,), -1), tables.new_zeros(tokens)
    if batch and width:
        first = fresh.cumsum(0) - fresh
        col = torch.arange(width, device=tables.device)
        take = (col >= held[:, None]) & (col < (held + fresh)[:, None]) & ok
        if free.shape[0]:
            pick = (first[:, None] + col - held[:, None]).clamp(0, free.shape[0] - 1)
            tables.copy_(torch.where(take, free[pick], tables))
        t = torch.arange(tokens, device=tables.device)
        seq = torch.searchsorted(start[1:], t, right=True).clamp(max=batch - 1)
        real = ok & (t < start[-1])
        positions = torch.where(real, ctx[seq] - new[seq] + t - start[seq], 0)
        slots = torch.where(real, tables[seq, (positions // bs).clamp(0, width - 1)] * bs + positions % bs, -1)
    return StepLayout(tables, torch.where(ok, held + fresh, held), slots, positions,
                      torch.where(ok, start, 0), counts)
