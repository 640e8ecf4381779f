"""An 8-bit paged KV cache: its pool, the append that quantises into it, and the attention
that reads it. A token takes half the bytes of a 16-bit pool, so a budget holds twice the
tokens and a decode step moves half the memory.

Format. A cached row (one token, one KV head, K or V) is head_dim e4m3 codes and one
power-of-two scale, an exponent byte: torch.float8_e4m3fn and torch.float8_e8m0fnu, so a
row's value is `codes.float() * scale.float()`. The scale is the least with which the row's
largest magnitude is at most e4m3's 448. A power of two costs no relative precision (e4m3 has
an exponent of its own) and makes code * scale exact in bf16 and fp32, as far as their normal
numbers go: magnitudes from 1.9375 * 2^127 on round up to 2^128, infinity there. A row with a value that
is not finite is stored as the NaN row: scale NaN, codes 0.

Backends follow CONFIG.attention, as for the 16- and 32-bit pools: "gather" runs tensor ops
on any device (in fp32, on exact values), "hip" libpagedkv's kernels, never falling back.
The reference has no such cache; the contract of the attention is core/attention.py's.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from inference_server import native
from inference_server.config import CONFIG
from inference_server.core.attention import _gather_ragged, check_contract
from inference_server.core.attention_hip import (_ALONE, _WORKSPACES, _attached_start, _on_device, _query_start,
                                                 _step_facts)
from inference_server.core.kv_pool import ModelDims, PagedKVPool

CODES, SCALES = torch.float8_e4m3fn, torch.float8_e8m0fnu
_NAN_SCALE = 255
_QUERY_DTYPES = (torch.float32, torch.float16, torch.bfloat16)


class Kv8(NamedTuple):
    """One layer's K or V, or rows of it. Any strides; the kernels are fastest on the ones of
    Kv8Pool (rows of codes together, a head's scales of a block together)."""

    codes: torch.Tensor     # float8_e4m3fn [num_blocks, block_size, kv_heads, head_dim]
    scales: torch.Tensor    # float8_e8m0fnu [num_blocks, block_size, kv_heads]


def kv8_quantize(x: torch.Tensor) -> Kv8:
    """The rows x [..., head_dim] as the cache holds them."""
    x = x.float()
    m, e = torch.frexp(x.abs().amax(-1))                      # largest = m 2^e, m in [1/2, 1)
    b = (e + (127 - 9) + (m > 0.875)).clamp(min=0)            # 448 = 0.875 * 2^9
    b = torch.where(m == 0, 0, b)
    finite = torch.isfinite(x).all(-1)
    # One rounding: the product by a power of two is exact.
    y = torch.where(finite[..., None], x * torch.exp2((127 - b).float())[..., None], 0.0)
    b = torch.where(finite, b, _NAN_SCALE).to(torch.uint8)
    return Kv8(y.to(CODES), b.view(SCALES))


def kv8_dequantize(rows: Kv8) -> torch.Tensor:
    """fp32 values of cached rows."""
    return rows.codes.float() * rows.scales.float()[..., None]


def _check_cache(name: str, cache: Kv8) -> None:
    codes, scales = cache
    if codes.dim() != 4:
        raise ValueError(f"{name} codes must be [blocks, block_size, kv_heads, dim], got {tuple(codes.shape)}")
    if scales.shape != codes.shape[:3]:
        raise ValueError(f"{name} scales must be {tuple(codes.shape[:3])}, got {tuple(scales.shape)}")
    if codes.dtype is not CODES or scales.dtype is not SCALES:
        raise ValueError(f"{name} must be {CODES} codes and {SCALES} scales, got {codes.dtype} and {scales.dtype}")
    if scales.device != codes.device:
        raise ValueError(f"{name} codes are on {codes.device}, its scales on {scales.device}")


def _check_pair(k: Kv8, v: Kv8) -> torch.Size:
    """The caches' shape, checked; messages for what is wrong are found only if something is."""
    (kc, ks), (vc, vs) = k, v
    shape = kc.shape
    if (len(shape) == 4 and vc.shape == shape and kc.dtype is CODES and vc.dtype is CODES and ks.dtype is SCALES
            and vs.dtype is SCALES and ks.shape == vs.shape == shape[:3]
            and kc.get_device() == vc.get_device() == ks.get_device() == vs.get_device()):
        return shape
    _check_cache("k_cache", k)
    _check_cache("v_cache", v)
    if vc.shape != shape:
        raise ValueError(f"k_cache {tuple(shape)} and v_cache {tuple(vc.shape)} differ")
    raise ValueError(f"k_cache is on {kc.device}, v_cache on {vc.device}")


def _pointers(k: Kv8, v: Kv8) -> tuple | None:
    """The kernels' view of a cache: base pointers and strides, one set for K and V; None
    where it has no such view (codes' inner stride, or strides that differ)."""
    (kc, ks), (vc, vs) = k, v
    c, s = kc.stride(), ks.stride()
    if c[3] != 1 or vc.stride() != c or vs.stride() != s:
        return None
    return (kc.data_ptr(), vc.data_ptr(), c[0], c[1], c[2], ks.data_ptr(), vs.data_ptr(), s[0], s[1], s[2])


# ----------------------------------------------------------------------- append
def kv8_append(k_cache: Kv8, v_cache: Kv8, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor,
               host_slots: torch.Tensor | None = None) -> None:
    """Quantise rows k / v [T, kv_heads, head_dim] (fp32, fp16 or bf16, any strides) into flat
    slots [T] (block * block_size + offset) of one layer's cache. Slots are distinct.

    A slot outside the cache raises IndexError where the host knows the slots: `host_slots`,
    the same values on the CPU, or slots on the CPU themselves. On the device alone they are
    not read back: the kernel skips such rows (-1 is a padding row's slot)."""
    n_blocks, bs, heads, dim = _check_pair(k_cache, v_cache)
    shape = k.shape
    if len(shape) != 3 or shape[1] != heads or shape[2] != dim or v.shape != shape:
        raise ValueError(f"append rows {tuple(k.shape)} and {tuple(v.shape)} do not match cache rows [{heads}, {dim}]")
    if k.dtype not in _QUERY_DTYPES or v.dtype is not k.dtype:
        raise ValueError(f"append rows must both be float32, float16 or bfloat16, got {k.dtype} and {v.dtype}")
    n_tok = shape[0]
    if slots.dim() != 1 or slots.shape[0] != n_tok:
        raise ValueError(f"slots must be [{n_tok}], got {tuple(slots.shape)}")
    codes = k_cache[0]
    if not k.get_device() == v.get_device() == codes.get_device():
        raise ValueError(f"k is on {k.device}, v on {v.device}, the cache on {codes.device}")
    known = host_slots if host_slots is not None else slots if slots.device.type == "cpu" else None
    if known is not None:
        if known.shape != slots.shape:
            raise ValueError(f"host_slots must be [{n_tok}], got {tuple(known.shape)}")
        if known.dtype is not torch.long or known.device.type != "cpu" or not known.is_contiguous():
            known = known.to(device="cpu", dtype=torch.long).contiguous()
    if CONFIG.kv_backend != "hip":
        _append_torch(Kv8(*k_cache), Kv8(*v_cache), k, v, slots, known)
        return
    native.require_gpu(codes, "kv8_append")
    if n_tok == 0:
        return
    where = _pointers(k_cache, v_cache)
    if where is None:
        raise ValueError("kv8_append needs K and V caches of equal strides with unit head_dim stride; got "
                         f"{k_cache[0].stride()} / {v_cache[0].stride()} and scales {k_cache[1].stride()} / "
                         f"{v_cache[1].stride()}")
    dev = codes.device
    with native.on_device(dev):
        st = k.stride()
        if st[2] != 1 or v.stride() != st:
            k, v = k.contiguous(), v.contiguous()
            st = k.stride()
        slots = _on_device(slots, dev).contiguous()
        rc = native.lib().pkv_kv8_append(
            *where, n_blocks, bs, heads, dim, k.data_ptr(), v.data_ptr(), st[0], st[1], slots.data_ptr(),
            None if known is None else known.data_ptr(), n_tok, native.DTYPE_CODES[k.dtype], native.stream_handle(dev))
        if rc == native.PKV_ERANGE:
            raise IndexError(native.lib().pkv_last_error().decode())
        native.check(rc, "pkv_kv8_append")


def _append_torch(k_cache, v_cache, k, v, slots, known) -> None:
    n_blocks, bs = k_cache.codes.shape[:2]
    slots = slots.to(k_cache.codes.device, torch.long)
    if known is not None:
        if known.numel() and (int(known.min()) < 0 or int(known.max()) >= n_blocks * bs):
            raise IndexError(f"slot index outside [0, {n_blocks * bs})")
    else:
        keep = (slots >= 0) & (slots < n_blocks * bs)
        k, v, slots = k[keep], v[keep], slots[keep]
    at = (slots // bs, slots % bs)
    for cache, rows in ((k_cache, k), (v_cache, v)):
        new = kv8_quantize(rows)
        for to, x in zip(cache, new):
            to.view(torch.uint8)[at] = x.view(torch.uint8)


# ----------------------------------------------------------------------- attention
def paged_attention_kv8(query: torch.Tensor, k_cache: Kv8, v_cache: Kv8, block_tables: torch.Tensor,
                        context_lens: torch.Tensor, query_lens: torch.Tensor, scale: float) -> torch.Tensor:
    """`core.attention.paged_attention` over an 8-bit cache: query [T, heads, head_dim] in
    fp32, fp16 or bf16, the batch's packed new tokens (a prompt, a chunk behind a cached
    context, one token of a decode step, or a mix); block_tables [B, W], context_lens and
    query_lens [B] as there, same checks and messages. Returns [T, heads, head_dim] in the
    query's dtype.

    Softmax and sums are in fp32; of a weight 16 bits at least (24 for fp32 queries) meet the
    values; the output is rounded once. A key that a query does not see does not reach it, NaN
    rows included. (A code that is NaN itself, which the append never writes, may.) Lengths with
    host copies attached (attach_host) are checked without a device round trip."""
    backend = CONFIG.attention
    if backend == "hip":
        return _attention_hip(query, k_cache, v_cache, block_tables, context_lens, query_lens, scale)
    if backend == "gather":
        return _attention_gather(query, Kv8(*k_cache), Kv8(*v_cache), block_tables, context_lens, query_lens, scale)
    if backend == "triton":
        raise NotImplementedError("ATTENTION=triton: this MI355X build ships no Triton kernel; use ATTENTION=hip "
                                  "(libpagedkv CDNA4 kernels) or ATTENTION=gather")
    raise ValueError(f"unknown ATTENTION={backend!r}; expected 'gather', 'triton' or 'hip'")


def _check_query(query: torch.Tensor, cache: Kv8) -> None:
    heads, dim = query.shape[1:]
    kv, pool_dim = cache[0].shape[2:]
    if query.dtype not in _QUERY_DTYPES:
        raise ValueError(f"query must be float32, float16 or bfloat16, got {query.dtype}")
    if query.get_device() != cache[0].get_device():
        raise ValueError(f"the cache is on {cache[0].device}, query is on {query.device}")
    if dim != pool_dim:
        raise ValueError(f"query head_dim {dim} != cache head_dim {pool_dim}")
    if heads % kv:
        raise ValueError(f"{heads} query heads not divisible by {kv} kv heads")


def _attention_gather(query, k_cache, v_cache, tables, ctx, qlens, scale):
    _check_pair(k_cache, v_cache)
    if tables.dim() != 2:
        raise ValueError(f"block_tables must be [batch, width], got {tuple(tables.shape)}")
    check_contract(query.dim(), tuple(query.shape), 4, tuple(k_cache.codes.shape), tables.shape, ctx.shape, qlens.shape,
                   lambda: (int(qlens.sum()), bool((qlens > ctx).any()),
                            bool(((-(-ctx // k_cache.codes.shape[1])) > tables.shape[1]).any())))
    _check_query(query, k_cache)
    if bool((qlens < 0).any()):
        raise ValueError("query_lens must not be negative")
    if query.shape[0] == 0:
        return torch.empty_like(query)
    # The blocks that some query sees, once each. The other entries may hold anything.
    blocks = torch.where(qlens > 0, -(-ctx // k_cache.codes.shape[1]), 0).to(tables.device)
    seen = torch.arange(tables.shape[1], device=tables.device) < blocks[:, None]
    used, number = torch.unique(tables[seen].to(query.device, torch.long), return_inverse=True)
    where = torch.zeros(tables.shape, dtype=torch.long, device=query.device)
    where[seen.to(query.device)] = number
    k, v = (Kv8(c.codes.view(torch.uint8)[used].view(CODES), c.scales.view(torch.uint8)[used].view(SCALES))
            for c in (k_cache, v_cache))
    keys, vals = kv8_dequantize(k), kv8_dequantize(v)
    # A NaN row of V makes every query that sees it NaN. As NaN scores it does so, and reaches
    # no other: a weight of 0 times NaN would.
    hurt = (v.scales.view(torch.uint8) == _NAN_SCALE)[..., None]
    keys, vals = torch.where(hurt, torch.nan, keys), torch.where(hurt, 0.0, vals)
    return _gather_ragged(query.float(), keys, vals, where, ctx, qlens, scale).to(query.dtype)


def _attention_hip(query, k_cache, v_cache, tables, context_lens, query_lens, scale):
    native.require_gpu(query, "paged_attention_kv8")
    c_shape = _check_pair(k_cache, v_cache)
    q_shape, t_shape = query.shape, tables.shape
    n_blocks, block_size, n_kv, head_dim = c_shape
    if len(t_shape) != 2:
        raise ValueError(f"block_tables must be [batch, width], got {tuple(t_shape)}")
    n_seqs, width = t_shape
    facts: dict | None = None

    def values():
        nonlocal facts
        facts = _step_facts(context_lens, query_lens, block_size, width)
        if "negative" not in facts:
            facts["negative"] = bool((facts["hql"] < 0).any())
        return facts["total"], facts["q_gt_c"], facts["too_few_blocks"]

    check_contract(len(q_shape), q_shape, 4, c_shape, t_shape, context_lens.shape, query_lens.shape, values)
    _check_query(query, k_cache)
    if facts["negative"]:
        raise ValueError("query_lens must not be negative")
    dev, (n_tok, n_heads, _) = query.device, q_shape
    with native.on_device(dev):
        out = torch.empty(q_shape, dtype=query.dtype, device=dev)
        if n_tok == 0 or n_seqs == 0:
            return out
        q_st = query.stride()
        if q_st[2] != 1:
            query = query.contiguous()
            q_st = query.stride()
        where = _pointers(k_cache, v_cache)
        if where is None:
            k_cache, v_cache = (Kv8(*(t.contiguous() for t in c)) for c in (k_cache, v_cache))
            where = _pointers(k_cache, v_cache)
        tables = _on_device(tables, dev)
        t_st = tables.stride()
        if t_st[1] != 1:
            tables = tables.contiguous()
            t_st = tables.stride()
        ctx_dev = _on_device(context_lens, dev).contiguous()
        stream = native.stream_handle(dev)
        qsl, starts = None, None
        if not facts["all_decode"]:
            starts = _attached_start(query_lens, dev)
            if starts is None:
                starts = _query_start(facts, context_lens, dev, stream)
            qsl = starts.data_ptr()
        lib = native.lib()
        max_q, max_ctx = facts["max_q"], facts["max_ctx"]
        lens = (facts["hctx"].data_ptr(), facts["hql"].data_ptr())
        # Workspace for contexts that are cut, sized by a step's first layer.
        key = ("kv8", n_heads, n_kv, head_dim, n_tok)
        ws_bytes = facts["split_ws"].get(key)
        if ws_bytes is None:
            ws_bytes = facts["split_ws"][key] = lib.pkv_kv8_attention_workspace_bytes(
                n_seqs, n_heads, n_kv, head_dim, n_tok, max_q, max_ctx, *lens)
        ws_ptr, ws_size = None, 0
        with _WORKSPACES.turn(dev, stream) if ws_bytes else _ALONE:
            if ws_bytes:
                # A capture's calls have one of their own: replays of graphs that were captured on
                # one stream may overlap.
                capturing = torch.cuda.is_current_stream_capturing()
                ws = (_WORKSPACES.of_capture if capturing else _WORKSPACES.partials)(dev, stream, ws_bytes)
                # Not what it has: the cut, and with it the output's bits, go by the call alone.
                ws_ptr, ws_size = ws.data_ptr(), ws_bytes
            rc = lib.pkv_kv8_attention(
                out.data_ptr(), n_heads * head_dim, head_dim, query.data_ptr(), q_st[0], q_st[1],
                *where, n_blocks, block_size, n_kv, head_dim,
                tables.data_ptr(), t_st[0], width, ctx_dev.data_ptr(), qsl,
                n_seqs, n_heads, n_tok, max_q, max_ctx, *lens,
                float(scale), native.DTYPE_CODES[query.dtype], ws_ptr, ws_size, stream)
        native.check(rc, "pkv_kv8_attention")
        return out


# ----------------------------------------------------------------------- pool
class Kv8Pool(PagedKVPool):
    """The preallocated blocks of an 8-bit cache. `dims` is the model's (its dtype is that of
    queries and appended rows). `k[l]` / `v[l]` are uint8 [num_blocks, block_bytes]: a block of
    a layer is one slab, its codes [block_size, kv_heads, head_dim], then its scales
    [kv_heads, block_size], padded to 128 bytes, so that block copies and swaps move codes and
    scales together; `layer(l)` is the layer's K and V as the append and the attention take
    them."""

    def __init__(self, dims: ModelDims, num_blocks: int = CONFIG.num_blocks, block_size: int = CONFIG.block_size,
                 device: str = CONFIG.device) -> None:
        self.row_bytes = block_size * dims.num_kv_heads * dims.head_dim
        self._slab_bytes = -(-(self.row_bytes + block_size * dims.num_kv_heads) // 128) * 128
        super().__init__(dims, num_blocks, block_size, device)
        self._layers = [(self._view(k), self._view(v)) for k, v in zip(self.k, self.v)]

    def _allocate(self) -> list[torch.Tensor]:
        shape = (self.num_blocks, self._slab_bytes)
        return [torch.zeros(shape, dtype=torch.uint8, device=self.device) for _ in range(self.dims.num_layers)]

    def _view(self, slab: torch.Tensor) -> Kv8:
        bs, heads, dim, block = self.block_size, self.dims.num_kv_heads, self.dims.head_dim, self._slab_bytes
        return Kv8(slab.view(CODES).as_strided((self.num_blocks, bs, heads, dim), (block, heads * dim, dim, 1)),
                   slab.view(SCALES).as_strided((self.num_blocks, bs, heads), (block, 1, bs), self.row_bytes))

    def layer(self, layer: int) -> tuple[Kv8, Kv8]:
        return self._layers[layer]

    @property
    def nbytes(self) -> int:
        return 2 * self.dims.num_layers * self.num_blocks * self._slab_bytes

    @property
    def block_bytes(self) -> int:
        return self._slab_bytes

    def _slot_tensors(self) -> list[torch.Tensor]:
        return [t.view(torch.uint8) for layer in self._layers for cache in layer for t in cache]

    def _slot_bytes(self) -> tuple[int, int]:
        return self.row_bytes // self.block_size, self.dims.num_kv_heads

    def _host_shape(self, n: int) -> tuple[tuple[int, ...], torch.dtype]:
        return (2 * self.dims.num_layers, n, self._slab_bytes), torch.uint8

    def append(self, layer: int, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor,
               host_slots: torch.Tensor | None = None) -> None:
        """As PagedKVPool.append, quantising the rows."""
        if slots.device.type != "cpu":
            self.check_slots(slots, host_slots)
        kv8_append(*self._layers[layer], k, v, slots)

    def describe(self) -> str:
        return super().describe()[:-1] + " as e4m3)"

    def release(self) -> None:
        super().release()
        self._layers = []
