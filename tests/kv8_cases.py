"""Inputs and tolerances shared by the tests of the 8-bit cache."""

from __future__ import annotations

from types import SimpleNamespace

import numpy as np
import torch

from inference_server.core.kv8 import CODES, SCALES, Kv8
from oracle import kv8 as oracle

HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
#: Least step of the type's subnormals.
LEAST = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133}


def slab(n_blocks, bs, kv, d, device):
    """A cache laid out as Kv8Pool's blocks."""
    rows = bs * kv
    block = -(-rows * (d + 1) // 128) * 128
    raw = torch.zeros(n_blocks, block, dtype=torch.uint8, device=device)
    return Kv8(raw.view(CODES).as_strided((n_blocks, bs, kv, d), (block, kv * d, d, 1)),
               raw.view(SCALES).as_strided((n_blocks, bs, kv), (block, 1, bs), rows * d))


def put(cache, codes, scales):
    cache.codes.view(torch.uint8).copy_(torch.from_numpy(codes))
    cache.scales.view(torch.uint8).copy_(torch.from_numpy(scales))
    return cache


def batch(lens, *, heads, kv, d, bs, dtype, seed=0, device="cpu", layout=slab, width=None, spare=3):
    """`lens`: (cached, new) of each sequence. Slots past a context hold bytes of no meaning."""
    rng = np.random.default_rng(seed)
    cached, new = np.array(lens, dtype=np.int64).T
    ctx = cached + new
    need = -(-ctx // bs)
    n_blocks = int(need.sum()) + spare
    ids = rng.permutation(n_blocks)
    width = max(1, int(need.max())) if width is None else width
    tables = np.zeros((len(lens), width), dtype=np.int64)
    at = 0
    for i, n in enumerate(need):
        tables[i, :n] = ids[at:at + n]
        at += n
    s = SimpleNamespace(ctx=ctx, new=new, tables=tables, dtype=dtype, scale=d ** -0.5)
    raw = []
    for _ in range(2):
        codes = rng.integers(0, 256, (n_blocks, bs, kv, d), dtype=np.uint8)     # NaN codes too
        scales = rng.integers(0, 256, (n_blocks, bs, kv), dtype=np.uint8)
        for i, n in enumerate(ctx):
            pos = np.arange(n)
            blk, row = tables[i, pos // bs], pos % bs
            c = rng.integers(0, 256, (n, kv, d), dtype=np.uint8)
            # Magnitudes up to 1.75 * 2^(-8..-4 + 8): codes uniform in their exponents.
            codes[blk, row] = np.where(c & 127 == 127, 0, c)
            scales[blk, row] = rng.integers(127 - 10, 127 - 6, (n, kv), dtype=np.uint8)
        raw.append((codes, scales))
    s.k_raw, s.v_raw = raw
    s.k, s.v = (put(layout(n_blocks, bs, kv, d, device), *r) for r in raw)
    s.q = (torch.from_numpy(rng.standard_normal((int(new.sum()), heads, d))) * 1.5).to(dtype).to(device)
    s.args = (torch.from_numpy(tables).to(device), torch.from_numpy(ctx).to(device), torch.from_numpy(new).to(device))
    return s


def check(s, out, scale=None, rows=slice(None), raws=None):
    """out against the exact attention: an output rounding; a rounding of each weight to the
    type (16 bits), on the sum of their parts; and what fp32 leaves. fp16 weights, the largest
    of them 2^7 at least, are off by up to half a subnormal step, 2^-25, where they are small:
    2^-32 of each value, as the weights' sum is no less than the largest."""
    k_raw, v_raw = raws or (s.k_raw, s.v_raw)
    want, size, slack, flat = oracle.attention(s.q.double().cpu().numpy(), k_raw, v_raw, s.tables, s.ctx, s.new,
                                         s.scale if scale is None else scale)
    u = HALF_STEP[s.dtype]
    tol = u * np.abs(want) + (u + slack) * size + LEAST[s.dtype] + (2.0 ** -32 * flat if s.dtype is torch.float16 else 0)
    got = out.double().cpu().numpy()
    assert got.shape == want.shape
    nan = np.isnan(want)
    assert np.array_equal(np.isnan(got[rows]), nan[rows])
    off = np.where(nan, 0.0, np.abs(got - want) - tol)[rows]
    assert off.size == 0 or off.max() <= 0, f"off by {off.max():.3g} more than {tol.max():.3g}"
