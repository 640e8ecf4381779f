"""Oracle of the 8-bit paged cache, in 64 bits and without the product's code: the e4m3 and
e8m0 values by their definition, quantisation by comparing with every code, attention over
the exact cached values, and a bound on what fp32 arithmetic may be off.
"""

from __future__ import annotations

import numpy as np

#: Values of the 128 non-negative e4m3 codes: bias 7, 3 bits of mantissa, subnormals below
#: 2^-6, no infinity, the last code NaN.
E4M3 = np.array([(b % 8) * 2.0 ** -9 if b < 8 else (8 + b % 8) * 2.0 ** (b // 8 - 10) for b in range(127)] + [np.nan])


def code_values(codes: np.ndarray) -> np.ndarray:
    return np.where(codes & 128, -E4M3[codes & 127], E4M3[codes & 127])


def scale_values(scales: np.ndarray) -> np.ndarray:
    return np.where(scales == 255, np.nan, np.exp2(scales.astype(np.float64) - 127))


def quantize(x: np.ndarray) -> tuple[np.ndarray, np.ndarray]:
    """(codes, scale bytes) of rows x [..., dim] of finite or other values (float64)."""
    codes = np.zeros(x.shape, dtype=np.uint8)
    scales = np.full(x.shape[:-1], 255, dtype=np.uint8)
    for at in np.ndindex(x.shape[:-1]):
        row = x[at]
        if not np.isfinite(row).all():
            continue
        b = next(b for b in range(255) if np.abs(row).max() <= 448 * 2.0 ** (b - 127))
        y = np.abs(row) * 2.0 ** (127 - b)
        off = np.abs(y[:, None] - E4M3[None, :127])
        near = off.min(1, keepdims=True)
        # Of two codes as near, the even one.
        code = np.where(off == near, np.arange(127) + 1000 * (np.arange(127) % 2), 10 ** 6).argmin(1)
        codes[at] = code | np.where(np.signbit(row), 128, 0)
        scales[at] = b
    return codes, scales


def attention(q, k, v, tables, ctx, qlens, scale):
    """q [T, H, D] float64, k / v = (codes, scales) uint8 arrays [NB, bs, Hkv(, D)]. Returns
    (out, size, slack, flat): the exact output; sum of p |v|; the relative error that fp32 dot
    products of any order, exponentials and sums may put on the weights; and sum of |v|."""
    heads, dim = q.shape[1:]
    bs, kv = k[0].shape[1:3]
    out = np.zeros(q.shape)
    size, flat = np.zeros(q.shape), np.zeros(q.shape)
    slack = np.zeros(q.shape[:2] + (1,))
    at = 0
    for i, (n, m) in enumerate(zip(ctx, qlens)):
        pos = np.arange(n)
        blocks, rows = tables[i][pos // bs], pos % bs
        keys, vals = (code_values(c[blocks, rows]) * scale_values(s[blocks, rows])[..., None] for c, s in (k, v))
        for t in range(m):
            seen = n - m + t + 1
            if seen <= 0:
                continue
            for h in range(heads):
                kk, vv = keys[:seen, h // (heads // kv)], vals[:seen, h // (heads // kv)]
                s = kk @ q[at + t, h] * scale
                w = np.exp(s - s.max())
                p = w / w.sum()
                out[at + t, h] = p @ vv
                size[at + t, h] = p @ np.abs(vv)
                flat[at + t, h] = np.abs(vv).sum(0)
                # |error of a score| <= (dim + 8) half steps of the sum of its terms' sizes; it
                # enters a weight and the sum of weights.
                reach = (np.abs(kk) @ np.abs(q[at + t, h])).max() * abs(scale)
                slack[at + t, h] = 2.0 ** -24 * (2 * (dim + 8) * reach + seen + 8)
        at += m
    return out, size, slack, flat
