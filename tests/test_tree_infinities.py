"""Infinities in V under keys whose weight is nothing in fp32 beside the row's largest: the rows that see them have them,
whichever wave, run or group of lanes held the key and whichever held the largest weight."""

from __future__ import annotations

import math

import pytest
import torch

from inference_server.config import CONFIG
from inference_server.core.token_tree import paged_tree_attention
from tree_cases import BF16, F16, F32, batch, check

BACKENDS = [pytest.param("gather", id="gather"), pytest.param("hip", id="hip", marks=pytest.mark.gpu)]

#: (cached, nodes): rows of one wave, of two, of four; a context that is cut, and one that is not, since more than
#: 256 sequences never are.
LENS = [pytest.param([(300, 9), (130, 3)], id="one"), pytest.param([(300, 40)], id="two"), pytest.param([(300, 90)], id="four"),
        pytest.param([(6000, 12)], id="cut"), pytest.param([(2500, 12)] + [(0, 1)] * 256, id="uncut")]


@pytest.mark.parametrize("backend", BACKENDS)
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("d", [32, 64, 128, 40, 160])
@pytest.mark.parametrize("lens", LENS)
@pytest.mark.parametrize("largest", [0, 0.9, 1])
def test_infinities_below_the_largest_weight(monkeypatch, backend, dtype, d, lens, largest):
    """One key 200 nats above all others (2^-288 of it is 0 in fp32), at the start, inside or at the end of the
    cached ones, or the first node."""
    monkeypatch.setattr(CONFIG, "attention", backend)
    device = "cuda" if backend == "hip" else "cpu"
    s = batch(lens, heads=4, kv=2, d=d, bs=16, dtype=dtype, device="cpu", seed=d)
    s.q[..., 0] = 1
    for i, (c, m) in enumerate(lens[:2]):
        where = lambda p: (int(s.tables[i, p // 16]), p % 16)  # noqa: E731
        for p in range(c + m):
            s.k[where(p)][:, 0] = 0
        top = int(largest * c)
        s.k[where(top)][:, 0] = 200 * d ** 0.5
        # One in every 16 keys or so, each in a dim of its own; two of opposite signs in the last dim.
        at = [p for p in [1, 17, 40, 70, 100, c // 3, c // 2, c - 1, c + 1, c + m - 1] if p != top and p < c + m]
        for n, p in enumerate(sorted(set(at))):
            s.v[where(p)][n % 2, n] = math.inf if n % 3 else -math.inf
        for n, p in enumerate(sorted(set(at))[1:3]):
            s.v[where(p)][0, d - 1] = (math.inf, -math.inf)[n]
    s.q, s.k, s.v = s.q.to(device), s.k.to(device), s.v.to(device)
    s.masks, s.args = s.masks.to(device), tuple(t.to(device) for t in s.args)
    out = paged_tree_attention(s.q, s.k, s.v, *s.args, s.masks, s.scale)
    assert torch.isinf(out).any() and torch.isnan(out).any() and torch.isfinite(out).any()
    check(s, out)


@pytest.mark.parametrize("backend", BACKENDS)
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("d", [1, 7, 24, 40, 72, 160, 272, 48, 64, 128])
@pytest.mark.parametrize("lens", LENS[:1] + LENS[3:4])
def test_infinities_in_k_that_make_a_score_lowest(monkeypatch, backend, dtype, d, lens):
    """K of -infinity in its first dim, against queries of 1 there: the key weighs nothing, as one 400 nats below the others
    (e^-400 is 0 in fp32), to the bit."""
    monkeypatch.setattr(CONFIG, "attention", backend)
    device = "cuda" if backend == "hip" else "cpu"
    s = batch(lens, heads=4, kv=2, d=d, bs=16, dtype=dtype, device="cpu", seed=d)
    s.q[..., 0] = 1
    low = s.k.clone()
    for i, (c, m) in enumerate(lens):
        for p in [0, 5, 16, 33, c // 2, c - 1, c, c + m - 1]:
            at = (int(s.tables[i, p // 16]), p % 16)
            low[at][:, 0] = -400 * d ** 0.5
            s.k[at][:, 0] = -math.inf
    s.q, s.v, s.masks = s.q.to(device), s.v.to(device), s.masks.to(device)
    s.args = tuple(t.to(device) for t in s.args)
    outs = [paged_tree_attention(s.q, k.to(device), s.v, *s.args, s.masks, s.scale) for k in (s.k, low)]
    assert torch.isfinite(outs[1]).all() and torch.equal(*outs)
    s.k = low
    check(s, outs[1])
