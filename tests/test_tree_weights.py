"""How much of a row's small weights tree attention keeps: one key that takes nearly all of the softmax
and has a V of zero, and a long tail of keys far below it that makes up the whole output."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from inference_server.config import CONFIG
from inference_server.core.token_tree import paged_tree_attention
from oracle import tree as oracle
from tree_cases import BF16, F16, HALF_STEP, LEAST, PIECES, batch

BACKENDS = [pytest.param("gather", id="gather"), pytest.param("hip", id="hip", marks=pytest.mark.gpu)]

#: (cached, nodes): rows of one wave, of two, of four; a context that is cut; one that is not, since more than 256
#: sequences never are.
LENS = [pytest.param([(700, 9), (130, 3)], id="one"), pytest.param([(700, 40)], id="two"), pytest.param([(700, 90)], id="four"),
        pytest.param([(6000, 70)], id="cut"), pytest.param([(3000, 70)] + [(0, 1)] * 256, id="uncut")]


def tailed(lens, below, spread, d, dtype, device):
    """Queries that read K's first element alone: scores are that element, exactly."""
    rng = np.random.default_rng(int(100 * below))
    s = batch(lens, heads=2, kv=2, d=d, bs=16, dtype=dtype, device="cpu", seed=d)
    s.q.zero_()
    s.q[..., 0] = 1
    s.scale = 1.0
    for i, (c, m) in enumerate(lens):
        pos = np.arange(c + m)
        at = (s.tables[i, pos // 16], pos % 16)
        score = -below - spread * rng.random((c + m, 2))
        value = rng.uniform(0.5, 1.5, (c + m, 2, d))
        if c:
            score[3], value[3] = 0, 0
        s.k[at + (slice(None), 0)] = torch.from_numpy(score).to(dtype)
        s.v[at] = torch.from_numpy(value).to(dtype)
    s.q, s.k, s.v = s.q.to(device), s.k.to(device), s.v.to(device)
    s.masks, s.args = s.masks.to(device), tuple(t.to(device) for t in s.args)
    return s


@pytest.mark.parametrize("backend", BACKENDS)
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("d", [64, 128, 40])
@pytest.mark.parametrize("lens", LENS)
@pytest.mark.parametrize("below,spread", [(10, 0), (12.25, 0), (14.75, 0), (16.5, 0), (17.25, 0), (11, 6)])
def test_a_tail_far_below_the_largest_weight(monkeypatch, backend, dtype, d, lens, below, spread):
    """Weights down to e^-17.25 = 2^-24.9 of the largest. Off by, relative to the output:
    half a step of the type; what its two pieces leave of a weight; weights in fp32, whose exponents of up to 2^6 are
    rounded twice (2^-18) and the exponential once (2^-23), above and below the line: 2^-16 in all; n keys summed 16 at a
    time in two pieces, n / 8 roundings, and some more where waves and runs meet, above and below the line.
    fp16 pieces end at 2^-24 times 2^-12 of the row's largest weight: half of that, absolute, a key."""
    monkeypatch.setattr(CONFIG, "attention", backend)
    s = tailed(lens, below, spread, d, dtype, "cuda" if backend == "hip" else "cpu")
    got = paged_tree_attention(s.q, s.k, s.v, *s.args, s.masks, s.scale).double().cpu().numpy()
    want, size, _, flat = oracle.attention(s.q.double().cpu().numpy(), s.k.double().cpu().numpy(), s.v.double().cpu().numpy(),
                                           s.tables, s.ctx, s.new, s.sees, s.scale)
    u, n = HALF_STEP[dtype], int(s.ctx.max())
    sums = 2 * (n / 8 + 64) * 2.0 ** -24
    tol = u * want + (1 + u) * (PIECES[dtype] + 2.0 ** -16 + sums) * size + LEAST[dtype]
    if dtype is F16:
        tol = tol + 2.0 ** -37 * flat
    off = np.abs(got - want) - tol
    at = np.unravel_index(off.argmax(), off.shape)
    assert off.max() <= 0, f"{got[at]:.6g} for {want[at]:.6g}, within {tol[at]:.3g}"


@pytest.mark.parametrize("backend", BACKENDS)
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("d", [64, 40])
@pytest.mark.parametrize("lens", LENS[2:4])
@pytest.mark.parametrize("scale,step", [(1.0, 4.0), (2.0 ** 11, 2.0 ** -9), (2.0 ** 13, 2.0 ** -11), (2.0 ** 15, 2.0 ** -12)])
@pytest.mark.parametrize("sign", [1, -1])
def test_scores_that_rise_from_far_off(monkeypatch, backend, dtype, d, lens, scale, step, sign):
    """Scores of up to 2^26, 4 or 8 apart, that rise along the context: products and sums are exact in fp32, the
    weights as above. Scores off by an exponent's rounding would make weights of more than fp16 holds."""
    monkeypatch.setattr(CONFIG, "attention", backend)
    device = "cuda" if backend == "hip" else "cpu"
    s = batch(lens, heads=2, kv=2, d=d, bs=16, dtype=dtype, device="cpu", seed=d)
    s.q.zero_()
    s.q[..., :2] = 1
    s.scale = scale
    (c, m), = lens
    pos = np.arange(c + m)
    at = (s.tables[0, pos // 16], pos % 16)
    rises = np.repeat(step * (16 * pos // (c + m))[:, None], 2, 1)
    s.k[at + (slice(None), 0)] = sign * 2.0 ** 11
    s.k[at + (slice(None), 1)] = torch.from_numpy(rises).to(dtype)
    s.v[at] = torch.from_numpy(np.random.default_rng(d).uniform(0.5, 1.5, (c + m, 2, d))).to(dtype)
    s.q, s.k, s.v = s.q.to(device), s.k.to(device), s.v.to(device)
    s.masks, s.args = s.masks.to(device), tuple(t.to(device) for t in s.args)
    got = paged_tree_attention(s.q, s.k, s.v, *s.args, s.masks, scale).double().cpu().numpy()
    want, size, _, flat = oracle.attention(s.q.double().cpu().numpy(), s.k.double().cpu().numpy(), s.v.double().cpu().numpy(),
                                           s.tables, s.ctx, s.new, s.sees, scale)
    u = HALF_STEP[dtype]
    sums = 2 * ((c + m) / 8 + 64) * 2.0 ** -24
    tol = u * want + (1 + u) * (PIECES[dtype] + 2.0 ** -16 + sums) * size + LEAST[dtype]
    if dtype is F16:
        tol = tol + 2.0 ** -37 * flat
    off = np.abs(got - want) - tol
    at = np.unravel_index(off.argmax(), off.shape)
    assert off.max() <= 0, f"{got[at]:.6g} for {want[at]:.6g}, within {tol[at]:.3g}"
