"""Tree attention over fp32 pools is in fp32 throughout: few keys, so that nothing hides a product of fewer bits."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from inference_server.config import CONFIG
from inference_server.core.token_tree import paged_tree_attention
from tree_cases import F32, batch

BACKENDS = [pytest.param("gather", id="gather"), pytest.param("hip", id="hip", marks=pytest.mark.gpu)]
U = 2.0 ** -24


def pieces(x):
    """x in two bf16 pieces: 16 bits of it."""
    hi = torch.from_numpy(x).bfloat16().double()
    return (hi + (torch.from_numpy(x) - hi).bfloat16().double()).numpy()


@pytest.mark.parametrize("backend", BACKENDS)
@pytest.mark.parametrize("d", [32, 48, 64, 80, 96, 112, 128, 40, 160])
@pytest.mark.parametrize("nodes", [3, 24, 40])
def test_products_and_sums_have_24_bits(monkeypatch, backend, d, nodes):
    """Tolerances, with U half a step: a dot product is d roundings of sums that are about t = |(q_e k_e)_e| in size, each with a
    standard deviation below 0.6 U of it: 4 U t sqrt(d) is more than six of their sum's. Exponents round twice and the
    exponential once: (2 |s| + 4) U of a weight. Each enters the output by the key's distance from it; n keys are
    summed in n roundings and joined in eight at most, above and below the line. q, k or v of 16 bits are not within them."""
    monkeypatch.setattr(CONFIG, "attention", backend)
    device = "cuda" if backend == "hip" else "cpu"
    lens = [(c, nodes if i < 3 else 2) for i, c in enumerate((3, 0, 6, 1, 2, 5, 9, 4, 7, 12, 3, 5, 8))]
    s = batch(lens, heads=4, kv=2, d=d, bs=16, dtype=F32, device=device, seed=d + nodes)
    scale = 3 * d ** -0.5
    got = paged_tree_attention(s.q, s.k, s.v, *s.args, s.masks, scale).double().cpu().numpy()
    q, k, v = (x.double().cpu().numpy() for x in (s.q, s.k, s.v))
    over = {"result": 0.0, "q and k of 16 bits": 0.0, "v of 16 bits": 0.0}
    t = 0
    for i, (c, m) in enumerate(lens):
        for node in range(m):
            pos = np.array([*range(c), *(c + j for j in s.sees[t])])
            for head in range(4):
                kk, vv = (x[s.tables[i, pos // 16], pos % 16, head // 2] for x in (k, v))

                def attend(q, kk, vv):
                    x = kk @ q * scale
                    p = np.exp(x - x.max())
                    return x, p / p.sum(), p / p.sum() @ vv

                x, p, want = attend(q[t, head], kk, vv)
                size = np.sqrt((q[t, head] ** 2 * kk ** 2).sum(1))
                slack = p * (4 * U * d ** 0.5 * size * scale + (2 * np.abs(x) + 4) * U)
                tol = slack @ np.abs(vv - want) + U * (2 * (len(pos) + 8) * (p @ np.abs(vv)) + np.abs(want)) + 2.0 ** -149
                for name, out in (("result", got[t, head]), ("q and k of 16 bits", attend(pieces(q[t, head]), pieces(kk), vv)[2]),
                                  ("v of 16 bits", attend(q[t, head], kk, pieces(vv))[2])):
                    over[name] = max(over[name], (np.abs(out - want) / tol).max())
            t += 1
    assert over["result"] <= 1, over
    assert min(over["q and k of 16 bits"], over["v of 16 bits"]) > 1, over
