"""What one query holds or sees does not reach another: NaN rows behind a query among few tokens of a
sequence, and queries that are not finite."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from inference_server.config import CONFIG
from inference_server.core.kv8 import paged_attention_kv8
from kv8_cases import batch, check, put

BACKENDS = [pytest.param("gather", id="gather"), pytest.param("hip", id="hip", marks=pytest.mark.gpu)]
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.fixture(params=BACKENDS)
def device(request, monkeypatch):
    monkeypatch.setattr(CONFIG, "attention", request.param)
    return "cuda" if request.param == "hip" else "cpu"


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d,bs", [(32, 8), (40, 16), (64, 16), (80, 16), (128, 16), (128, 4)])
@pytest.mark.parametrize("cached", [0, 61, 600])
@pytest.mark.parametrize("which", ["k", "v"])
def test_nan_rows_behind_a_query_of_few_tokens(device, dtype, d, bs, cached, which):
    s = batch([(cached, 4), (7, 1)], heads=4, kv=2, d=d, bs=bs, dtype=dtype, device=device)
    raw, cache = (s.k_raw, s.k) if which == "k" else (s.v_raw, s.v)
    at = cached + 2                                             # the third of the four tokens, and the last
    blk = s.tables[0, at // bs]
    raw[0][blk, at % bs, 1] = 0
    raw[1][blk, at % bs, 1] = 255
    put(cache, *raw)
    out = paged_attention_kv8(s.q, s.k, s.v, *s.args, s.scale)
    check(s, out)
    nan = out.isnan().any(-1).cpu()
    assert nan[2:4, 2:].all() and not nan[:2].any() and not nan[:, :2].any() and not nan[4].any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [40, 64, 128])
@pytest.mark.parametrize("lens", [[(30, 1), (5, 1)], [(600, 4), (9, 2)], [(40, 60), (1500, 30)]],
                         ids=["single", "few", "many"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_queries_that_are_not_finite(device, dtype, d, lens, bad):
    s = batch(lens, heads=4, kv=2, d=d, bs=16, dtype=dtype, device=device)
    want = paged_attention_kv8(s.q, s.k, s.v, *s.args, s.scale)
    rows = int(s.new.sum())
    tok, head = rows // 2, 1
    s.q[tok, head, d // 2] = bad
    out = paged_attention_kv8(s.q, s.k, s.v, *s.args, s.scale)
    others = torch.ones(rows, 4, dtype=torch.bool, device=out.device)
    others[tok, head] = False
    assert torch.equal(out[others], want[others])
    if np.isnan(bad):
        assert out[tok, head].isnan().all()
