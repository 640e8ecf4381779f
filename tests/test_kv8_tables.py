"""Table entries that no query reads: behind a context's last block, and in rows of sequences
without queries. They may hold anything, as in core.attention.paged_attention."""

from __future__ import annotations

import pytest
import torch

from inference_server.config import CONFIG
from inference_server.core.kv8 import paged_attention_kv8
from kv8_cases import batch, check

BACKENDS = [pytest.param("gather", id="gather"), pytest.param("hip", id="hip", marks=pytest.mark.gpu)]


@pytest.fixture(params=BACKENDS)
def device(request, monkeypatch):
    monkeypatch.setattr(CONFIG, "attention", request.param)
    return "cuda" if request.param == "hip" else "cpu"


@pytest.mark.parametrize("junk", [-1, -(10 ** 12), 10 ** 6, 10 ** 15])
@pytest.mark.parametrize("lens", [[(0, 1), (15, 1), (16, 1), (40, 1)], [(0, 17), (31, 1), (40, 0), (16, 3)]],
                         ids=["single", "chunks"])
@pytest.mark.parametrize("d", [32, 40])
def test_entries_that_no_query_reads(device, junk, lens, d):
    s = batch(lens, heads=4, kv=2, d=d, bs=16, dtype=torch.float32, device=device, width=8)
    tables, ctx, new = s.args[0].clone(), *s.args[1:]
    for i, n in enumerate(s.ctx):
        tables[i, -(-int(n) // 16) if s.new[i] else 0:] = junk
    check(s, paged_attention_kv8(s.q, s.k, s.v, tables, ctx, new, s.scale))
    # Tables on the other side of the bus, and of another integer type.
    check(s, paged_attention_kv8(s.q, s.k, s.v, tables.cpu(), ctx, new, s.scale))
    if abs(junk) < 2 ** 31:
        check(s, paged_attention_kv8(s.q, s.k, s.v, tables.int(), ctx, new, s.scale))


def test_entries_that_queries_read_are_followed_or_refused_on_the_cpu(monkeypatch):
    monkeypatch.setattr(CONFIG, "attention", "gather")
    s = batch([(15, 1), (20, 1)], heads=4, kv=2, d=32, bs=16, dtype=torch.float32)
    tables = s.args[0].clone()
    tables[1, 1] = s.k.codes.shape[0]
    with pytest.raises(IndexError):
        paged_attention_kv8(s.q, s.k, s.v, tables, *s.args[1:], s.scale)


@pytest.mark.parametrize("d", [32, 40])
def test_negative_query_lengths_are_refused(device, d):
    s = batch([(5, 1), (3, 1)], heads=4, kv=2, d=d, bs=8, dtype=torch.float16, device=device)
    new = torch.tensor([-1, 3], device=s.q.device)
    with pytest.raises(ValueError, match="must not be negative"):
        paged_attention_kv8(s.q, s.k, s.v, *s.args[:2], new, s.scale)
