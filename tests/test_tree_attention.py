"""Attention of drafted trees over the paged pool, on tensor ops and on the kernels, against the
exact attention over the keys that each token sees (64 bits)."""

from __future__ import annotations

import math
import threading

import numpy as np
import pytest
import torch

from inference_server.config import CONFIG
from inference_server.core.attention import paged_attention
from inference_server.core.attention_hip import attach_host, attach_query_start
from inference_server.core.token_tree import paged_tree_attention
from tree_cases import BF16, F16, F32, batch, check

BACKENDS = [pytest.param("gather", id="gather"), pytest.param("hip", id="hip", marks=pytest.mark.gpu)]


@pytest.fixture(params=BACKENDS)
def device(request, monkeypatch):
    monkeypatch.setattr(CONFIG, "attention", request.param)
    return "cuda" if request.param == "hip" else "cpu"


def call(s, **kw):
    return paged_tree_attention(s.q, s.k, s.v, *s.args, s.masks, kw.get("scale", s.scale))


#: (cached, nodes): few rows a sequence, with empty sequences and empty caches; more rows; many.
FEW = [(0, 1), (3, 4), (40, 0), (63, 1), (64, 7), (0, 9), (100, 3), (15, 2)]
SOME = [(0, 30), (31, 33), (127, 17), (0, 0), (200, 25)]
MANY = [(50, 70), (0, 129), (65, 64)]
LENS = [pytest.param(FEW, id="few"), pytest.param(SOME, id="some"), pytest.param(MANY, id="many")]
HEADS = [(4, 4), (6, 2), (16, 2), (5, 1), (3, 3), (12, 4)]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("d", [32, 48, 64, 80, 96, 112, 128])
@pytest.mark.parametrize("lens", LENS)
def test_head_dims(device, dtype, d, lens):
    heads, kv = HEADS[(d // 16) % len(HEADS)]
    s = batch(lens, heads=heads, kv=kv, d=d, bs=16, dtype=dtype, device=device, seed=d)
    check(s, call(s))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("heads,kv", [(4, 4), (6, 2), (16, 2), (33, 1), (20, 1), (12, 12)])
@pytest.mark.parametrize("lens", LENS)
def test_head_layouts(device, dtype, heads, kv, lens):
    s = batch(lens[:3], heads=heads, kv=kv, d=64, bs=16, dtype=dtype, device=device, seed=heads)
    check(s, call(s))


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("bs", [1, 4, 8, 24, 32, 64, 128])
@pytest.mark.parametrize("lens", LENS)
def test_block_sizes(device, dtype, bs, lens):
    s = batch(lens, heads=4, kv=2, d=64, bs=bs, dtype=dtype, device=device, seed=bs, width=600 // bs + 1)
    check(s, call(s))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("d", [1, 7, 16, 24, 40, 72, 160, 256, 512])
def test_other_head_dims(device, dtype, d):
    s = batch(FEW, heads=4, kv=2, d=d, bs=16, dtype=dtype, device=device, seed=d)
    check(s, call(s))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("kind", ["chain", "any", "none"])
@pytest.mark.parametrize("lens", LENS + [pytest.param([(n, m) for n in (0, 1, 50, 126, 127, 128) for m in (1, 2, 62, 65)],
                                                      id="edges")])
@pytest.mark.parametrize("d", [64, 128, 40])
def test_masks(device, dtype, kind, lens, d):
    """Chains (causal), any bits (a row that sees nothing, a node that sees later ones), none."""
    s = batch(lens, heads=2, kv=1, d=d, bs=16, dtype=dtype, device=device, seed=d, kind=kind)
    check(s, call(s))


@pytest.mark.parametrize("lens", LENS)
def test_a_chain_is_causal_attention(device, lens):
    s = batch([(c, n) for c, n in lens if n], heads=4, kv=2, d=64, bs=16, dtype=F32, device=device, kind="chain")
    # Both are as near the exact attention as `check` says.
    for out in (call(s), paged_attention(s.q, s.k, s.v, *s.args, s.scale)):
        check(s, out)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("d", [64, 128, 40])
@pytest.mark.parametrize("lens", LENS)
@pytest.mark.parametrize("kind", ["tree", "any"])
def test_what_is_not_seen_does_not_reach_a_row(device, dtype, d, lens, kind):
    """NaN and infinities in drafted K and V: rows that see them are hurt as the definition says
    (V's in their dims alone), the others not at all."""
    for what in ("k", "v"):
        s = batch(lens, heads=4, kv=2, d=d, bs=16, dtype=dtype, device=device, seed=d, kind=kind)
        rng = np.random.default_rng(5)
        for i, (c, m) in enumerate(lens):
            for j in range(m):
                if rng.random() < 0.3:
                    at = (int(s.tables[i, (c + j) // 16]), (c + j) % 16, int(rng.integers(0, 2)))
                    value = rng.choice([math.nan, math.inf, -math.inf]) if what == "v" else math.nan
                    (s.k if what == "k" else s.v)[at][int(rng.integers(0, d))] = float(value)
        check(s, call(s))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("d", [64, 40])
def test_values_in_the_cached_part_that_are_not_finite(device, dtype, d):
    s = batch([(40, 5), (40, 5)], heads=2, kv=1, d=d, bs=16, dtype=dtype, device=device)
    s.v[int(s.tables[0, 1]), 3, 0, 9] = math.inf
    s.k[int(s.tables[1, 1]), 3, 0, 9] = math.nan
    out = call(s)
    assert torch.isinf(out[:5, :, 9]).all() and torch.isfinite(out[:5, :, :9]).all() and torch.isnan(out[5:]).all()


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("lens", LENS)
@pytest.mark.parametrize("d", [64, 40])
def test_strides(device, dtype, lens, d):
    """Queries as the executor hands them over, pools that are slices of wider tensors and of other axis
    orders, masks and tables among wider rows."""
    s = batch(lens, heads=4, kv=2, d=d, bs=16, dtype=dtype, device=device, seed=3)
    want = call(s)
    check(s, want)
    q = s.q.transpose(0, 1).contiguous().transpose(0, 1)
    wide = torch.cat([s.q, s.q, s.q], -1)[..., d:2 * d]
    odd = torch.empty(s.q.numel() + 1, dtype=dtype, device=device)[1:].view(s.q.shape).copy_(s.q)
    for other in (q, wide, odd):
        s.q = other
        check(s, call(s))
    tables, ctx, new = s.args
    s.args = (torch.cat([tables, tables], 1)[:, :tables.shape[1]], torch.stack([ctx, ctx], 1)[:, 0], new)
    s.masks = torch.cat([s.masks, torch.full_like(s.masks, -1)], 1)[:, :s.masks.shape[1]]
    check(s, call(s))
    s.masks = torch.stack([s.masks, ~s.masks], 2)[..., 0]
    check(s, call(s))
    k, v = s.k, s.v
    s.k, s.v = (torch.stack([x, x + 1])[0] for x in (k, v))
    check(s, call(s))
    s.k, s.v = (x.transpose(1, 2).contiguous().transpose(1, 2) for x in (k, v))       # heads before slots
    check(s, call(s))
    both = torch.stack([k, v], 2)                                                     # [blocks, slots, 2, heads, dim]
    s.k, s.v = both[:, :, 0], both[:, :, 1]
    check(s, call(s))
    s.k, s.v = k, both[:, :, 1]                                                       # of different strides
    check(s, call(s))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("scale", [0.01, 1.0, -0.125, 0.0])
def test_scales(device, dtype, scale):
    s = batch(SOME, heads=4, kv=2, d=64, bs=16, dtype=dtype, device=device)
    check(s, call(s, scale=scale), scale=scale)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lens", [[(3000, 5)], [(2500, 24), (10, 3)], [(1500, 60), (4000, 2)], [(2100, 130)]], ids=str)
def test_long_contexts(device, dtype, d, lens):
    s = batch(lens, heads=4, kv=1, d=d, bs=16, dtype=dtype, device=device, seed=d)
    check(s, call(s))


@pytest.mark.parametrize("dtype", [F16, F32])
def test_masks_of_more_words_than_a_sequence_needs(device, dtype):
    s = batch(SOME, heads=2, kv=2, d=64, bs=16, dtype=dtype, device=device, words=5)
    s.masks[:, 1:] = -1                                   # of no node
    check(s, call(s))


def test_refusals(device):
    s = batch(FEW, heads=4, kv=2, d=64, bs=16, dtype=F16, device=device)
    tables, ctx, new = s.args

    def refused(match, *, q=s.q, k=s.k, v=s.v, tables=tables, ctx=ctx, new=new, masks=s.masks):
        with pytest.raises(ValueError, match=match):
            paged_tree_attention(q, k, v, tables, ctx, new, masks, 0.125)

    refused("must be", q=s.q[0])
    refused("must be", k=s.k[0])
    refused("differ", v=s.v[:, :8])
    refused("dtype", k=s.k.float(), v=s.v.float())
    refused("head_dim", q=s.q[..., :32])
    refused("divisible", q=s.q[:, :3])
    refused("masks must be", masks=s.masks[:-1])
    refused("masks must be", masks=s.masks[:, 0])
    refused("int64", masks=s.masks.int())
    refused("sum to", new=new + 1, ctx=ctx + 10)
    refused("exceeds", ctx=ctx * 0)
    refused("more blocks", ctx=ctx + 10 ** 6)
    refused("words", masks=s.masks[:, :0])
    worse = new.clone()
    worse[0], worse[1] = -1, new[1] + 2
    refused("negative", new=worse)
    refused("block_tables", tables=tables[:, :, None])
    empty = paged_tree_attention(s.q[:0], s.k, s.v, tables[:0], ctx[:0], new[:0], s.masks[:0], 0.125)
    assert empty.shape == (0, 4, 64)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("d", [64, 40])
def test_strides_of_one_row_of_masks(device, dtype, d):
    """A lone row's stride means nothing, and may be anything."""
    s = batch([(70, 1)], heads=4, kv=2, d=d, bs=16, dtype=dtype, device=device, words=3)
    row = s.masks.reshape(3)
    for masks in (s.masks, row[:, None].t(), row.as_strided((1, 3), (0, 1)), torch.stack([row, ~row], 1)[:, 0][None],
                  row[:1].as_strided((1, 1), (0, 5)), row[:1].as_strided((1, 1), (0, 0))):
        s.masks = masks
        check(s, call(s))


# ------------------------------------------------------------------ GPU only
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("d", [64, 128])
def test_captured_calls_replay(monkeypatch, dtype, d):
    """Two graphs captured on one stream, replayed on two at once, with eager calls between them;
    contexts that are cut among them."""
    monkeypatch.setattr(CONFIG, "attention", "hip")
    cases = [batch([(3000, 5), (70, 9)], heads=4, kv=1, d=d, bs=16, dtype=dtype, device="cuda", seed=1),
             batch([(2000, 40)], heads=4, kv=1, d=d, bs=16, dtype=dtype, device="cuda", seed=2)]
    for s in cases:
        tables, ctx, new = s.args
        attach_host(ctx, ctx.cpu()), attach_host(new, new.cpu())
        attach_query_start(new, s.start)
    want = [call(s) for s in cases]
    for s, w in zip(cases, want):
        check(s, w)
    stream, other = torch.cuda.Stream(), torch.cuda.Stream()
    graphs, outs = [], []
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        for s in cases:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=stream):
                outs.append(call(s))
            graphs.append(g)
    for _ in range(5):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            graphs[0].replay()
        with torch.cuda.stream(other):
            graphs[1].replay()
        eager = call(cases[0])
        torch.cuda.synchronize()
        for o, w in zip([*outs, eager], [*want, want[0]]):
            assert torch.equal(o, w)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_lengths_that_only_the_device_knows(monkeypatch, dtype):
    """Host copies that are bounds, as a captured step has them: the device's lengths count. Rows
    behind the last sequence stay as they may."""
    monkeypatch.setattr(CONFIG, "attention", "hip")
    s = batch([(700, 20), (50, 3), (90, 17)], heads=4, kv=2, d=64, bs=16, dtype=dtype, device="cuda")
    pad = 24
    s.q = torch.cat([s.q, torch.full_like(s.q[:pad], math.nan)])
    s.masks = torch.cat([s.masks, torch.full_like(s.masks[:pad], -1)])
    tables, ctx, new = s.args
    width = tables.shape[1] * 16
    attach_host(ctx, torch.full((3,), width)), attach_host(new, torch.tensor([24, 20, 20]))
    attach_query_start(new, s.start)
    out = call(s)
    s.q = s.q[:40]
    check(s, out[:40])
    s.q = torch.cat([s.q, s.q[:pad]])
    new.sub_(new)                                          # a refused step: nothing to do
    s.start.zero_()
    call(s)
    torch.cuda.synchronize()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("d", [64, 128])
def test_block_ids_outside_the_pool_are_not_followed(monkeypatch, dtype, d):
    monkeypatch.setattr(CONFIG, "attention", "hip")
    s = batch([(300, 20), (1500, 6), (50, 70)], heads=4, kv=2, d=d, bs=16, dtype=dtype, device="cuda")
    good = call(s)
    s.args[0][0, 3], s.args[0][1, 0], s.args[0][0, 5] = -1, 10 ** 9, 2 ** 40
    out = call(s)
    assert torch.isfinite(out[20 + 6:]).all() and torch.equal(out[26:], good[26:])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_a_pool_past_4_gib(monkeypatch, dtype):
    """Blocks whose bytes lie beyond 32 bits."""
    monkeypatch.setattr(CONFIG, "attention", "hip")
    s = batch([(200, 9)], heads=8, kv=8, d=128, bs=16, dtype=dtype, device="cuda")
    want = call(s)
    per = s.k[0].numel() * s.k.element_size()
    n = (5 << 30) // per
    k, v = (torch.empty(n, *x.shape[1:], dtype=dtype, device="cuda") for x in (s.k, s.v))
    tables = s.args[0].clone()
    for j in range(14):
        at = n - 1 - 3 * j
        k[at], v[at] = s.k[tables[0, j]], s.v[tables[0, j]]
        tables[0, j] = at
    s.k, s.v, s.args = k, v, (tables, *s.args[1:])
    assert torch.equal(call(s), want)


@pytest.mark.gpu
def test_a_call_repeats_bit_for_bit_on_any_stream(monkeypatch):
    monkeypatch.setattr(CONFIG, "attention", "hip")
    for dtype in (F32, F16, BF16):
        s = batch([(3000, 30), (500, 7), (0, 64)], heads=8, kv=2, d=64, bs=16, dtype=dtype, device="cuda")
        want = call(s)
        torch.cuda.synchronize()
        with torch.cuda.stream(torch.cuda.Stream()):
            outs = [call(s) for _ in range(4)]
        torch.cuda.synchronize()
        for o in outs:
            assert torch.equal(o, want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_calls_of_two_threads(monkeypatch, dtype):
    """Threads with streams of their own, calls that cut their contexts."""
    monkeypatch.setattr(CONFIG, "attention", "hip")
    cases = [batch([(3000 + 500 * i, 5 + i), (70, 9)], heads=4, kv=1, d=64, bs=16, dtype=dtype, device="cuda", seed=i)
             for i in range(2)]
    want = [call(s) for s in cases]
    for s, w in zip(cases, want):
        check(s, w)
    torch.cuda.synchronize()
    got = [[], []]

    def run(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            got[i] += [call(cases[i]) for _ in range(20)]
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for outs, w in zip(got, want):
        assert len(outs) == 20
        for o in outs:
            assert torch.equal(o, w)
