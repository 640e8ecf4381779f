"""What is queued behind a step layout that was refused: appends do nothing, attention that is given
the layout's query starts does nothing, and attention that is not reads nothing outside the
cache (its rows mean nothing)."""

from __future__ import annotations

import pytest
import torch

from inference_server import native
from inference_server.config import CONFIG
from inference_server.core.attention_hip import attach_host, attach_query_start
from inference_server.core.kv8 import Kv8Pool, kv8_append, paged_attention_kv8
from inference_server.core.kv_pool import ModelDims
from inference_server.core.step_layout import step_layout

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def hip_backend(monkeypatch):
    monkeypatch.setattr(CONFIG, "attention", "hip")


def attention(q, pool, tables, ctx, start, new, bound, ws):
    """The library's call into rows of 7, with query starts also where every sequence has one token."""
    (kc, ks), (vc, vs) = pool.layer(0)
    out = torch.full_like(q, 7.0)
    tokens, heads, d = q.shape
    n, bs, kv = len(ctx), pool.block_size, pool.dims.num_kv_heads
    hctx, hnew = torch.full((n,), bound), torch.tensor(new)
    native.check(native.lib().pkv_kv8_attention(
        out.data_ptr(), heads * d, d, q.data_ptr(), heads * d, d, kc.data_ptr(), vc.data_ptr(), *kc.stride()[:3],
        ks.data_ptr(), vs.data_ptr(), *ks.stride(), kc.shape[0], bs, kv, d, tables.data_ptr(), tables.stride(0),
        tables.shape[1], ctx.data_ptr(), start.data_ptr(), n, heads, tokens, max(new), bound, hctx.data_ptr(),
        hnew.data_ptr(), d ** -0.5, native.DTYPE_CODES[q.dtype], ws.data_ptr(), ws.numel(),
        torch.cuda.current_stream().cuda_stream), "pkv_kv8_attention")
    return out


@pytest.mark.parametrize("d", [40, 64, 128])
@pytest.mark.parametrize("new", [[1, 1, 1], [1, 30, 5]], ids=["single", "chunks"])
def test_nothing_follows_a_refused_layout(d, new):
    heads, kv, bs, cached = 4, 2, 16, 2100
    pool = Kv8Pool(ModelDims(1, kv, d, torch.float16), num_blocks=500, block_size=bs, device="cuda")
    width, tokens, bound = 200, sum(new), 200 * bs
    # Held blocks of 1 to 396; what stands behind them was never given out.
    tables = torch.full((3, width), 10 ** 12, dtype=torch.long)
    held = [-(-cached // bs)] * 3
    for i, h in enumerate(held):
        tables[i, :h] = torch.arange(i * h, (i + 1) * h)
    tables = tables.cuda()
    before = tables.clone()
    ctx = torch.tensor([cached + m + 20 for m in new]).cuda()       # two blocks each are missing
    new_d = torch.tensor(new).cuda()
    lay = step_layout(tables, torch.tensor(held).cuda(), ctx, new_d, torch.tensor([499, 498]).cuda(), bs, tokens)
    counts = lay.counts.tolist()
    assert counts[0] == 0 and counts[1] > 2 and counts[2] == 0
    assert torch.equal(tables, before) and (lay.slots == -1).all() and not lay.query_start.any()
    g = torch.Generator(device="cuda").manual_seed(0)
    rows = torch.randn(tokens, kv, d, device="cuda", generator=g).half()
    q = torch.randn(tokens, heads, d, device="cuda", generator=g).half()
    kv8_append(*pool.layer(0), rows, rows, lay.slots)
    assert not pool.k[0].any() and not pool.v[0].any()
    ws = torch.zeros(1 << 24, dtype=torch.uint8, device="cuda")
    out = attention(q, pool, tables, ctx, lay.query_start, new, bound, ws)
    assert (out == 7.0).all() and not ws[:1 << 18].any()
    # Through the entry point, with bounds attached and with and without the layout's starts.
    attach_host(ctx, torch.full((3,), bound))
    attach_host(new_d, torch.tensor(new))
    for _ in range(2):
        assert paged_attention_kv8(q, *pool.layer(0), tables, ctx, new_d, d ** -0.5).shape == q.shape
        attach_query_start(new_d, lay.query_start)
    torch.cuda.synchronize()
    # The same step with blocks enough runs.
    lay = step_layout(tables, torch.tensor(held).cuda(), ctx, new_d, torch.arange(400, 500).cuda(), bs, tokens)
    assert lay.counts.tolist()[0] == counts[1]
    kv8_append(*pool.layer(0), rows, rows, lay.slots)
    assert pool.k[0].any()
    out = attention(q, pool, lay.block_tables, ctx, lay.query_start, new, bound, ws)
    assert out.isfinite().all() and not (out == 7.0).any()
