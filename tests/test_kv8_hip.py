"""The 8-bit cache's kernels on the GPU: the append bit for bit against the format's
definition, attention against the exact attention over the cached values (64 bits), and the
operators together as a step uses them."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from inference_server.config import CONFIG
from inference_server.core.attention_hip import attach_host, attach_query_start
from inference_server.core.kv8 import CODES, SCALES, Kv8, Kv8Pool, kv8_append, kv8_quantize, paged_attention_kv8
from inference_server.core.kv_pool import ModelDims
from inference_server.core.step_layout import step_layout
from kv8_cases import batch, check, put, slab
from oracle import kv8 as oracle
from test_kv8 import hard_rows

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.fixture(autouse=True)
def hip_backend(monkeypatch):
    monkeypatch.setattr(CONFIG, "attention", "hip")


def plain(n_blocks, bs, kv, d, device):
    """Codes and scales as two contiguous tensors."""
    return Kv8(torch.zeros(n_blocks, bs, kv, d, dtype=torch.uint8, device=device).view(CODES),
               torch.zeros(n_blocks, bs, kv, dtype=torch.uint8, device=device).view(SCALES))


def head_major(n_blocks, bs, kv, d, device):
    """[blocks, heads, slots, dim]: another order of the axes, and rows at odd addresses."""
    raw = torch.zeros(n_blocks * kv * bs * (d + 1) + 1, dtype=torch.uint8, device=device)[1:]
    return Kv8(raw.view(n_blocks, kv, bs, d + 1)[..., :d].view(CODES).transpose(1, 2),
               raw.view(n_blocks, kv, bs, d + 1)[..., d].view(SCALES).transpose(1, 2))


def call(s, **kw):
    return paged_attention_kv8(s.q, s.k, s.v, *s.args, kw.get("scale", s.scale))


# ------------------------------------------------------------------ append
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("d", [1, 7, 24, 32, 64, 80, 128, 200, 512])
@pytest.mark.parametrize("layout", [slab, plain, head_major])
def test_append_is_the_formats_definition(dtype, d, layout):
    x = torch.cat([hard_rows(d, dtype), torch.randn(23, d, generator=torch.Generator().manual_seed(d)).to(dtype)])
    n = x.shape[0] // 3 * 3
    x = x[:n].view(-1, 3, d)
    v = x.flip(0).contiguous()
    caches = [layout(9, 8, 3, d, "cuda") for _ in range(2)]
    slots = torch.randperm(72, generator=torch.Generator().manual_seed(1))[:x.shape[0]]
    kv8_append(*caches, x.cuda(), v.cuda(), slots.cuda(), host_slots=slots)
    for cache, rows in zip(caches, (x, v)):
        want_codes, want_scales = np.zeros((72, 3, d), np.uint8), np.zeros((72, 3), np.uint8)
        want_codes[slots], want_scales[slots] = oracle.quantize(rows.double().numpy())
        assert np.array_equal(cache.scales.view(torch.uint8).cpu().reshape(72, 3).numpy(), want_scales)
        assert np.array_equal(cache.codes.view(torch.uint8).cpu().reshape(72, 3, d).numpy(), want_codes)


def test_append_takes_strided_rows_and_skips_padding():
    qkv = torch.randn(40, 3, 5, 48, device="cuda").half()
    odd = torch.randn(40, 2, 5, 49, device="cuda").half()[..., 1:]
    for k, v in ((qkv[:, 1], qkv[:, 2]), (odd[:, 0], odd[:, 1]), (qkv[:, 1].transpose(0, 1).contiguous().transpose(0, 1), odd[:, 1])):
        caches = [slab(4, 16, 5, 48, "cuda") for _ in range(2)]
        slots = torch.randperm(64)[:40]
        slots[[3, 7]], slots[9] = torch.tensor([-1, 64]), 10 ** 12
        kv8_append(*caches, k, v, slots.cuda())
        keep = (slots >= 0) & (slots < 64)
        for c, rows in zip(caches, (k, v)):
            want = kv8_quantize(rows[keep.cuda()])
            got = Kv8(*(t.view(torch.uint8).reshape(64, *t.shape[2:]) for t in c))
            assert torch.equal(got.codes[slots[keep]], want.codes.view(torch.uint8))
            assert torch.equal(got.scales[slots[keep]], want.scales.view(torch.uint8))
            rest = torch.ones(64, dtype=torch.bool)
            rest[slots[keep]] = False
            assert not got.codes[rest].any() and not got.scales[rest].any()
    with pytest.raises(IndexError):
        kv8_append(*caches, k, v, slots.cuda(), host_slots=slots)
    with pytest.raises(ValueError, match="equal strides"):
        kv8_append(caches[0], plain(4, 16, 5, 48, "cuda"), k, v, slots.cuda())
    kv8_append(*caches, k[:0], v[:0], slots[:0].cuda())


# ------------------------------------------------------------------ attention
SINGLE = [(n - 1, 1) for n in (1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 300)]
CHUNKS = [(0, 1), (0, 40), (15, 1), (16, 3), (40, 0), (31, 130), (500, 2), (64, 64), (0, 65)]
HEADS = [(4, 4), (6, 2), (16, 2), (5, 1), (20, 1), (3, 3)]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("d", [32, 48, 64, 80, 96, 112, 128])
@pytest.mark.parametrize("lens", [SINGLE, CHUNKS], ids=["single", "chunks"])
def test_head_dims(dtype, d, lens):
    heads, kv = HEADS[(d // 16) % len(HEADS)]
    s = batch(lens, heads=heads, kv=kv, d=d, bs=16, dtype=dtype, device="cuda", seed=d)
    check(s, call(s))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("heads,kv", HEADS + [(33, 1), (12, 12), (64, 2)])
@pytest.mark.parametrize("lens", [SINGLE, CHUNKS[:6]], ids=["single", "chunks"])
def test_head_layouts(dtype, heads, kv, lens):
    s = batch(lens, heads=heads, kv=kv, d=64, bs=16, dtype=dtype, device="cuda", seed=heads)
    check(s, call(s))


@pytest.mark.parametrize("bs", [1, 2, 4, 8, 24, 32, 64, 128])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lens", [SINGLE, CHUNKS], ids=["single", "chunks"])
def test_block_sizes(bs, d, lens):
    s = batch(lens, heads=8, kv=4, d=d, bs=bs, dtype=BF16, device="cuda", seed=bs, width=700 // bs + 1)
    check(s, call(s))


@pytest.mark.parametrize("d", [1, 8, 40, 100, 160, 256, 300, 512])
@pytest.mark.parametrize("lens", [SINGLE, CHUNKS[:6]], ids=["single", "chunks"])
def test_other_head_dims(d, lens):
    s = batch(lens, heads=4, kv=2, d=d, bs=16, dtype=F16, device="cuda", seed=d)
    check(s, call(s))


@pytest.mark.parametrize("layout", [plain, head_major])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("lens", [SINGLE, CHUNKS], ids=["single", "chunks"])
def test_other_strides(layout, dtype, lens):
    s = batch(lens, heads=6, kv=3, d=64, bs=16, dtype=dtype, device="cuda", layout=layout)
    want = call(s)
    check(s, want)
    # The queries as the model hands them over: a transposed view; and rows of odd addresses.
    s.q = s.q.transpose(0, 1).contiguous().transpose(0, 1)
    check(s, call(s))
    wide = torch.empty(*s.q.shape[:2], 67, dtype=dtype, device="cuda")
    wide[..., 1:65] = s.q
    s.q = wide[..., 1:65]
    check(s, call(s))
    # K and V caches of other strides than each other.
    s.v = put(slab(*s.v.codes.shape, "cuda"), *s.v_raw)
    check(s, call(s))


@pytest.mark.parametrize("scale", [0.0, -0.2, 1.0, 1e-30])
@pytest.mark.parametrize("lens", [SINGLE, CHUNKS[:6]], ids=["single", "chunks"])
def test_softmax_scales(scale, lens):
    s = batch(lens, heads=4, kv=2, d=64, bs=16, dtype=F16, device="cuda")
    check(s, call(s, scale=scale), scale=scale)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("lens", [[(4999, 1), (3, 1), (1200, 1)], [(7000, 1)], [(6000, 7), (0, 3), (900, 30)],
                                  [(2500, 200)]], ids=["decode", "lone", "tails", "chunk"])
@pytest.mark.parametrize("d", [64, 128])
def test_long_contexts(dtype, lens, d):
    s = batch(lens, heads=4, kv=2, d=d, bs=16, dtype=dtype, device="cuda")
    check(s, call(s))


@pytest.mark.parametrize("lens", [[(n % 97, 1) for n in range(300)], [(n % 50, n % 4) for n in range(300)],
                                  [(n % 7, 1) for n in range(1500)]], ids=["single", "chunks", "many"])
def test_many_sequences(lens):
    s = batch(lens, heads=4, kv=2, d=64, bs=8, dtype=BF16, device="cuda")
    check(s, call(s))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("lens", [[(20, 30)], [(48, 1), (49, 1)]], ids=["chunk", "single"])
def test_nan_rows_reach_only_the_queries_that_see_them(dtype, lens):
    s = batch(lens, heads=4, kv=2, d=64, bs=16, dtype=dtype, device="cuda")
    for raw, cache, pos in ((s.k_raw, s.k, 30), (s.v_raw, s.v, 49)):
        blk = s.tables[-1, pos // 16]
        raw[0][blk, pos % 16, 1] = 0
        raw[1][blk, pos % 16, 1] = 255
        put(cache, *raw)
    check(s, call(s))


def test_scales_at_the_ends_of_their_range():
    """Rows of tiny and huge values in one context, each type in its own range."""
    for dtype, low, high in ((F32, 20, 200), (BF16, 20, 200), (F16, 108, 130)):
        for lens in ([(40, 1)], [(10, 40)]):
            s = batch(lens, heads=2, kv=2, d=64, bs=16, dtype=dtype, device="cuda")
            rng = np.random.default_rng(0)
            s.v_raw[1][:] = rng.integers(low, high, s.v_raw[1].shape)
            s.v_raw[0][s.v_raw[0] & 127 == 127] = 1
            s.k_raw[0][s.k_raw[0] & 127 == 127] = 1
            s.k_raw[1][:] = rng.integers(max(low, 60), 119, s.k_raw[1].shape)
            put(s.k, *s.k_raw)
            put(s.v, *s.v_raw)
            check(s, call(s))


def test_block_ids_outside_the_cache_are_not_followed():
    """Ids past the pool and below 0, inside a context and behind it: other sequences' rows
    are right, and nothing is read out of bounds (the rows of the bad one mean nothing)."""
    for lens in ([(40, 1), (50, 1), (33, 1)], [(40, 9), (50, 20), (33, 1)]):
        for bs in (16, 24):
            s = batch(lens, heads=4, kv=2, d=64, bs=bs, dtype=BF16, device="cuda", width=6)
            bad = s.args[0].clone()
            bad[1, :3] = torch.tensor([-1, 10 ** 15, s.k.codes.shape[0]])
            bad[:, 4:] = -(10 ** 12)
            out = paged_attention_kv8(s.q, s.k, s.v, bad, *s.args[1:], s.scale)
            rows = np.ones(int(s.new.sum()), dtype=bool)
            rows[s.new[0]:s.new[0] + s.new[1]] = False
            check(s, out, rows=rows)


def padded(s, tokens, seqs, ctx=None):
    """The batch as a captured step holds it: bounds attached, more rows and sequences."""
    n = len(s.ctx)
    q = torch.randn(tokens, *s.q.shape[1:], device="cuda").to(s.dtype)
    q[:s.q.shape[0]] = s.q
    tables = torch.zeros(seqs, s.tables.shape[1], dtype=torch.long, device="cuda")
    tables[:n] = s.args[0]
    ctx, new = torch.zeros(seqs, dtype=torch.long, device="cuda"), torch.zeros(seqs, dtype=torch.long, device="cuda")
    ctx[:n], new[:n] = s.args[1], s.args[2]
    return q, tables, ctx, new


def test_padding_rows_and_sequences():
    s = batch(CHUNKS, heads=4, kv=2, d=64, bs=16, dtype=BF16, device="cuda")
    real = int(s.new.sum())
    q, tables, ctx, new = padded(s, real + 70, len(s.ctx) + 3)
    host = torch.zeros(len(ctx), dtype=torch.long)
    host[:len(s.ctx)] = torch.from_numpy(s.new)
    host[-1] = 70                                               # a bound: the device says 0
    attach_host(ctx, torch.full((len(ctx),), s.tables.shape[1] * 16))
    attach_host(new, host)
    attach_query_start(new, torch.cat([new.new_zeros(1), new.cumsum(0)]))
    check(s, paged_attention_kv8(q, s.k, s.v, tables, ctx, new, s.scale)[:real])


@pytest.mark.parametrize("d,bs", [(64, 16), (40, 16)])
def test_rows_without_a_key_are_zero(d, bs):
    s = batch(SINGLE, heads=4, kv=2, d=d, bs=bs, dtype=F16, device="cuda")
    q, tables, ctx, _ = padded(s, len(s.ctx) + 2, len(s.ctx) + 2)
    one = torch.ones(len(ctx), dtype=torch.long)
    attach_host(ctx, torch.full((len(ctx),), s.tables.shape[1] * bs))
    new = attach_host(one.cuda(), one)
    out = paged_attention_kv8(q, s.k, s.v, tables, ctx, new, s.scale)
    check(s, out[:-2])
    assert not out[-2:].any()


@pytest.mark.parametrize("lens", [SINGLE + [(2000, 1)], CHUNKS + [(2000, 3)]], ids=["single", "chunks"])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_replayed_from_a_graph(lens, dtype):
    """Captured once (two calls, one workspace), replayed on other lengths within the bounds,
    with eager work between; every replay against the eager result."""
    s = batch(lens, heads=8, kv=2, d=64, bs=16, dtype=dtype, device="cuda")
    tables, ctx, new = s.args
    bound = torch.full((len(lens),), s.tables.shape[1] * 16)
    attach_host(ctx, bound)
    attach_host(new, torch.from_numpy(s.new))
    attach_query_start(new, torch.cat([new.new_zeros(1), new.cumsum(0)]))
    eager = call(s)
    check(s, eager)
    stream = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        first = call(s)
        second = paged_attention_kv8(s.q * 0.5, s.k, s.v, tables, ctx, new, s.scale)
    half = paged_attention_kv8(s.q * 0.5, s.k, s.v, tables, ctx, new, s.scale)
    for _ in range(3):
        for out in (first, second):
            out.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(first, eager) and torch.equal(second, half)
        assert torch.equal(call(s), eager)
    # Shorter contexts than captured (the same new tokens).
    full = s.ctx.copy()
    s.ctx = np.maximum(full // 2, s.new)
    ctx.copy_(torch.from_numpy(s.ctx))
    graph.replay()
    torch.cuda.synchronize()
    check(s, first)
    ctx.copy_(torch.from_numpy(full))


def test_streams_and_repeated_calls():
    """Calls that overlap on two streams, and many on one: the same bits each time."""
    a = batch([(3000, 1), (10, 1)], heads=8, kv=2, d=128, bs=16, dtype=BF16, device="cuda")
    b = batch([(2500, 5), (1, 1)], heads=8, kv=2, d=128, bs=16, dtype=BF16, device="cuda", seed=1)
    want = [call(a), call(b)]
    check(a, want[0])
    check(b, want[1])
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for i in range(40):
        s, st = (a, b)[i % 2], streams[i // 2 % 2]
        with torch.cuda.stream(st):
            got.append((i % 2, call(s)))
    torch.cuda.synchronize()
    assert all(torch.equal(out, want[k]) for k, out in got)


@pytest.mark.parametrize("lens", [[(600, 1), (5, 1)], [(600, 40), (5, 3)]], ids=["single", "chunks"])
def test_rows_beyond_4_gib(lens):
    """A cache of more than 2^32 bytes, the batch's blocks at both of its ends."""
    bs, kv, d = 16, 8, 128
    s = batch(lens, heads=16, kv=kv, d=d, bs=bs, dtype=BF16, device="cuda")
    n = 300_000                                                 # x 16.1 KiB: 4.9 GB each
    small = s.k.codes.shape[0]
    big = [slab(n, bs, kv, d, "cuda") for _ in range(2)]
    move = np.where(np.arange(small) % 2, np.arange(small), n - 1 - np.arange(small))
    for cache, (codes, scales) in zip(big, (s.k_raw, s.v_raw)):
        at = torch.from_numpy(move).cuda()
        cache.codes.view(torch.uint8)[at] = torch.from_numpy(codes).cuda()
        cache.scales.view(torch.uint8)[at] = torch.from_numpy(scales).cuda()
    tables = torch.from_numpy(move[s.tables]).cuda()
    check(s, paged_attention_kv8(s.q, *big, tables, *s.args[1:], s.scale))
    x = torch.randn(2, kv, d, device="cuda").half()
    slots = torch.tensor([3, n * bs - 1])
    kv8_append(*big, x, x, slots.cuda(), host_slots=slots)
    want = kv8_quantize(x)
    for c in big:
        assert torch.equal(c.codes.view(torch.uint8)[slots // bs, slots % bs], want.codes.view(torch.uint8))


def test_sequences_that_share_blocks():
    """Forks of one prompt: tables with the same ids, one of them an expanded view."""
    s = batch([(100, 1)], heads=4, kv=2, d=64, bs=16, dtype=F16, device="cuda")
    one = call(s)
    q = s.q.expand(6, -1, -1)
    out = paged_attention_kv8(q, s.k, s.v, s.args[0].expand(6, -1), s.args[1].expand(6), s.args[2].expand(6), s.scale)
    for row in out:
        assert torch.allclose(row.float(), one[0].float(), rtol=2 ** -9, atol=2 ** -9)


# ------------------------------------------------------------------ together
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_steps_of_layout_append_and_attention(dtype):
    """Three steps of four requests on the GPU: tables and slots from lengths, the append into
    them, attention over what has been appended, against a dense computation over the
    quantised rows of each request's whole history."""
    heads, kv, d, bs, n = 8, 2, 64, 16, 4
    pool = Kv8Pool(ModelDims(1, kv, d, dtype), num_blocks=64, block_size=bs, device="cuda")
    g = torch.Generator().manual_seed(5)
    free = torch.randperm(64, generator=g).cuda()
    tables = torch.zeros(n, 16, dtype=torch.long, device="cuda")
    held = torch.zeros(n, dtype=torch.long, device="cuda")
    history = [[] for _ in range(n)]
    lens = np.zeros(n, dtype=np.int64)
    for new in ([17, 1, 40, 100], [1, 1, 1, 1], [1, 33, 0, 5], [1, 1, 1, 1]):
        lens += new
        tokens = sum(new)
        ctx_d, new_d = torch.from_numpy(lens.copy()).cuda(), torch.tensor(new).cuda()
        lay = step_layout(tables, held, ctx_d, new_d, free, bs, tokens)
        taken = int(lay.counts[0])
        assert lay.counts.tolist() == [taken, taken, 0]
        held, free = lay.held, free[taken:]
        q, k, v = (torch.randn(tokens, h, d, generator=g).to(dtype) for h in (heads, kv, kv))
        kv8_append(*pool.layer(0), k.cuda(), v.cuda(), lay.slots)
        out = paged_attention_kv8(q.cuda(), *pool.layer(0), lay.block_tables, ctx_d, new_d, d ** -0.5)
        at = 0
        raws = [(np.zeros((n, 200, kv, d), np.uint8), np.zeros((n, 200, kv), np.uint8)) for _ in range(2)]
        for i, m in enumerate(new):
            history[i] += [(k[t], v[t]) for t in range(at, at + m)]
            at += m
            for raw, which in zip(raws, (0, 1)):
                rows = kv8_quantize(torch.stack([x[which] for x in history[i]]))
                raw[0][i, :len(history[i])] = rows.codes.view(torch.uint8).numpy()
                raw[1][i, :len(history[i])] = rows.scales.view(torch.uint8).numpy()

        class S:
            pass

        s = S()
        s.q, s.k_raw, s.v_raw, s.dtype, s.scale = q, raws[0], raws[1], dtype, d ** -0.5
        s.tables, s.ctx, s.new = np.arange(n)[:, None], lens.copy(), np.array(new)
        check(s, out)


def test_a_refused_layout_leaves_the_cache_alone():
    """A free list that is short: the append and attention queued behind it do nothing."""
    pool = Kv8Pool(ModelDims(1, 2, 64, F16), num_blocks=4, block_size=16, device="cuda")
    long = lambda *v: torch.tensor(v, device="cuda")  # noqa: E731
    lay = step_layout(torch.zeros(1, 8, dtype=torch.long, device="cuda"), long(0), long(50), long(50), long(0, 1, 2), 16, 50)
    assert lay.counts.tolist() == [0, 4, 0]
    rows = torch.randn(50, 2, 64, device="cuda").half()
    kv8_append(*pool.layer(0), rows, rows, lay.slots)
    assert not pool.k[0].any() and not pool.v[0].any()


def test_pool_moves_codes_and_scales_together():
    pool = Kv8Pool(ModelDims(3, 2, 48, BF16), num_blocks=10, block_size=8, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(0)
    for t in pool.k + pool.v:
        t.random_(0, 256, generator=g)
    before = [t.clone() for t in pool.k + pool.v]
    pool.copy_blocks([(1, 9), (4, 0)])
    host = pool.swap_out([4, 2, 7])
    pool.swap_in(host, [3, 5, 6])
    for t, b in zip(pool.k + pool.v, before):
        want = b.clone()
        want[[9, 0]] = b[[1, 4]]
        want[[3, 5, 6]] = b[[4, 2, 7]]
        assert torch.equal(t, want)


def test_graphs_of_one_stream_replayed_side_by_side():
    """Two graphs captured on one stream, each with contexts that are cut, replayed at the same
    time on two others: each capture has its own workspace."""
    batches = [batch([(6000, 1), (3000, 1)], heads=8, kv=2, d=128, bs=16, dtype=BF16, device="cuda", seed=k)
               for k in range(2)]
    for s in batches:
        attach_host(s.args[1], torch.from_numpy(s.ctx))
        attach_host(s.args[2], torch.from_numpy(s.new))
    stream, want, graphs = torch.cuda.Stream(), [], []
    for s in batches:
        with torch.cuda.stream(stream):
            want.append(call(s))
        torch.cuda.synchronize()
        check(s, want[-1])
    for s in batches:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            outs = [call(s) for _ in range(8)]
        graphs.append((graph, outs))
    sides = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        for (graph, outs), side in zip(graphs, sides):
            with torch.cuda.stream(side):
                for o in outs:
                    o.fill_(float("nan"))
                graph.replay()
        torch.cuda.synchronize()
        for (_, outs), w in zip(graphs, want):
            assert all(torch.equal(o, w) for o in outs)


@pytest.mark.parametrize("d,told", [(64, (1, 0)), (128, (0, 0)), (64, (900, 1)), (128, (100000, 1))])
def test_host_lengths_only_decide_the_cut(d, told):
    """The library's call with host lengths that are not the device's: shorter and longer
    contexts, sequences without queries that have some."""
    from inference_server import native

    s = batch([(3000, 1), (70, 2), (0, 1), (2000, 2)] * 5, heads=4, kv=2, d=d, bs=16, dtype=BF16, device="cuda")
    (kc, ks), (vc, vs) = s.k, s.v
    out, n = torch.full_like(s.q, 7.0), len(s.ctx)
    tables, ctx, new = s.args
    start = torch.cat([new.new_zeros(1), new.cumsum(0)])
    for last in (0, 1):                         # all of them told wrongly; the last one rightly
        hctx, hnew = torch.full((n,), told[0]), torch.full((n,), told[1])
        if last:
            hctx[-1], hnew[-1] = int(s.ctx[-1]), int(s.new[-1])
        sizes = (n, 4, 2, d, s.q.shape[0], 2, 100000, hctx.data_ptr(), hnew.data_ptr())
        lib = native.lib()
        ws = torch.zeros(max(1, lib.pkv_kv8_attention_workspace_bytes(*sizes)), dtype=torch.uint8, device="cuda")
        rc = lib.pkv_kv8_attention(
            out.data_ptr(), 4 * d, d, s.q.data_ptr(), 4 * d, d, kc.data_ptr(), vc.data_ptr(), *kc.stride()[:3],
            ks.data_ptr(), vs.data_ptr(), *ks.stride(), kc.shape[0], 16, 2, d, tables.data_ptr(), tables.stride(0),
            tables.shape[1], ctx.data_ptr(), start.data_ptr(), n, 4, s.q.shape[0], 2, 100000, hctx.data_ptr(),
            hnew.data_ptr(), s.scale, native.DTYPE_CODES[BF16], ws.data_ptr(), ws.numel(),
            torch.cuda.current_stream().cuda_stream)
        native.check(rc, "pkv_kv8_attention")
        check(s, out)
        assert not ws[:1 << 18].any()
        out.fill_(7.0)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("lens", [[(2999, 1), (0, 1), (1200, 1)], [(900, 300), (0, 3), (700, 30)]],
                         ids=["few", "many"])
@pytest.mark.parametrize("d,bs", [(40, 16), (101, 16), (256, 16), (512, 16), (64, 24)])
def test_long_contexts_of_other_shapes(dtype, lens, d, bs):
    """Shapes of no matrix kernel, few and many rows, a NaN row among the last keys."""
    s = batch(lens, heads=8, kv=2, d=d, bs=bs, dtype=dtype, device="cuda")
    for raw, cache, pos in ((s.k_raw, s.k, s.ctx[0] - 1), (s.v_raw, s.v, s.ctx[2] - 1)):
        row = 0 if cache is s.k else 2
        blk = s.tables[row, pos // bs]
        raw[0][blk, pos % bs, 1] = 0
        raw[1][blk, pos % bs, 1] = 255
        put(cache, *raw)
    check(s, call(s))


def test_more_sequences_than_the_decode_kernel_takes():
    s = batch([(n % 19, 1) for n in range(2500)], heads=4, kv=2, d=64, bs=16, dtype=BF16, device="cuda")
    check(s, call(s))
