"""The 8-bit cache on the CPU: its format, the torch backend of its append and attention, its
pool, and what the entry points refuse."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from inference_server.config import CONFIG
from inference_server.core.kv8 import (CODES, SCALES, Kv8, Kv8Pool, kv8_append, kv8_dequantize, kv8_quantize,
                                       paged_attention_kv8)
from inference_server.core.kv_pool import ModelDims
from kv8_cases import batch, check, slab
from oracle import kv8 as oracle


@pytest.fixture(autouse=True)
def gather_backend(monkeypatch):
    monkeypatch.setattr(CONFIG, "attention", "gather")


def hard_rows(dim, dtype):
    """Rows at the borders of the format: zeros, ties between codes, the largest magnitude just
    at and past a scale's reach, tiny and huge rows, and rows that are not finite."""
    top = torch.finfo(dtype).max
    rows = [torch.zeros(dim), torch.full((dim,), -0.0), torch.full((dim,), top), torch.full((dim,), torch.finfo(dtype).tiny)]
    for big in (1.75, 1.7578125, 2.0, 1.0, 448.0, 449.0):
        r = torch.linspace(-1, 1, dim) * big
        r[0] = big
        rows.append(r)
    mid = torch.from_numpy((oracle.E4M3[1:127] + oracle.E4M3[:126]) / 2).float()
    r = mid[torch.arange(dim) % 126].clone()
    r[0] = 448.0
    rows.append(r)                                             # every element a tie (as fp32 and bf16 hold it)
    for bad in (float("nan"), float("inf"), -float("inf")):
        r = torch.ones(dim)
        r[dim // 2] = bad
        rows.append(r)
    return torch.stack(rows).to(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim", [1, 7, 64])
def test_quantize_is_the_formats_definition(dtype, dim):
    x = torch.cat([hard_rows(dim, dtype), torch.randn(20, dim, generator=torch.Generator().manual_seed(1)).to(dtype)])
    got = kv8_quantize(x)
    codes, scales = oracle.quantize(x.double().numpy())
    assert np.array_equal(got.scales.view(torch.uint8).numpy(), scales)
    assert np.array_equal(got.codes.view(torch.uint8).numpy()[scales != 255], codes[scales != 255])
    assert not got.codes.view(torch.uint8).numpy()[scales == 255].any()
    assert kv8_dequantize(got)[scales == 255].isnan().all()


def test_append_and_pool_round_trip():
    pool = Kv8Pool(ModelDims(2, 3, 8, torch.float16), num_blocks=6, block_size=4, device="cpu")
    assert pool.block_bytes % 128 == 0 and pool.nbytes == 4 * 6 * pool.block_bytes
    x = torch.randn(2, 9, 3, 8, generator=torch.Generator().manual_seed(0)).half()
    slots = torch.randperm(24, generator=torch.Generator().manual_seed(1))[:9]
    pool.append(1, x[0], x[1], slots)
    for c, rows in zip(pool.layer(1), x):
        want = kv8_quantize(rows)
        assert torch.equal(c.codes.view(torch.uint8)[slots // 4, slots % 4], want.codes.view(torch.uint8))
        assert torch.equal(c.scales.view(torch.uint8)[slots // 4, slots % 4], want.scales.view(torch.uint8))
    assert not pool.k[0].any() and not pool.v[0].any()
    before = [t.clone() for t in pool.k + pool.v]
    pool.copy_blocks([(int(slots[0]) // 4, (int(slots[0]) // 4 + 1) % 6)])
    for t, b in zip(pool.k + pool.v, before):
        assert torch.equal(t[(int(slots[0]) // 4 + 1) % 6], b[int(slots[0]) // 4])
    host = pool.swap_out([3, 1])
    assert len(host) == 2 and host.nbytes == 4 * 2 * pool.block_bytes
    pool.swap_in(host, [0, 5])
    for t, h in zip(pool.k + pool.v, host.k + host.v):
        assert torch.equal(t[[0, 5]], h)
    with pytest.raises(ValueError):
        pool.swap_in(host, [0])
    with pytest.raises(IndexError):
        pool.append(0, x[0], x[1], slots + 24)


LENS = [(0, 1), (0, 17), (15, 1), (16, 3), (40, 0), (31, 33)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads,kv,d,bs", [(4, 4, 32, 16), (6, 2, 40, 8), (5, 1, 64, 24)])
def test_attention(dtype, heads, kv, d, bs):
    s = batch(LENS, heads=heads, kv=kv, d=d, bs=bs, dtype=dtype)
    check(s, paged_attention_kv8(s.q, s.k, s.v, *s.args, s.scale))
    decode = batch([(n, 1) for n in (0, 1, 15, 16, 70)], heads=heads, kv=kv, d=d, bs=bs, dtype=dtype, seed=1)
    check(decode, paged_attention_kv8(decode.q, decode.k, decode.v, *decode.args, decode.scale))


def test_nan_rows_reach_only_the_queries_that_see_them():
    s = batch([(20, 30)], heads=4, kv=2, d=32, bs=16, dtype=torch.float32)
    for raw, cache, pos in ((s.k_raw, s.k, 30), (s.v_raw, s.v, 40)):
        blk = s.tables[0, pos // 16]
        raw[0][blk, pos % 16, 1] = 0
        raw[1][blk, pos % 16, 1] = 255
        cache.codes.view(torch.uint8).copy_(torch.from_numpy(raw[0]))
        cache.scales.view(torch.uint8).copy_(torch.from_numpy(raw[1]))
    out = paged_attention_kv8(s.q, s.k, s.v, *s.args, s.scale)
    check(s, out)
    assert not out[:10].isnan().any() and out[10:, 2:].isnan().all() and not out[:, :2].isnan().any()


def test_refusals():
    s = batch([(5, 2), (3, 1)], heads=4, kv=2, d=32, bs=8, dtype=torch.float16)
    tables, ctx, new = s.args
    call = lambda **kw: paged_attention_kv8(**{**dict(query=s.q, k_cache=s.k, v_cache=s.v, block_tables=tables,  # noqa: E731
                                                      context_lens=ctx, query_lens=new, scale=0.1), **kw})
    with pytest.raises(ValueError, match="num_tokens, heads, dim"):
        call(query=s.q[0])
    with pytest.raises(ValueError, match="batch, width"):
        call(block_tables=tables[0])
    with pytest.raises(ValueError, match="sum to"):
        call(query=s.q[:2])
    with pytest.raises(ValueError, match="exceeds context_len"):
        call(context_lens=ctx * 0)
    with pytest.raises(ValueError, match="more blocks"):
        call(context_lens=ctx + 100)
    with pytest.raises(ValueError, match="head_dim"):
        call(query=s.q[..., :16])
    with pytest.raises(ValueError, match="not divisible"):
        call(query=s.q[:, :3])
    with pytest.raises(ValueError, match="query must be"):
        call(query=s.q.double())
    with pytest.raises(ValueError, match="scales must be"):
        call(k_cache=Kv8(s.k.codes, s.k.scales[:, :4]))
    with pytest.raises(ValueError, match="codes and"):
        call(v_cache=Kv8(s.v.codes.view(torch.uint8), s.v.scales))
    with pytest.raises(ValueError, match="differ"):
        call(v_cache=slab(1, 8, 2, 32, "cpu"))
    rows = torch.zeros(2, 2, 32)
    with pytest.raises(ValueError, match="do not match"):
        kv8_append(s.k, s.v, rows[:, :1], rows[:, :1], torch.tensor([0, 1]))
    with pytest.raises(ValueError, match="slots must be"):
        kv8_append(s.k, s.v, rows, rows, torch.tensor([0]))
    with pytest.raises(ValueError, match="must both be"):
        kv8_append(s.k, s.v, rows.double(), rows.double(), torch.tensor([0, 1]))
    with pytest.raises(IndexError):
        kv8_append(s.k, s.v, rows, rows, torch.tensor([0, -1]))
    with pytest.raises(ValueError, match="host_slots"):
        kv8_append(s.k, s.v, rows, rows, torch.tensor([0, 1]), host_slots=torch.tensor([0]))


@pytest.mark.parametrize("backend,error", [("hip", NotImplementedError), ("triton", NotImplementedError), ("x", ValueError)])
def test_backends_without_a_device(monkeypatch, backend, error):
    monkeypatch.setattr(CONFIG, "attention", backend)
    s = batch([(5, 2)], heads=2, kv=2, d=32, bs=8, dtype=torch.float16)
    with pytest.raises(error):
        paged_attention_kv8(s.q, s.k, s.v, *s.args, 0.1)
    if backend == "hip":
        with pytest.raises(error):
            kv8_append(s.k, s.v, s.q, s.q, torch.tensor([0, 1]))


def test_library_refuses_bad_sizes():
    from inference_server import native

    handle = native.load_library()
    append = lambda nb=1, d=64, t=1, dt=0: handle.pkv_kv8_append(  # noqa: E731
        None, None, 1, 1, 1, None, None, 1, 1, 1, nb, 16, 1, d, None, None, 1, 1, None, None, t, dt, None)
    assert append() == append(nb=0) == append(t=-1) == append(dt=3) == native.PKV_EINVAL
    assert append(d=513) == native.PKV_EUNSUPPORTED
    attend = lambda heads=2, kv=2, d=64, seqs=1, tok=1, dt=0, width=1: handle.pkv_kv8_attention(  # noqa: E731
        None, 1, 1, None, 1, 1, None, None, 1, 1, 1, None, None, 1, 1, 1, 1, 16, kv, d, None, 1, width, None, None,
        seqs, heads, tok, 1, 16, None, None, 1.0, dt, None, 0, None)
    assert attend(tok=0, seqs=0) == native.PKV_OK
    assert attend() == attend(heads=3) == attend(tok=2) == attend(dt=9) == attend(seqs=-1) == native.PKV_EINVAL
    assert attend(d=513) == attend(width=1 << 40) == native.PKV_EUNSUPPORTED
    assert append(nb=1 << 60) == native.PKV_EUNSUPPORTED
    layout = lambda seqs=2, stride=4, width=4, bs=16: handle.pkv_step_layout(  # noqa: E731
        None, stride, width, None, None, None, seqs, None, 0, bs, 0, None, None, None, None, None, None)
    assert layout() == layout(stride=3) == layout(bs=0) == layout(seqs=-1) == native.PKV_EINVAL
    assert layout(width=1 << 31, stride=1 << 31) == native.PKV_EUNSUPPORTED
    assert append(t=0) == native.PKV_OK and handle.pkv_last_error() == b""
