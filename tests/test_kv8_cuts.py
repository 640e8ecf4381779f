"""Decode and chunks over the 8-bit cache where contexts are cut and merged, one test for each way in
which a batch is cut: runs of a workgroup and of a wave, inside a sequence, in batches of up to
64 sequences and of more; and even runs over the ends of sequences. Which way a batch goes follows
from the rules of the plan, restated below."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from inference_server import native
from inference_server.config import CONFIG
from inference_server.core.attention_hip import attach_host
from inference_server.core.kv8 import paged_attention_kv8
from kv8_cases import batch, check, put

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
COUNTERS = 256 * 1024


@pytest.fixture(autouse=True)
def hip_backend(monkeypatch):
    monkeypatch.setattr(CONFIG, "attention", "hip")


def workspace(s, heads, kv, d, bound=None):
    ctx = torch.from_numpy(s.ctx if bound is None else np.full_like(s.ctx, bound))
    new = torch.from_numpy(s.new).contiguous()
    return native.lib().pkv_kv8_attention_workspace_bytes(
        len(s.ctx), heads, kv, d, int(s.new.sum()), int(s.new.max()), int(ctx.max()), ctx.data_ptr(), new.data_ptr())


def partials(s, heads, kv, d, bound=None):
    """How many partials per KV head the decode plan makes of a batch; 0: it is not cut. By the
    plan's rules, and checked to have room in the workspace that the library asks for."""
    ctx, n = s.ctx if bound is None else np.full_like(s.ctx, bound), len(s.ctx)
    keys = 64 if d <= 64 else 32
    units = np.maximum(-(-ctx // keys), 1)[s.new > 0]
    if d > 64 and units.sum() * keys * kv >= 768 * 768:                  # even runs
        numbers = 2 * (512 // kv)
    else:
        waves = n * kv >= 768                                            # a run is a wave's
        runs = int((-(-units // (4 if waves else 8))).sum())
        numbers = 0 if runs <= n else min(runs, max(768 * (4 if waves else 1) // kv, 2 * n))
    room = numbers * kv * int(s.new.max()) * (heads // kv) * (d + 2) * 4
    assert workspace(s, heads, kv, d, bound) >= (COUNTERS + room if numbers else 0)
    return numbers


def nan_rows(s, seq, k_at, v_at, bs):
    """Keys k_at of sequence seq become NaN rows of K, v_at of V, in KV head 0."""
    for raw, cache, at in ((s.k_raw, s.k, k_at), (s.v_raw, s.v, v_at)):
        blk = s.tables[seq, at // bs]
        raw[0][blk, at % bs, 0] = 0
        raw[1][blk, at % bs, 0] = 255
        put(cache, *raw)


def mixed(n, every, long, short=60, new=1):
    """n sequences, every so-manieth one with a long context."""
    return [(long - 7 * (i // every) if i % every == every - 1 else i % short, 1 + i % new) for i in range(n)]


def twice(s):
    """Two calls of one workspace: the same bits."""
    out = paged_attention_kv8(s.q, s.k, s.v, *s.args, s.scale)
    again = paged_attention_kv8(s.q, s.k, s.v, *s.args, s.scale)
    assert torch.equal(out, again) or bool(torch.isnan(out).any())
    return out


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("d,bs", [(32, 16), (64, 16), (64, 8), (80, 16), (128, 16), (128, 4)])
@pytest.mark.parametrize("n,new", [(50, 1), (100, 1), (300, 1), (100, 3)])
def test_workgroup_runs(dtype, d, bs, n, new):
    """Fewer (sequence, KV head) pairs than workgroups; up to 64 sequences and more, one and two
    sequences a thread."""
    heads, kv = 4, 2
    s = batch(mixed(n, 25, 2300, new=new), heads=heads, kv=kv, d=d, bs=bs, dtype=dtype, device="cuda", seed=n)
    assert partials(s, heads, kv, d) > n and n * kv < 768
    check(s, twice(s))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("d,bs", [(48, 16), (64, 16), (64, 4), (96, 16), (128, 16), (128, 8)])
@pytest.mark.parametrize("n,heads,kv,new", [(64, 12, 12, 1), (400, 4, 2, 1), (400, 4, 2, 2)])
def test_wave_runs(dtype, d, bs, n, heads, kv, new):
    """At least as many (sequence, KV head) pairs as workgroups: a run is a wave's."""
    s = batch(mixed(n, n // 4, 1500, new=new), heads=heads, kv=kv, d=d, bs=bs, dtype=dtype, device="cuda", seed=n)
    assert partials(s, heads, kv, d) > n and n * kv >= 768
    check(s, twice(s))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("d,bs", [(80, 16), (80, 8), (96, 16), (112, 32), (112, 4), (128, 16), (128, 8)])
@pytest.mark.parametrize("n,bound,new", [(20, 100_000, 1), (20, 100_000, 4), (300, 4_000, 1)])
def test_even_runs(dtype, d, bs, n, bound, new):
    """Bounds of the contexts decide that the runs are even; the contexts are shorter."""
    heads, kv = 4, 2
    s = batch(mixed(n, max(2, n // 8), 2500, new=new), heads=heads, kv=kv, d=d, bs=bs, dtype=dtype, device="cuda",
              seed=n, width=bound // bs)
    assert partials(s, heads, kv, d, bound) == 2 * (512 // kv)
    attach_host(s.args[1], torch.full((n,), bound))
    attach_host(s.args[2], torch.from_numpy(s.new))
    check(s, twice(s))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("which", ["k", "v", "all"])
@pytest.mark.parametrize("n,heads,kv", [(3, 4, 2), (100, 4, 2), (64, 12, 12)])
def test_runs_of_nan_rows(dtype, d, which, n, heads, kv):
    """A part of a context, longer than a run, or all of it, whose scores are all NaN."""
    s = batch(mixed(n, n // 3, 2300), heads=heads, kv=kv, d=d, bs=16, dtype=dtype, device="cuda")
    assert partials(s, heads, kv, d) > n
    seq = n // 3 - 1
    none, some, every = np.arange(0), np.arange(500, 1300), np.arange(s.ctx[seq])
    nan_rows(s, seq, *{"k": (some, none), "v": (none, some), "all": (every, none)}[which], 16)
    out = twice(s)
    check(s, out)
    row = int(s.new[:seq].sum())
    assert out[row, :heads // kv].isnan().all() and not out[row, heads // kv:].isnan().any()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("which", ["k", "v", "all"])
@pytest.mark.parametrize("d", [80, 128])
def test_even_runs_of_nan_rows(dtype, which, d):
    s = batch(mixed(20, 5, 2500), heads=4, kv=2, d=d, bs=16, dtype=dtype, device="cuda", width=6250)
    assert partials(s, 4, 2, d, 100_000) == 512
    attach_host(s.args[1], torch.full((20,), 100_000))
    attach_host(s.args[2], torch.from_numpy(s.new))
    none, some, every = np.arange(0), np.arange(500, 1300), np.arange(s.ctx[9])
    nan_rows(s, 9, *{"k": (some, none), "v": (none, some), "all": (every, none)}[which], 16)
    out = twice(s)
    check(s, out)
    assert out[9, :2].isnan().all() and not out[9, 2:].isnan().any()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("which", ["k", "v", "all", "hidden"])
@pytest.mark.parametrize("d", [64, 128])
def test_chunks_of_nan_rows(dtype, which, d):
    """A cut context of a chunk: parts all NaN, all of it NaN, and NaN rows that only the chunk's
    last tokens see."""
    heads, kv = 4, 2
    s = batch([(2500, 40), (10, 30)], heads=heads, kv=kv, d=d, bs=16, dtype=dtype, device="cuda")
    assert workspace(s, heads, kv, d) > 0
    none, some, every, last = np.arange(0), np.arange(500, 1800), np.arange(2540), np.arange(2530, 2540)
    nan_rows(s, 0, *{"k": (some, none), "v": (none, some), "all": (every, none), "hidden": (none, last)}[which], 16)
    out = twice(s)
    check(s, out)
    seen = out[30:40] if which == "hidden" else out[:40]
    assert seen[:, :2].isnan().all() and not out[:, 2:].isnan().any() and not out[40:].isnan().any()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_contexts_cut_at_every_length(dtype):
    """Contexts one key apart around the ends of units and runs."""
    lens = [(n - 1, 1) for n in (255, 256, 257, 511, 512, 513, 543, 544, 545, 767, 768, 769, 2047, 2048, 2049)]
    for heads, kv, d in ((4, 4, 128), (2, 2, 64), (16, 1, 96)):
        s = batch(lens, heads=heads, kv=kv, d=d, bs=16, dtype=dtype, device="cuda")
        assert partials(s, heads, kv, d) > len(lens)
        check(s, twice(s))
