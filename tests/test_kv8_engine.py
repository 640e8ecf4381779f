"""The paged engine on an 8-bit cache (KV_CACHE=fp8): its steps run the append and the
attention of core/kv8.py, and copies, swaps, prefix sharing and step graphs carry the cache's
blocks as they carry the others."""

from __future__ import annotations

import pytest
import torch

from inference_server.config import CONFIG
from inference_server.core.kv8 import Kv8Pool, kv8_dequantize, kv8_quantize
from inference_server.core.kv_pool import ModelDims
from inference_server.core.paged_executor import PagedExecutor
from inference_server.core.sequence import Sequence
from inference_server.core.block_allocator import BlockAllocator
from inference_server.core.block_table import BlockTable
from inference_server.engine.paged import PagedEngine
from inference_server.model import load
from test_engine import _requests


@pytest.fixture
def fp8(monkeypatch):
    monkeypatch.setattr(CONFIG, "attention", "gather")
    monkeypatch.setattr(CONFIG, "kv_cache", "fp8")
    for name in ("decode_graphs", "prefill_graphs", "preemption"):
        monkeypatch.setattr(CONFIG, name, getattr(CONFIG, name))
    return monkeypatch


def run(reqs, device="cpu", blocks=128, **kw):
    model, tok = load(small=True, device=device)
    engine = PagedEngine(model, tok, num_blocks=blocks, block_size=16, device=device, **kw)
    assert isinstance(engine.pool, Kv8Pool)
    res = engine.run(reqs)
    graphs = engine.executor.graphs
    replays = graphs.replays if graphs else 0
    engine.shutdown()
    return res, replays


@pytest.mark.parametrize("mode", ["recompute", "swap"])
def test_preemption_does_not_change_tokens(fp8, mode):
    reqs = _requests(n=6, max_tokens=20)
    ref, _ = run(reqs)
    CONFIG.preemption = mode
    tight, _ = run(reqs, blocks=9)
    assert tight.stats["preemptions"] > 0 and (tight.stats["swaps"] > 0) == (mode == "swap")
    assert tight.outputs == ref.outputs


def test_prefix_sharing_does_not_change_tokens(fp8):
    reqs = _requests(n=6, prefix=list(range(100, 148)), max_tokens=10)
    shared, _ = run(reqs, prefix_caching=True)
    assert shared.outputs == run(reqs, prefix_caching=False)[0].outputs


def test_unknown_cache_is_refused(fp8):
    fp8.setattr(CONFIG, "kv_cache", "int3")
    with pytest.raises(ValueError, match="KV_CACHE"):
        run(_requests(n=1))


def test_step_stores_what_the_model_projects(fp8):
    """One prompt pass: every layer's cached rows are the quantised K and V of that layer."""
    model, tok = load(small=True)
    pool = Kv8Pool(ModelDims.from_model(model, torch.float32), num_blocks=8, block_size=16, device="cpu")
    seen = {}
    append = Kv8Pool.append
    fp8.setattr(Kv8Pool, "append", lambda self, layer, k, v, *a, **kw: (seen.update({layer: (k.clone(), v.clone())}),
                                                                       append(self, layer, k, v, *a, **kw)))
    seq = Sequence(seq_id="a", prompt_token_ids=list(range(20)), max_tokens=4)
    seq.block_table = BlockTable(BlockAllocator(8), block_size=16)
    seq.block_table.ensure_capacity(20)
    PagedExecutor(model, tok, pool).execute([seq])
    slots = torch.from_numpy(seq.block_table.slots(20))
    for layer, rows in seen.items():
        for cache, x in zip(pool.layer(layer), rows):
            got = kv8_dequantize(cache)[slots // 16, slots % 16]
            assert torch.equal(got, kv8_dequantize(kv8_quantize(x)))
            # At most half a step of e4m3 off, 2^-4 of the value, or of the least normal code's.
            assert ((got - x).abs() <= 2 ** -4 * x.abs().maximum(x.abs().amax(-1, keepdim=True) / 448 * 2 ** -5)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("graphs", [False, True])
def test_hip_tokens_identical_to_gather(fp8, graphs):
    """fp32: both backends attend to the same cached values in fp32."""
    reqs = _requests(n=6, max_tokens=20)
    ref, _ = run(reqs, device="cuda")
    fp8.setattr(CONFIG, "attention", "hip")
    CONFIG.decode_graphs = CONFIG.prefill_graphs = graphs
    got, replays = run(reqs, device="cuda")
    assert (replays > 0) == graphs
    assert got.outputs == ref.outputs


@pytest.mark.gpu
@pytest.mark.parametrize("mode", ["recompute", "swap"])
def test_hip_under_preemption(fp8, mode):
    fp8.setattr(CONFIG, "attention", "hip")
    reqs = _requests(n=6, max_tokens=20, prefix=list(range(32)))
    ref, _ = run(reqs, device="cuda")
    CONFIG.preemption = mode
    tight, _ = run(reqs, device="cuda", blocks=11)
    assert tight.stats["preemptions"] > 0 and (tight.stats["swaps"] > 0) == (mode == "swap")
    assert tight.outputs == ref.outputs
