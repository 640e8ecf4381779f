"""A call's cut, and with it its bits and its time, goes by the call alone: not by how large a workspace
earlier calls of the stream have left, nor by whether it is captured."""

from __future__ import annotations

import pytest
import torch

from inference_server.config import CONFIG
from inference_server.core.attention_hip import _WORKSPACES, attach_host
from inference_server.core.kv8 import CODES, SCALES, Kv8, paged_attention_kv8
from kv8_cases import batch, check, slab

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def hip_backend(monkeypatch):
    monkeypatch.setattr(CONFIG, "attention", "hip")


def plain(n_blocks, bs, kv, d, device):
    """Codes and scales as two contiguous tensors: a block's scales of a head are not together."""
    return Kv8(torch.zeros(n_blocks, bs, kv, d, dtype=torch.uint8, device=device).view(CODES),
               torch.zeros(n_blocks, bs, kv, dtype=torch.uint8, device=device).view(SCALES))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("layout", [slab, plain])
@pytest.mark.parametrize("lens", [[(5000, 1), (2000, 1), (30, 1)], [(4000, 3), (1, 2)], [(3000, 60)]],
                         ids=["single", "few", "chunk"])
def test_earlier_calls_do_not_change_a_call(dtype, layout, lens):
    s = batch(lens, heads=4, kv=2, d=64, bs=16, dtype=dtype, device="cuda", layout=layout)
    tables, ctx, new = s.args
    attach_host(ctx, torch.from_numpy(s.ctx))
    attach_host(new, torch.from_numpy(s.new))
    call = lambda: paged_attention_kv8(s.q, s.k, s.v, tables, ctx, new, s.scale)  # noqa: E731
    stream, dev = torch.cuda.current_stream().cuda_stream, s.q.device
    torch.cuda.synchronize()
    _WORKSPACES.reset()
    first = call()
    check(s, first)
    _WORKSPACES.partials(dev, stream, 1 << 27)
    assert torch.equal(call(), first)
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    if int(s.new.max()) > 1:
        call()                                   # the capture takes the query starts of a call before it
    with torch.cuda.graph(graph, stream=side):
        out = call()
    for _ in range(2):
        out.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, first)
