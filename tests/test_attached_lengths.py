"""What may be attached to a step's lengths: host copies of their shape, query starts as the kernels
read them. The library reads both by address, as many entries as the batch has sequences."""

from __future__ import annotations

import pytest
import torch

from inference_server.config import CONFIG
from inference_server.core.attention import paged_attention
from inference_server.core.attention_hip import _step_facts, attach_host, attach_query_start
from inference_server.core.kv8 import paged_attention_kv8
from kv8_cases import batch


@pytest.mark.gpu
@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("cache", ["8-bit", "16-bit"])
def test_host_copies_of_another_shape_are_refused(monkeypatch, which, cache):
    monkeypatch.setattr(CONFIG, "attention", "hip")
    s = batch([(5, 1), (3, 1), (40, 1)], heads=4, kv=2, d=32, bs=8, dtype=torch.float16, device="cuda")
    tables, *lens = s.args
    pool = torch.zeros(s.k.codes.shape, dtype=torch.float16, device="cuda")
    call = lambda: (paged_attention_kv8(s.q, s.k, s.v, tables, *lens, s.scale) if cache == "8-bit"  # noqa: E731
                    else paged_attention(s.q, pool, pool, tables, *lens, s.scale))
    good = [torch.from_numpy(s.ctx), torch.from_numpy(s.new)]
    for t, h in zip(lens, good):
        attach_host(t, h)
    assert call().shape == s.q.shape
    three = torch.tensor([1, 1, 1])
    for bad in (three[:2], torch.tensor([1, 1, 1, 0]), torch.tensor(3)):
        attach_host(lens[which], bad + 40 if which == 0 else bad)
        with pytest.raises(ValueError, match="host copies"):
            call()
    attach_host(lens[which], good[which])
    assert call().shape == s.q.shape


def test_facts_of_a_step_need_copies_of_its_shape():
    lens, ones = torch.tensor([3, 4, 5]), torch.tensor([1, 1, 1])

    class OnDevice(torch.Tensor):           # says it is on a device, as far as the facts ask
        device = torch.device("cuda")

    ctx, new = lens.as_subclass(OnDevice), ones.as_subclass(OnDevice)
    attach_host(ctx, lens)
    attach_host(new, ones)
    assert _step_facts(ctx, new, 16, 1)["total"] == 3
    for bad in (torch.tensor([3, 4]), torch.tensor([1, 1, 1, 1]), torch.tensor(3)):
        for pair in ((bad, ones), (lens, bad), (bad, bad)):
            with pytest.raises(ValueError, match="host copies"):
                _step_facts(attach_host(ctx, pair[0]), attach_host(new, pair[1]), 16, 1)


def test_query_starts_that_the_kernels_cannot_read_are_refused():
    lens = torch.tensor([3, 4, 5])
    starts = torch.tensor([0, 3, 7, 12])
    assert attach_query_start(lens, starts) is lens
    for bad in (starts.int(), starts.double(), starts[:-1], starts.repeat(2), starts[None],
                starts.repeat_interleave(2)[::2], starts.to("meta")):
        with pytest.raises(ValueError, match="query_start"):
            attach_query_start(lens, bad)
