"""What may be attached to a step's lengths: host copies of their shape, query starts as the kernels
read them. The library reads both by address, as many entries as the batch has sequences."""

from __future__ import annotations

import pytest
import torch

from inference_server.core.attention_hip import attach_host, attach_query_start


def test_host_copies_of_another_shape_are_refused():
    lens = torch.tensor([3, 4, 5])
    assert attach_host(lens, torch.tensor([9, 9, 9])) is lens
    for bad in (torch.tensor([3, 4]), torch.tensor([[3, 4, 5]]), torch.tensor(12)):
        with pytest.raises(ValueError, match="host copy"):
            attach_host(lens, bad)


def test_query_starts_that_the_kernels_cannot_read_are_refused():
    lens = torch.tensor([3, 4, 5])
    starts = torch.tensor([0, 3, 7, 12])
    assert attach_query_start(lens, starts) is lens
    for bad in (starts.int(), starts.double(), starts[:-1], starts.repeat(2), starts[None],
                starts.repeat_interleave(2)[::2], starts.to("meta")):
        with pytest.raises(ValueError, match="query_start"):
            attach_query_start(lens, bad)
