"""What attention over the 8-bit cache keeps of its softmax weights and cached values: 16 bits of
a weight at least, whatever the query's type and however many rows a sequence has, and all of a
cached row, also far outside fp16's range."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from inference_server.config import CONFIG
from inference_server.core.kv8 import paged_attention_kv8
from kv8_cases import HALF_STEP, LEAST, batch, put
from oracle import kv8 as oracle

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16

BACKENDS = [pytest.param("gather", id="gather"), pytest.param("hip", id="hip", marks=pytest.mark.gpu)]


@pytest.fixture(params=BACKENDS)
def device(request, monkeypatch):
    monkeypatch.setattr(CONFIG, "attention", request.param)
    return "cuda" if request.param == "hip" else "cpu"


def tight(s, out, scale):
    """An output rounding of half a step, and on each weight what two bf16 pieces leave of it (three:
    what fp32 has): the second one is half a step off, 2^-8 of what the first one, half a step
    off, has left."""
    want, size, slack, _ = oracle.attention(s.q.double().cpu().numpy(), s.k_raw, s.v_raw, s.tables, s.ctx, s.new, scale)
    u, piece = HALF_STEP[s.dtype], 2.0 ** -24 if s.dtype is F32 else 2.0 ** -16
    tol = u * np.abs(want) + (1 + u) * (piece + slack) * size + LEAST[s.dtype]
    off = np.abs(out.double().cpu().numpy() - want) - tol
    assert off.max() <= 0, f"off by {off.max():.3g} more than {tol.flat[off.argmax()]:.3g}"


#: Of few rows and of many; a context that is cut.
FEW, MANY, CUT = [(0, 2), (1, 1), (5, 2), (40, 1)], [(0, 40), (3, 30), (0, 17), (20, 18)], [(1500, 24)]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("d,bs", [(32, 16), (48, 8), (64, 16), (80, 32), (128, 16), (128, 8), (40, 16)])
@pytest.mark.parametrize("lens", [FEW, MANY, CUT], ids=["few", "many", "cut"])
def test_weights_keep_16_bits(device, dtype, d, bs, lens):
    """Keys that score nearly alike under values of +-1: sums that cancel, so that what is lost of
    a weight stands in the output."""
    s = batch(lens, heads=2, kv=2, d=d, bs=bs, dtype=dtype, device=device, seed=d + bs)
    rng = np.random.default_rng(d)
    s.k_raw[1][:] = 127 - 13
    s.v_raw[0][:] = np.where(rng.random(s.v_raw[0].shape) < 0.5, 0x38, 0xb8)
    s.v_raw[1][:] = 127
    s.k_raw[0][s.k_raw[0] & 127 == 127] = 1
    put(s.k, *s.k_raw)
    put(s.v, *s.v_raw)
    tight(s, paged_attention_kv8(s.q, s.k, s.v, *s.args, s.scale), s.scale)


@pytest.mark.parametrize("b,q_size,scale", [(127 + 10, 2.0 ** -18, 0.125), (127 - 30, 1000.0, 1024.0)],
                         ids=["huge", "tiny"])
@pytest.mark.parametrize("lens", [FEW, MANY, CUT], ids=["few", "many", "cut"])
def test_fp16_queries_take_keys_of_any_size(device, b, q_size, scale, lens):
    s = batch(lens, heads=2, kv=2, d=64, bs=16, dtype=F16, device=device)
    s.k_raw[0][s.k_raw[0] & 127 == 127] = 1
    s.k_raw[1][:] = b
    put(s.k, *s.k_raw)
    s.q = (s.q.float() * q_size).half()
    tight(s, paged_attention_kv8(s.q, s.k, s.v, *s.args, scale), scale)
