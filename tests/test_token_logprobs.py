"""Log probabilities of tokens, ranks, entropies and alternatives against 64 bits, on tensor ops and on
the kernel."""

from __future__ import annotations

import math
import threading

import numpy as np
import pytest
import torch

from inference_server.config import CONFIG
from inference_server.core.sampling import MAX_TOP, token_logprobs
from oracle import tree as oracle
from tree_cases import BF16, F16, F32

BACKENDS = [pytest.param("gather", id="gather"), pytest.param("hip", id="hip", marks=pytest.mark.gpu)]
E = 2.0 ** -24


@pytest.fixture(params=BACKENDS)
def device(request, monkeypatch):
    monkeypatch.setattr(CONFIG, "attention", request.param)
    return "cuda" if request.param == "hip" else "cpu"


def check(logits, ids, got, top):
    """Whole numbers are equal. A weight e^(x - m) is off by the rounding of its exponent, |x - m| log2(e)
    (with log2(e)'s own: 3 roundings of it) and 2 of its own; weights below e^-40 do not count,
    so that a sum is off by (3 * 40 * 1.5 + 2) roundings and one for each of the additions behind one
    another in a lane, at most vocab / 256 or, on the CPU, of a pairwise sum, and 16 to merge, of itself. The
    logarithm takes that as it is; x - m rounds once, the result twice."""
    x = logits.double().cpu().numpy()
    lp, rank, entropy, top_lp, top_ids = oracle.logprobs(x, ids.cpu().numpy(), top)
    assert np.array_equal(got.ranks.cpu().numpy(), rank)
    assert np.array_equal(got.top_ids.cpu().numpy(), top_ids)
    sum_off = (182 + logits.shape[1] / 256 + 16) * E
    for a, want in ((got.logprobs, lp), (got.top_logprobs, top_lp)):
        a = a.double().cpu().numpy()
        with np.errstate(invalid="ignore"):
            off = np.abs(a - want) - (sum_off + 3 * E * (np.abs(want) + 20))
        same = (a == want) | (np.isnan(a) & np.isnan(want))
        assert np.all(same | (off <= 0)), np.nanmax(off)
    # ln s - t / s: s and t off by that much each, of |t| / s <= 40 + ln(vocab).
    a = got.entropy.double().cpu().numpy()
    spread = np.where(np.isnan(entropy), 0, entropy) + 1
    off = np.abs(a - entropy) - 3 * (sum_off + 4 * E) * spread
    assert np.array_equal(np.isnan(a), np.isnan(entropy)) and np.all(np.isnan(a) | (off <= 0)), np.nanmax(off)


def rows(n, vocab, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, vocab, generator=g) * 2.5
    x.scatter_add_(1, torch.randint(0, vocab, (n, 4), generator=g), torch.rand(n, 4, generator=g) * 8 + 2)
    return x.to(dtype), torch.randint(0, vocab, (n,), generator=g)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("vocab", [1, 2, 7, 8, 9, 63, 64, 65, 255, 257, 1000, 2049, 8191, 8192, 8200, 20000, 50257])
@pytest.mark.parametrize("n,top", [(1, 5), (3, 0), (2, 64), (5, 1), (70, 20)])
def test_logprobs(device, dtype, vocab, n, top):
    if device == "cpu" and n * vocab > 200_000:
        n = max(1, 200_000 // vocab)
    x, ids = rows(n, vocab, dtype, vocab + n)
    top = min(top, vocab)
    check(x, ids, token_logprobs(x.to(device), ids.to(device), top), top)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n", [1, 3, 40, 600])
def test_rows_at_any_address_and_stride(device, dtype, n):
    vocab = 1001
    wide = torch.zeros(n, vocab + 37, dtype=dtype)
    for first in (0, 1, 3, 5, 8, 13):
        x, ids = rows(n, vocab, dtype, first)
        where = wide.to(device)
        where.fill_(float("nan"))                # nothing beside the rows counts
        where[:, first:first + vocab] = x.to(device)
        check(x, ids, token_logprobs(where[:, first:first + vocab], ids.to(device), 9), 9)
    x, ids = rows(n, vocab, dtype)
    check(x, ids, token_logprobs(x.t().contiguous().to(device).t(), ids.to(device), 9), 9)
    two = torch.stack([x, x + 1], 1).to(device)[:, 0]
    check(x, ids, token_logprobs(two, torch.stack([ids, ids], 1).to(device)[:, 1], 3), 3)


PATTERNS = {
    "equal": lambda v: torch.zeros(v),
    "ascending": lambda v: torch.arange(v) / 64.0,
    "descending": lambda v: -torch.arange(v) / 64.0,
    "two values": lambda v: (torch.arange(v) % 3 == 1).float(),
    "zeros of both signs": lambda v: torch.where(torch.arange(v) % 2 == 0, 0.0, -0.0),
    "steps of 512": lambda v: (torch.arange(v) // 512).float(),
    "a block of large ones": lambda v: torch.where((torch.arange(v) // 700) == 1, 5.0 + torch.arange(v) % 7, -1.0),
    "every 64th": lambda v: torch.where(torch.arange(v) % 64 == 5, torch.arange(v) / 1000.0, -3.0),
    "lowest value": lambda v: torch.where(torch.arange(v) % 5 == 0, torch.arange(v) / 1000.0, torch.finfo(F16).min),
    "one": lambda v: torch.where(torch.arange(v) == v // 2, 80.0, -80.0),
    "three left": lambda v: torch.where((torch.arange(v) + 1) % (v // 3) == 0, torch.arange(v) / 1000.0, -math.inf),
    "few left, first ids": lambda v: torch.where(torch.arange(v) < 4, 1.0, -math.inf),
    "large": lambda v: 30000.0 + 16 * (torch.arange(v) % 11),
}


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("pattern", PATTERNS, ids=str)
@pytest.mark.parametrize("vocab", [300, 8192, 50257])
@pytest.mark.parametrize("n", [2, 520])
def test_patterns(device, dtype, pattern, vocab, n):
    """Ties by index, lists that overflow, rows with fewer tokens than alternatives asked for."""
    if device == "cpu":
        n = 2
    x = PATTERNS[pattern](vocab).to(dtype)
    for top in (1, 20, 64):
        ids = torch.tensor([0, vocab // 2])
        got = token_logprobs(x.to(device).expand(n, vocab).contiguous(), ids.repeat(n // 2).to(device), top)
        first = min(n, 8)
        check(x.expand(first, vocab), ids.repeat(first // 2), type(got)(*(t[:first] for t in got)), top)
        for t in got:                          # rows of one alignment (mod 16 bytes) are alike
            assert torch.equal(t, t[:first].repeat(n // first, *[1] * (t.dim() - 1)))


@pytest.mark.parametrize("vocab", [100, 8192, 50257])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_rows_without_a_distribution_and_odd_ids(device, dtype, vocab):
    x, ids = rows(8, vocab, dtype)
    x[0, vocab - 1] = math.nan
    x[1] = -math.inf
    x[2, 3] = math.inf
    x[3, 0], x[3, vocab // 2] = math.nan, math.inf
    x[4, 1:] = -math.inf
    ids[4], ids[5], ids[6], ids[7] = 2, -1, vocab, 10 ** 12
    got = token_logprobs(x.to(device), ids.to(device), 12)
    check(x, ids, got, 12)
    assert got.ranks.tolist()[:4] == [0] * 4 and got.ranks.tolist()[5:] == [0] * 3
    assert got.logprobs[4].item() == -math.inf and got.ranks[4].item() == 2
    # One token is left: s = 2^r and t = r 2^r against a reference within half of it, |r| <= 1/2, and
    # log2 s - t / s is two values near r, each off by two roundings of it.
    assert got.top_ids[4].tolist() == list(range(12)) and 0.0 <= got.entropy[4].item() <= 4 * E * 0.5


def test_fp32_logits_at_the_types_ends(device):
    low, high = torch.finfo(F32).min, torch.finfo(F32).max
    x = torch.full((4, 3000), low)
    x[1, 7] = 0.0
    x[2, ::2] = high
    x[3] = torch.randn(3000)
    x[3, ::3] = low
    ids = torch.tensor([5, 7, 2, 1])
    got = token_logprobs(x.to(device), ids.to(device), 6)
    check(x, ids, got, 6)
    assert abs(got.logprobs[0].item() + math.log(3000)) < 1e-5 and abs(got.logprobs[2].item() + math.log(1500)) < 1e-5


@pytest.mark.parametrize("n", [1, 3, 600])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_logits_of_any_size(device, dtype, n):
    """Sizes at which fp32 products with log2(e) no longer tell neighbours apart, in one place of a row, all
    over it, among others and among masked ones."""
    vocab = 9000
    x = torch.zeros(9, vocab)
    g = torch.Generator().manual_seed(0)
    x[0] = torch.randn(vocab, generator=g)
    x[0, 8000] = 1e12
    x[1, 5], x[1, 8500] = 6e8, 6e8 + 64
    x[2] = -1e10
    x[2, 100], x[2, 8999] = -2e9, -2e9
    x[3] = -1e9
    x[3, 4000:4010] = torch.arange(10.0)
    x[4] = -math.inf
    x[4, 7], x[4, 8000] = -3e38, -3e38
    x[5] = torch.randn(vocab, generator=g) * 1e6
    x[6] = 4e8 + 32 * torch.randint(0, 4, (vocab,), generator=g)
    x[7, 8990] = math.nan
    x[7, 3] = 1e30
    x[8, 3000:] = -1e9
    x = x.to(dtype)
    ids = torch.tensor([8000, 8500, 100, 4003, 7, 11, 5, 2, 10])
    every = x.repeat(-(-n // 9), 1)[:max(n, 9)].to(device)
    got = token_logprobs(every, ids.repeat(-(-n // 9))[:max(n, 9)].to(device), 9)
    check(x, ids, type(got)(*(t[:9] for t in got)), 9)
    for r in range(9) if n == 1 else ():
        one = token_logprobs(x[r:r + 1].to(device), ids[r:r + 1].to(device), 9)
        check(x[r:r + 1], ids[r:r + 1], one, 9)


def test_many_short_rows(device):
    x, ids = rows(70_000 if device == "cuda" else 3000, 5, BF16)
    check(x, ids, token_logprobs(x.to(device), ids.to(device), 5), 5)


def test_one_row_for_all(device):
    """Rows of stride 0."""
    x, ids = rows(1, 9000, F32)
    ids = torch.arange(40) * 200
    x = x.expand(40, -1)
    check(x, ids, token_logprobs(x[:1].to(device).expand(40, -1), ids.to(device), 3), 3)


@pytest.mark.gpu
def test_logits_past_2_31_elements(monkeypatch):
    monkeypatch.setattr(CONFIG, "attention", "hip")
    vocab, n = 50257, 43_000
    x, ids = rows(2, vocab, F16)
    big = torch.zeros(n, vocab, dtype=F16, device="cuda")
    big[n - 2:] = x.cuda()
    at = torch.zeros(n, dtype=torch.long, device="cuda")
    at[n - 2:] = ids.cuda()
    got = token_logprobs(big, at, 7)
    check(x, ids, type(got)(*(t[n - 2:] for t in got)), 7)
    same = type(got)(*(t[:1] for t in got))
    check(torch.zeros(1, vocab), ids[:1] * 0, same, 7)
    for t, s in zip(got, same):
        assert torch.equal(t[:n - 2], s.expand_as(t[:n - 2]))


@pytest.mark.gpu
def test_calls_of_two_threads(monkeypatch):
    """Threads with streams of their own, rows in pieces."""
    monkeypatch.setattr(CONFIG, "attention", "hip")
    cases = [tuple(t.cuda() for t in rows(3 + i, 50257, F16, i)) for i in range(2)]
    want = [token_logprobs(*c, 10) for c in cases]
    torch.cuda.synchronize()
    got = [[], []]

    def run(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            got[i] += [token_logprobs(*cases[i], 10) for _ in range(30)]
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for outs, w in zip(got, want):
        assert len(outs) == 30
        for o in outs:
            assert all(torch.equal(a, b) for a, b in zip(o, w))


def test_refusals(device):
    x, ids = torch.zeros(3, 100, device=device), torch.zeros(3, dtype=torch.long, device=device)
    for bad in ((x[0], ids, 0), (x, ids[:2], 0), (x, ids.int(), 0), (x, ids[None], 0), (x.double(), ids, 0),
                (x, ids, -1), (x, ids, MAX_TOP + 1), (x[:, :10], ids, 11), (x[:, :0], ids, 0)):
        with pytest.raises(ValueError):
            token_logprobs(*bad)
    got = token_logprobs(x[:0], ids[:0], 5)
    assert got.logprobs.shape == (0,) and got.top_ids.shape == (0, 5)


@pytest.mark.gpu
def test_captured_calls_replay(monkeypatch):
    """Two graphs captured on one stream, replayed on two at once, with eager calls between."""
    monkeypatch.setattr(CONFIG, "attention", "hip")
    cases = [rows(4, 50257, F16, 1), rows(9, 50257, F16, 2)]
    dev = [(x.cuda(), i.cuda()) for x, i in cases]
    want = [token_logprobs(*d, 10) for d in dev]
    stream = torch.cuda.Stream()
    graphs, outs = [], []
    with torch.cuda.stream(stream):
        torch.cuda.synchronize()
        for d in dev:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=stream):
                outs.append(token_logprobs(*d, 10))
            graphs.append(g)
    other = torch.cuda.Stream()
    for _ in range(5):
        for o in outs:
            for t in o:
                t.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            graphs[0].replay()
        with torch.cuda.stream(other):
            graphs[1].replay()
        token_logprobs(*dev[0], 10)
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            for a, b in zip(o, w):
                assert torch.equal(a, b)
