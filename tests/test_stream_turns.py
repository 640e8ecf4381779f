"""Host threads that share a stream. A call with cut contexts is two launches, of which the second
reads what the first one left in the stream's workspace: no other call that uses the workspace
may come between them. On the CPU, with a library that only watches who is inside it; then on the
GPU with the real one."""

from __future__ import annotations

import contextlib
import threading
import time
from concurrent.futures import ThreadPoolExecutor

import pytest
import torch

from inference_server import native
from inference_server.config import CONFIG
from inference_server.core import attention_hip
from inference_server.core.attention_hip import _Workspaces, attach_host, attach_query_start
from inference_server.core.kv8 import paged_attention_kv8
from inference_server.core.attention import paged_attention
from kv8_cases import batch, check

BF16 = torch.bfloat16


class Watcher:
    """Stands for the library: calls take a while, and note how many of a stream are inside."""

    def __init__(self, meet=None):
        self.inside, self.most, self.lock, self.meet = {}, 0, threading.Lock(), meet

    def __getattr__(self, name):
        if name.endswith("_workspace_bytes"):
            return lambda *a: 1 << 19
        if name.endswith("_can_split"):
            return lambda *a: 1

        def call(*args):
            stream = args[-1]
            with self.lock:
                self.inside[stream] = self.inside.get(stream, 0) + 1
                self.most = max(self.most, self.inside[stream])
            if self.meet is not None:
                self.meet.wait(10)
            time.sleep(0.01)
            with self.lock:
                self.inside[stream] -= 1
            return native.PKV_OK

        return call


@pytest.fixture
def watcher(monkeypatch):
    w = Watcher()
    here = threading.local()
    monkeypatch.setattr(CONFIG, "attention", "hip")
    monkeypatch.setattr(native, "lib", lambda: w)
    monkeypatch.setattr(native, "require_gpu", lambda *a: None)
    monkeypatch.setattr(native, "on_device", lambda dev: contextlib.nullcontext())
    monkeypatch.setattr(native, "stream_handle", lambda dev: getattr(here, "stream", 7))
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    fresh = _Workspaces()
    monkeypatch.setattr(attention_hip, "_WORKSPACES", fresh)
    monkeypatch.setattr("inference_server.core.kv8._WORKSPACES", fresh)
    w.here = here
    return w


def calls(device="cpu", seed=0):
    """A chunk and a decode step over the 8-bit cache and over a 16-bit pool, ready to be called."""
    found = []
    for lens in ([(2500, 40), (3, 1)], [(3000, 1), (10, 1)]):
        s = batch(lens, heads=8, kv=2, d=64, bs=16, dtype=BF16, device=device, seed=seed)
        tables, ctx, new = (t.clone() for t in s.args)
        attach_host(ctx, torch.from_numpy(s.ctx))
        attach_host(new, torch.from_numpy(s.new))
        attach_query_start(new, torch.cat([new.new_zeros(1), new.cumsum(0)]))
        g = torch.Generator().manual_seed(seed)
        pool = [torch.randn(s.k.codes.shape, generator=g).to(BF16).to(device) for _ in range(2)]
        found.append((s, lambda s=s, a=(tables, ctx, new): paged_attention_kv8(s.q, s.k, s.v, *a, s.scale)))
        found.append((None, lambda s=s, p=pool, a=(tables, ctx, new): paged_attention(s.q, *p, *a, s.scale)))
    return found


def test_calls_of_one_stream_take_turns(watcher):
    work = [f for _, f in calls()] * 6
    with ThreadPoolExecutor(8) as pool:
        list(pool.map(lambda f: f(), work))
    assert watcher.most == 1


def test_streams_do_not_wait_for_each_other(watcher):
    """Two calls that each return only once the other one is inside the library."""
    watcher.meet = threading.Barrier(2)

    def on(stream, f):
        watcher.here.stream = stream
        f()

    one = calls()[0][1]
    with ThreadPoolExecutor(2) as pool:
        list(pool.map(on, (1, 2), (one, one)))
    assert watcher.most == 1


def test_an_error_ends_its_turn(watcher, monkeypatch):
    one = calls()[0][1]
    monkeypatch.setattr(native, "check", lambda rc, what: (_ for _ in ()).throw(RuntimeError("refused")))
    for _ in range(2):
        with pytest.raises(RuntimeError, match="refused"):
            one()


@pytest.mark.gpu
def test_threads_on_one_stream(monkeypatch):
    monkeypatch.setattr(CONFIG, "attention", "hip")
    work = [c for seed in range(3) for c in calls("cuda", seed)]
    want = []
    for s, f in work:
        want.append(f())
        if s is not None:
            check(s, want[-1])
    torch.cuda.synchronize()

    def many(k):
        return [(i, work[i][1]()) for j in range(20) for i in [(j * 5 + k) % len(work)]]

    with ThreadPoolExecutor(4) as pool:
        got = [x for xs in pool.map(many, range(4)) for x in xs]
    torch.cuda.synchronize()
    assert all(torch.equal(out, want[i]) for i, out in got)
