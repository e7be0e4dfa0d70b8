"""CPU checks of the workspaces that the entry points keep between calls: whose they are and how
long they live. The device's part (streams, capture, memory) is replaced by stand-ins."""
import gc
import threading
import weakref

import pytest
import torch

from specdec import _lib


@pytest.fixture
def fake(monkeypatch):
    """Workspaces in host memory on stream 0; the list of those that were prepared."""
    prepared = []

    def workspace(nbytes, device, prepare=True):
        ws = torch.empty(max(int(nbytes), 1), dtype=torch.uint8)
        if prepare:
            prepared.append(ws.data_ptr())
        return ws

    monkeypatch.setattr(_lib, "workspace", workspace)
    monkeypatch.setattr(_lib, "prepare", lambda ws: prepared.append(ws.data_ptr()))
    monkeypatch.setattr(_lib, "_stream", lambda device: 0)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    return prepared


KINDS = ["prefix_attn", "logprobs", "to_probs", "sample", "residual", "verify", "draft", "greedy"]


def _in_thread(f):
    out = []
    t = threading.Thread(target=lambda: out.append(f()))
    t.start()
    t.join()
    return out[0]


@pytest.mark.parametrize("kind", KINDS)
def test_threads_on_one_stream_have_workspaces_of_their_own(fake, kind):
    """The kernels of one call hand data over in its workspace, and those of two threads' calls
    may be queued in turn."""
    got, both = {}, threading.Barrier(3)

    def call(name):
        got[name] = _lib.cached_workspace(1000, "cuda:0", kind)
        both.wait()          # both threads live
        got[name, "again"] = _lib.cached_workspace(900, "cuda:0", kind)
        both.wait()

    ts = [threading.Thread(target=call, args=(n,)) for n in "ab"]
    for t in ts:
        t.start()
    both.wait()
    got["main"] = _lib.cached_workspace(1000, "cuda:0", kind)
    both.wait()
    for t in ts:
        t.join()
    assert len({got[n].data_ptr() for n in ("a", "b", "main")}) == 3
    for n in "ab":           # kept for the thread's next calls
        assert got[n, "again"] is got[n]
    assert _lib.cached_workspace(1000, "cuda:0", kind) is got["main"]


def test_workspaces_end_with_their_thread(fake):
    kept = _in_thread(lambda: weakref.ref(_lib.cached_workspace(64, "cuda:0", "logprobs")))
    gc.collect()
    assert kept() is None


def test_reset_reaches_every_thread(fake):
    """reset_workspaces prepares those of the prepared kinds of all threads that live."""
    mine = _lib.cached_workspace(64, "cuda:0", "verify")
    other, have, done = [], threading.Event(), threading.Event()

    def run():
        other.append(_lib.cached_workspace(64, "cuda:0", "draft"))
        _lib.cached_workspace(64, "cuda:0", "sample")
        have.set()
        done.wait()

    t = threading.Thread(target=run)
    t.start()
    have.wait()
    fake.clear()
    _lib.reset_workspaces()
    done.set()
    t.join()
    assert {mine.data_ptr(), other[0].data_ptr()} <= set(fake)
    assert _lib.cached_workspace(64, "cuda:0", "sample").data_ptr() not in fake


def test_large_scratch_is_not_kept(fake):
    """One call over very many tokens does not hold its gigabytes for the thread's life, nor drop
    the workspace of the ordinary calls; prepared kinds, which a call would have to prepare
    again, are kept at any size."""
    at = _lib.KEEP_BYTES
    small = _lib.cached_workspace(1 << 20, "cuda:0", "prefix_attn")
    large = weakref.ref(_lib.cached_workspace(at + 1, "cuda:0", "prefix_attn"))
    gc.collect()
    assert large() is None
    assert _lib.cached_workspace(1 << 20, "cuda:0", "prefix_attn") is small
    whole = _lib.cached_workspace(at, "cuda:0", "prefix_attn")
    assert _lib.cached_workspace(1 << 20, "cuda:0", "prefix_attn") is whole
    held = _lib.cached_workspace(at + 1, "cuda:0", "verify")
    assert _lib.cached_workspace(at + 1, "cuda:0", "verify") is held
