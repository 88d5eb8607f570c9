"""The pool of workspaces, with workspaces that are only sizes: what is reused, replaced and kept."""
from __future__ import annotations

import threading
import types

import pytest

DEVICE = types.SimpleNamespace(index=0)


class Fake:
    def __init__(self, device, nbytes, capture=0):
        self.nbytes, self.capture, self.captured = nbytes, capture, False

    def ready(self):
        return True


@pytest.fixture
def pool(monkeypatch):
    """Sets the stream and the capture that calls find themselves in."""
    from svdflash_b200.kernels import ops
    now = types.SimpleNamespace(stream=7, capture=0, waits=0, ops=ops)

    def wait():
        assert not now.capture, "waiting for a stream inside a capture"
        now.waits += 1
    for name in ("_ws_pool", "_ws_captures"):
        monkeypatch.setattr(ops, name, {})
    monkeypatch.setattr(ops, "_ws_kept", [])
    monkeypatch.setattr(ops, "_Workspace", Fake)
    monkeypatch.setattr(ops, "_raw_stream", lambda index: now.stream)
    monkeypatch.setattr(ops, "_capture_id", lambda index, stream: now.capture)
    monkeypatch.setattr(ops.torch.cuda, "current_stream", lambda device: types.SimpleNamespace(synchronize=wait))
    now.get = lambda nbytes: ops.workspace_for(DEVICE, nbytes)
    return now


def test_one_a_stream_grown_on_demand(pool):
    small = pool.get(1 << 21)
    assert pool.get(100) is small and pool.waits == 0
    large = pool.get(1 << 22)
    assert large is not small and pool.get(1 << 21) is large and pool.waits == 1
    pool.stream = 8
    assert pool.get(100) is not large
    assert pool.ops._ws_kept == []                     # nothing holds what only calls used


def test_what_a_capture_used_outlives_its_replacement(pool):
    small = pool.get(1 << 21)
    pool.capture = 3
    assert pool.get(1 << 20) is small
    pool.capture = 0
    assert pool.get(1 << 22) is not small
    assert [ws for _, ws in pool.ops._ws_kept] == [small]


def test_a_capture_never_waits_and_gets_its_own(pool):
    small = pool.get(1 << 21)
    pool.capture = 3
    own = pool.get(1 << 22)
    assert own is not small and own.capture == 3
    assert pool.get(1 << 21) is small                  # what is large enough is shared with calls, as ever
    assert pool.get((1 << 21) + 1) is own
    pool.capture = 4                                   # another graph: set up by its own replays
    assert pool.get(1 << 22) is not own
    pool.capture = 0
    later = pool.get(1 << 22)                          # and calls never get one that only a replay sets up
    assert later.capture == 0
    assert pool.get(1) is later


def test_a_capture_on_a_stream_without_one(pool):
    pool.capture = 5
    own = pool.get(10)
    assert own.capture == 5 and pool.get(1000) is own and pool.ops._ws_pool == {}
    pool.capture = 0
    assert pool.get(10).capture == 0


def _in_thread(call):
    got = []
    thread = threading.Thread(target=lambda: got.append(call()))
    thread.start()
    thread.join()
    return got[0]


def test_threads_on_one_stream_do_not_share(pool):
    """A call's launches meet in its workspace, and another thread's launches may come between them."""
    mine, meet = pool.get(100), threading.Barrier(3)
    theirs = []

    def work():
        ws = pool.get(100)
        theirs.append(ws)
        meet.wait()
        assert pool.get(100) is ws
        meet.wait()
    threads = [threading.Thread(target=work) for _ in range(2)]
    for t in threads:
        t.start()
    meet.wait()
    assert pool.get(100) is mine
    meet.wait()
    for t in threads:
        t.join()
    assert len({id(ws) for ws in theirs + [mine]}) == 3


def test_threads_that_have_ended_leave_theirs(pool):
    """Short-lived threads do not pile workspaces up; one that is too small for its heir grows."""
    mine = pool.get(100)
    first = _in_thread(lambda: pool.get(1 << 21))
    assert first is not mine
    for _ in range(5):
        assert _in_thread(lambda: pool.get(1 << 21)) is first
    larger = _in_thread(lambda: pool.get(1 << 22))
    assert larger is not first and pool.waits == 1
    pool.stream = 8
    assert _in_thread(lambda: pool.get(100)) is not larger     # of another stream
    pool.stream = 7
    assert pool.get(100) is mine and len(pool.ops._ws_pool) == 3
