"""The operators' torch binding called from several host threads, with a stand-in
for the library: no call may be given device memory that another may still use."""
import gc
import importlib
import struct
import threading
import weakref

import pytest

torch = pytest.importorskip("torch")

NEED = 1 << 16


class Library:
    """Entry points that refuse a call without NEED bytes of workspace, as the
    library's do, and meet at a barrier inside a call that is taken."""

    def __init__(self, layout, ws_at, parties):
        self.layout, self.ws_at = layout, ws_at
        self.inside = threading.Barrier(parties, timeout=20)
        self.lock, self.taken = threading.Lock(), []

    def mx_op(self, packed, stream):
        values = self.layout.unpack(packed)
        ws, size = values[self.ws_at], values[self.ws_at + 1]
        if not ws or size < NEED:
            return -1
        with self.lock:
            self.taken.append((ws, size))
        self.inside.wait()
        return 0

    def mx_op_workspace(self, packed, need):
        need._obj.value = NEED
        return 0


@pytest.fixture
def ops(monkeypatch):
    ops = importlib.import_module("maxim-rs_b200.ops")
    monkeypatch.setattr(ops, "_kept", ops._Kept())  # nothing of the stand-in's stays behind
    monkeypatch.setattr(ops, "_cuda_device", lambda: 0)
    monkeypatch.setattr(ops, "_cuda_stream", lambda device: 0)
    monkeypatch.setattr(ops, "_cuda_capturing", lambda: False)
    empty = torch.empty
    monkeypatch.setattr(ops.torch, "empty", lambda size, dtype, device: empty(size, dtype=dtype))
    return ops


def test_threads_on_one_stream_have_workspaces_of_their_own(ops, monkeypatch):
    layout, calls, threads = struct.Struct("<2Q2q"), 3, 4
    lib = Library(layout, 2, threads)
    monkeypatch.setattr(ops._native, "lib", lambda: lib)
    errors = []

    def work():
        try:
            for _ in range(calls):
                ops._launch("mx_op", layout, [1, 2, 0, 0], 0, 2)
        except Exception as e:  # a thread's assertion would be lost
            errors.append(e)

    run = [threading.Thread(target=work) for _ in range(threads)]
    for t in run:
        t.start()
    for t in run:
        t.join()
    assert not errors, errors
    # The barrier lets `threads` calls through at a time: those that are in
    # flight together must not overlap.
    assert len(lib.taken) == threads * calls
    for i in range(0, len(lib.taken), threads):
        spans = sorted(lib.taken[i:i + threads])
        assert all(a + n <= b for (a, n), (b, _) in zip(spans, spans[1:])), spans


def test_a_thread_keeps_its_workspace(ops, monkeypatch):
    layout = struct.Struct("<2Q2q")
    lib = Library(layout, 2, 1)
    monkeypatch.setattr(ops._native, "lib", lambda: lib)
    for _ in range(3):
        ops._launch("mx_op", layout, [1, 2, 0, 0], 0, 2)
    assert len(set(lib.taken)) == 1


def test_kept_workspaces_can_be_released(ops, monkeypatch):
    """By the thread that keeps them; another thread's go with it."""
    layout = struct.Struct("<2Q2q")
    monkeypatch.setattr(ops._native, "lib", lambda: Library(layout, 2, 1))
    made = []
    empty = ops.torch.empty

    def recording(*a, **kw):
        t = empty(*a, **kw)
        made.append(weakref.ref(t))
        return t

    monkeypatch.setattr(ops.torch, "empty", recording)

    def call():
        ops._launch("mx_op", layout, [1, 2, 0, 0], 0, 2)

    call()
    t = threading.Thread(target=call)
    t.start()
    t.join()
    gc.collect()
    assert [r() is not None for r in made] == [True, False]
    ops.release_workspaces()
    gc.collect()
    assert made[0]() is None
    call()
    assert len(made) == 3
