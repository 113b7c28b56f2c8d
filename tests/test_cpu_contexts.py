"""Contexts of host threads and objects, against a library that only remembers
(the host logic needs no device)."""
import ctypes as C
import threading
import types

import pytest

torch = pytest.importorskip("torch")

from pixal3d.cpp_b200 import _lib as L
from pixal3d.cpp_b200 import ops


class Library:
    """Handles, and the stream each was last given."""

    def __init__(self):
        self.streams, self.made, self.destroyed = {}, [], []

    def _new(self, out, kind):
        handle = 100 + len(self.made)
        self.made.append(kind)
        out._obj.value = handle
        return 0

    def p3d_ctx_create(self, device, stream, out):
        return self._new(out, "create")

    def p3d_ctx_fork(self, ctx, stream, out):
        return self._new(out, "fork")

    def p3d_ctx_set_stream(self, h, s):
        self.streams[h.value] = s.value
        return 0

    def p3d_ctx_destroy(self, h):
        self.destroyed.append(h.value)
        return 0


@pytest.fixture
def library(monkeypatch):
    fake = Library()
    monkeypatch.setattr(ops.L, "lib", fake)
    monkeypatch.setattr(ops, "_CTX", {})
    if hasattr(ops, "_MINE"):
        monkeypatch.setattr(ops, "_MINE", threading.local())
    # torch's current stream is a thread's own
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: types.SimpleNamespace(cuda_stream=threading.get_ident()))
    yield fake


def test_a_thread_does_not_move_another_threads_context(library):
    """Between binding a context and the call that launches on it, another
    thread binds too: the first one's stream stays its own."""
    bound, done, seen = threading.Event(), threading.Event(), {}

    def first():
        c = ops.ctx(0)
        bound.set()
        done.wait(10)
        seen["first"] = (library.streams[c.h.value], threading.get_ident())

    def second():
        bound.wait(10)
        c = ops.ctx(0)
        seen["second"] = (library.streams[c.h.value], threading.get_ident())
        done.set()

    threads = [threading.Thread(target=f) for f in (first, second)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert all(stream == thread for stream, thread in seen.values()), seen


def test_threads_share_one_root_and_keep_their_context(library):
    handles = []

    def work():
        handles.append({ops.ctx(0).h.value for _ in range(5)})

    threads = [threading.Thread(target=work) for _ in range(8)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert all(len(h) == 1 for h in handles)
    assert library.made.count("create") == 1  # one fault flag a device


def test_an_objects_context_is_its_own_and_ends_with_it(library):
    mine, own = ops.ctx(0), ops.new_ctx(0)
    assert mine.h.value != own.h.value and ops.ctx(0) is mine
    handle = own.h.value
    del own
    assert handle in library.destroyed and mine.h.value not in library.destroyed


def test_fork_refuses_null():
    h = C.c_void_p()
    assert L.lib.p3d_ctx_fork(None, None, C.byref(h)) == L.P3D_ERR_INVALID
