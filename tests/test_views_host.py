"""What becomes of a view's tensor and of its stream's order when the view goes, with a library that only takes notes."""
import gc
import os
import subprocess
import sys
import threading

import pytest

from onyxia_b200 import _ffi, backend, ir


class Notes:
    """The session's entry points; `refuses`: streams that cannot be waited for."""

    def __init__(self):
        self.calls, self.refuses = [], set()

    def ox_session_num_outputs(self, h):
        return 1

    def ox_session_device_view(self, h, t, stream, ptr):
        self.calls.append(("view", stream))
        return 0

    def ox_session_after_stream(self, h, stream):
        self.calls.append(("after", stream, threading.get_ident()))
        return 7 if stream in self.refuses else 0

    def ox_session_sync(self, h):
        self.calls.append(("sync",))
        return 0

    def ox_session_free(self, h):
        self.calls.append(("free",))


class Tensor:
    released = 0
    handle = None

    def __init__(self, dtype=ir.F32):
        self.dtype = dtype

    def describe(self):
        return self.dtype, (2, 3)

    def clone(self):
        return Tensor()

    def __del__(self):
        type(self).released += 1


@pytest.fixture
def session(monkeypatch):
    notes = Notes()
    monkeypatch.setattr(_ffi, "cuda_lib", lambda: notes)
    s = backend.CudaSession(1)
    Tensor.released = 0
    yield s, notes
    s.close()


def test_a_view_that_goes_orders_the_session_and_lets_its_tensor_go(session):
    s, notes = session
    v, t = s.view(Tensor(), 5), None
    released = Tensor.released
    del v, t
    gc.collect()
    assert notes.calls[-1] == ("after", 5, threading.get_ident()) and Tensor.released == released + 1


def test_the_tensor_stays_where_the_stream_cannot_be_waited_for(session):
    s, notes = session
    notes.refuses.add(6)
    v = s.view(Tensor(), 6)
    released = Tensor.released
    del v
    gc.collect()
    assert notes.calls[-1][0] == "after" and Tensor.released == released  # its memory may not come back to the pool
    s.close()
    gc.collect()
    assert Tensor.released == released + 1


def test_a_view_that_goes_on_another_thread_is_ended_by_the_sessions_next_call(session):
    s, notes = session
    held = [s.view(Tensor(), 5)]
    released = Tensor.released
    other = threading.Thread(target=held.clear)
    other.start()
    other.join()
    gc.collect()
    assert not [c for c in notes.calls if c[0] == "after"] and Tensor.released == released
    assert s._h == 1  # what every call begins with
    gc.collect()
    assert notes.calls[-1] == ("after", 5, threading.get_ident()) and Tensor.released == released + 1


def test_the_types_that_arrays_know(session):
    s, _ = session
    for dtype, kind in ((ir.F32, "<f4"), (ir.F16, "<f2"), (ir.BF16, "<i2"), (ir.I64, "<i8"), (ir.I32, "<i4"), (ir.U32, "<u4"), (ir.U8, "|u1"), (ir.I8, "|i1"), (ir.BOOL, "|b1")):
        assert s.view(Tensor(dtype)).__cuda_array_interface__["typestr"] == kind
    for dtype in (ir.U4, ir.I4):
        with pytest.raises(ValueError, match="4-bit"):
            s.view(Tensor(dtype))


def test_views_of_a_closed_session_ask_nothing_of_it(session):
    s, notes = session
    v = s.view(Tensor(), 5)
    s.close()
    del v
    gc.collect()
    assert notes.calls[-1] == ("free",)


def test_views_that_are_held_until_the_interpreter_ends_go_quietly():
    here = os.path.dirname(os.path.abspath(__file__))
    program = ("import sys\nimport test_views_host as t\nfrom onyxia_b200 import _ffi, backend\nnotes = t.Notes()\n_ffi.cuda_lib = lambda: notes\nsys.held = backend.CudaSession(1).view(t.Tensor(), 5)\n"
               "held = backend.CudaSession(1).view(t.Tensor(), 5)\n")
    r = subprocess.run([sys.executable, "-c", program], capture_output=True, text=True, env=dict(os.environ, PYTHONPATH=os.pathsep.join([here, os.path.dirname(here)])))
    assert r.returncode == 0 and r.stderr == ""
