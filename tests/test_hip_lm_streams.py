"""Streams and recorded graphs of the operators of language models: the null stream, and what is ordered when the launch
stream changes."""
import ctypes as C

import numpy as np
import pytest

EINVAL = 1
gpu = pytest.mark.gpu


@pytest.fixture(scope="module")
def rt():
    from swcompiler_amd.hip import runtime
    return runtime()


@gpu
def test_the_null_stream(rt):
    """events, timers and copies on the null stream; it is named by its handle, and refused for recording"""
    x = rt.upload(np.zeros(1000, np.float32))
    rt.sync()
    rt.use_default_stream()
    try:
        assert rt.lib.swc_hip_stream() == 1       # hipStreamLegacy: what swc_hip_set_stream takes
        rt._check(rt.lib.swc_hip_set_stream(rt.lib.swc_hip_stream()), "set_stream")
        rt._check(rt.lib.swc_hip_timer_begin(), "timer")
        rt._check(rt.lib.swc_hip_event_record(0), "event")
        rt._check(rt.lib.swc_hip_fill_f(x.ptr, 3.0, x.size), "fill")
        rt._check(rt.lib.swc_hip_event_record(1), "event")
        rt._check(rt.lib.swc_hip_timer_end(), "timer")
        assert np.all(x.numpy() == 3)
        assert rt.lib.swc_hip_timer_elapsed_ms() >= rt.lib.swc_hip_event_elapsed_ms(0, 1) >= 0
        assert rt.lib.swc_hip_graph_begin() == EINVAL and b"null stream" in rt.lib.swc_hip_last_error()
    finally:
        rt.sync()
        rt._check(rt.lib.swc_hip_set_stream(None), "set_stream")
    assert rt.lib.swc_hip_stream() not in (None, 0, 1)


class Busy:
    """some 20 ms of products on whatever stream the library launches on"""

    def __init__(self, rt):
        self.rt, self.n = rt, 4096
        self.a, self.b, self.c = (rt.empty((self.n, self.n)) for _ in range(3))
        for x in (self.a, self.b):
            rt._check(rt.lib.swc_hip_fill_f(x.ptr, 1.0, self.n * self.n), "fill")

    def __call__(self):
        for _ in range(20):
            self.rt.matrixMatrixFCActAdd(self.a, self.b, out=self.c)


@gpu
def test_a_change_of_stream_waits(rt):
    """what was launched before the launch stream changes has ended when later work runs: from the library's own stream
    to the null stream and back, and to a stream of the caller's"""
    busy, x = Busy(rt), rt.upload(np.zeros(1000, np.float32))
    hiprt = C.CDLL("libamdhip64.so.7")
    stream = C.c_void_p()
    assert hiprt.hipStreamCreateWithFlags(C.byref(stream), 1) == 0
    to = {"null": rt.use_default_stream, "own": lambda: rt._check(rt.lib.swc_hip_set_stream(None), "set_stream"),
          "caller's": lambda: rt._check(rt.lib.swc_hip_set_stream(stream), "set_stream")}
    try:
        for value, name in enumerate(("null", "own", "caller's"), 1):
            busy()
            rt._check(rt.lib.swc_hip_fill_f(x.ptr, float(value), x.size), "fill")
            to[name]()
            assert np.all(x.numpy() == value), name      # (copied on the new stream)
    finally:
        rt.sync()
        to["own"]()
        hiprt.hipStreamDestroy(stream)


@gpu
def test_a_new_state_survives_a_change_of_stream(rt):
    """the counter that adamw_state clears on one stream is counted on the next"""
    busy = Busy(rt)
    try:
        for _ in range(3):
            busy()
            state = rt.adamw_state()
            rt.use_default_stream()
            rt.adamwAdvance(state, 0.9, 0.99)
            rt.adamwAdvance(state, 0.9, 0.99)
            assert state.numpy()[0] == 2
            rt._check(rt.lib.swc_hip_set_stream(None), "set_stream")
    finally:
        rt._check(rt.lib.swc_hip_set_stream(None), "set_stream")


@gpu
def test_no_change_of_stream_while_recording(rt):
    graph = C.c_void_p()
    rt._check(rt.lib.swc_hip_graph_begin(), "begin")
    try:
        assert rt.lib.swc_hip_set_stream(C.c_void_p(1)) == EINVAL and b"recorded" in rt.lib.swc_hip_last_error()
    finally:
        rt._check(rt.lib.swc_hip_graph_end(C.byref(graph)), "end")
    rt._check(rt.lib.swc_hip_graph_destroy(graph), "destroy")
