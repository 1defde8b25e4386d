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
