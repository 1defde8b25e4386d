"""Streams and recorded graphs of the operators of language models: the null stream, and what is ordered when the launch
stream changes."""
import ctypes as C
import os
import subprocess
import sys

import numpy as np
import pytest

EINVAL = 1
gpu = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def run_with_torch(program):
    """in a process of its own: torch brings its own HIP runtime, which has to be the first one loaded"""
    done = subprocess.run([sys.executable, "-u", "-c", program], cwd=ROOT, capture_output=True, text=True, timeout=110)
    assert done.returncode == 0 and done.stdout.endswith("done\n"), done.stdout[-1000:] + done.stderr[-2000:]


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


RECORDED_BY_TORCH = """
import torch
assert torch.cuda.is_available()
from swcompiler_amd.hip import SwcHipError, runtime
rt = runtime()
rt.use_default_stream()
gen = torch.Generator().manual_seed(3)
ints = lambda *s: torch.randint(-3, 4, s, generator=gen).to("cuda", torch.bfloat16)
m, n, k = 70, 301, 75          # (rows off the 16-byte grid: both operands are copied into the workspace)
a, b = ints(m, k), ints(k, n)
c = torch.empty(m, n, dtype=torch.bfloat16, device="cuda")
large, weight = ints(3000, 1001), ints(1001, 3001)
side = torch.cuda.Stream()
rt.matrixMatrixFCActAdd(a, b, out=c)
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph, stream=side):
    rt._check(rt.lib.swc_hip_set_stream(side.cuda_stream), "set_stream")
    rt.matrixMatrixFCActAdd(a, b, None, "relu", out=c)
    try:                       # more than the buffer holds: refused, and the recording goes on
        rt.matrixMatrixFCActAdd(large, weight, out=torch.empty(3000, 3001, dtype=torch.bfloat16, device="cuda"))
    except SwcHipError as e:
        assert "while a graph is recorded" in str(e), e
    else:
        raise AssertionError("a workspace was allocated during a recording")
torch.cuda.synchronize()
rt.use_default_stream()
for i in range(4):
    print("replay", i, flush=True)
    # the library's buffer is replaced by a larger one; what was freed would be reused here
    big = torch.empty(3000 - i, 3001, dtype=torch.bfloat16, device="cuda")
    rt.matrixMatrixFCActAdd(large[i:], weight, out=big)
    other = [torch.full((1 << 18,), float("nan"), device="cuda") for _ in range(64)]
    a.copy_(ints(m, k))
    c.fill_(7)
    graph.replay()
    torch.cuda.synchronize()
    want = (a.float() @ b.float()).clamp(min=0).bfloat16()
    assert torch.equal(c, want), (c - want).abs().max()
    assert all(bool(x.isnan().all()) for x in other)
    assert torch.equal(big, (large[i:].float() @ weight.float()).bfloat16())
print("done")
"""


@gpu
def test_a_graph_recorded_by_torch_keeps_its_workspace():
    """ops recorded into a torch graph replay correctly after a larger call has replaced the library's own workspace"""
    run_with_torch(RECORDED_BY_TORCH)
