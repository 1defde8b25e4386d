"""Streams and recorded graphs of the operators of language models: the null stream, what is ordered when the launch stream
changes, and calls with torch tensors."""
import ctypes as C
import os
import subprocess
import sys

import numpy as np
import pytest

from swcompiler_amd import hip
from swcompiler_amd.hip import SwcHipError

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


# ------------------------------------------------------------------------- torch's streams: who waits for whom (no device)
class _FakeTorch:
    """as much of torch as the binding asks about streams, and a log of what it is told"""

    def __init__(self, current=0, device=0, capturing=()):
        self.log, self.now, self.device, self.capturing = [], current, device, capturing
        self.cuda, self._C = self, self

    def stream_of(self, handle):
        fake = self

        class Stream:
            cuda_stream = handle

            def wait_stream(self, other):
                fake.log.append(f"{handle} waits for {other.cuda_stream}")

            def __enter__(self):
                self.before, fake.now = fake.now, handle

            def __exit__(self, *_):
                fake.now = self.before
        return Stream()

    def _cuda_getDevice(self):
        return self.device

    def _cuda_getCurrentRawStream(self, device):
        return self.now

    def current_stream(self, device):
        return self.stream_of(self.now)

    def default_stream(self, device):
        return self.stream_of(0)

    def ExternalStream(self, handle, device):
        return self.stream_of(handle)

    def stream(self, s):
        return s

    def is_current_stream_capturing(self):
        return self.now in self.capturing


class _FakeTensor:
    dtype, shape = "torch.float32", (4, 8)

    def get_device(self):
        return 0

    def data_ptr(self):
        return 1 << 20

    def is_contiguous(self):
        return True

    def numel(self):
        return 32


class _FakeLib:
    def __init__(self, fake, stream):
        self.fake, self.handle = fake, stream

    def swc_hip_stream(self):
        return self.handle

    def __getattr__(self, name):
        return lambda *args: self.fake.log.append("call") or 0


def call_with(monkeypatch, ours, **kw):
    fake = _FakeTorch(**kw)
    monkeypatch.setitem(sys.modules, "torch", fake)
    rt = object.__new__(hip.SwcHip)
    rt.device, rt.lib = 0, _FakeLib(fake, ours)
    a, b, c = _FakeTensor(), _FakeTensor(), _FakeTensor()
    b.shape, c.shape = (8, 8), (4, 8)
    try:
        rt.matrixMatrixFCActAdd(a, b, out=c)
        first, fake.log = fake.log, []
        rt.adamw([a], [a], [a], [a], _state(), 1e-3, 0.9, 0.99, 1e-8, 0.0)
        assert fake.log == first
        return first
    finally:
        hip._TORCH_KINDS.clear()


def _state():
    x = _FakeTensor()
    x.dtype, x.shape = "torch.int32", (hip.ADAMW_STATE_WORDS,)
    return x


def test_calls_with_torch_operands_are_ordered(monkeypatch):
    assert call_with(monkeypatch, 1) == ["call"]                   # both the null stream
    assert call_with(monkeypatch, 77, current=77) == ["call"]
    assert call_with(monkeypatch, 77) == ["77 waits for 0", "call", "0 waits for 77"]
    assert call_with(monkeypatch, 1, current=5) == ["0 waits for 5", "call", "5 waits for 0"]
    assert call_with(monkeypatch, 77, capturing=(77,)) == ["call"]     # recorded by the library: ordered where launched


def test_a_refused_call_leaves_nothing_behind(monkeypatch):
    """a call with torch tensors that is refused does not make the next one, without any, ask torch"""
    fake = _FakeTorch(current=5, capturing=(5,))
    monkeypatch.setitem(sys.modules, "torch", fake)
    rt = object.__new__(hip.SwcHip)
    rt.device, rt.lib = 0, _FakeLib(fake, 77)
    rt._malloc, rt._free = lambda nbytes: 1 << 20, lambda ptr: None
    a, b = _FakeTensor(), _FakeTensor()
    try:
        with pytest.raises(SwcHipError, match="do not multiply"):
            rt.matrixMatrixFCActAdd(a, b)
        d = hip.DeviceArray(rt, (4, 4))
        rt.matrixMatrixFCActAdd(d, d, out=hip.DeviceArray(rt, (4, 4)))
        assert fake.log == ["call"]
        b.shape = (8, 8)
        rt.lib.handle, fake.log = None, []          # shut down: the library is asked, and refuses
        rt.matrixMatrixFCActAdd(a, b, out=_FakeTensor())
        assert fake.log == ["call"]
    finally:
        hip._TORCH_KINDS.clear()


def test_torch_operands_are_refused_where_they_cannot_be_ordered(monkeypatch):
    with pytest.raises(SwcHipError, match="torch is recording a graph on another stream"):
        call_with(monkeypatch, 77, current=5, capturing=(5,))
    with pytest.raises(SwcHipError, match="the current device is 1, the runtime's 0"):
        call_with(monkeypatch, 1, device=1)


TORCH_STREAMS = """
import torch
assert torch.cuda.is_available()
from swcompiler_amd.hip import SwcHipError, runtime
rt = runtime()
gen = torch.Generator().manual_seed(3)
n = 2048
ints = lambda *s: torch.randint(-2, 3, s, generator=gen).to("cuda")
eye, w = torch.eye(n, device="cuda"), ints(64, 200).bfloat16()
side = torch.cuda.Stream()
torch.cuda.synchronize()


def late(value):
    # `value` behind some milliseconds of torch's work
    x = eye
    for _ in range(30):
        x = x @ eye
    return value * x[:1, :1].bfloat16()


def check(name):
    for i in range(5):
        a = late(ints(70, 64).bfloat16())
        c = torch.full((70, 200), 7, device="cuda", dtype=torch.bfloat16)
        rt.matrixMatrixFCActAdd(a, w, None, "relu", out=c)
        got = c.float()                       # torch's next work reads the result ...
        want = (a.float() @ w.float()).clamp(min=0).bfloat16().float()
        del a, c                              # ... and its allocator reuses the operands
        junk = [torch.full((70, 200), float("nan"), device="cuda", dtype=torch.bfloat16) for _ in range(8)]
        g = late(ints(300).bfloat16())[0] * 0.5
        p, m, v = (torch.zeros(300, device="cuda") for _ in range(3))
        state = torch.zeros(8, dtype=torch.int32, device="cuda")
        rt.adamwAdvance(state, 0.9, 0.99)
        rt.adamw([p], [g], [m], [v], state, 1e-3, 0.9, 0.99, 1e-8, 0.0)
        steps, mean = state[0].clone(), m * 10
        torch.cuda.current_stream().synchronize()
        assert torch.equal(got, want), name
        assert int(steps) == 1 and torch.allclose(mean, g.float(), rtol=1e-5), name


for library in ("own", "null"):
    if library == "null":
        rt.use_default_stream()
    print("library on its", library, "stream", flush=True)
    check(library + ", torch on its default stream")
    with torch.cuda.stream(side):
        check(library + ", torch on a side stream")
torch.cuda.synchronize()
graph, c = torch.cuda.CUDAGraph(), torch.empty(70, 200, device="cuda", dtype=torch.bfloat16)
a = ints(70, 64).bfloat16()
with torch.cuda.graph(graph):
    c.fill_(1)
    try:
        rt.matrixMatrixFCActAdd(a, w, out=c)
    except SwcHipError as e:
        assert "torch is recording" in str(e), e
    else:
        raise AssertionError("an op that the graph would lack")
print("done")
"""


@gpu
def test_torch_streams():
    """torch on its default and on a side stream, the library on its own and on the null stream: results are ordered with
    the work before and behind the calls, no synchronisation between them"""
    run_with_torch(TORCH_STREAMS)
