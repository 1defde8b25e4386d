"""ctypes binding of libswc_hip.so (C ABI declared in include/swc_hip.h).

Method names and argument order mirror the reference's CPU kernels
(src/codegen/utils/kernels.h) — the same correspondence the C ABI keeps — so a
parity test reads like a call sequence of the reference's generated program.
Data lives in DeviceArray objects (device memory + shape); numpy arrays cross
only through upload()/download().  The operators of language models take torch tensors too, as
they are, and order themselves with the work on torch's current stream; a program
that uses torch imports it before this library is loaded (torch brings a HIP
runtime of its own, and a process has one).  Sharing a stream
(use_default_stream) saves the waits between the two.

No fallback: a missing library or device raises SwcHipError.
"""
import ctypes as C
import os
import sys

import numpy as np

_HERE = os.path.dirname(os.path.abspath(__file__))

EXPORTS = [
    "swc_hip_init", "swc_hip_shutdown", "swc_hip_malloc", "swc_hip_free", "swc_hip_h2d", "swc_hip_d2h",
    "swc_hip_d2d", "swc_hip_copy_h2d_async", "swc_hip_copy_wait_ops", "swc_hip_ops_wait_copies", "swc_hip_copy_sync", "swc_hip_fill_f", "swc_hip_sync", "swc_hip_last_error", "swc_hip_stream",
    "swc_hip_set_stream", "swc_hip_device_name", "swc_hip_timer_begin", "swc_hip_timer_end",
    "swc_hip_timer_elapsed_ms", "swc_hip_event_record", "swc_hip_event_elapsed_ms", "swc_hip_graph_begin",
    "swc_hip_graph_end", "swc_hip_graph_launch", "swc_hip_graph_destroy", "swc_hip_device_cus", "swc_hip_last_kernel", "swc_hip_reload_switches",
    "swc_hip_enable_auto_workspace", "swc_hip_conv2dGrad_workspace_bytes", "swc_hip_matrixSoftmaxWithLoss_workspace_bytes",
    "swc_hip_matrixMatrixFCBias_noalloc_f",
    "swc_hip_matrixMatrixMul_f", "swc_hip_batchedadd_f", "swc_hip_relu_f",
    "swc_hip_vecAdd_f", "swc_hip_conv2d_f", "swc_hip_batchnormalization_f", "swc_hip_maxpool_f",
    "swc_hip_maxpool_argmax_f", "swc_hip_avgpool_f", "swc_hip_transpose4d_f", "swc_hip_transpose2d_f",
    "swc_hip_matrixSoftmax_f", "swc_hip_matrixTanh_f", "swc_hip_argMax_i", "swc_hip_accuracy_i", "swc_hip_fill_i",
    "swc_hip_matrixMatrixFCBias_f", "swc_hip_vecAddRelu_f", "swc_hip_batchnormRelu_f",
    "swc_hip_batchnormReluMaxpool_f", "swc_hip_conv2dFused_f", "swc_hip_conv2dFusedAdd_f",
    "swc_hip_conv2dFusedMaxpool_f", "swc_hip_conv2dFusedMaxpool_workspace_bytes",
    "swc_hip_set_workspace", "swc_hip_matrixMatrixFCBiasSoftmax_f", "swc_hip_gemm_workspace_bytes", "swc_hip_conv2d_workspace_bytes", "swc_hip_host_malloc", "swc_hip_host_free", "swc_hip_matrixTrans_f", "swc_hip_matrixTanhGrad_f", "swc_hip_matrixSoftmaxWithLoss_f",
    "swc_hip_matrixSoftmaxGrad_f", "swc_hip_matrixSoftmaxWithLossGrad_f", "swc_hip_conv2dGrad_f",
    "swc_hip_maxpoolGrad_f", "swc_hip_batchedreduceadd_f", "swc_hip_sgd_f", "swc_hip_reluGrad_f",
    "swc_hip_matrixMatrixFCActAdd_f", "swc_hip_matrixMatrixFCActAdd_bf", "swc_hip_matrixMatrixFCActAdd_workspace_bytes",
    "swc_hip_matrixMatrixFCActAddGrad_f", "swc_hip_matrixMatrixFCActAddGrad_bf",
    "swc_hip_matrixMatrixFCActAddGrad_workspace_bytes",
    "swc_hip_matrixFCSoftmaxWithLoss_f", "swc_hip_matrixFCSoftmaxWithLoss_bf",
    "swc_hip_matrixFCSoftmaxWithLoss_workspace_bytes", "swc_hip_matrixFCSoftmaxWithLossGrad_f",
    "swc_hip_matrixFCSoftmaxWithLossGrad_bf", "swc_hip_matrixFCSoftmaxWithLossGrad_workspace_bytes",
    "swc_hip_adamwAdvance", "swc_hip_adamw_f", "swc_hip_adamw_bf", "swc_hip_adamw8_f", "swc_hip_adamw8_bf",
]

ACTIVATIONS = {"none": 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4}   # the SWC_HIP_ACT_* values
ADAMW_STATE_WORDS = 8     # SWC_HIP_ADAMW_STATE_BYTES in 32-bit words
ADAMW_BLOCK = 256         # elements that share a scale of the 8-bit states


class SwcHipError(RuntimeError):
    pass


def lib_path():
    return os.path.join(_HERE, "libswc_hip.so")


def load_library():
    """dlopen the in-tree library; raises if it has not been built."""
    path = lib_path()
    if not os.path.exists(path):
        raise SwcHipError(f"{path} is missing: build it with `python -m swcompiler_amd.build` "
                          "(there is no CPU fallback)")
    lib = C.CDLL(path)
    vp, sz, i32, f32 = C.c_void_p, C.c_size_t, C.c_int, C.c_float
    szp = C.POINTER(C.c_size_t)
    f64 = C.c_double
    fc = [i32, i32, i32, vp, i32, vp, i32, vp, i32, vp, i32, vp, i32, vp, i32]
    fc_grad = [i32, i32, i32, vp, i32, vp, i32, vp, i32, vp, i32, i32, vp, i32, vp, i32, vp]
    loss = [i32, i32, i32, vp, i32, vp, i32, vp, vp, vp, vp, vp]
    loss_grad = [i32, i32, i32, vp, i32, vp, i32, vp, vp, vp, vp, vp, i32, vp, i32, vp]
    adamw_tail = [vp, szp, vp, f32, f64, f64, f32, f32, vp, vp]
    sig = {
        "swc_hip_init": (i32, [i32]),
        "swc_hip_shutdown": (i32, []),
        "swc_hip_reload_switches": (i32, []),
        "swc_hip_malloc": (vp, [sz]),
        "swc_hip_free": (i32, [vp]),
        "swc_hip_h2d": (i32, [vp, vp, sz]),
        "swc_hip_d2h": (i32, [vp, vp, sz]),
        "swc_hip_d2d": (i32, [vp, vp, sz]),
        "swc_hip_fill_f": (i32, [vp, f32, sz]),
        "swc_hip_copy_h2d_async": (i32, [vp, vp, sz]),
        "swc_hip_copy_wait_ops": (i32, []),
        "swc_hip_ops_wait_copies": (i32, []),
        "swc_hip_copy_sync": (i32, []),
        "swc_hip_sync": (i32, []),
        "swc_hip_last_error": (C.c_char_p, []),
        "swc_hip_stream": (vp, []),
        "swc_hip_set_stream": (i32, [vp]),
        "swc_hip_device_name": (C.c_char_p, []),
        "swc_hip_timer_begin": (i32, []),
        "swc_hip_timer_end": (i32, []),
        "swc_hip_timer_elapsed_ms": (f32, []),
        "swc_hip_event_record": (i32, [i32]),
        "swc_hip_event_elapsed_ms": (f32, [i32, i32]),
        "swc_hip_graph_begin": (i32, []),
        "swc_hip_graph_end": (i32, [C.POINTER(vp)]),
        "swc_hip_graph_launch": (i32, [vp]),
        "swc_hip_graph_destroy": (i32, [vp]),
        "swc_hip_device_cus": (i32, []),
        "swc_hip_last_kernel": (C.c_char_p, []),
        "swc_hip_enable_auto_workspace": (i32, [i32]),
        "swc_hip_conv2dGrad_workspace_bytes": (sz, [szp] * 6 + [sz]),
        "swc_hip_matrixSoftmaxWithLoss_workspace_bytes": (sz, [i32, i32]),
        "swc_hip_matrixMatrixFCBias_noalloc_f": (i32, [i32, i32, i32, vp, i32, vp, i32, vp, vp, i32, i32]),
        "swc_hip_matrixMatrixMul_f": (i32, [i32, i32, i32, vp, i32, vp, i32, vp, i32]),
        "swc_hip_batchedadd_f": (i32, [vp, vp, vp, sz, sz]),
        "swc_hip_relu_f": (i32, [vp, vp, sz]),
        "swc_hip_vecAdd_f": (i32, [i32, vp, vp, vp]),
        "swc_hip_conv2d_f": (i32, [vp, vp, vp, vp, szp, szp, szp, szp, szp, szp, szp, sz]),
        "swc_hip_batchnormalization_f": (i32, [vp, vp, vp, vp, vp, vp, szp, f32]),
        "swc_hip_maxpool_f": (i32, [vp, vp, szp, szp, szp, szp, szp]),
        "swc_hip_maxpool_argmax_f": (i32, [vp, vp, vp, szp, szp, szp, szp, szp]),
        "swc_hip_avgpool_f": (i32, [vp, vp, szp, szp, szp, szp, szp]),
        "swc_hip_transpose4d_f": (i32, [vp, vp, szp, szp, szp]),
        "swc_hip_transpose2d_f": (i32, [vp, vp, szp, szp, szp]),
        "swc_hip_matrixSoftmax_f": (i32, [i32, i32, vp, i32, vp, i32]),
        "swc_hip_matrixTanh_f": (i32, [i32, i32, vp, i32, vp, i32]),
        "swc_hip_argMax_i": (i32, [vp, vp, i32, i32, i32]),
        "swc_hip_accuracy_i": (i32, [vp, vp, vp, i32, i32]),
        "swc_hip_fill_i": (i32, [vp, i32, sz]),
        "swc_hip_matrixMatrixFCBias_f": (i32, [i32, i32, i32, vp, i32, vp, i32, vp, vp, i32, i32]),
        "swc_hip_matrixMatrixFCBiasSoftmax_f": (i32, [i32, i32, i32, vp, i32, vp, i32, vp, vp, i32]),
        "swc_hip_vecAddRelu_f": (i32, [i32, vp, vp, vp]),
        "swc_hip_batchnormRelu_f": (i32, [vp, vp, vp, vp, vp, vp, szp, f32]),
        "swc_hip_batchnormReluMaxpool_f": (i32, [vp, vp, vp, vp, vp, vp, szp, f32, szp, szp, szp, szp]),
        "swc_hip_conv2dFused_f": (i32, [vp, vp, vp, vp, szp, szp, szp, szp, szp, szp, szp, sz,
                                        vp, vp, vp, vp, f32, i32]),
        "swc_hip_conv2dFusedAdd_f": (i32, [vp, vp, vp, vp, szp, szp, szp, szp, szp, szp, szp, sz,
                                        vp, vp, vp, vp, f32, vp, i32]),
        "swc_hip_conv2dFusedMaxpool_f": (i32, [vp, vp, vp, vp, szp, szp, szp, szp, szp, szp, szp, sz,
                                            vp, vp, vp, vp, f32, i32, szp, szp, szp, szp]),
        "swc_hip_conv2dFusedMaxpool_workspace_bytes": (sz, [szp] * 6 + [sz] + [szp] * 4),
        "swc_hip_set_workspace": (i32, [vp, sz]),
        "swc_hip_host_malloc": (vp, [sz]),
        "swc_hip_host_free": (i32, [vp]),
        "swc_hip_gemm_workspace_bytes": (sz, [i32, i32, i32]),
        "swc_hip_conv2d_workspace_bytes": (sz, [szp] * 6 + [sz]),
        "swc_hip_matrixTrans_f": (i32, [i32, i32, vp, i32, vp, i32]),
        "swc_hip_matrixTanhGrad_f": (i32, [i32, i32, vp, i32, vp, i32, vp, i32]),
        "swc_hip_matrixSoftmaxWithLoss_f": (i32, [i32, i32, vp, i32, vp, i32, vp, vp]),
        "swc_hip_matrixSoftmaxGrad_f": (i32, [i32, i32, vp, i32, vp, i32, vp]),
        "swc_hip_matrixSoftmaxWithLossGrad_f": (i32, [i32, i32, vp, i32, vp, i32, vp]),
        "swc_hip_conv2dGrad_f": (i32, [vp, vp, vp, vp, vp, vp, szp, szp, szp, szp, szp, szp, szp, sz]),
        "swc_hip_maxpoolGrad_f": (i32, [vp, vp, vp, szp, szp, szp, szp, szp]),
        "swc_hip_batchedreduceadd_f": (i32, [vp, vp, sz, sz]),
        "swc_hip_sgd_f": (i32, [sz, vp, vp, vp, vp, f32, f32, f32, sz]),
        "swc_hip_reluGrad_f": (i32, [vp, vp, vp, sz]),
        "swc_hip_matrixMatrixFCActAdd_f": (i32, fc),
        "swc_hip_matrixMatrixFCActAdd_bf": (i32, fc),
        "swc_hip_matrixMatrixFCActAdd_workspace_bytes": (sz, [i32] * 4),
        "swc_hip_matrixMatrixFCActAddGrad_f": (i32, fc_grad),
        "swc_hip_matrixMatrixFCActAddGrad_bf": (i32, fc_grad),
        "swc_hip_matrixMatrixFCActAddGrad_workspace_bytes": (sz, [i32] * 4),
        "swc_hip_matrixFCSoftmaxWithLoss_f": (i32, loss),
        "swc_hip_matrixFCSoftmaxWithLoss_bf": (i32, loss),
        "swc_hip_matrixFCSoftmaxWithLoss_workspace_bytes": (sz, [i32] * 4),
        "swc_hip_matrixFCSoftmaxWithLossGrad_f": (i32, loss_grad),
        "swc_hip_matrixFCSoftmaxWithLossGrad_bf": (i32, loss_grad),
        "swc_hip_matrixFCSoftmaxWithLossGrad_workspace_bytes": (sz, [i32] * 4),
        "swc_hip_adamwAdvance": (i32, [vp, f64, f64]),
        "swc_hip_adamw_f": (i32, [i32] + [vp] * 4 + adamw_tail),
        "swc_hip_adamw_bf": (i32, [i32] + [vp] * 4 + adamw_tail),
        "swc_hip_adamw8_f": (i32, [i32] + [vp] * 6 + adamw_tail),
        "swc_hip_adamw8_bf": (i32, [i32] + [vp] * 6 + adamw_tail),
    }
    for name, (res, args) in sig.items():
        fn = getattr(lib, name)
        fn.restype, fn.argtypes = res, args
    return lib


def _dims(seq):
    return (C.c_size_t * len(seq))(*[int(v) for v in seq])


def pool_out_dims(idims, kernels, strides, pads):
    """src/op/dlOp/dlOp.cpp:195-196: o = (i + pad_begin + pad_end - k) / s + 1, pads = {t,l,b,r}."""
    n, h, w, c = idims
    return (n, (h + pads[0] + pads[2] - kernels[0]) // strides[0] + 1,
            (w + pads[1] + pads[3] - kernels[1]) // strides[1] + 1, c)


def _int32(x, what):
    """x where the library takes a 32-bit int (ctypes would cut a larger one off without a word)"""
    if x > 0x7fffffff:
        raise SwcHipError(f"{what}: {x} is beyond 2^31 - 1")
    return x


class _Arg:
    """What an op needs of an operand: its address, shape, element type and row stride.  Operands are DeviceArrays or
    torch tensors on the runtime's device (taken as they are: any row stride, columns contiguous)."""

    __slots__ = ("ptr", "shape", "type", "ld")

    def __init__(self, rt, x, what, name):
        try:
            self.shape = shape = x.shape
        except AttributeError:
            raise _no_operand(x, what, name) from None
        self.ld = shape[-1] if shape else 1
        if isinstance(x, DeviceArray):
            self.ptr, self.type = x.ptr, _NUMPY_TYPES.get(x.dtype.name)
            return
        self.ptr, self.type = _torch_operand(rt, x, what, name)
        if x.is_contiguous():
            return
        stride = x.stride()
        if len(shape) > 2 or (shape[-1] > 1 and stride[-1] != 1):
            raise SwcHipError(f"{what}: {name}: the elements of a row are not contiguous (strides {stride})")
        if len(shape) == 2 and shape[0] > 1:
            self.ld = stride[0]
            if self.ld < shape[1]:
                raise SwcHipError(f"{what}: {name}: rows overlap (stride {self.ld}, {shape[1]} columns)")
            _int32(self.ld, f"{what}: {name}: row stride")

    @property
    def size(self):
        n = 1
        for d in self.shape:
            n *= d
        return n


def _no_operand(x, what, name):
    return SwcHipError(f"{what}: {name}: expected a DeviceArray or a torch tensor on the GPU, got {type(x).__name__}")


def _torch_operand(rt, x, what, name):
    """-> (address, element type) of a torch tensor on the runtime's device"""
    try:
        if x.get_device() != rt.device:
            raise SwcHipError(f"{what}: {name}: the tensor is on {x.device}, the runtime on device {rt.device}")
        kind = _TORCH_KINDS.get(x.dtype)
        ptr = x.data_ptr()
    except AttributeError:
        raise _no_operand(x, what, name) from None
    if kind is None:
        kind = _TORCH_KINDS[x.dtype] = _TORCH_TYPES.get(str(x.dtype), "?")
    rt._torch_given = True
    return ptr or None, kind


_NULL_STREAM = 1      # the library's name for the null stream (hipStreamLegacy); torch's is 0
_TORCH_KINDS = {}     # torch.dtype -> element type, filled as they are met (this module does not import torch)
_NUMPY_TYPES = {"float32": "f32", "int32": "i32", "uint16": "bf16", "uint8": "u8"}   # bfloat16 travels as its bits
_TORCH_TYPES = {"torch.float32": "f32", "torch.int32": "i32", "torch.bfloat16": "bf16", "torch.uint16": "bf16",
                "torch.uint8": "u8", "torch.float8_e4m3fn": "u8"}


class DeviceArray:
    """A device allocation with a shape and dtype (float32, int32, uint16 for bfloat16 bits, or uint8)."""

    def __init__(self, rt, shape, dtype=np.float32):
        self.rt = rt
        self.shape = tuple(int(s) for s in shape)
        self.dtype = np.dtype(dtype)
        self.size = int(np.prod(self.shape)) if self.shape else 1
        self.nbytes = self.size * self.dtype.itemsize
        self.ptr = rt._malloc(self.nbytes)

    def reshape(self, *shape):
        view = object.__new__(DeviceArray)
        view.__dict__.update(self.__dict__)
        shape = tuple(shape[0]) if len(shape) == 1 and not np.isscalar(shape[0]) else tuple(shape)
        if -1 in shape:
            known = int(np.prod([s for s in shape if s != -1]))
            shape = tuple(self.size // known if s == -1 else s for s in shape)
        view.shape = tuple(int(s) for s in shape)
        assert int(np.prod(view.shape)) == self.size
        view._base = self  # keep the owner alive; views never free
        return view

    def numpy(self):
        return self.rt.download(self)

    def offset_view(self, first, shape):
        """A view starting `first` elements in (to exercise unaligned pointers)."""
        view = self.reshape(self.shape)
        view.shape = tuple(int(s) for s in shape)
        view.size = int(np.prod(view.shape))
        assert first + view.size <= self.size
        view.nbytes = view.size * self.dtype.itemsize
        view.ptr = self.ptr + first * self.dtype.itemsize
        return view

    def free(self):
        if getattr(self, "_base", None) is None and self.ptr:
            self.rt._free(self.ptr)
        self.ptr = None

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass


class SwcHip:
    """One process-wide runtime: device 0 unless told otherwise."""

    _torch_given = False   # whether an operand of the call being made is a torch tensor

    def __init__(self, device=0, auto_workspace=True):
        """auto_workspace: let the library keep (and grow) a scratch buffer of its own, as a harness that calls
        ops of many shapes wants; False: ops that need scratch fail until set_workspace() provides it, as in a
        generated program."""
        self.lib = load_library()
        self._check(self.lib.swc_hip_init(device), "swc_hip_init")
        self._check(self.lib.swc_hip_enable_auto_workspace(int(auto_workspace)), "swc_hip_enable_auto_workspace")
        self.device = device
        self._pinned = {}   # address of a pinned numpy array -> the pointer to free
        self._bench_lib = None

    def enable_auto_workspace(self, on):
        self._check(self.lib.swc_hip_enable_auto_workspace(int(on)), "swc_hip_enable_auto_workspace")

    def last_kernel(self):
        """the kernel variant the last FC/GEMM or convolution call dispatched to"""
        return self.lib.swc_hip_last_kernel().decode()

    def device_cus(self):
        return int(self.lib.swc_hip_device_cus())

    def reload_switches(self):
        """have the library read the SWC_HIP_* environment variables again (it reads them once, at init)"""
        self._check(self.lib.swc_hip_reload_switches(), "swc_hip_reload_switches")

    def use_default_stream(self):
        """launch on the device's default (null) stream, the one torch uses unless told otherwise, behind what was launched on
        the library's own stream (work on a stream of the caller's own is not waited for)"""
        self._check(self.lib.swc_hip_set_stream(C.c_void_p(_NULL_STREAM)), "swc_hip_set_stream")

    # -- plumbing --------------------------------------------------------
    def _check(self, rc, what):
        if rc != 0:
            raise SwcHipError(f"{what} failed ({rc}): {self.lib.swc_hip_last_error().decode()}")

    def _malloc(self, nbytes):
        p = self.lib.swc_hip_malloc(nbytes)
        if not p:
            raise SwcHipError(self.lib.swc_hip_last_error().decode())
        return p

    def _free(self, ptr):
        self.lib.swc_hip_free(ptr)

    def device_name(self):
        return self.lib.swc_hip_device_name().decode()

    def empty(self, shape, dtype=np.float32):
        return DeviceArray(self, shape, dtype)

    def upload(self, host):
        host = np.ascontiguousarray(host)
        assert host.dtype in (np.float32, np.int32, np.uint16, np.uint8)
        d = DeviceArray(self, host.shape, host.dtype)
        self._check(self.lib.swc_hip_h2d(d.ptr, host.ctypes.data, host.nbytes), "swc_hip_h2d")
        return d

    def download(self, d):
        host = np.empty(d.shape, d.dtype)
        self._check(self.lib.swc_hip_d2h(host.ctypes.data, d.ptr, d.nbytes), "swc_hip_d2h")
        return host

    def upload_into(self, d, host):
        """h2d into an existing allocation of the same size"""
        host = np.ascontiguousarray(host)
        assert host.nbytes == d.nbytes
        self._check(self.lib.swc_hip_h2d(d.ptr, host.ctypes.data, host.nbytes), "swc_hip_h2d")

    def download_into(self, host, d):
        assert host.nbytes == d.nbytes and host.flags.c_contiguous
        self._check(self.lib.swc_hip_d2h(host.ctypes.data, d.ptr, d.nbytes), "swc_hip_d2h")

    def d2d(self, dst, src):
        """device-to-device copy on the op stream (asynchronous)"""
        assert dst.nbytes == src.nbytes
        self._check(self.lib.swc_hip_d2d(dst.ptr, src.ptr, src.nbytes), "swc_hip_d2d")

    # uploads on the library's second stream (see include/swc_hip.h)
    def copy_h2d_async(self, d, pinned_host):
        assert pinned_host.nbytes == d.nbytes
        self._check(self.lib.swc_hip_copy_h2d_async(d.ptr, pinned_host.ctypes.data, d.nbytes), "swc_hip_copy_h2d_async")

    def copy_wait_ops(self):
        self._check(self.lib.swc_hip_copy_wait_ops(), "swc_hip_copy_wait_ops")

    def ops_wait_copies(self):
        self._check(self.lib.swc_hip_ops_wait_copies(), "swc_hip_ops_wait_copies")

    def copy_sync(self):
        self._check(self.lib.swc_hip_copy_sync(), "swc_hip_copy_sync")

    def _bench(self):
        """the bench-only helper library (include/swc_hip_bench.h), loaded on first use"""
        if self._bench_lib is None:
            path = os.path.join(_HERE, "libswc_hip_bench.so")
            if not os.path.exists(path):
                raise SwcHipError(f"{path} is missing: build it with `python -m swcompiler_amd.build`")
            self._bench_lib = C.CDLL(path)
            self._bench_lib.swc_hip_bench_probe_mfma_f32.restype = C.c_int
            self._bench_lib.swc_hip_bench_probe_mfma_f32.argtypes = [C.c_void_p, C.c_int, C.c_void_p, C.c_size_t, C.c_int,
                                                                     C.POINTER(C.c_float), C.POINTER(C.c_double)]
            self._bench_lib.swc_hip_bench_clock_watch_start.restype = C.c_int
            self._bench_lib.swc_hip_bench_clock_watch_start.argtypes = [C.c_void_p, C.c_int, C.c_int]
            self._bench_lib.swc_hip_bench_clock_watch_wait.restype = C.c_int
            self._bench_lib.swc_hip_bench_clock_watch_wait.argtypes = []
        return self._bench_lib

    def shader_clock_ghz(self, fn, op_ms, watch_ms=4.0):
        """The shader clock (GHz) while `fn` — which enqueues one op of about op_ms on the library's stream — runs
        back to back: a one-wavefront watcher of the bench-only library notes the 100 MHz wall clock and the shader
        clock counter every ~3.5 us on a stream of its own for watch_ms; fn is enqueued often enough to outlast it;
        the figure is the median over consecutive samples of the middle 80 % of the watch."""
        import numpy as np
        lib = self._bench()
        n = max(16, int(watch_ms * 1e3 / 3.6))
        samples = self.empty((4 * n,))          # 2 n 64-bit words
        self.sync()
        rc = lib.swc_hip_bench_clock_watch_start(samples.ptr, n, 1)
        if rc != 0:
            raise SwcHipError(f"swc_hip_bench_clock_watch_start failed (hipError {rc})")
        for _ in range(max(3, int(1.5 * watch_ms / max(op_ms, 1e-3)) + 2)):
            fn()
        rc = lib.swc_hip_bench_clock_watch_wait()
        self.sync()
        if rc != 0:
            raise SwcHipError(f"swc_hip_bench_clock_watch_wait failed (hipError {rc})")
        s = samples.numpy().view(np.uint64).reshape(n, 2).astype(np.float64)
        samples.free()
        s = s[n // 10: n - n // 10]
        d = np.diff(s, axis=0)
        return float(np.median(0.1 * d[:, 1] / d[:, 0]))

    def probe_mfma_tflops(self, iters=2000):
        """fp32 MFMA rate a register-only loop sustains (TFLOP/s) and its duration in ms; runs the bench-only
        helper library (include/swc_hip_bench.h) on the library's stream"""
        self._bench()
        self.sync()
        scratch = self.empty((512 * 512,))
        ms, flop = C.c_float(), C.c_double()
        rc = self._bench_lib.swc_hip_bench_probe_mfma_f32(self.lib.swc_hip_stream(), self.device_cus(), scratch.ptr,
                                                          scratch.size, iters, C.byref(ms), C.byref(flop))
        if rc != 0:
            raise SwcHipError(f"swc_hip_bench_probe_mfma_f32 failed (hipError {rc})")
        scratch.free()
        return flop.value / (ms.value * 1e-3) / 1e12, ms.value

    def sync(self):
        self._check(self.lib.swc_hip_sync(), "swc_hip_sync")

    def timer_begin(self):
        self._check(self.lib.swc_hip_timer_begin(), "swc_hip_timer_begin")

    def timer_end_ms(self):
        self._check(self.lib.swc_hip_timer_end(), "swc_hip_timer_end")
        return float(self.lib.swc_hip_timer_elapsed_ms())

    def event_record(self, slot):
        self._check(self.lib.swc_hip_event_record(slot), "swc_hip_event_record")

    def event_elapsed_ms(self, first, second):
        ms = float(self.lib.swc_hip_event_elapsed_ms(first, second))
        if ms < 0:
            raise SwcHipError("swc_hip_event_elapsed_ms failed: " + self.lib.swc_hip_last_error().decode())
        return ms

    def capture(self, fn):
        """Records the ops `fn()` issues into a HIP graph; returns a handle for graph_launch()."""
        self._check(self.lib.swc_hip_graph_begin(), "swc_hip_graph_begin")
        try:
            fn()
        finally:
            handle = C.c_void_p()
            rc = self.lib.swc_hip_graph_end(C.byref(handle))
        self._check(rc, "swc_hip_graph_end")
        return handle

    def graph_launch(self, handle):
        self._check(self.lib.swc_hip_graph_launch(handle), "swc_hip_graph_launch")

    def graph_destroy(self, handle):
        self._check(self.lib.swc_hip_graph_destroy(handle), "swc_hip_graph_destroy")

    # -- ops (device in, device out) -------------------------------------
    def matrixMatrixMul(self, a, b, out=None):
        m, k = a.shape
        k2, n = b.shape
        assert k == k2
        out = out if out is not None else self.empty((m, n))
        self._check(self.lib.swc_hip_matrixMatrixMul_f(m, n, k, a.ptr, k, b.ptr, n, out.ptr, n), "matrixMatrixMul_f")
        return out

    def batchedadd(self, batch, slice_, out=None):
        rows, cols = batch.shape
        out = out if out is not None else self.empty(batch.shape)
        self._check(self.lib.swc_hip_batchedadd_f(out.ptr, batch.ptr, slice_.ptr, rows, cols), "batchedadd_f")
        return out

    def fcbias(self, a, w, bias, relu=False, softmax=False, out=None):
        """a @ w + bias, then ReLU or the row softmax (the fused calls of the HIP target)"""
        m, k = a.shape
        k2, n = w.shape
        assert k == k2 and not (relu and softmax)
        out = out if out is not None else self.empty((m, n))
        bptr = bias.ptr if bias is not None else None
        if softmax:
            self._check(self.lib.swc_hip_matrixMatrixFCBiasSoftmax_f(m, n, k, a.ptr, k, w.ptr, n, bptr, out.ptr, n),
                        "matrixMatrixFCBiasSoftmax_f")
        else:
            self._check(self.lib.swc_hip_matrixMatrixFCBias_f(m, n, k, a.ptr, k, w.ptr, n, bptr, out.ptr, n, int(relu)),
                        "matrixMatrixFCBias_f")
        return out

    def fcbias_noalloc(self, a, w, bias, relu=False, out=None):
        """fcbias through the entry point that allocates nothing (fixed scratch inside the library)"""
        m, k = a.shape
        k2, n = w.shape
        assert k == k2
        out = out if out is not None else self.empty((m, n))
        bptr = bias.ptr if bias is not None else None
        self._check(self.lib.swc_hip_matrixMatrixFCBias_noalloc_f(m, n, k, a.ptr, k, w.ptr, n, bptr, out.ptr, n, int(relu)),
                    "matrixMatrixFCBias_noalloc_f")
        return out

    def relu(self, x, out=None):
        out = out if out is not None else self.empty(x.shape)
        self._check(self.lib.swc_hip_relu_f(x.ptr, out.ptr, x.size), "relu_f")
        return out

    def vecAdd(self, a, b, out=None, relu=False):
        assert a.shape == b.shape
        out = out if out is not None else self.empty(a.shape)
        fn = self.lib.swc_hip_vecAddRelu_f if relu else self.lib.swc_hip_vecAdd_f
        self._check(fn(a.size, a.ptr, b.ptr, out.ptr), "vecAdd_f")
        return out

    def matrixTanh(self, a, out=None):
        m, n = a.shape
        out = out if out is not None else self.empty(a.shape)
        self._check(self.lib.swc_hip_matrixTanh_f(m, n, a.ptr, n, out.ptr, n), "matrixTanh_f")
        return out

    def matrixSoftmax(self, a, out=None):
        m, n = a.shape
        out = out if out is not None else self.empty(a.shape)
        self._check(self.lib.swc_hip_matrixSoftmax_f(m, n, a.ptr, n, out.ptr, n), "matrixSoftmax_f")
        return out

    def argMax(self, x, top_k):
        m, n = x.shape
        out = self.empty((m, top_k), np.int32)
        self._check(self.lib.swc_hip_argMax_i(x.ptr, out.ptr, m, n, top_k), "argMax_i")
        return out

    def accuracy(self, pred, label, counters):
        """adds this batch to the device counters [hits, rows] (int32[2]) and returns them"""
        m, n = pred.shape
        self._check(self.lib.swc_hip_accuracy_i(pred.ptr, label.ptr, counters.ptr, m, n), "accuracy_i")
        return counters

    def fill_i(self, t, value):
        self._check(self.lib.swc_hip_fill_i(t.ptr, int(value), t.size), "fill_i")
        return t

    def conv2d(self, x, filt, bias, kernels=None, strides=(1, 1), pads=(0, 0, 0, 0), group=1, bn=None,
               eps=1e-5, relu=False, out=None, residual=None, pool=None):
        """bn = (mean, var, scale, bias) DeviceArrays to fuse inference batchnorm; pool = (kernels, strides[, pads])
        to max-pool the result in the same call (the result is then the pooled tensor)."""
        if kernels is None:
            kernels = filt.shape[1:3]
        n, oh, ow, _ = pool_out_dims(x.shape, kernels, strides, pads)
        odims = (n, oh, ow, filt.shape[0])
        if pool is not None:
            assert residual is None
            pk, ps = pool[0], pool[1]
            pp = pool[2] if len(pool) > 2 else (0, 0, 0, 0)
            pdims = pool_out_dims(odims, pk, ps, pp)
            out = out if out is not None else self.empty(pdims)
            ptrs = [p.ptr for p in bn] if bn is not None else [None] * 4
            self._check(self.lib.swc_hip_conv2dFusedMaxpool_f(
                out.ptr, x.ptr, filt.ptr, bias.ptr, _dims(odims), _dims(x.shape), _dims(filt.shape), _dims(bias.shape),
                _dims(kernels), _dims(strides), _dims(pads), group, *ptrs, eps, int(relu), _dims(pdims), _dims(pk),
                _dims(ps), _dims(pp)), "conv2dFusedMaxpool_f")
            return out
        out = out if out is not None else self.empty(odims)
        shp = (_dims(odims), _dims(x.shape), _dims(filt.shape), _dims(bias.shape), _dims(kernels),
               _dims(strides), _dims(pads))
        if residual is not None:
            assert tuple(residual.shape) == tuple(odims)
            ptrs = [p.ptr for p in bn] if bn is not None else [None] * 4
            rc = self.lib.swc_hip_conv2dFusedAdd_f(out.ptr, x.ptr, filt.ptr, bias.ptr, *shp, group, *ptrs,
                                                   eps, residual.ptr, int(relu))
        elif bn is None and not relu:
            rc = self.lib.swc_hip_conv2d_f(out.ptr, x.ptr, filt.ptr, bias.ptr, *shp, group)
        else:
            ptrs = [p.ptr for p in bn] if bn is not None else [None] * 4
            rc = self.lib.swc_hip_conv2dFused_f(out.ptr, x.ptr, filt.ptr, bias.ptr, *shp, group, *ptrs,
                                                eps, int(relu))
        self._check(rc, "conv2d_f")
        return out

    def batchnormalization(self, x, mean, var, scale, bias, eps, relu=False, out=None):
        out = out if out is not None else self.empty(x.shape)
        fn = self.lib.swc_hip_batchnormRelu_f if relu else self.lib.swc_hip_batchnormalization_f
        self._check(fn(out.ptr, x.ptr, mean.ptr, var.ptr, scale.ptr, bias.ptr, _dims(x.shape), eps),
                    "batchnormalization_f")
        return out

    def maxpool(self, x, kernels, strides, pads=(0, 0, 0, 0), out=None):
        odims = pool_out_dims(x.shape, kernels, strides, pads)
        out = out if out is not None else self.empty(odims)
        self._check(self.lib.swc_hip_maxpool_f(x.ptr, out.ptr, _dims(x.shape), _dims(odims), _dims(kernels),
                                               _dims(strides), _dims(pads)), "maxpool_f")
        return out

    def avgpool(self, x, kernels, strides, pads=(0, 0, 0, 0), out=None):
        odims = pool_out_dims(x.shape, kernels, strides, pads)
        out = out if out is not None else self.empty(odims)
        self._check(self.lib.swc_hip_avgpool_f(x.ptr, out.ptr, _dims(x.shape), _dims(odims), _dims(kernels),
                                               _dims(strides), _dims(pads)), "avgpool_f")
        return out

    def transpose(self, x, shuffle, out=None):
        """out axis a = in axis shuffle[a] (2-D or 4-D)."""
        odims = tuple(x.shape[s] for s in shuffle)
        out = out if out is not None else self.empty(odims)
        fn = self.lib.swc_hip_transpose4d_f if len(x.shape) == 4 else self.lib.swc_hip_transpose2d_f
        self._check(fn(x.ptr, out.ptr, _dims(x.shape), _dims(odims), _dims(shuffle)), "transpose_f")
        return out

    def maxpool_argmax(self, x, kernels, strides, pads=(0, 0, 0, 0)):
        odims = pool_out_dims(x.shape, kernels, strides, pads)
        out, idx = self.empty(odims), self.empty(odims, np.int32)
        self._check(self.lib.swc_hip_maxpool_argmax_f(x.ptr, out.ptr, idx.ptr, _dims(x.shape), _dims(odims),
                                                      _dims(kernels), _dims(strides), _dims(pads)),
                    "maxpool_argmax_f")
        return out, idx

    def batchnormReluMaxpool(self, x, mean, var, scale, bias, eps, kernels, strides, pads=(0, 0, 0, 0), out=None):
        odims = pool_out_dims(x.shape, kernels, strides, pads)
        out = out if out is not None else self.empty(odims)
        self._check(self.lib.swc_hip_batchnormReluMaxpool_f(out.ptr, x.ptr, mean.ptr, var.ptr, scale.ptr, bias.ptr,
                                                            _dims(x.shape), eps, _dims(odims), _dims(kernels),
                                                            _dims(strides), _dims(pads)), "batchnormReluMaxpool_f")
        return out


    # -- training kernels ------------------------------------------------
    def matrixTrans(self, a):
        m, n = a.shape
        out = self.empty((n, m))
        self._check(self.lib.swc_hip_matrixTrans_f(m, n, a.ptr, n, out.ptr, m), "matrixTrans_f")
        return out

    def matrixTanhGrad(self, out_, out_grad):
        m, n = out_.shape
        ig = self.empty(out_.shape)
        self._check(self.lib.swc_hip_matrixTanhGrad_f(m, n, ig.ptr, n, out_.ptr, n, out_grad.ptr, n), "matrixTanhGrad_f")
        return ig

    def matrixSoftmaxWithLoss(self, a, selected):
        """-> (probabilities DeviceArray, loss as a python float)"""
        m, n = a.shape
        out, loss = self.empty(a.shape), self.empty((1,))
        self._check(self.lib.swc_hip_matrixSoftmaxWithLoss_f(m, n, a.ptr, n, out.ptr, n, selected.ptr, loss.ptr),
                    "matrixSoftmaxWithLoss_f")
        return out, float(loss.numpy()[0])

    def matrixSoftmaxGrad(self, prob, selected, with_loss=False):
        m, n = prob.shape
        ig = self.empty(prob.shape)
        fn = self.lib.swc_hip_matrixSoftmaxWithLossGrad_f if with_loss else self.lib.swc_hip_matrixSoftmaxGrad_f
        self._check(fn(m, n, ig.ptr, n, prob.ptr, n, selected.ptr), "matrixSoftmaxGrad_f")
        return ig

    def conv2dGrad(self, x, filt, out_grad, kernels=None, strides=(1, 1), pads=(0, 0, 0, 0), group=1, out=None):
        if kernels is None:
            kernels = filt.shape[1:3]
        ig, fg, bg = out if out is not None else (self.empty(x.shape), self.empty(filt.shape), self.empty((filt.shape[0],)))
        self._check(self.lib.swc_hip_conv2dGrad_f(ig.ptr, fg.ptr, bg.ptr, out_grad.ptr, x.ptr, filt.ptr,
                                                  _dims(out_grad.shape), _dims(x.shape), _dims(filt.shape),
                                                  _dims(bg.shape), _dims(kernels), _dims(strides), _dims(pads), group),
                    "conv2dGrad_f")
        return ig, fg, bg

    def maxpoolGrad(self, x, out_grad, kernels, strides, pads=(0, 0, 0, 0), out=None):
        ig = out.reshape(x.shape) if out is not None else self.empty(x.shape)
        self._check(self.lib.swc_hip_maxpoolGrad_f(ig.ptr, out_grad.ptr, x.ptr, _dims(x.shape), _dims(out_grad.shape),
                                                   _dims(kernels), _dims(strides), _dims(pads)), "maxpoolGrad_f")
        return ig

    def batchedreduceadd(self, batch):
        ns, ss = batch.shape
        out = self.empty((ns,))
        self._check(self.lib.swc_hip_batchedreduceadd_f(out.ptr, batch.ptr, ns, ss), "batchedreduceadd_f")
        return out

    def sgd(self, w, dw, mom, lr, decay, momentum, batch, out=None):
        """updates out (default: w itself, as the generated call passes it) and mom in place"""
        out = w if out is None else out
        self._check(self.lib.swc_hip_sgd_f(w.size, out.ptr, w.ptr, dw.ptr, mom.ptr, lr, decay, momentum, batch), "sgd_f")
        return out, mom

    def reluGrad(self, src, dest_grad, out=None):
        out = out if out is not None else self.empty(src.shape)
        self._check(self.lib.swc_hip_reluGrad_f(out.ptr, src.ptr, dest_grad.ptr, src.size), "reluGrad_f")
        return out

    # -- operators of language models (matrices fp32 or bfloat16; DeviceArrays or torch tensors) --
    def _launch(self, what, fn, *args):
        """The library's call.  With torch tensors among the operands it comes behind the work on torch's current stream,
        and that stream's later work (and whatever reuses the operands' memory there) behind it."""
        if self._torch_given:
            self._torch_given = False
            # (half a microsecond a call: torch.cuda's own forms of these questions take three times that)
            torch = sys.modules["torch"]
            device, theirs, ours = torch._C._cuda_getDevice(), torch._C._cuda_getCurrentRawStream(self.device), self.lib.swc_hip_stream()
            if device != self.device:
                raise SwcHipError(f"{what}: the current device is {device}, the runtime's {self.device}")
            if theirs != ours and ours and (theirs or ours != _NULL_STREAM):   # (none: the library is shut down, and says so)
                return self._launch_between(what, torch, ours, fn, args)
        rc = fn(*args)
        if rc:
            self._check(rc, what)

    def _launch_between(self, what, torch, ours, fn, args):
        """_launch where torch's stream is not the library's"""
        theirs = torch.cuda.current_stream(self.device)
        if torch.cuda.is_current_stream_capturing():
            raise SwcHipError(f"{what}: torch is recording a graph on another stream than the library's: name it with "
                              "swc_hip_set_stream first")
        ours = torch.cuda.default_stream(self.device) if ours == _NULL_STREAM else torch.cuda.ExternalStream(ours, self.device)
        with torch.cuda.stream(ours):
            recording = torch.cuda.is_current_stream_capturing()
        if recording:   # (into a graph, which is ordered where it is launched)
            return self._check(fn(*args), what)
        ours.wait_stream(theirs)
        rc = fn(*args)
        theirs.wait_stream(ours)
        self._check(rc, what)

    def _arg(self, x, what, name, types, shape=None):
        """the operand as an _Arg; None for None"""
        if x is None:
            return None
        a = _Arg(self, x, what, name)
        if a.type not in types:
            raise SwcHipError(f"{what}: {name}: element type {a.type or x.dtype} is not one of {', '.join(types)}")
        if shape is not None and a.shape != shape:
            raise SwcHipError(f"{what}: {name}: shape {tuple(a.shape)}, expected {shape}")
        return a

    def _out(self, out, shape, like):
        return out if out is not None else self.empty(shape, np.float32 if like == "f32" else np.uint16)

    def _product(self, a, b, what):
        self._torch_given = False
        a, b = self._arg(a, what, "a", ("f32", "bf16")), self._arg(b, what, "b", ("f32", "bf16"))
        if len(a.shape) != 2 or len(b.shape) != 2 or a.shape[1] != b.shape[0] or a.type != b.type:
            raise SwcHipError(f"{what}: a {a.shape} {a.type} and b {b.shape} {b.type} do not multiply")
        (m, k), n = a.shape, b.shape[1]
        _int32(m if m > n and m > k else n if n > k else k, what)
        return a, b, m, n, k, (a.type,), "_f" if a.type == "f32" else "_bf"

    @staticmethod
    def _activation(act):
        if act not in ACTIVATIONS:
            raise SwcHipError(f"unknown activation {act!r}: one of {', '.join(ACTIVATIONS)}")
        return ACTIVATIONS[act]

    def matrixMatrixFCActAdd(self, a, b, bias=None, act="none", residual=None, preact=None, out=None):
        """act(a b + bias) + residual; preact receives a b + bias"""
        what = "matrixMatrixFCActAdd"
        a, b, m, n, k, t, suffix = self._product(a, b, what)
        act = self._activation(act)
        out = self._out(out, (m, n), t[0])
        c = self._arg(out, what, "out", t, (m, n))
        bias, r = self._arg(bias, what, "bias", t, (n,)), self._arg(residual, what, "residual", t, (m, n))
        z = self._arg(preact, what, "preact", t, (m, n))
        self._launch(what, getattr(self.lib, "swc_hip_matrixMatrixFCActAdd" + suffix),
                     m, n, k, a.ptr, a.ld, b.ptr, b.ld, bias and bias.ptr, act, r and r.ptr, r.ld if r else 0, z and z.ptr,
                     z.ld if z else 0, c.ptr, c.ld)
        return out

    def matrixMatrixFCActAddGrad(self, dc, a, b, preact=None, act="none", da=None, db=None, dbias=None):
        """the gradients of matrixMatrixFCActAdd into those of da, db and dbias that are given; all three, new, if none is"""
        what = "matrixMatrixFCActAddGrad"
        a, b, m, n, k, t, suffix = self._product(a, b, what)
        act = self._activation(act)
        if da is None and db is None and dbias is None:
            da, db, dbias = self._out(None, (m, k), t[0]), self._out(None, (k, n), t[0]), self._out(None, (n,), t[0])
        g, z = self._arg(dc, what, "dc", t, (m, n)), self._arg(preact, what, "preact", t, (m, n))
        ga, gb = self._arg(da, what, "da", t, (m, k)), self._arg(db, what, "db", t, (k, n))
        gbias = self._arg(dbias, what, "dbias", t, (n,))
        self._launch(what, getattr(self.lib, "swc_hip_matrixMatrixFCActAddGrad" + suffix),
                     m, n, k, g.ptr, g.ld, a.ptr, a.ld, b.ptr, b.ld, z and z.ptr, z.ld if z else 0, act, ga and ga.ptr,
                     ga.ld if ga else 0, gb and gb.ptr, gb.ld if gb else 0, gbias and gbias.ptr)
        return da, db, dbias

    def matrixFCSoftmaxWithLoss(self, a, b, bias, selected, row_loss=None, lse=None, loss=None):
        """-> (loss, row_loss, lse) of the softmax over the rows of a b + bias, whose logits are never stored"""
        what = "matrixFCSoftmaxWithLoss"
        a, b, m, n, k, t, suffix = self._product(a, b, what)
        loss, row_loss, lse = self._out(loss, (), "f32"), self._out(row_loss, (m,), "f32"), self._out(lse, (m,), "f32")
        bias, sel = self._arg(bias, what, "bias", t, (n,)), self._arg(selected, what, "selected", ("i32",), (m,))
        one = self._arg(loss, what, "loss", ("f32",))
        if one.size != 1:
            raise SwcHipError(f"{what}: loss: shape {one.shape}, expected one value")
        rl, ls = self._arg(row_loss, what, "row_loss", ("f32",), (m,)), self._arg(lse, what, "lse", ("f32",), (m,))
        self._launch(what, getattr(self.lib, "swc_hip_matrixFCSoftmaxWithLoss" + suffix),
                     m, n, k, a.ptr, a.ld, b.ptr, b.ld, bias and bias.ptr, sel.ptr, rl.ptr, ls.ptr, one.ptr)
        return loss, row_loss, lse

    def matrixFCSoftmaxWithLossGrad(self, a, b, bias, selected, lse, row_grad=None, da=None, db=None, dbias=None):
        """the gradients of the rows' losses (times row_grad) into those of da, db and dbias that are given; all three,
        new, if none is"""
        what = "matrixFCSoftmaxWithLossGrad"
        a, b, m, n, k, t, suffix = self._product(a, b, what)
        if da is None and db is None and dbias is None:
            da, db, dbias = self._out(None, (m, k), t[0]), self._out(None, (k, n), t[0]), self._out(None, (n,), t[0])
        bias, sel = self._arg(bias, what, "bias", t, (n,)), self._arg(selected, what, "selected", ("i32",), (m,))
        ls, rg = self._arg(lse, what, "lse", ("f32",), (m,)), self._arg(row_grad, what, "row_grad", ("f32",), (m,))
        ga, gb = self._arg(da, what, "da", t, (m, k)), self._arg(db, what, "db", t, (k, n))
        gbias = self._arg(dbias, what, "dbias", t, (n,))
        self._launch(what, getattr(self.lib, "swc_hip_matrixFCSoftmaxWithLossGrad" + suffix),
                     m, n, k, a.ptr, a.ld, b.ptr, b.ld, bias and bias.ptr, sel.ptr, ls.ptr, rg and rg.ptr, ga and ga.ptr, ga.ld if ga else 0,
                     gb and gb.ptr, gb.ld if gb else 0, gbias and gbias.ptr)
        return da, db, dbias

    def adamw_state(self):
        """a new step counter for adamwAdvance, at zero"""
        state = self.empty((ADAMW_STATE_WORDS,), np.int32)
        self._check(self.lib.swc_hip_fill_i(state.ptr, 0, ADAMW_STATE_WORDS), "swc_hip_fill_i")
        return state

    def _state(self, state, what):
        return self._arg(state, what, "state", ("i32",), (ADAMW_STATE_WORDS,)).ptr

    def adamwAdvance(self, state, beta1, beta2):
        """begins a step: counts it and prepares the bias corrections of the updates that follow"""
        self._torch_given = False
        state = self._state(state, "adamwAdvance")
        self._launch("adamwAdvance", self.lib.swc_hip_adamwAdvance, state, beta1, beta2)

    def _adamw(self, what, w, dw, states, scales, copies, state, lr, beta1, beta2, eps, decay, lr_factor, grad_factor):
        count = len(w)
        self._torch_given = False

        def addresses(values, types, sizes, name):
            """-> (array of addresses, element counts, the type of all)"""
            if len(values) != count:
                raise SwcHipError(f"{what}: lists of different lengths")
            try:   # torch tensors of one known type that need no further word
                kinds = {x.dtype for x in values}
                kind = _TORCH_KINDS.get(kinds.pop()) if len(kinds) == 1 else None
                if kind in types and all([x.is_contiguous() and x.get_device() == self.device for x in values]):
                    found = [x.numel() for x in values]
                    if sizes is None or found == sizes:
                        self._torch_given = True
                        return (C.c_void_p * count)(*[x.data_ptr() for x in values]), found, kind
            except AttributeError:
                pass
            out, found, kind = [], [], types[0]
            for i, x in enumerate(values):
                if x is None and name == "copies":
                    out.append(None)
                    continue
                if isinstance(x, DeviceArray):
                    ptr, t, n = x.ptr, _NUMPY_TYPES.get(x.dtype.name), x.size
                else:
                    (ptr, t), n = _torch_operand(self, x, what, f"{name} of tensor {i}"), x.numel()
                    if not x.is_contiguous():
                        raise SwcHipError(f"{what}: {name} of tensor {i} is not contiguous")
                if t not in types:
                    raise SwcHipError(f"{what}: {name} of tensor {i}: element type {t} is not one of {', '.join(types)}")
                if sizes is not None and n != sizes[i]:
                    raise SwcHipError(f"{what}: {name} of tensor {i}: {n} elements, expected {sizes[i]}")
                if i and t != kind:
                    raise SwcHipError(f"{what}: {name} of different types")
                kind = t
                out.append(ptr)
                found.append(n)
            return (C.c_void_p * count)(*out), found, kind

        pw, sizes, _ = addresses(w, ("f32",), None, "w")
        pg, _, dtype = addresses(dw, ("f32", "bf16"), sizes, "dw")
        held = ("u8",) if scales else ("f32",)
        pm, pv = addresses(states[0], held, sizes, "mom")[0], addresses(states[1], held, sizes, "var")[0]
        if scales:
            blocks = [-(-n // ADAMW_BLOCK) for n in sizes]
            pms, pvs = (addresses(x, ("f32",), blocks, name)[0] for x, name in zip(scales, ("mom_scale", "var_scale")))
            pointers = [pw, pg, pm, pms, pv, pvs]
        else:
            pointers = [pw, pg, pm, pv]
        pointers.append(None if copies is None else addresses(copies, ("bf16",), sizes, "copies")[0])
        sizes = (C.c_size_t * count)(*sizes)
        factors = [self._arg(x, what, "factor", ("f32",)) for x in (lr_factor, grad_factor)]
        if any(x is not None and x.size != 1 for x in factors):
            raise SwcHipError(f"{what}: a factor is one value")
        one = [x and x.ptr for x in factors]
        fn = getattr(self.lib, f"swc_hip_{what}" + ("_bf" if dtype == "bf16" else "_f"))
        self._launch(what, fn, count, *pointers, sizes, self._state(state, what), lr, beta1, beta2, eps, decay, *one)

    def adamw(self, w, dw, mom, var, state, lr, beta1, beta2, eps, decay, copies=None, lr_factor=None, grad_factor=None):
        """one AdamW step of the tensors in the lists w, dw, mom, var (and their bfloat16 copies), in place"""
        self._adamw("adamw", w, dw, [mom, var], [], copies, state, lr, beta1, beta2, eps, decay, lr_factor, grad_factor)

    def adamw8(self, w, dw, mom, mom_scale, var, var_scale, state, lr, beta1, beta2, eps, decay, copies=None, lr_factor=None,
               grad_factor=None):
        """the same with the states in 8 bits and a scale per ADAMW_BLOCK elements"""
        self._adamw("adamw8", w, dw, [mom, var], [mom_scale, var_scale], copies, state, lr, beta1, beta2, eps, decay,
                    lr_factor, grad_factor)

    def pinned_empty(self, shape, dtype=np.float32):
        """a numpy array in page-locked host memory (kept alive by the returned array; freed with free_pinned)"""
        n = int(np.prod(shape)) * np.dtype(dtype).itemsize
        ptr = self.lib.swc_hip_host_malloc(max(n, 1))
        if not ptr:
            raise SwcHipError("swc_hip_host_malloc: " + self.lib.swc_hip_last_error().decode())
        buf = (C.c_char * max(n, 1)).from_address(ptr)
        arr = np.frombuffer(buf, dtype=dtype, count=int(np.prod(shape))).reshape(shape)
        self._pinned[arr.ctypes.data] = ptr
        return arr

    def free_pinned(self, arr):
        self._check(self.lib.swc_hip_host_free(self._pinned.pop(arr.ctypes.data)), "swc_hip_host_free")

    def gemm_workspace_bytes(self, m, n, k):
        """scratch bytes an m x n x k FC/GEMM call uses on this device (0 unless it is split over K)"""
        return int(self.lib.swc_hip_gemm_workspace_bytes(m, n, k))

    def conv2d_maxpool_workspace_bytes(self, xshape, fshape, strides, pads, pool, group=1):
        n, oh, ow, _ = pool_out_dims(xshape, fshape[1:3], strides, pads)
        odims = (n, oh, ow, fshape[0])
        pk, ps = pool[0], pool[1]
        pp = pool[2] if len(pool) > 2 else (0, 0, 0, 0)
        pdims = pool_out_dims(odims, pk, ps, pp)
        return int(self.lib.swc_hip_conv2dFusedMaxpool_workspace_bytes(
            _dims(odims), _dims(xshape), _dims(fshape), _dims(fshape[1:3]), _dims(strides), _dims(pads), group, _dims(pdims),
            _dims(pk), _dims(ps), _dims(pp)))

    def conv2d_workspace_bytes(self, xshape, fshape, strides=(1, 1), pads=(0, 0, 0, 0), group=1):
        """scratch bytes a conv2d call of these shapes uses on this device (0 if every tile is computed whole)"""
        odims = pool_out_dims(xshape, fshape[1:3], strides, pads)[:3] + (fshape[0],)
        return int(self.lib.swc_hip_conv2d_workspace_bytes(_dims(odims), _dims(xshape), _dims(fshape), _dims(fshape[1:3]),
                                                           _dims(strides), _dims(pads), group))

    def conv2dGrad_workspace_bytes(self, xshape, fshape, strides=(1, 1), pads=(0, 0, 0, 0), group=1):
        odims = pool_out_dims(xshape, fshape[1:3], strides, pads)[:3] + (fshape[0],)
        return int(self.lib.swc_hip_conv2dGrad_workspace_bytes(_dims(odims), _dims(xshape), _dims(fshape),
                                                               _dims(fshape[1:3]), _dims(strides), _dims(pads), group))

    def set_workspace(self, arr):
        """give the library a DeviceArray to use as scratch (None: its own buffer again)"""
        if arr is None:
            self._check(self.lib.swc_hip_set_workspace(None, 0), "swc_hip_set_workspace")
        else:
            self._check(self.lib.swc_hip_set_workspace(arr.ptr, arr.nbytes), "swc_hip_set_workspace")


_RT = None


def runtime():
    """The process-wide SwcHip instance (created on first use)."""
    global _RT
    if _RT is None:
        _RT = SwcHip(0)
    return _RT
