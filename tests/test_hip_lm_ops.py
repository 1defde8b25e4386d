"""The operators of language models against plain implementations in 64 bits: the fully connected layer with its
activation and second summand, the softmax loss over a large vocabulary that stores no logits, the AdamW step.

Tolerances.  u = 2^-24 is half a step of fp32, 2^-8 of bfloat16 (relative).  A sum of k products in fp32, in any order,
is off by at most (k + 1) u sum |a b| (products of bfloat16 values are exact); activations move an error in their
argument by at most their largest slope (1.13) and add some roundings of their own, at most 16 u |z| here; a result is
rounded once to its type.  Where dZ is held in bfloat16 each of its values brings 2^-8 of itself into the sums behind it.
Integer-valued operands small enough for every sum to be exact are compared bit for bit: that is what shows a wrong or
lost element at the edge of a tile.
"""
import ctypes as C
import os
import re
import subprocess
import sys

import numpy as np
import pytest
from scipy.special import erf, expit

from swcompiler_amd import hip
from swcompiler_amd.hip import ACTIVATIONS, ADAMW_BLOCK, SwcHipError

U = 2.0 ** -24
gpu = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


# ------------------------------------------------------------------------------------------------------ bfloat16
def to_bf16(x):
    """float array -> bits of the nearest bfloat16 (ties to even)"""
    b = np.ascontiguousarray(x, np.float32).view(np.uint32).astype(np.uint64)
    out = ((b + 0x7FFF + ((b >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(np.asarray(x, np.float32)), np.uint16(0x7FC0), out)


def from_bf16(bits):
    return (np.ascontiguousarray(bits, np.uint16).astype(np.uint32) << 16).view(np.float32)


class Kind:
    """an element type of the matrices: host values, their device form, half a step"""

    def __init__(self, name):
        self.name = name
        self.half = 2.0 ** -8 if name == "bf16" else U
        self.numpy = np.uint16 if name == "bf16" else np.float32

    def values(self, x):
        """the nearest values of the type, in fp32"""
        return from_bf16(to_bf16(x)).reshape(np.shape(x)) if self.name == "bf16" else np.asarray(x, np.float32)

    def up(self, rt, x):
        return rt.upload(to_bf16(x) if self.name == "bf16" else np.asarray(x, np.float32))

    def down(self, d):
        return from_bf16(d.numpy()).reshape(d.shape) if self.name == "bf16" else d.numpy()

    def suffix(self):
        return "_bf" if self.name == "bf16" else "_f"


BF, F32 = Kind("bf16"), Kind("f32")
KINDS = [pytest.param(k, id=k.name) for k in (BF, F32)]


@pytest.fixture(scope="module")
def rt():
    from swcompiler_amd.hip import runtime
    return runtime()


def act64(z, act):
    if act == "relu":
        return np.where(z > 0, z, 0.0)
    if act == "gelu":
        return 0.5 * z * (1 + erf(z / np.sqrt(2)))
    if act == "gelu_tanh":
        return 0.5 * z * (1 + np.tanh(np.sqrt(2 / np.pi) * (z + 0.044715 * z ** 3)))
    if act == "silu":
        return z * expit(z)
    return z


def slope64(z, act):
    if act == "relu":
        return (z > 0).astype(np.float64)
    if act == "gelu":
        return 0.5 * (1 + erf(z / np.sqrt(2))) + z * np.exp(-0.5 * z * z) / np.sqrt(2 * np.pi)
    if act == "gelu_tanh":
        c = np.sqrt(2 / np.pi)
        t = np.tanh(c * (z + 0.044715 * z ** 3))
        return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z)
    if act == "silu":
        p = expit(z)
        return p * (1 + z * (1 - p))
    return np.ones_like(z)


def within(got, want, bound, what):
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    assert got.shape == want.shape, f"{what}: {got.shape} against {want.shape}"
    off = np.abs(got - want)
    bad = ~(off <= bound)
    if bad.any():
        at = np.unravel_index(np.argmax(np.where(bad, off, -1)), got.shape)
        raise AssertionError(f"{what}: {bad.sum()} of {got.size} out of bounds; at {at}: {got[at]!r} against {want[at]!r}, "
                             f"bound {np.broadcast_to(bound, got.shape)[at]!r}")


# -------------------------------------------------------------------------------------------- refusals (no device)
LIB = None


def lib():
    global LIB
    if LIB is None:
        LIB = hip.load_library()
    return LIB


EINVAL, EUNSUPPORTED, ENOTINIT = 1, 2, 4
P = C.c_void_p(1 << 20)   # an address that is never followed: every call below is refused before it starts work
Q = C.c_void_p(2 << 20)
R = C.c_void_p(3 << 20)
S, T = C.c_void_p(4 << 20), C.c_void_p(5 << 20)


def fc_args(m=4, n=8, k=8, a=P, lda=8, b=Q, ldb=8, bias=None, act=0, res=None, ldr=0, pre=None, ldp=0, c=R, ldc=8):
    return m, n, k, a, lda, b, ldb, bias, act, res, ldr, pre, ldp, c, ldc


def fc_grad_args(m=4, n=8, k=8, dc=P, lddc=8, a=Q, lda=8, b=Q, ldb=8, pre=None, ldp=0, act=0, da=R, ldda=8, db=None, lddb=0,
                 dbias=None):
    return m, n, k, dc, lddc, a, lda, b, ldb, pre, ldp, act, da, ldda, db, lddb, dbias


def loss_args(m=4, n=8, k=8, a=P, lda=8, b=Q, ldb=8, bias=None, sel=Q, row=R, lse=S, loss=T):
    return m, n, k, a, lda, b, ldb, bias, sel, row, lse, loss


def loss_grad_args(m=4, n=8, k=8, a=P, lda=8, b=Q, ldb=8, bias=None, sel=Q, lse=Q, grad=None, da=R, ldda=8, db=None, lddb=0,
                   dbias=None):
    return m, n, k, a, lda, b, ldb, bias, sel, lse, grad, da, ldda, db, lddb, dbias


REFUSED = [
    ("matrixMatrixFCActAdd", fc_args, [dict(m=-1), dict(act=5), dict(act=-1), dict(a=None), dict(c=None), dict(lda=7),
                                       dict(ldb=7), dict(ldc=7), dict(res=Q, ldr=7), dict(pre=Q, ldp=7), dict(c=P), dict(c=Q),
                                       dict(pre=R, ldp=8), dict(bias=R), dict(pre=P, ldp=8), dict(bias=P, pre=P, ldp=8),
                                       dict(res=R, ldr=9), dict(res=P, pre=P, ldp=8, ldr=8)]),
    ("matrixMatrixFCActAddGrad", fc_grad_args, [dict(n=-1), dict(act=9), dict(dc=None), dict(act=2), dict(act=2, pre=P, ldp=7),
                                                dict(b=None), dict(db=R, lddb=8, a=None), dict(lddc=7), dict(ldda=7),
                                                dict(db=R, lddb=7), dict(da=P), dict(db=Q, lddb=8), dict(dbias=P),
                                                dict(db=R, lddb=8), dict(dbias=R), dict(da=None, db=R, lddb=8, dbias=R)]),
    ("matrixFCSoftmaxWithLoss", loss_args, [dict(k=-1), dict(sel=None), dict(a=None), dict(b=None), dict(lda=7), dict(ldb=7),
                                            dict(row=None), dict(lse=None), dict(loss=None), dict(k=0),
                                            dict(lse=R), dict(loss=R), dict(loss=S)]),
    ("matrixFCSoftmaxWithLossGrad", loss_grad_args, [dict(m=-1), dict(sel=None), dict(lse=None), dict(a=None), dict(ldda=7),
                                                     dict(db=R, lddb=7), dict(da=P), dict(dbias=Q), dict(k=0),
                                                     dict(db=R, lddb=8), dict(dbias=R), dict(da=None, db=R, lddb=8, dbias=R)]),
]


@pytest.mark.parametrize("suffix", ["_f", "_bf"])
@pytest.mark.parametrize("name,make,cases", REFUSED, ids=[r[0] for r in REFUSED])
def test_refused_arguments(name, make, cases, suffix):
    fn = getattr(lib(), "swc_hip_" + name + suffix)
    for change in cases:
        assert fn(*make(**change)) == EINVAL, change
        assert name.encode() in lib().swc_hip_last_error(), change


def test_refused_sizes():
    far = (1 << 31) // 512
    assert lib().swc_hip_matrixMatrixFCActAdd_bf(*fc_args(lda=far)) == EUNSUPPORTED
    assert lib().swc_hip_matrixMatrixFCActAddGrad_bf(*fc_grad_args(ldb=far)) == EUNSUPPORTED
    assert lib().swc_hip_matrixFCSoftmaxWithLoss_bf(*loss_args(ldb=far)) == EUNSUPPORTED
    assert lib().swc_hip_matrixFCSoftmaxWithLoss_f(*loss_args(m=5_000_000)) == EUNSUPPORTED
    assert lib().swc_hip_matrixFCSoftmaxWithLossGrad_bf(*loss_grad_args(m=5_000_000)) == EUNSUPPORTED
    assert lib().swc_hip_matrixMatrixFCActAdd_f(*fc_args(m=(1 << 30) + 1)) == EUNSUPPORTED
    assert lib().swc_hip_matrixMatrixFCActAddGrad_f(*fc_grad_args(m=(1 << 30) + 1)) == EUNSUPPORTED
    # (a matrix that is not needed has no row length to be refused for, the dimension has)
    assert lib().swc_hip_matrixMatrixFCActAddGrad_bf(*fc_grad_args(k=far, a=None, lda=0, ldda=far)) == EUNSUPPORTED
    assert lib().swc_hip_matrixMatrixFCActAdd_bf(*fc_args(n=far, k=0, ldc=far)) == EUNSUPPORTED


def test_adamw_refuses_sizes_and_repeats():
    for name in ("adamw_f", "adamw8_bf"):
        assert adamw_call(name, sizes=(17179868161,)) == EUNSUPPORTED
    two, sizes = (C.c_void_p * 2)(P.value, P.value), (C.c_size_t * 2)(5, 5)
    call = lambda w, n: lib().swc_hip_adamw_f(2, w, two, two, two, None, n, P, 1e-3, 0.9, 0.99, 1e-8, 0.0, None, None)   # noqa: E731
    assert call(two, sizes) == EINVAL and b"twice" in lib().swc_hip_last_error()


def adamw_call(name, count=1, w=P, dw=P, mom=P, var=P, scale=P, sizes=(5,), state=P, lr=1e-3, beta1=0.9, beta2=0.99, eps=1e-8,
               decay=0.0):
    one = (C.c_void_p * 1)
    arr = lambda p: None if p == "none" else one(p.value if p else None)   # noqa: E731
    states = [arr(mom), arr(scale), arr(var), arr(scale)] if "8" in name else [arr(mom), arr(var)]
    return getattr(lib(), "swc_hip_" + name)(count, arr(w), arr(dw), *states, None, (C.c_size_t * 1)(*sizes), state, lr, beta1,
                                             beta2, eps, decay, None, None)


@pytest.mark.parametrize("name", ["adamw_f", "adamw_bf", "adamw8_f", "adamw8_bf"])
def test_adamw_refused_arguments(name):
    nan = float("nan")
    for change in (dict(count=-1), dict(w="none"), dict(dw="none"), dict(mom="none"), dict(var="none"), dict(w=None),
                   dict(dw=None), dict(mom=None), dict(var=None), dict(state=None), dict(beta1=1.0), dict(beta1=-0.1),
                   dict(beta2=1.0), dict(beta2=nan), dict(eps=-1.0), dict(eps=nan), dict(lr=nan), dict(decay=nan)):
        assert adamw_call(name, **change) == EINVAL, change
    if "8" in name:
        assert adamw_call(name, scale=None) == EINVAL and adamw_call(name, scale="none") == EINVAL
    assert lib().swc_hip_adamwAdvance(None, 0.9, 0.99) == EINVAL
    assert lib().swc_hip_adamwAdvance(P, 1.0, 0.99) == EINVAL


def test_header_constants():
    text = open(os.path.join(ROOT, "include", "swc_hip.h")).read()
    for name, value in ACTIVATIONS.items():
        assert re.search(r"SWC_HIP_ACT_%s = %d\b" % (name.upper(), value), text)
    assert "#define SWC_HIP_ADAMW_BLOCK %du" % ADAMW_BLOCK in text
    assert "#define SWC_HIP_ADAMW_STATE_BYTES %du" % (4 * hip.ADAMW_STATE_WORDS) in text


class _NoDevice(hip.SwcHip):
    """the binding's own checks, without a device: the library is never reached"""

    def __init__(self):
        self.device = 0
        self.lib = None

    def _malloc(self, nbytes):
        return 1 << 20

    def _free(self, ptr):
        pass


def test_binding_refuses():
    rt = _NoDevice()
    e = lambda *shape, dtype=np.float32: hip.DeviceArray(rt, shape, dtype)   # noqa: E731
    with pytest.raises(SwcHipError, match="do not multiply"):
        rt.matrixMatrixFCActAdd(e(4, 8), e(9, 8))
    with pytest.raises(SwcHipError, match="do not multiply"):
        rt.matrixMatrixFCActAdd(e(4, 8), e(8, 8, dtype=np.uint16))
    with pytest.raises(SwcHipError, match="unknown activation"):
        rt.matrixMatrixFCActAdd(e(4, 8), e(8, 8), act="swish")
    with pytest.raises(SwcHipError, match="bias: shape"):
        rt.matrixMatrixFCActAdd(e(4, 8), e(8, 8), bias=e(7))
    with pytest.raises(SwcHipError, match="residual: shape"):
        rt.matrixMatrixFCActAdd(e(4, 8), e(8, 8), residual=e(8))
    with pytest.raises(SwcHipError, match="element type"):
        rt.matrixMatrixFCActAdd(e(4, 8), e(8, 8), bias=e(8, dtype=np.uint16))
    with pytest.raises(SwcHipError, match="dc: shape"):
        rt.matrixMatrixFCActAddGrad(e(4, 9), e(4, 8), e(8, 8))
    with pytest.raises(SwcHipError, match="selected: element type"):
        rt.matrixFCSoftmaxWithLoss(e(4, 8), e(8, 8), None, e(4))
    with pytest.raises(SwcHipError, match="loss: shape"):
        rt.matrixFCSoftmaxWithLoss(e(4, 8), e(8, 8), None, e(4, dtype=np.int32), loss=e(2))
    with pytest.raises(SwcHipError, match="lse: shape"):
        rt.matrixFCSoftmaxWithLossGrad(e(4, 8), e(8, 8), None, e(4, dtype=np.int32), e(5))
    with pytest.raises(SwcHipError, match="expected a DeviceArray"):
        rt.matrixMatrixFCActAdd(np.zeros((4, 8), np.float32), e(8, 8))
    state = e(8, dtype=np.int32)
    with pytest.raises(SwcHipError, match="different lengths"):
        rt.adamw([e(3)], [e(3)], [e(3)], [], state, 1e-3, 0.9, 0.99, 1e-8, 0.0)
    with pytest.raises(SwcHipError, match="elements, expected"):
        rt.adamw([e(3)], [e(4)], [e(3)], [e(3)], state, 1e-3, 0.9, 0.99, 1e-8, 0.0)
    with pytest.raises(SwcHipError, match="elements, expected 2"):
        u = lambda n: e(n, dtype=np.uint8)   # noqa: E731
        rt.adamw8([e(257)], [e(257)], [u(257)], [e(1)], [u(257)], [e(2)], state, 1e-3, 0.9, 0.99, 1e-8, 0.0)
    with pytest.raises(SwcHipError, match="a factor is one value"):
        rt.adamw([e(3)], [e(3)], [e(3)], [e(3)], state, 1e-3, 0.9, 0.99, 1e-8, 0.0, grad_factor=e(2))
    with pytest.raises(SwcHipError, match="beyond 2"):
        rt.matrixMatrixFCActAdd(e(1 << 31, 1), e(1, 1))
    with pytest.raises(SwcHipError, match="state: shape"):
        rt.adamwAdvance(e(7, dtype=np.int32), 0.9, 0.99)


def test_torch_operands_are_checked():
    torch = pytest.importorskip("torch")
    rt = _NoDevice()
    with pytest.raises(SwcHipError, match="the tensor is on cpu"):
        rt.matrixMatrixFCActAdd(torch.zeros(4, 8), torch.zeros(8, 8))


# ------------------------------------------------------------------------------ the fully connected layer, forward
def small_ints(rng, *shape, top=3):
    return rng.integers(-top, top + 1, shape).astype(np.float32)


# one row to several tiles of every height, widths and depths at, next to and far from multiples of 8, 16, 64, 128, 256
FC_SHAPES = [(1, 1, 1), (1, 8, 8), (2, 3, 5), (1, 4096, 520), (5, 257, 1000), (16, 128, 64), (17, 130, 72), (31, 1000, 33),
             (32, 127, 64), (33, 200, 136), (64, 128, 512), (65, 72, 264), (70, 301, 75), (100, 65, 2048), (128, 128, 128),
             (129, 255, 63), (200, 511, 300), (256, 256, 64), (257, 300, 65), (300, 513, 1000), (513, 260, 96), (1000, 2056, 520),
             (1025, 4104, 200), (4097, 4360, 72),
             # a last round of large tiles left to smaller ones: of the layer, of its weights' gradient
             (2048, 8400, 1000), (1000, 8400, 2048)]


@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("m,n,k", FC_SHAPES)
def test_fc_integers_bit_exact(rt, kind, m, n, k):
    print("case fc integers", kind.name, m, n, k, flush=True)
    rng = np.random.default_rng(m * 7 + n * 3 + k)
    # sums stay below 2^24 / 4 in fp32; for bfloat16 the last rounding is the only one
    a, b = small_ints(rng, m, k), small_ints(rng, k, n)
    bias, res = small_ints(rng, n, top=9), small_ints(rng, m, n, top=9)
    z = a.astype(np.float64) @ b + bias
    for act in ("none", "relu"):
        pre = rt.empty((m, n), kind.numpy)
        c = rt.matrixMatrixFCActAdd(kind.up(rt, a), kind.up(rt, b), kind.up(rt, bias), act, kind.up(rt, res), pre)
        np.testing.assert_array_equal(kind.down(pre), kind.values(z))
        np.testing.assert_array_equal(kind.down(c), kind.values(act64(z, act) + res))
    plain = rt.matrixMatrixFCActAdd(kind.up(rt, a), kind.up(rt, b))
    np.testing.assert_array_equal(kind.down(plain), kind.values(z - bias))


# few rows: the forms for decoding and the first sizes beyond them; contractions of less than a wavefront's share to several
# rounds of all of them, whole slices and not, and past the longest of them
FEW_SHAPES = [(2, 520, 64), (8, 33, 72), (3, 1000, 1088), (4, 72, 2056), (5, 264, 3080), (8, 130, 4096), (1, 48, 8192), (8, 40, 8192),
              (8, 72, 8200), (9, 520, 4096), (2, 4104, 1028), (4, 4099, 513)]


@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("pad", [0, 8, 3])
@pytest.mark.parametrize("m,n,k", FEW_SHAPES)
def test_fc_few_rows_bit_exact(rt, kind, pad, m, n, k):
    print("case fc few", kind.name, pad, m, n, k, flush=True)
    rng = np.random.default_rng(m * 7 + n * 3 + k)
    a, b, res = small_ints(rng, m, k), small_ints(rng, k, n), small_ints(rng, m, n, top=9)
    bias = small_ints(rng, n)
    dbias = kind.up(rt, bias)
    da, pa = strided(rt, kind, a, k + pad)
    db, pb = strided(rt, kind, b, n + pad)
    dr, pr = strided(rt, kind, res, n + pad)
    dz, pz = strided(rt, kind, np.zeros((m, n)), n + pad)
    dc, pc = strided(rt, kind, np.zeros((m, n)), n + pad)
    fn = getattr(rt.lib, "swc_hip_matrixMatrixFCActAdd" + kind.suffix())
    rt._check(fn(m, n, k, pa, k + pad, pb, n + pad, dbias.ptr, 1, pr, n + pad, pz, n + pad, pc, n + pad), "fc")
    z = a.astype(np.float64) @ b + bias
    for d, want in ((dz, z), (dc, np.maximum(z, 0) + res)):
        inside, beside, behind = rows_of(kind, d, m, n, n + pad)
        np.testing.assert_array_equal(inside, kind.values(want))
        assert np.all(np.isnan(beside)) and np.all(np.isnan(behind))


def fc_bound(a, b, bias, res, z, value, kind):
    k = a.shape[1]
    size = np.abs(a).astype(np.float64) @ np.abs(b).astype(np.float64) + (0 if bias is None else np.abs(bias))
    e = 1.13 * (k + 2) * U * size + 16 * U * np.abs(z)
    r = 0 if res is None else np.abs(res)
    e = e + 2 * U * (np.abs(value) + r)
    return e + kind.half * (np.abs(value + (0 if res is None else res)) + e)


@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("act", list(ACTIVATIONS))
@pytest.mark.parametrize("m,n,k", [(1, 1000, 512), (7, 72, 40), (130, 264, 200), (300, 520, 1024), (1100, 1032, 96)])
def test_fc_activations(rt, kind, act, m, n, k):
    print("case fc", kind.name, act, m, n, k, flush=True)
    rng = np.random.default_rng(m + n + k)
    a, b = kind.values(rng.standard_normal((m, k))), kind.values(rng.standard_normal((k, n)) * 2 / np.sqrt(k))
    bias, res = kind.values(rng.standard_normal(n)), kind.values(rng.standard_normal((m, n)))
    for has_bias, has_res in ((True, True), (False, False), (True, False)):
        z = a.astype(np.float64) @ b.astype(np.float64) + (bias if has_bias else 0)
        c = rt.matrixMatrixFCActAdd(kind.up(rt, a), kind.up(rt, b), kind.up(rt, bias) if has_bias else None, act,
                                    kind.up(rt, res) if has_res else None)
        value = act64(z, act)
        want = value + (res if has_res else 0)
        within(kind.down(c), want, fc_bound(a, b, bias if has_bias else None, res if has_res else None, z, value, kind), act)


@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("act", list(ACTIVATIONS))
def test_fc_activation_values(rt, kind, act):
    """the activation itself over its whole range: one product with 1, far values and those next to zero"""
    z = kind.values(np.concatenate([np.linspace(-60, 60, 4001), [0.0, -0.0, 1e-30, -1e-30, 1e30, 300.0, -300.0, 88.0, -88.0, 6.0,
                                                                   -6.0]]))
    a = np.zeros((8, 8), np.float32)
    a[0, 0] = 1
    b = np.zeros((8, len(z)), np.float32)
    b[0] = z
    got = kind.down(rt.matrixMatrixFCActAdd(kind.up(rt, a), kind.up(rt, b), act=act))[0]
    z = z.astype(np.float64)
    want = act64(z, act)
    within(got, want, kind.half * np.abs(want) + 16 * U * np.minimum(np.abs(z), 8) + 16 * U * np.abs(want) + 1e-37, act)


@gpu
@pytest.mark.parametrize("kind", KINDS)
def test_fc_non_finite(rt, kind):
    """an infinity or NaN reaches the elements of its row or column and no others"""
    rng = np.random.default_rng(0)
    a, b = small_ints(rng, 70, 72), small_ints(rng, 72, 136) + 10
    res = small_ints(rng, 70, 136)
    a[3, 5], a[66, 71] = np.inf, np.nan
    res[8, 9] = -np.inf
    for act in ("none", "gelu", "gelu_tanh", "silu", "relu"):
        got = kind.down(rt.matrixMatrixFCActAdd(kind.up(rt, a), kind.up(rt, b), None, act, kind.up(rt, res)))
        assert np.all(got[3] == np.inf) and got[8, 9] == -np.inf
        if act == "relu":   # as relu_f: NaN > 0 is false
            np.testing.assert_array_equal(got[66], res[66])
        else:
            assert np.all(np.isnan(got[66]))
        rest = np.ones_like(got, bool)
        rest[3] = rest[66] = False
        rest[8, 9] = False
        assert np.all(np.isfinite(got[rest]))


def strided(rt, kind, x, ld, first=0):
    """x in rows of ld, starting `first` elements into an allocation, on a ground of NaN -> (base array, address)"""
    rows, cols = x.shape
    ground = np.full(first + rows * ld + 8, np.nan, np.float32)
    flat = ground[first:first + rows * ld].reshape(rows, ld)
    flat[:, :cols] = x
    d = kind.up(rt, ground)
    return d, d.ptr + first * d.dtype.itemsize


def rows_of(kind, d, rows, cols, ld, first=0):
    flat = kind.down(d)[first:first + rows * ld].reshape(rows, ld)
    return flat[:, :cols], flat[:, cols:], kind.down(d)[first + rows * ld:]


@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("pad,first", [(0, 0), (8, 0), (3, 0), (8, 8), (5, 3), (1, 1)])
@pytest.mark.parametrize("m,n,k", [(1, 72, 72), (33, 200, 136), (66, 131, 77), (300, 520, 264)])
def test_fc_strides_and_alignment(rt, kind, pad, first, m, n, k):
    """row strides of their own on every matrix and any alignment; what lies around them is neither read into a result
    (it is NaN) nor written"""
    print("case fc strides", kind.name, pad, first, m, n, k, flush=True)
    rng = np.random.default_rng(m + pad * 5 + first)
    a, b, res = small_ints(rng, m, k), small_ints(rng, k, n), small_ints(rng, m, n, top=9)
    bias = small_ints(rng, n)
    dbias = kind.up(rt, bias)
    da, pa = strided(rt, kind, a, k + pad, first)
    db, pb = strided(rt, kind, b, n + pad, first)
    dr, pr = strided(rt, kind, res, n + 2 * pad, first)
    dz, pz = strided(rt, kind, np.zeros((m, n)), n + pad, first)
    dc, pc = strided(rt, kind, np.zeros((m, n)), n + 2 * pad, first)
    fn = getattr(rt.lib, "swc_hip_matrixMatrixFCActAdd" + kind.suffix())
    rt._check(fn(m, n, k, pa, k + pad, pb, n + pad, dbias.ptr, 1, pr, n + 2 * pad, pz, n + pad, pc, n + 2 * pad), "fc")
    z = a.astype(np.float64) @ b + bias
    for d, ld, want in ((dz, n + pad, z), (dc, n + 2 * pad, np.maximum(z, 0) + res)):
        inside, beside, behind = rows_of(kind, d, m, n, ld, first)
        np.testing.assert_array_equal(inside, kind.values(want))
        assert np.all(np.isnan(beside)) and np.all(np.isnan(behind)) and np.all(np.isnan(kind.down(d)[:first]))


@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("m,n,k", [(3, 40, 1024), (300, 520, 264)])
def test_fc_residual_in_place(rt, kind, m, n, k):
    """C may be the second summand itself (x += layer(h))"""
    rng = np.random.default_rng(3)
    a, b, x = small_ints(rng, m, k), small_ints(rng, k, n), small_ints(rng, m, n, top=9)
    c = kind.up(rt, x)
    rt.matrixMatrixFCActAdd(kind.up(rt, a), kind.up(rt, b), None, "relu", c, out=c)
    np.testing.assert_array_equal(kind.down(c), kind.values(np.maximum(a.astype(np.float64) @ b, 0) + x))


@gpu
@pytest.mark.parametrize("kind", KINDS)
def test_fc_empty(rt, kind):
    fn = getattr(rt.lib, "swc_hip_matrixMatrixFCActAdd" + kind.suffix())
    assert fn(*fc_args(m=0, a=None, b=None, c=None)) == 0
    assert fn(*fc_args(n=0, a=None, b=None, c=None)) == 0
    bias, res = np.arange(-4, 4, dtype=np.float32), np.ones((3, 8), np.float32)
    c, z, dbias, dres = rt.empty((3, 8), kind.numpy), rt.empty((3, 8), kind.numpy), kind.up(rt, bias), kind.up(rt, res)
    rt._check(fn(3, 8, 0, None, 0, None, 0, dbias.ptr, 1, dres.ptr, 8, z.ptr, 8, c.ptr, 8), "fc")
    np.testing.assert_array_equal(kind.down(z), np.broadcast_to(bias, (3, 8)))
    np.testing.assert_array_equal(kind.down(c), np.maximum(bias, 0) + res)
    grad = getattr(rt.lib, "swc_hip_matrixMatrixFCActAddGrad" + kind.suffix())
    ga, gb, gbias = (rt.upload(np.full(s, 7, kind.numpy)) for s in ((1, 8), (8, 8), (8,)))
    ones = kind.up(rt, np.ones((8, 8)))
    rt._check(grad(0, 8, 8, None, 8, None, 8, ones.ptr, 8, None, 0, 0, ga.ptr, 8, gb.ptr, 8, gbias.ptr), "grad")
    assert np.all(kind.down(gb) == 0) and np.all(kind.down(gbias) == 0)


# --------------------------------------------------------------------------- the fully connected layer, gradients
@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("m,n,k", FC_SHAPES)
def test_fc_grad_integers_bit_exact(rt, kind, m, n, k):
    print("case fc grad integers", kind.name, m, n, k, flush=True)
    rng = np.random.default_rng(m + n * 5 + k * 3)
    dc, a, b, pre = small_ints(rng, m, n), small_ints(rng, m, k), small_ints(rng, k, n), small_ints(rng, m, n)
    for act in ("none", "relu"):
        dz = dc * (pre > 0) if act == "relu" else dc
        da, db, dbias = rt.matrixMatrixFCActAddGrad(kind.up(rt, dc), kind.up(rt, a), kind.up(rt, b),
                                                    kind.up(rt, pre) if act == "relu" else None, act)
        np.testing.assert_array_equal(kind.down(da), kind.values(dz.astype(np.float64) @ b.T))
        np.testing.assert_array_equal(kind.down(db), kind.values(a.T.astype(np.float64) @ dz))
        np.testing.assert_array_equal(kind.down(dbias), kind.values(dz.sum(0, dtype=np.float64)))


@gpu
def test_fc_beyond_32_bits(rt):
    """a matrix of 2.8e9 elements, written by the layer and read by its gradients: C = A B in exact small integers, so that
    dA = C B^T = A (B B^T), dB = A^T C = (A^T A) B and the column sums are known without C"""
    rng = np.random.default_rng(41)
    m, n, k = 70001, 40000, 8
    a, b = small_ints(rng, m, k, top=2), small_ints(rng, k, n, top=2)     # |C| <= 32; sums below 2^24 / 2
    da_, db_ = BF.up(rt, a), BF.up(rt, b)
    c = rt.empty((m, n), np.uint16)
    rt.matrixMatrixFCActAdd(da_, db_, out=c)
    a, b = a.astype(np.float64), b.astype(np.float64)
    for row in (0, 1, 53686, 53687, 53688, 69999, 70000):     # 53687 n passes 2^31
        got = from_bf16(c.offset_view(row * n, (n,)).numpy())
        np.testing.assert_array_equal(got, a[row] @ b)
    ga, gb, gbias = (BF.down(x) for x in rt.matrixMatrixFCActAddGrad(c, da_, db_))
    np.testing.assert_array_equal(ga, BF.values(a @ (b @ b.T)))
    np.testing.assert_array_equal(gb, BF.values((a.T @ a) @ b))
    np.testing.assert_array_equal(gbias, BF.values(a.sum(0) @ b))


@gpu
def test_fc_grad_many_rows(rt):
    """more rows than a grid's second direction has workgroups of 32 (65535): exact integers all the same"""
    rng = np.random.default_rng(9)
    m, n, k = 65535 * 32 + 1, 8, 8
    dc, a, b = (rng.integers(-1, 2, s).astype(np.float32) for s in ((m, n), (m, k), (k, n)))
    da, db, dbias = (x.numpy() for x in rt.matrixMatrixFCActAddGrad(rt.upload(dc), rt.upload(a), rt.upload(b)))
    np.testing.assert_array_equal(da, dc @ b.T)
    np.testing.assert_array_equal(db, a.T.astype(np.float64) @ dc)
    np.testing.assert_array_equal(dbias, dc.sum(0, dtype=np.float64))


def fc_grad_bounds(dz, a, b, kind, slack):
    """slack: how far a value of dZ may be off, relative to |dC|"""
    m, n = dz.shape
    err = slack + (2.0 ** -8 * np.abs(dz) if kind.name == "bf16" else 0)
    size = np.abs(dz) + err
    ea = err @ np.abs(b).T + (n + 1) * U * (size @ np.abs(b).T)
    eb = np.abs(a).T @ err + (m + 1) * U * (np.abs(a).T @ size)
    es = slack.sum(0) + (m + 1) * U * size.sum(0)
    return ea, eb, es


@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("act", list(ACTIVATIONS))
@pytest.mark.parametrize("m,n,k", [(1, 64, 512), (75, 200, 136), (300, 520, 264)])
def test_fc_grad_activations(rt, kind, act, m, n, k):
    print("case fc grad", kind.name, act, m, n, k, flush=True)
    rng = np.random.default_rng(m * 3 + n + k)
    dc, a = kind.values(rng.standard_normal((m, n))), kind.values(rng.standard_normal((m, k)))
    b, pre = kind.values(rng.standard_normal((k, n))), kind.values(rng.standard_normal((m, n)) * 3)
    pre[0, :8] = kind.values([0.0, -0.0, 50.0, -50.0, 1e20, -1e20, 8.0, -8.0])
    dz = dc.astype(np.float64) * slope64(pre.astype(np.float64), act)
    if act != "none":
        dz[0, 4:6] = [dc[0, 4], 0.0]   # (the formulas in 64 bits overflow there)
    da, db, dbias = rt.matrixMatrixFCActAddGrad(kind.up(rt, dc), kind.up(rt, a), kind.up(rt, b), kind.up(rt, pre), act)
    # a slope is at most 1.13 and its formula rounds some 16 times values of at most 1.5
    slack = 24 * U * np.abs(dc).astype(np.float64)
    a64, b64 = a.astype(np.float64), b.astype(np.float64)
    for got, want, e in zip((da, db, dbias), (dz @ b64.T, a64.T @ dz, dz.sum(0)), fc_grad_bounds(dz, a64, b64, kind, slack)):
        within(kind.down(got), want, e + kind.half * (np.abs(want) + e), act)


@pytest.mark.parametrize("act", list(ACTIVATIONS))
def test_slopes_are_derivatives(act):
    """the slopes the gradients are held to, against differences of the activations"""
    z, h = np.linspace(-7, 7, 1000) + 0.0005, 1e-5
    diff = (act64(z + h, act) - act64(z - h, act)) / (2 * h)
    np.testing.assert_allclose(slope64(z, act), diff, atol=1e-8)


@gpu
def test_fc_grad_by_differences(rt):
    """the fp32 gradients against differences of the fp32 forward call, summed against a random direction in 64 bits"""
    rng = np.random.default_rng(11)
    m, n, k, act = 20, 24, 12, "gelu"
    a, b, bias = (rng.standard_normal(s).astype(np.float32) for s in ((m, k), (k, n), (n,)))
    w = rng.standard_normal((m, n)).astype(np.float32)
    pre = rt.empty((m, n))
    rt.matrixMatrixFCActAdd(rt.upload(a), rt.upload(b), rt.upload(bias), act, None, pre)
    da, db, dbias = rt.matrixMatrixFCActAddGrad(rt.upload(w), rt.upload(a), rt.upload(b), pre, act)

    def f(a, b, bias):
        return float((rt.matrixMatrixFCActAdd(rt.upload(a), rt.upload(b), rt.upload(bias), act).numpy().astype(np.float64) * w).sum())

    h = 2.0 ** -7
    z = a.astype(np.float64) @ b + bias
    e = fc_bound(a, b, bias, None, z, act64(z, act), F32) * 1.1     # of a value of the forward call, a little off z too
    for i, (x, g) in enumerate(((a, da), (b, db), (bias, dbias))):
        d = rng.choice([-1.0, 1.0], x.shape).astype(np.float32)
        up, down = [a, b, bias], [a, b, bias]
        up[i], down[i] = (x + np.float32(h) * d), (x - np.float32(h) * d)
        want = (f(*up) - f(*down)) / (2 * h)
        got = float((g.numpy().astype(np.float64) * d).sum())
        # the difference: the third derivative of gelu, z phi(z) (z^2 - 4), is below 0.8; z moves by at most h s; and the
        # two values' own errors over 2 h
        s = (np.broadcast_to(np.abs(b).sum(0), (m, n)), np.broadcast_to(np.abs(a).sum(1)[:, None], (m, n)), np.ones((m, n)))[i]
        bound = (np.abs(w) * (0.8 * s ** 3 * h * h / 6 + e / h)).sum() + 1e-5 * abs(want)
        assert abs(got - want) <= bound, (i, got, want, bound)


@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("pad,first", [(0, 0), (8, 8), (3, 1)])
@pytest.mark.parametrize("m,n,k", [(33, 200, 136), (66, 131, 77), (300, 264, 520)])
def test_fc_grad_strides(rt, kind, pad, first, m, n, k):
    print("case fc grad strides", kind.name, pad, first, m, n, k, flush=True)
    rng = np.random.default_rng(m + pad)
    dc, a, b, pre = small_ints(rng, m, n), small_ints(rng, m, k), small_ints(rng, k, n), small_ints(rng, m, n)
    _keep, p = zip(*(strided(rt, kind, x, x.shape[1] + pad, first) for x in (dc, a, b, pre)))
    ga, pga = strided(rt, kind, np.zeros((m, k)), k + pad, first)
    gb, pgb = strided(rt, kind, np.zeros((k, n)), n + pad, first)
    fn = getattr(rt.lib, "swc_hip_matrixMatrixFCActAddGrad" + kind.suffix())
    rt._check(fn(m, n, k, p[0], n + pad, p[1], k + pad, p[2], n + pad, p[3], n + pad, 1, pga, k + pad, pgb, n + pad, None), "grad")
    dz = (dc * (pre > 0)).astype(np.float64)
    for d, rows, cols, want in ((ga, m, k, dz @ b.T), (gb, k, n, a.T @ dz)):
        inside, beside, behind = rows_of(kind, d, rows, cols, cols + pad, first)
        np.testing.assert_array_equal(inside, kind.values(want))
        assert np.all(np.isnan(beside)) and np.all(np.isnan(behind))


@gpu
@pytest.mark.parametrize("kind", KINDS)
def test_fc_grad_each_alone(rt, kind):
    """any of the three gradients alone is what it is among the others, bit for bit"""
    rng = np.random.default_rng(8)
    m, n, k = 130, 200, 72
    x = [kind.up(rt, rng.standard_normal(s)) for s in ((m, n), (m, k), (k, n), (m, n))]
    every = [d.numpy() for d in rt.matrixMatrixFCActAddGrad(*x, "silu")]
    for i, shape in enumerate(((m, k), (k, n), (n,))):
        out = rt.empty(shape, kind.numpy)
        rt.matrixMatrixFCActAddGrad(*x, "silu", **{("da", "db", "dbias")[i]: out})
        np.testing.assert_array_equal(out.numpy(), every[i])


# ----------------------------------------------------------------------------------------- loss without logits
def loss64(a, b, bias, sel, row_grad=None):
    """loss, row losses, lse and the three gradients, by the definition, over the rows that count alone"""
    m, n = a.shape[0], b.shape[1]
    a, b = a.astype(np.float64), b.astype(np.float64)
    rows = np.flatnonzero((sel >= 0) & (sel < n))
    z = a[rows] @ b + (0 if bias is None else bias.astype(np.float64))
    top = z.max(1, initial=-np.inf) if len(rows) else np.zeros(0)
    lse_r = top + np.log(np.exp(z - top[:, None]).sum(1))
    row, lse = np.zeros(m), np.zeros(m)
    lse[rows] = lse_r
    row[rows] = lse_r - z[np.arange(len(rows)), sel[rows]]
    p = np.exp(z - lse_r[:, None])
    p[np.arange(len(rows)), sel[rows]] -= 1
    if row_grad is not None:
        p *= row_grad[rows][:, None]
    da = np.zeros(a.shape)
    da[rows] = p @ b.T
    return (row.sum() / max(1, len(rows)), row, lse, da, a[rows].T @ p, p.sum(0)), (rows, z, p)


def check_loss(rt, kind, a, b, bias, sel, row_grad=None, grad=True):
    up = lambda x: None if x is None else kind.up(rt, x)   # noqa: E731
    da_, db_, dsel, dbias_ = up(a), up(b), rt.upload(sel.astype(np.int32)), up(bias)
    loss, row, lse = rt.matrixFCSoftmaxWithLoss(da_, db_, dbias_, dsel)
    (wl, wr, wlse, wda, wdb, wdbias), (rows, z, p) = loss64(a, b, bias, sel, row_grad)
    k, n = b.shape
    # logits: an fp32 sum of k products; lse: as far off as the worst logit, plus the sum of exponentials (hardware
    # exponential and the additions, together below 2^-19 relative) and its logarithm
    size = np.abs(a[rows]).astype(np.float64) @ np.abs(b).astype(np.float64) + (0 if bias is None else np.where(np.isfinite(bias), np.abs(bias), 0))
    ez = (k + 2) * U * size.max(1, initial=0.0)
    el = np.zeros(len(sel))
    el[rows] = ez + 2.0 ** -19 + 2 * U * np.abs(wlse[rows])
    within(lse.numpy(), wlse, el, "lse")
    er = np.zeros(len(sel))
    er[rows] = el[rows] + ez + 2 * U * (np.abs(wlse[rows]) + np.abs(wr[rows]))
    within(row.numpy(), wr, er, "row loss")
    within(loss.numpy().reshape(()), wl, (er.sum() / max(1, len(rows))) + 2 * U * abs(wl), "loss")
    if not grad:
        return
    g = None if row_grad is None else rt.upload(row_grad.astype(np.float32))
    ga, gb, gbias = rt.matrixFCSoftmaxWithLossGrad(da_, db_, dbias_, dsel, lse, g)
    up_g = np.abs(row_grad[rows])[:, None] if row_grad is not None else 1.0
    prob = np.exp(z - wlse[rows][:, None])
    # (a probability below 2^-126, the least normal fp32, may be held as zero, and its products with it: the exact value is
    # then off by at most 2^-126 of the factors behind it)
    err = up_g * prob * (ez + el[rows] + 2.0 ** -20)[:, None] + 2 * U * np.abs(p) + up_g * 2.0 ** -126
    if kind.name == "bf16":
        err = err + 2.0 ** -8 * (np.abs(p) + err)
    big = np.abs(p) + err
    a64, b64 = np.abs(a[rows]).astype(np.float64), np.abs(b).astype(np.float64)
    ea = np.zeros(a.shape)
    ea[rows] = err @ b64.T + (n + 2) * U * (big @ b64.T)
    eb = a64.T @ err + (len(rows) + 2) * U * (a64.T @ big)
    es = err.sum(0) + (len(rows) + 2) * U * big.sum(0)
    for name, got, want, e in (("da", ga, wda, ea), ("db", gb, wdb, eb), ("dbias", gbias, wdbias, es)):
        within(kind.down(got), want, e + kind.half * (np.abs(want) + e) + 2.0 ** -126, name)


LOSS_SHAPES = [(1, 1, 8), (1, 100, 8), (2, 3, 1), (5, 33, 40), (17, 64, 64), (33, 1000, 64), (64, 257, 72), (70, 301, 75),
               (130, 4100, 136), (257, 513, 200), (300, 50, 264), (520, 20003, 96), (1000, 2056, 520),
               (2048, 8401, 1000)]


@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("m,n,k", LOSS_SHAPES)
def test_loss_and_gradients(rt, kind, m, n, k):
    print("case loss", kind.name, m, n, k, flush=True)
    rng = np.random.default_rng(m + n + k)
    a, b = kind.values(rng.standard_normal((m, k))), kind.values(rng.standard_normal((k, n)) * 2 / np.sqrt(k))
    bias = kind.values(rng.standard_normal(n)) if m % 2 else None
    check_loss(rt, kind, a, b, bias, rng.integers(0, n, m))


@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("m,n,k,share", [(70, 301, 72, 0.5), (300, 1000, 64, 0.9), (33, 40, 16, 1.0), (1030, 130, 40, 0.3),
                                         (4096, 70, 24, 0.1), (4097, 70, 24, 0.1), (6000, 100, 19, 0.6),
                                         (5000, 320, 64, 0.2), (2048, 700, 200, 0.5), (28, 1000, 320, 0.3), (28, 9000, 65, 0.3),
                                         (600, 130, 1028, 0.2)])
def test_loss_rows_left_out(rt, kind, m, n, k, share):
    """rows whose class lies outside the vocabulary bring nothing, whatever they hold: here infinities and NaN"""
    print("case loss left out", kind.name, m, n, k, share, flush=True)
    rng = np.random.default_rng(m)
    a, b = kind.values(rng.standard_normal((m, k))), kind.values(rng.standard_normal((k, n)))
    sel = rng.integers(0, n, m)
    out = rng.random(m) < share if share < 1 else np.ones(m, bool)
    sel[out] = rng.choice([-1, -100, n, n + 7, -2 ** 31, 2 ** 31 - 1], out.sum())
    a[out] = rng.choice(np.array([np.nan, np.inf, -np.inf], np.float32), (out.sum(), k))
    grad = rng.standard_normal(m).astype(np.float32)
    grad[out] = np.nan
    with np.errstate(invalid="ignore"):
        check_loss(rt, kind, a, b, kind.values(rng.standard_normal(n)), sel, grad)


@gpu
@pytest.mark.parametrize("kind,m", [pytest.param(F32, 2900, id="f32"), pytest.param(BF, 5800, id="bf16")])
def test_loss_gradient_in_pieces(rt, kind, m):
    """a vocabulary whose dz does not fit the workspace's 256 MiB at once: two pieces, the second of 260 classes"""
    rng = np.random.default_rng(31)
    n, k = 23300, 16
    a, b = kind.values(rng.standard_normal((m, k))), kind.values(rng.standard_normal((k, n)) / 2)
    sel = rng.integers(-1, n, m)
    sel[:40] = rng.integers(23040, n, 40)
    check_loss(rt, kind, a, b, kind.values(rng.standard_normal(n)), sel, rng.standard_normal(m).astype(np.float32))


@gpu
@pytest.mark.parametrize("kind", KINDS)
def test_loss_classes_ruled_out(rt, kind):
    """a bias of minus infinity rules classes out (the padding of a vocabulary): whole blocks of them, whole tiles"""
    rng = np.random.default_rng(5)
    m, n, k = 70, 1300, 72
    a, b = kind.values(rng.standard_normal((m, k))), kind.values(rng.standard_normal((k, n)))
    bias = kind.values(rng.standard_normal(n))
    bias[40:900] = -np.inf
    bias[1290:] = -np.inf
    check_loss(rt, kind, a, b, bias, rng.choice(np.flatnonzero(np.isfinite(bias)), m))
    # the type's lowest value does the same, without infinities
    bias[~np.isfinite(bias)] = kind.values(-3.3e38)
    (wl, wr, wlse, *_), _ = loss64(a, b, bias, np.zeros(m, int))
    _, row, lse = rt.matrixFCSoftmaxWithLoss(kind.up(rt, a), kind.up(rt, b), kind.up(rt, bias), rt.upload(np.zeros(m, np.int32)))
    within(lse.numpy(), wlse, 1e-4, "lse")
    within(row.numpy(), wr, 2e-4, "row loss")


@gpu
@pytest.mark.parametrize("kind", KINDS)
def test_loss_far_logits(rt, kind):
    """logits in the thousands: only their distance counts"""
    rng = np.random.default_rng(6)
    m, n, k = 40, 500, 64
    a, b = kind.values(rng.standard_normal((m, k)) * 30), kind.values(rng.standard_normal((k, n)) * 10)
    check_loss(rt, kind, a, b, None, rng.integers(0, n, m))


@gpu
@pytest.mark.parametrize("kind", KINDS)
def test_loss_non_finite_row(rt, kind):
    """a NaN in a row that counts is its row's alone"""
    rng = np.random.default_rng(7)
    a, b = small_ints(rng, 40, 16), small_ints(rng, 16, 300)
    a[3, 4] = np.nan
    sel = rng.integers(0, 300, 40).astype(np.int32)
    _, row, lse = rt.matrixFCSoftmaxWithLoss(kind.up(rt, a), kind.up(rt, b), None, rt.upload(sel))
    for x in (row.numpy(), lse.numpy()):
        assert np.isnan(x[3]) and np.all(np.isfinite(np.delete(x, 3)))
    ga, _, _ = rt.matrixFCSoftmaxWithLossGrad(kind.up(rt, a), kind.up(rt, b), None, rt.upload(sel), lse)
    g = kind.down(ga)
    assert np.all(np.isnan(g[3])) and np.all(np.isfinite(np.delete(g, 3, 0)))


@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("pad,first", [(8, 8), (3, 1)])
@pytest.mark.parametrize("m,n,k", [(33, 200, 136), (70, 301, 75), (300, 1000, 64)])
def test_loss_strides(rt, kind, pad, first, m, n, k):
    print("case loss strides", kind.name, pad, first, m, n, k, flush=True)
    rng = np.random.default_rng(m)
    a, b = kind.values(rng.standard_normal((m, k))), kind.values(rng.standard_normal((k, n)))
    sel = rt.upload(rng.integers(-1, n, m).astype(np.int32))
    loss, row, lse = rt.matrixFCSoftmaxWithLoss(kind.up(rt, a), kind.up(rt, b), None, sel)
    ga, gb, _ = rt.matrixFCSoftmaxWithLossGrad(kind.up(rt, a), kind.up(rt, b), None, sel, lse)
    da, pa = strided(rt, kind, a, k + pad, first)
    db, pb = strided(rt, kind, b, n + pad, first)
    out = [rt.empty((m,)), rt.empty((m,)), rt.empty((1,))]
    lib_ = rt.lib
    s = kind.suffix()
    rt._check(getattr(lib_, "swc_hip_matrixFCSoftmaxWithLoss" + s)(m, n, k, pa, k + pad, pb, n + pad, None, sel.ptr,
                                                                   *(o.ptr for o in out)), "loss")
    # the same products over the same values: the same sums but for the order of copies that are cut differently
    np.testing.assert_allclose(out[0].numpy(), row.numpy(), rtol=1e-5, atol=1e-4)
    np.testing.assert_allclose(out[1].numpy(), lse.numpy(), rtol=1e-5, atol=1e-4)
    sga, pga = strided(rt, kind, np.zeros((m, k)), k + pad, first)
    sgb, pgb = strided(rt, kind, np.zeros((k, n)), n + pad, first)
    rt._check(getattr(lib_, "swc_hip_matrixFCSoftmaxWithLossGrad" + s)(m, n, k, pa, k + pad, pb, n + pad, None, sel.ptr, lse.ptr,
                                                                       None, pga, k + pad, pgb, n + pad, None), "grad")
    for d, rows, cols, want in ((sga, m, k, ga), (sgb, k, n, gb)):
        inside, beside, behind = rows_of(kind, d, rows, cols, cols + pad, first)
        np.testing.assert_allclose(inside, kind.down(want), rtol=4 * kind.half, atol=1e-3)
        assert np.all(np.isnan(beside)) and np.all(np.isnan(behind))


@gpu
@pytest.mark.parametrize("kind", KINDS)
def test_loss_empty(rt, kind):
    fn = getattr(rt.lib, "swc_hip_matrixFCSoftmaxWithLoss" + kind.suffix())
    loss = rt.upload(np.full(1, 7, np.float32))
    rt._check(fn(*loss_args(m=0, a=None, sel=None, row=None, lse=None, loss=loss.ptr)), "loss")
    assert loss.numpy()[0] == 0
    row, lse, sel = rt.upload(np.full(4, 7, np.float32)), rt.upload(np.full(4, 7, np.float32)), rt.upload(np.zeros(4, np.int32))
    rt._check(fn(*loss_args(n=0, a=None, b=None, sel=sel.ptr, row=row.ptr, lse=lse.ptr, loss=loss.ptr)), "loss")
    assert np.all(row.numpy() == 0) and np.all(lse.numpy() == 0)
    grad = getattr(rt.lib, "swc_hip_matrixFCSoftmaxWithLossGrad" + kind.suffix())
    gb, gbias = rt.upload(np.full((8, 8), 7, kind.numpy)), rt.upload(np.full(8, 7, kind.numpy))
    rt._check(grad(*loss_grad_args(m=0, a=None, b=None, sel=None, lse=None, da=None, db=gb.ptr, lddb=8, dbias=gbias.ptr)), "grad")
    assert np.all(kind.down(gb) == 0) and np.all(kind.down(gbias) == 0)


@gpu
def test_loss_gradient_by_differences(rt):
    """fp32: the gradient of the sum of the rows' losses against differences of the forward call"""
    rng = np.random.default_rng(13)
    m, n, k = 12, 50, 16
    a, b = rng.standard_normal((m, k)).astype(np.float32), rng.standard_normal((k, n)).astype(np.float32)
    sel = rt.upload(rng.integers(0, n, m).astype(np.int32))
    _, _, lse = rt.matrixFCSoftmaxWithLoss(rt.upload(a), rt.upload(b), None, sel)
    ga, gb, _ = rt.matrixFCSoftmaxWithLossGrad(rt.upload(a), rt.upload(b), None, sel, lse)

    def f(a, b):
        return float(rt.matrixFCSoftmaxWithLoss(rt.upload(a), rt.upload(b), None, sel)[1].numpy().astype(np.float64).sum())

    h = 2.0 ** -8
    e = ((k + 2) * U * (np.abs(a) @ np.abs(b)).max(1) + 2.0 ** -19 + 1e-6).sum() * 2      # of the sum of the rows' losses
    for x, g, other, s in ((a, ga, lambda y: f(y, b), np.abs(b).sum(0).max()), (b, gb, lambda y: f(a, y), np.abs(a).sum(1))):
        d = rng.choice([-1.0, 1.0], x.shape).astype(np.float32)
        want = (other(x + np.float32(h) * d) - other(x - np.float32(h) * d)) / (2 * h)
        got = float((g.numpy().astype(np.float64) * d).sum())
        # a row's loss along a line is a cumulant generating function: its third derivative is the third cumulant of values
        # between -s and s, at most (2 s)^3 / (6 sqrt 3)
        bound = (np.broadcast_to(2 * s, m) ** 3 / (6 * 3 ** 0.5)).sum() * h * h / 6 + e / h + 1e-5 * abs(want)
        assert abs(got - want) <= bound, (got, want, bound)


# --------------------------------------------------------------------------------------------------------- AdamW
RATES = dict(lr=3e-3, beta1=0.9, beta2=0.99, eps=1e-8, decay=0.1)


def adamw64(w, g, m, v, t, lr, beta1, beta2, eps, decay):
    m = beta1 * m + (1 - beta1) * g
    v = beta2 * v + (1 - beta2) * g * g
    w = w * (1 - lr * decay) - lr * (m / (1 - beta1 ** t)) / (np.sqrt(v / (1 - beta2 ** t)) + eps)
    return w, m, v


SIZES = [[1], [255, 1, 7], [256, 0, 1024, 1025, 3], [5000] * 3, list(range(1, 150)), [100003, 17]]


@gpu
@pytest.mark.parametrize("grads", KINDS)
@pytest.mark.parametrize("sizes", SIZES, ids=[f"{len(s)}x{max(s)}" for s in SIZES])
def test_adamw_32(rt, grads, sizes):
    """three steps over many tensors; the bfloat16 copies of some of them"""
    print("case adamw", grads.name, len(sizes), max(sizes), flush=True)
    rng = np.random.default_rng(sum(sizes))
    w = [rng.standard_normal(s).astype(np.float32) for s in sizes]
    m, v = [np.zeros(s) for s in sizes], [np.zeros(s) for s in sizes]
    dw = [rt.upload(x) for x in w]
    dm, dv = ([rt.upload(np.zeros(s, np.float32)) for s in sizes] for _ in range(2))
    copies = [rt.upload(np.full(s, 0x7FC0, np.uint16)) if i % 3 != 1 else None for i, s in enumerate(sizes)]
    state = rt.adamw_state()
    w = [x.astype(np.float64) for x in w]
    for t in range(1, 4):
        g = [grads.values(rng.standard_normal(s) * 0.1) for s in sizes]
        rt.adamwAdvance(state, RATES["beta1"], RATES["beta2"])
        rt.adamw(dw, [grads.up(rt, x) for x in g], dm, dv, state, copies=copies, **RATES)
        for i, s in enumerate(sizes):
            w[i], m[i], v[i] = adamw64(w[i], g[i].astype(np.float64), m[i], v[i], t, **RATES)
    assert state.numpy()[0] == 3
    for i, s in enumerate(sizes):
        gw = dw[i].numpy()
        # per step: the states two roundings each of their size, w two of its own and the update's ten of the update
        within(dm[i].numpy(), m[i], 3 * 4 * U * (np.abs(m[i]) + 0.3), "mom")
        within(dv[i].numpy(), v[i], 3 * 4 * U * (v[i] + 0.01), "var")
        within(gw, w[i], 3 * (3 * U * np.abs(w[i]) + 20 * U * RATES["lr"] * 8), "w")
        if copies[i] is not None:
            np.testing.assert_array_equal(copies[i].numpy(), to_bf16(gw).reshape(-1))


@gpu
def test_adamw_factors(rt):
    """a schedule's factor and a clipping coefficient on the device"""
    rng = np.random.default_rng(2)
    w, g = rng.standard_normal(300).astype(np.float32), rng.standard_normal(300).astype(np.float32)
    dw, dm, dv = rt.upload(w), rt.upload(np.zeros(300, np.float32)), rt.upload(np.zeros(300, np.float32))
    state = rt.adamw_state()
    rt.adamwAdvance(state, RATES["beta1"], RATES["beta2"])
    rt.adamw([dw], [rt.upload(g)], [dm], [dv], state, lr_factor=rt.upload(np.array([0.5], np.float32)),
             grad_factor=rt.upload(np.array([0.25], np.float32)), **RATES)
    want, m, v = adamw64(w.astype(np.float64), 0.25 * g, 0, 0, 1, **dict(RATES, lr=RATES["lr"] / 2))
    within(dw.numpy(), want, 3 * U * np.abs(want) + 20 * U * RATES["lr"] * 8, "w")
    within(dm.numpy(), m, 4 * U * np.abs(m), "mom")


def e4m3_values():
    code = np.arange(128)
    e, f = code >> 3, code & 7
    v = np.where(e == 0, f * 2.0 ** -9, (8 + f) * 2.0 ** (e - 10))
    v[127] = np.nan
    return np.concatenate([v, -v])


E4M3 = e4m3_values()


def random20(number, step, tensor):
    x = (np.asarray(number, np.uint64) + tensor * 0x9E3779B9 + step * 0x85EBCA6B) & 0xFFFFFFFF
    x = ((x ^ (x >> np.uint64(16))) * np.uint64(0x7FEB352D)) & np.uint64(0xFFFFFFFF)
    x = ((x ^ (x >> np.uint64(15))) * np.uint64(0x846CA68B)) & np.uint64(0xFFFFFFFF)
    return (x ^ (x >> np.uint64(16))) >> np.uint64(12)


def blocks(x, n):
    return np.pad(x, (0, -n % ADAMW_BLOCK)).reshape(-1, ADAMW_BLOCK)


@gpu
@pytest.mark.parametrize("grads", KINDS)
@pytest.mark.parametrize("sizes", SIZES, ids=[f"{len(s)}x{max(s)}" for s in SIZES])
def test_adamw_8(rt, grads, sizes):
    """two steps with 8-bit states: the codes are the nearest (mom) or the randomly chosen neighbour (root of var) of the
    step in 64 bits; one that differs lies at a border to within fp32's rounding"""
    print("case adamw8", grads.name, len(sizes), max(sizes), flush=True)
    rng = np.random.default_rng(sum(sizes) + 1)
    w = [rng.standard_normal(s) for s in sizes]
    count = [-(-s // ADAMW_BLOCK) for s in sizes]
    dw = [rt.upload(x.astype(np.float32)) for x in w]
    m8, v8 = ([rt.upload(np.zeros(s, np.uint8)) for s in sizes] for _ in range(2))
    ms, vs = ([rt.upload(np.zeros(c, np.float32)) for c in count] for _ in range(2))
    state = rt.adamw_state()
    for t in (1, 2):
        before = [(d.numpy().astype(np.float64), E4M3[a.numpy()] * np.repeat(b.numpy(), ADAMW_BLOCK)[:s].astype(np.float64),
                   E4M3[c.numpy()] * np.repeat(e.numpy(), ADAMW_BLOCK)[:s].astype(np.float64))
                  for d, a, b, c, e, s in zip(dw, m8, ms, v8, vs, sizes)]
        g = [grads.values(rng.standard_normal(s) * 10.0 ** rng.uniform(-6, 0, s)) for s in sizes]
        rt.adamwAdvance(state, RATES["beta1"], RATES["beta2"])
        rt.adamw8(dw, [grads.up(rt, x) for x in g], m8, ms, v8, vs, state, **RATES)
        for i, s in enumerate(sizes):
            if not s:
                continue
            w0, m0, r0 = before[i]
            w1, m1, v1 = adamw64(w0, g[i].astype(np.float64), m0, r0 * r0, t, **RATES)
            root = np.sqrt(v1)
            within(dw[i].numpy(), w1, 3 * U * np.abs(w1) + 40 * U * (np.abs(w1 - w0) + 10 * RATES["lr"]), "w")
            top, peak = np.abs(blocks(m1, s)).max(1), blocks(root, s).max(1)
            np.testing.assert_allclose(ms[i].numpy(), top / 448, rtol=16 * U)
            np.testing.assert_allclose(vs[i].numpy(), peak / 448, rtol=16 * U)
            y = m1 * np.repeat(448 / top, ADAMW_BLOCK)[:s]
            grid = 2.0 ** (np.floor(np.log2(np.maximum(np.abs(y), 2.0 ** -6))) - 3)
            got = E4M3[m8[i].numpy()]
            within(got, y, grid * (0.5 + 1e-5) + 1e-5 * np.abs(y), "mom, in units of its scale")
            y = root * np.repeat(448 / peak, ADAMW_BLOCK)[:s]
            grid = 2.0 ** (np.floor(np.log2(np.maximum(y, 2.0 ** -6))) - 3)
            up = y / grid + random20(np.arange(s), t, i).astype(np.float64) * 2.0 ** -20
            want = np.where(y > 0, np.maximum(np.floor(up), 1), 0) * grid
            got = E4M3[v8[i].numpy()]
            differ = ~np.isclose(got, want, rtol=1e-9)
            border = np.abs(up - np.round(up)) < 32 * 64 * U   # values of up to 16 units, some 64 roundings
            assert np.all(border[differ]), "a root of the variance on the wrong side"
            assert np.all(got[root > 0] > 0)
            within(got, y, grid * (1 + 1e-5), "root of var, in units of its scale")


@gpu
def test_adamw_8_random_rounding_keeps_the_mean(rt):
    """a variance that decays by 0.1 % a step: to nearest it would stay for good, at random it decays on average.
    4096 elements at the same value (and one large one per block to hold the scale): the mean of the roots after 100 steps of
    sqrt(0.999) is within five standard errors; a step of a rounding moves by at most a 16th of the value, so a chain of
    100 has a standard deviation of at most sqrt(100 / 4) / 16 of it"""
    n = 4096
    w, g = np.zeros(n, np.float32), np.zeros(n, np.float32)
    code = np.full(n, 0x48, np.uint8)       # 4.0 of 448 ...
    code[::ADAMW_BLOCK] = 0x7E              # ... next to 448 itself, which its gradient keeps there
    g[::ADAMW_BLOCK] = 448
    dw, dg, m8, v8 = rt.upload(w), rt.upload(g), rt.upload(np.zeros(n, np.uint8)), rt.upload(code)
    ms, vs = rt.upload(np.zeros(n // ADAMW_BLOCK, np.float32)), rt.upload(np.full(n // ADAMW_BLOCK, 1.0, np.float32))
    state = rt.adamw_state()
    for _ in range(100):
        rt.adamwAdvance(state, 0.9, 0.999)
        rt.adamw8([dw], [dg], [m8], [ms], [v8], [vs], state, 1e-3, 0.9, 0.999, 1e-8, 0.0)
    scale = np.repeat(vs.numpy(), ADAMW_BLOCK)
    root = E4M3[v8.numpy()] * scale
    small = np.ones(n, bool)
    small[::ADAMW_BLOCK] = False
    want = 4.0 * 0.999 ** 50
    assert abs(root[small].mean() - want) <= 5 * (5 / 16 * 4.0) / np.sqrt(small.sum())
    assert np.unique(root[small]).size > 1


@gpu
def test_adamw_8_not_finite(rt):
    """an infinite or NaN gradient marks its own element and no other of its block; an all-zero block stays zero"""
    n = 700
    rng = np.random.default_rng(1)
    g = rng.standard_normal(n).astype(np.float32)
    g[5], g[300] = np.inf, np.nan
    g[512:] = 0
    dw, m8, v8 = rt.upload(np.ones(n, np.float32)), rt.upload(np.zeros(n, np.uint8)), rt.upload(np.zeros(n, np.uint8))
    ms, vs = rt.upload(np.zeros(3, np.float32)), rt.upload(np.zeros(3, np.float32))
    state = rt.adamw_state()
    rt.adamwAdvance(state, 0.9, 0.99)
    rt.adamw8([dw], [rt.upload(g)], [m8], [ms], [v8], [vs], state, **RATES)
    bad = np.zeros(n, bool)
    bad[[5, 300]] = True
    for d in (m8, v8):
        np.testing.assert_array_equal(np.isnan(E4M3[d.numpy()]), bad)
        assert np.all(d.numpy()[512:] == 0)
    assert np.all(np.isfinite(ms.numpy())) and ms.numpy()[2] == 0 and vs.numpy()[2] == 0
    assert np.all(np.isfinite(dw.numpy()[~bad]))


@gpu
@pytest.mark.parametrize("kind", KINDS)
def test_adamw_unaligned(rt, kind):
    """tensors at any element of an arena (next to each other, off the 16-byte grid): nothing outside them changes"""
    rng = np.random.default_rng(4)
    total, parts = 3000, [(1, 300), (303, 1), (304, 1025), (1331, 1600)]
    w, g = rng.standard_normal(total).astype(np.float32), kind.values(rng.standard_normal(total))
    dw, dg = rt.upload(w), kind.up(rt, g)
    dm, dv, dc = rt.upload(np.full(total, 7, np.float32)), rt.upload(np.full(total, 7, np.float32)), rt.upload(np.zeros(total, np.uint16))
    view = lambda d: [d.offset_view(at, (n,)) for at, n in parts]   # noqa: E731
    state = rt.adamw_state()
    rt.adamwAdvance(state, RATES["beta1"], RATES["beta2"])
    rt.adamw(view(dw), view(dg), view(dm), view(dv), state, copies=view(dc), **RATES)
    inside = np.zeros(total, bool)
    for at, n in parts:
        inside[at:at + n] = True
    want, m, v = adamw64(w.astype(np.float64), g.astype(np.float64), 7.0, 7.0, 1, **RATES)
    got = dw.numpy()
    np.testing.assert_array_equal(got[~inside], w[~inside])
    assert np.all(dm.numpy()[~inside] == 7) and np.all(dv.numpy()[~inside] == 7) and np.all(dc.numpy()[~inside] == 0)
    within(got[inside], want[inside], 3 * U * np.abs(want[inside]) + 40 * U, "w")
    np.testing.assert_array_equal(dc.numpy()[inside], to_bf16(got[inside]))


@gpu
@pytest.mark.parametrize("grads", KINDS)
def test_adamw_large(rt, grads):
    """a call large enough to go past the caches gives the bits of calls on its parts"""
    rng = np.random.default_rng(17)
    n, cut = 17_000_003, 5120 * ADAMW_BLOCK
    w, g = rng.standard_normal(n).astype(np.float32), grads.values(rng.standard_normal(n).astype(np.float32))
    state = rt.adamw_state()
    rt.adamwAdvance(state, RATES["beta1"], RATES["beta2"])
    dg = grads.up(rt, g)
    one, two = ([rt.upload(w), rt.upload(np.zeros(n, np.float32)), rt.upload(np.zeros(n, np.float32))] for _ in range(2))
    rt.adamw([one[0]], [dg], [one[1]], [one[2]], state, **RATES)
    for at, size in ((0, cut), (cut, 9_000_001), (cut + 9_000_001, n - cut - 9_000_001)):
        v = [x.offset_view(at, (size,)) for x in two]
        rt.adamw([v[0]], [dg.offset_view(at, (size,))], [v[1]], [v[2]], state, **RATES)
    for x, y in zip(one, two):
        np.testing.assert_array_equal(x.numpy(), y.numpy())
    # 8 bits: the random numbers are an element's in its tensor, so only the first part is the same
    count = -(-n // ADAMW_BLOCK)
    one, two = ([rt.upload(w), rt.upload(np.zeros(n, np.uint8)), rt.upload(np.zeros(n, np.uint8)), rt.upload(np.zeros(count, np.float32)),
                 rt.upload(np.zeros(count, np.float32))] for _ in range(2))
    rt.adamw8([one[0]], [dg], [one[1]], [one[3]], [one[2]], [one[4]], state, **RATES)
    v = [x.offset_view(0, (cut,)) for x in two[:3]] + [x.offset_view(0, (cut // ADAMW_BLOCK,)) for x in two[3:]]
    rt.adamw8([v[0]], [dg.offset_view(0, (cut,))], [v[1]], [v[3]], [v[2]], [v[4]], state, **RATES)
    for x, y in zip(one[:3], two):
        np.testing.assert_array_equal(x.numpy()[:cut], y.numpy()[:cut])
    assert one[0].numpy()[-1] != w[-1]


# ---------------------------------------------------------------- together, workspaces, graphs and streams
TORCH_VIEWS = """
import torch
assert torch.cuda.is_available()
from swcompiler_amd.hip import SwcHipError, runtime
rt = runtime()
gen = torch.Generator().manual_seed(3)
base = torch.randint(-3, 4, (80, 200), generator=gen).to("cuda", torch.bfloat16)
weight = torch.randint(-3, 4, (64, 136), generator=gen).to("cuda", torch.bfloat16)
out, pre = torch.zeros(70, 300, device="cuda", dtype=torch.bfloat16), torch.zeros(140, 136, device="cuda", dtype=torch.bfloat16)
torch.cuda.synchronize()
a, c, z = base[5:75, 3:67], out[:, 100:236], pre[::2]
rt.matrixMatrixFCActAdd(a, weight, None, "relu", None, z, c)
rt.sync()
want = a.float().cpu() @ weight.float().cpu()
assert torch.equal(z.float().cpu(), want.bfloat16().float())
assert torch.equal(c.float().cpu(), want.clamp(min=0).bfloat16().float())
assert not out[:, :100].any() and not out[:, 236:].any() and not pre[1::2].any()
rt.use_default_stream()     # torch's: no waits between its work and the library's
for _ in range(20):
    x = base[:70, :64] * 2
    y = torch.empty(70, 136, device="cuda", dtype=torch.bfloat16)
    rt.matrixMatrixFCActAdd(x, weight, out=y)
    y = y - (x.float() @ weight.float()).bfloat16()
    assert not y.any()
for bad, message in ((weight.t(), "not contiguous"), (a[:1].expand(70, 64), "rows overlap")):
    try:
        rt.matrixMatrixFCActAdd(bad, base[:bad.shape[1], :8].contiguous())
    except SwcHipError as e:
        assert message in str(e), e
    else:
        raise AssertionError(message)
print("views done")
"""


@gpu
def test_torch_views():
    """torch tensors as they are: columns of a wider one, rows of a longer one, outputs too; on torch's own stream.  In a
    process of its own: torch brings its own HIP runtime, which has to be the first one loaded"""
    done = subprocess.run([sys.executable, "-c", TORCH_VIEWS],
                          cwd=ROOT, capture_output=True, text=True, timeout=110)
    assert done.returncode == 0 and "views done" in done.stdout, done.stderr[-2000:]


def make_step(rt, rng, kind, m=150, d=72, h=200, n=1003):
    """a small language-model step: two layers with a residual, the loss, all gradients, AdamW on fp32 weights with
    bfloat16 copies feeding the products -> (run, parameters, everything the step writes)"""
    shapes = dict(w1=(d, h), b1=(h,), w2=(h, d), b2=(d,), head=(d, n))
    master = {k: rt.upload((rng.standard_normal(s) / np.sqrt(s[0])).astype(np.float32)) for k, s in shapes.items()}
    if kind is BF:
        weight = {k: rt.upload(to_bf16(v.numpy()).reshape(v.shape)) for k, v in master.items()}
    else:
        weight = master
    grad = {k: rt.empty(s, kind.numpy) for k, s in shapes.items()}
    mom, var = ({k: rt.upload(np.zeros(s, np.float32)) for k, s in shapes.items()} for _ in range(2))
    x = kind.up(rt, rng.standard_normal((m, d)))
    sel = rng.integers(0, n, m).astype(np.int32)
    sel[::5] = -1
    sel = rt.upload(sel)
    e = lambda *s: rt.empty(s, kind.numpy)   # noqa: E731
    z1, a1, y, dy, da1 = e(m, h), e(m, h), e(m, d), e(m, d), e(m, h)
    loss, row, lse = rt.empty((1,)), rt.empty((m,)), rt.empty((m,))
    state = rt.adamw_state()
    names = list(shapes)

    def run():
        rt.matrixMatrixFCActAdd(x, weight["w1"], weight["b1"], "gelu", None, z1, a1)
        rt.matrixMatrixFCActAdd(a1, weight["w2"], weight["b2"], "none", x, None, y)
        rt.matrixFCSoftmaxWithLoss(y, weight["head"], None, sel, row, lse, loss)
        rt.matrixFCSoftmaxWithLossGrad(y, weight["head"], None, sel, lse, None, dy, grad["head"])
        rt.matrixMatrixFCActAddGrad(dy, a1, weight["w2"], None, "none", da1, grad["w2"], grad["b2"])
        rt.matrixMatrixFCActAddGrad(da1, x, weight["w1"], z1, "gelu", None, grad["w1"], grad["b1"])
        rt.adamwAdvance(state, 0.9, 0.99)
        rt.adamw([master[k] for k in names], [grad[k] for k in names], [mom[k] for k in names], [var[k] for k in names], state,
                 1e-2, 0.9, 0.99, 1e-8, 0.01, copies=[weight[k] for k in names] if kind is BF else None)

    return run, (x, sel, master, weight), dict(loss=loss, row=row, lse=lse, state=state, y=y,
                                               **{"g_" + k: v for k, v in grad.items()}, **{"w_" + k: v for k, v in master.items()})


@gpu
@pytest.mark.parametrize("kind", KINDS)
def test_a_training_step(rt, kind):
    """the operators in sequence against the same step in 64 bits (gradients and losses of the first step)"""
    rng = np.random.default_rng(21)
    run, (x, sel, master, weight), out = make_step(rt, rng, kind)
    w = {k: kind.down(v).astype(np.float64) for k, v in weight.items()}
    x64, s = kind.down(x).astype(np.float64), sel.numpy()
    run()
    z1 = x64 @ w["w1"] + w["b1"]
    a1 = act64(z1, "gelu")
    y = a1 @ w["w2"] + w["b2"] + x64
    (loss, row, lse, dy, dhead, _), _ = loss64(y, w["head"], None, s)
    da1 = dy @ w["w2"].T
    dz1 = da1 * slope64(z1, "gelu")
    want = dict(loss=loss, row=row, lse=lse, y=y, g_head=dhead, g_w2=a1.T @ dy, g_b2=dy.sum(0), g_w1=x64.T @ dz1, g_b1=dz1.sum(0))
    # seven roundings lie between the input and the last gradient; the norm of what independent roundings do is at most
    # the number of them times half a step
    for name, value in want.items():
        got = out[name].numpy() if name in ("loss", "row", "lse") else kind.down(out[name])
        got = np.asarray(got, np.float64).reshape(np.shape(value))
        assert np.linalg.norm(got - value) <= (7 * kind.half if kind is BF else 1e-5) * np.linalg.norm(value), name
    before = {k: v.numpy() for k, v in master.items()}
    run()
    assert out["state"].numpy()[0] == 2
    assert all(np.any(before[k] != v.numpy()) for k, v in master.items())


@gpu
@pytest.mark.parametrize("kind", KINDS)
def test_a_recorded_step_replays(rt, kind):
    """a training step recorded into a graph: every replay, with eager steps of another model and synchronisation between,
    is bit for bit what the eager step does"""
    eager, _, want = make_step(rt, np.random.default_rng(22), kind)
    run, _, out = make_step(rt, np.random.default_rng(22), kind)
    other, _, _ = make_step(rt, np.random.default_rng(23), kind, m=90, n=2001)
    other(), run(), eager()           # (the workspace is large enough for all of them now)
    graph = C.c_void_p()
    rt._check(rt.lib.swc_hip_graph_begin(), "begin")
    try:
        run()
    finally:
        rt._check(rt.lib.swc_hip_graph_end(C.byref(graph)), "end")
    try:
        for _ in range(4):
            rt._check(rt.lib.swc_hip_graph_launch(graph), "launch")
            other()
            eager()
            rt.sync()
            for name in want:
                np.testing.assert_array_equal(out[name].numpy(), want[name].numpy(), err_msg=name)
    finally:
        rt._check(rt.lib.swc_hip_graph_destroy(graph), "destroy")


@gpu
@pytest.mark.parametrize("kind", KINDS)
def test_runs_are_bit_for_bit_the_same(rt, kind):
    """no result depends on the order in which workgroups finish"""
    first, _, a = make_step(rt, np.random.default_rng(24), kind, m=700, d=264, h=520, n=3001)
    second, _, b = make_step(rt, np.random.default_rng(24), kind, m=700, d=264, h=520, n=3001)
    for _ in range(3):
        first(), second()
    for name in a:
        np.testing.assert_array_equal(a[name].numpy(), b[name].numpy(), err_msg=name)


WORKSPACE_CASES = [(1, 72, 2048), (33, 200, 136), (70, 301, 75), (300, 520, 1024), (1100, 1032, 96)]


@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("m,n,k", WORKSPACE_CASES)
def test_workspace_queries(rt, kind, m, n, k):
    """each call runs on a workspace of exactly the queried size, at any alignment, and is refused one that is too small"""
    print("case workspace", kind.name, m, n, k, flush=True)
    rng = np.random.default_rng(m)
    bf = int(kind is BF)
    s = kind.suffix()
    sel, lse = rt.upload(rng.integers(0, n, m).astype(np.int32)), rt.empty((m,))
    row, loss = rt.empty((m,)), rt.empty((1,))
    for first in (0, 1):
        at = lambda rows, cols: strided(rt, kind, rng.standard_normal((rows, cols)), cols, first)   # noqa: E731
        (ka, a), (kb, b), (kc, c), (kga, ga), (kgb, gb), (kz, z) = at(m, k), at(k, n), at(m, n), at(m, k), at(k, n), at(m, n)
        bias, gbias = kind.up(rt, np.zeros(n)), rt.empty((n,), kind.numpy)
        calls = {
            "matrixMatrixFCActAdd": (m, n, k, a, k, b, n, bias.ptr, 2, z, n, None, 0, c, n),
            "matrixMatrixFCActAddGrad": (m, n, k, c, n, a, k, b, n, z, n, 2, ga, k, gb, n, gbias.ptr),
            "matrixFCSoftmaxWithLoss": (m, n, k, a, k, b, n, bias.ptr, sel.ptr, row.ptr, lse.ptr, loss.ptr),
            "matrixFCSoftmaxWithLossGrad": (m, n, k, a, k, b, n, bias.ptr, sel.ptr, lse.ptr, None, ga, k, gb, n, gbias.ptr),
        }
        for name, args in calls.items():
            need = getattr(rt.lib, f"swc_hip_{name}_workspace_bytes")(m, n, k, bf)
            buf = rt.upload(np.full(max(need, 16) + 4096, 0xA5, np.uint8))
            rt._check(rt.lib.swc_hip_set_workspace(buf.ptr, max(need, 16)), "set_workspace")
            try:
                rt._check(getattr(rt.lib, "swc_hip_" + name + s)(*args), name)
                assert np.all(buf.numpy()[max(need, 16):] == 0xA5), f"{name} wrote behind its workspace"
                if "Loss" in name:
                    rt._check(rt.lib.swc_hip_set_workspace(buf.ptr, 16), "set_workspace")
                    assert getattr(rt.lib, "swc_hip_" + name + s)(*args) == EINVAL
            finally:
                rt._check(rt.lib.swc_hip_set_workspace(None, 0), "set_workspace")
                rt.sync()


@gpu
@pytest.mark.parametrize("kind", KINDS)
def test_on_another_stream(rt, kind):
    """the calls go to the stream that swc_hip_set_stream names, all of their launches"""
    hiprt = C.CDLL("libamdhip64.so.7")
    stream = C.c_void_p()
    assert hiprt.hipStreamCreateWithFlags(C.byref(stream), 1) == 0
    eager, _, want = make_step(rt, np.random.default_rng(25), kind)
    run, _, out = make_step(rt, np.random.default_rng(25), kind)
    eager()
    rt.sync()
    rt._check(rt.lib.swc_hip_set_stream(stream), "set_stream")
    try:
        run()
        rt.sync()
        for name in want:
            np.testing.assert_array_equal(out[name].numpy(), want[name].numpy(), err_msg=name)
    finally:
        rt._check(rt.lib.swc_hip_set_stream(None), "set_stream")
        hiprt.hipStreamDestroy(stream)
