"""AdamW with its states in 8 bits: the mean under slow decays, copies, factors, tensors off the 16-byte grid, recorded steps
and long runs (helpers and the definition as in test_hip_lm_ops.py)."""
import ctypes as C

import numpy as np
import pytest

from tests.test_hip_lm_ops import E4M3, KINDS, SIZES, U, adamw64, blocks, random20, to_bf16, within
from swcompiler_amd.hip import ADAMW_BLOCK

gpu = pytest.mark.gpu
RATES = dict(lr=3e-3, beta1=0.9, beta2=0.99, eps=1e-8, decay=0.1)


@pytest.fixture(scope="module")
def rt():
    from swcompiler_amd.hip import runtime
    return runtime()


class Model:
    """tensors of the given sizes and their states on the device; first: offsets of every array from an allocation's start"""

    def __init__(self, rt, sizes, seed=0, first=None, copies=True, bits=8):
        rng = np.random.default_rng(seed)
        self.rt, self.sizes, self.bits = rt, sizes, bits
        self.state = rt.adamw_state()
        first = first or dict(w=0, g=0, mom=0, var=0, copy=0)
        self.arena = {}

        def views(name, values, counts, dtype, fill):
            at, starts = first.get(name, 0), []
            for c in counts:
                starts.append(at)
                at += c + first.get("gap", 0)
            host = np.full(at + 64, fill, dtype)
            inside = np.zeros(at + 64, bool)
            for s, c, v in zip(starts, counts, values):
                host[s:s + c], inside[s:s + c] = v, True
            d = rt.upload(host)
            self.arena[name] = (d, inside, fill)
            return [d.offset_view(s, (c,)) for s, c in zip(starts, counts)]

        zeros = lambda n: [0] * len(n)   # noqa: E731
        self.w = views("w", [rng.standard_normal(s) for s in sizes], sizes, np.float32, 7)
        held = np.uint8 if bits == 8 else np.float32
        self.mom, self.var = (views(n, zeros(sizes), sizes, held, 77) for n in ("mom", "var"))
        count = [-(-s // ADAMW_BLOCK) for s in sizes]
        self.ms, self.vs = (views(n, zeros(count), count, np.float32, 7) for n in ("ms", "vs"))
        self.copy = views("copy", [0x7FC0] * len(sizes), sizes, np.uint16, 77) if copies else None
        self.first, self.views = first, views

    def grads(self, kind, values):
        host = [kind.values(v) if kind.name == "f32" else to_bf16(v) for v in values]
        self.views("g", host, self.sizes, kind.numpy, 0)
        d, _, _ = self.arena["g"]
        at, out = self.first.get("g", 0), []
        for s in self.sizes:
            out.append(d.offset_view(at, (s,)))
            at += s + self.first.get("gap", 0)
        return out

    def step(self, g, lr_factor=None, grad_factor=None, **rates):
        r = dict(RATES, **rates)
        self.rt.adamwAdvance(self.state, r["beta1"], r["beta2"])
        more = dict(copies=self.copy, lr_factor=lr_factor, grad_factor=grad_factor, **r)
        if self.bits == 8:
            self.rt.adamw8(self.w, g, self.mom, self.ms, self.var, self.vs, self.state, **more)
        else:
            self.rt.adamw(self.w, g, self.mom, self.var, self.state, **more)

    def held(self):
        names = ("w", "mom", "var") + (("ms", "vs") if self.bits == 8 else ()) + (("copy",) if self.copy else ())
        return {n: [x.numpy() for x in getattr(self, n)] for n in names}


def same(a, b):
    for name in a:
        for i, (x, y) in enumerate(zip(a[name], b[name])):
            np.testing.assert_array_equal(x, y, err_msg=f"{name} of tensor {i}")


# ------------------------------------------------------------------------------------- the mean under a slow decay
@gpu
@pytest.mark.parametrize("grads", KINDS)
@pytest.mark.parametrize("beta1", [0.9374, 0.9375, 0.95, 0.99, 0.999])
def test_mean_codes(rt, grads, beta1):
    """three steps: below 15/16 the mean's codes are the nearest, from there on the neighbour that the random number chooses;
    one that differs lies at a border to within fp32's rounding"""
    print("case mean", grads.name, beta1, flush=True)
    sizes = [255, 1, 1025, 5000]
    rng = np.random.default_rng(3)
    m = Model(rt, sizes)
    for t in (1, 2, 3):
        before = [E4M3[a.numpy()] * np.repeat(b.numpy(), ADAMW_BLOCK)[:s].astype(np.float64) for a, b, s in zip(m.mom, m.ms, sizes)]
        g = [grads.values(rng.standard_normal(s) * 10.0 ** rng.uniform(-4, 0, s)) for s in sizes]
        m.step(m.grads(grads, g), beta1=beta1)
        for i, s in enumerate(sizes):
            mean = beta1 * before[i] + (1 - beta1) * g[i].astype(np.float64)
            top = np.abs(blocks(mean, s)).max(1)
            np.testing.assert_allclose(m.ms[i].numpy(), top / 448, rtol=16 * U)
            y = mean * np.repeat(448 / top, ADAMW_BLOCK)[:s]
            grid = 2.0 ** (np.floor(np.log2(np.maximum(np.abs(y), 2.0 ** -6))) - 3)
            got = E4M3[m.mom[i].numpy()]
            # (a mean whose two parts cancel is off by their roundings, two of either)
            size = (np.abs(beta1 * before[i]) + np.abs((1 - beta1) * g[i])) * np.repeat(448 / top, ADAMW_BLOCK)[:s]
            slack = 32 * U * (np.abs(y) + size) / grid
            if beta1 < 15 / 16:
                within(got, y, grid * (0.5 + slack), "mean to the nearest value")
                continue
            number = 0xFFFFFFFF ^ ((np.arange(s, dtype=np.uint64) + i * 0x9E3779B9 + t * 0x85EBCA6B) & 0xFFFFFFFF)
            up = np.abs(y) / grid + random20(number, 0, 0).astype(np.float64) * 2.0 ** -20
            want = np.floor(up) * grid * np.sign(y)
            differ = ~np.isclose(got, want, rtol=1e-9, atol=0)
            assert np.all((np.abs(up - np.round(up)) < slack)[differ]), "a mean on the wrong side"
            within(got, y, grid * (1 + slack), "mean up or down")


@gpu
@pytest.mark.parametrize("beta1", [0.95, 0.99])
@pytest.mark.parametrize("gradient", [8.0, 0.0, -4.0])
def test_a_slow_mean_follows_its_gradient(rt, beta1, gradient):
    """4080 means at 4 under a gradient that stays, in blocks whose scale one large element holds at 1.  To the nearest value they
    would stop where (1 - beta1) |g - mom| is below half the distance of two values (at 4, to 8 or to 0, from the first step
    for beta1 0.99).  Their average is within five standard errors of the exact mean: a rounding is between values at most 1
    apart (below 16), so its standard deviation at most 1/2, and earlier ones decay by beta1 a step"""
    n, steps = 4096, 200
    m = Model(rt, [n], copies=False)
    code, g = np.full(n, 0x48, np.uint8), np.full(n, gradient, np.float32)      # 4.0
    code[::ADAMW_BLOCK], g[::ADAMW_BLOCK] = 0x7E, 448
    m.mom, m.ms = [rt.upload(code)], [rt.upload(np.ones(n // ADAMW_BLOCK, np.float32))]
    dg = [rt.upload(g)]
    for _ in range(steps):
        m.step(dg, beta1=beta1, lr=0.0)
    small = np.ones(n, bool)
    small[::ADAMW_BLOCK] = False
    got = (E4M3[m.mom[0].numpy()] * np.repeat(m.ms[0].numpy(), ADAMW_BLOCK))[small]
    want = gradient + (4 - gradient) * beta1 ** steps
    assert abs(got.mean() - want) <= 5 * 0.5 / np.sqrt((1 - beta1 ** 2) * small.sum())


# ------------------------------------------------------------------- copies, factors, offsets, recorded and large steps
@gpu
@pytest.mark.parametrize("grads", KINDS)
@pytest.mark.parametrize("sizes", SIZES, ids=[f"{len(s)}x{max(s)}" for s in SIZES])
def test_copies(rt, grads, sizes):
    """copies of some of the tensors, whole blocks and short ones: w rounded to bfloat16; they change nothing else"""
    print("case copies", grads.name, len(sizes), max(sizes), flush=True)
    rng = np.random.default_rng(sum(sizes))
    with_, without = Model(rt, sizes), Model(rt, sizes, copies=False)
    with_.copy = [None if i % 3 == 1 else c for i, c in enumerate(with_.copy)]
    for _ in range(2):
        g = [rng.standard_normal(s) for s in sizes]
        with_.step(with_.grads(grads, g))
        without.step(without.grads(grads, g))
    for w, c in zip(with_.w, with_.copy):
        if c is not None:
            np.testing.assert_array_equal(c.numpy(), to_bf16(w.numpy()).reshape(-1))
    with_.copy = None
    same(with_.held(), without.held())


@gpu
@pytest.mark.parametrize("grads", KINDS)
@pytest.mark.parametrize("beta1", [0.9, 0.95])
def test_offsets(rt, grads, beta1):
    """every array at addresses of an element's alignment only (codes at odd bytes), with gaps: the bits of aligned arrays, and
    nothing beside the tensors changes"""
    sizes = [300, 1, 1025, 256, 0, 1600, 2048]
    rng = np.random.default_rng(4)
    plain, moved = Model(rt, sizes), Model(rt, sizes, first=dict(w=1, g=3, mom=1, var=3, ms=1, vs=3, copy=5, gap=3))
    for _ in range(3):
        g = [rng.standard_normal(s) for s in sizes]
        plain.step(plain.grads(grads, g), beta1=beta1)
        moved.step(moved.grads(grads, g), beta1=beta1)
    same(plain.held(), moved.held())
    for name, (d, inside, fill) in moved.arena.items():
        assert np.all(d.numpy()[~inside] == fill), name


@gpu
@pytest.mark.parametrize("grads", KINDS)
def test_factors(rt, grads):
    """factors on the device that are powers of two give the bits of a call with the rate and the gradients scaled"""
    sizes = [700, 33]
    rng = np.random.default_rng(2)
    one, two = Model(rt, sizes), Model(rt, sizes)
    half, quarter = (rt.upload(np.array([x], np.float32)) for x in (0.5, 0.25))
    for _ in range(2):
        g = [grads.values(rng.standard_normal(s)) for s in sizes]
        one.step(one.grads(grads, g), lr_factor=half, grad_factor=quarter, decay=0.0)
        two.step(two.grads(grads, [x / 4 for x in g]), lr=RATES["lr"] / 2, decay=0.0)
    same(one.held(), two.held())


@gpu
@pytest.mark.parametrize("grads", KINDS)
def test_a_recorded_step_goes_on(rt, grads):
    """a step recorded once and replayed counts, and is bit for bit the eager step: the random numbers are those of the step"""
    sizes = [5000, 257, 16]
    rng = np.random.default_rng(6)
    eager, recorded, other = Model(rt, sizes), Model(rt, sizes), Model(rt, [9000])
    g = [rng.standard_normal(s) for s in sizes]
    ge, gr, go = eager.grads(grads, g), recorded.grads(grads, g), other.grads(grads, [rng.standard_normal(9000)])
    for m, x in ((eager, ge), (recorded, gr), (other, go)):
        m.step(x, beta1=0.95)
    graph = C.c_void_p()
    rt._check(rt.lib.swc_hip_graph_begin(), "begin")
    try:
        recorded.step(gr, beta1=0.95)
    finally:
        rt._check(rt.lib.swc_hip_graph_end(C.byref(graph)), "end")
    try:
        for _ in range(4):
            rt._check(rt.lib.swc_hip_graph_launch(graph), "launch")
            other.step(go)
            eager.step(ge, beta1=0.95)
            rt.sync()
            same(eager.held(), recorded.held())
    finally:
        rt._check(rt.lib.swc_hip_graph_destroy(graph), "destroy")
    assert recorded.state.numpy()[0] == 5


@gpu
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("grads", KINDS)
def test_large(rt, grads, bits):
    """a call large enough to go past the caches (17 million elements) gives the bits, scales and copies of a small call on its
    first part, and every copy is its weight rounded"""
    n, cut = 17_000_003, 5120 * ADAMW_BLOCK
    rng = np.random.default_rng(17)
    one, two = Model(rt, [n], bits=bits), Model(rt, [n], bits=bits)
    g = rng.standard_normal(n, np.float32)
    go, gt = one.grads(grads, [g]), two.grads(grads, [g])
    two.w, gt, two.mom, two.var, two.copy = ([x[0].offset_view(0, (cut,))] for x in (two.w, gt, two.mom, two.var, two.copy))
    two.ms, two.vs = ([x[0].offset_view(0, (cut // ADAMW_BLOCK,))] for x in (two.ms, two.vs))
    for beta1 in (0.9, 0.95):
        one.step(go, beta1=beta1)
        two.step(gt, beta1=beta1)
    a, b = one.held(), two.held()
    np.testing.assert_array_equal(a["copy"][0], to_bf16(a["w"][0]))
    for name, value in b.items():
        np.testing.assert_array_equal(a[name][0][:value[0].size], value[0], err_msg=name)
    arena, inside, fill = one.arena["w"]
    assert np.all(arena.numpy()[~inside] == fill) and a["w"][0][-1] != two.arena["w"][0].numpy()[n - 1]


@gpu
@pytest.mark.parametrize("grads", KINDS)
@pytest.mark.parametrize("beta1", [0.9, 0.95])
def test_a_long_run(rt, grads, beta1):
    """40 steps: the first, from states of zero, has the weights that 32-bit states give, bit for bit; each later one the step in
    64 bits from the states as held before it, no drift and no neighbour's state; the copies stay the weights rounded"""
    sizes = [4096, 513]
    rng = np.random.default_rng(8)
    eight, full = Model(rt, sizes), Model(rt, sizes, bits=32)
    rates = dict(RATES, beta1=beta1)
    for t in range(1, 41):
        h = eight.held()
        g = [grads.values(rng.standard_normal(s) * 10.0 ** rng.uniform(-3, 0, s)) for s in sizes]
        eight.step(eight.grads(grads, g), beta1=beta1)
        if t == 1:
            full.step(full.grads(grads, g), beta1=beta1)
            same(dict(w=full.held()["w"]), dict(w=eight.held()["w"]))
        for i, s in enumerate(sizes):
            m0, r0 = (E4M3[h[a][i]] * np.repeat(h[b][i], ADAMW_BLOCK)[:s].astype(np.float64) for a, b in (("mom", "ms"), ("var", "vs")))
            w0 = h["w"][i].astype(np.float64)
            w1, m1, v1 = adamw64(w0, g[i].astype(np.float64), m0, r0 * r0, t, **rates)
            # three roundings of w; some forty of the update, whose mean is off by those of its two parts where they cancel
            parts = beta1 * np.abs(m0) + (1 - beta1) * np.abs(g[i])
            size = rates["lr"] * (parts / (1 - beta1 ** t)) / (np.sqrt(v1 / (1 - rates["beta2"] ** t)) + rates["eps"])
            within(eight.w[i].numpy(), w1, 3 * U * np.abs(w1) + 40 * U * (size + rates["lr"] * rates["decay"] * np.abs(w0)), f"w, step {t}")
    h = eight.held()
    for w, c in zip(h["w"], h["copy"]):
        np.testing.assert_array_equal(c, to_bf16(w))
