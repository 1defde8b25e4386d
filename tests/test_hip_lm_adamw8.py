"""AdamW with its states in 8 bits: the mean under slow decays (helpers and the definition as in test_hip_lm_ops.py)."""
import numpy as np
import pytest

from tests.test_hip_lm_ops import E4M3, KINDS, U, blocks, random20, to_bf16, within
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
