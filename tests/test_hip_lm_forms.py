"""Operators of language models: forms, sizes and values beside the ones that test_hip_lm_ops.py takes (whose helpers and
tolerances hold here too)."""
import numpy as np
import pytest

from tests.test_hip_lm_ops import BF, F32, KINDS, U, rows_of, small_ints, strided, within

gpu = pytest.mark.gpu


@pytest.fixture(scope="module")
def rt():
    from swcompiler_amd.hip import runtime
    return runtime()


# ------------------------------------------------------------------------------- every tile, cut and remainder in use
# Exact integers in fp32, so that an element, a slice of the contraction or a range of it that is lost or taken twice shows.
# The shapes are the smallest that reach each tile with each layout and end, whole and cut along the contraction, and with
# columns left to smaller tiles; `kernel`: what has to have run, so that another choice of tiles does not drop it unseen.
DEEP, BIG, LOW = "product<bf16,256x256,4,3,2,", "product<bf16,256x256,8,3,2,", "product<bf16,64x128,4,3,3,"
FORWARD = [(5645, 720, 3880, "product<bf16,256x256,8,3,2,kn> x"), (165, 16952, 9, LOW), (5916, 2704, 820, LOW),
           (67, 2856, 3496, LOW + "kn> x"), (7866, 2568, 536, ""), (2838, 65, 4307, ""), (732, 6795, 2468, ""), (210, 12505, 8, ""),
           (3789, 5832, 264, ""), (66, 4097, 1568, ""), (6362, 3764, 1317, ""), (66, 4352, 3792, ""), (512, 4096, 1000, LOW + "kn> x1")]
# (m, n, k, dA's kernel, dB's kernel)
GRADIENTS = [(4097, 6200, 2050, DEEP + "kk> x1", BIG + "mn> x1"), (1400, 50264, 1032, DEEP + "kk> x8", ""),
             (4104, 6150, 4099, LOW + "kk> x1", ""), (6102, 11416, 704, "", DEEP + "mn> x1"), (8675, 8558, 130, BIG + "kk> x", ""),
             (7651, 12244, 540, DEEP + "kk> x", ""), (4628, 196, 2810, BIG + "kk> x1", ""), (4642, 8, 791, LOW + "kk> x1", ""),
             (4437, 8, 653, "", ""), (806, 8, 6649, "", ""), (3866, 536, 5416, "", ""), (4560, 472, 3760, "", ""),
             (4251, 814, 4072, "", ""), (7751, 247, 2728, "", ""), (4550, 1563, 6268, "", ""), (736, 2280, 7072, "", ""),
             (4054, 156, 4175, "", ""), (4033, 16592, 224, "", BIG + "mn> x"), (770, 12070, 1336, "", LOW + "mn> x1"),
             (525, 4214, 4928, "", ""), (2275, 3536, 1472, "", ""), (255, 5064, 4351, "", ""), (1315, 10552, 2216, "", ""),
             (3048, 3462, 72, LOW + "kk> x", ""), (8020, 1431, 65, "", LOW + "mn> x"), (813, 8728, 72, "", ""), (2222, 6212, 68, "", ""),
             (1358, 8, 37, "", ""), (37, 1384, 40, "", ""), (1800, 1597, 33, "", ""), (1, 1487, 34, "", ""), (1482, 9, 9, "", ""),
             (1, 12648, 216, "", ""), (1, 16784, 160, "", ""), (1, 14344, 328, "", "")]


def ran(rt, kind, kernel):
    if kernel and kind is BF:
        assert rt.last_kernel().startswith(kernel), rt.last_kernel()


@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("m,n,k,kernel", FORWARD)
def test_forward_tiles(rt, kind, m, n, k, kernel):
    print("case forward", kind.name, m, n, k, flush=True)
    rng = np.random.default_rng(m + n + k)
    a, b, bias, res = (small_ints(rng, *s) for s in ((m, k), (k, n), (n,), (m, n)))
    pre = rt.empty((m, n), kind.numpy)
    c = rt.matrixMatrixFCActAdd(kind.up(rt, a), kind.up(rt, b), kind.up(rt, bias), "relu", kind.up(rt, res), pre)
    ran(rt, kind, kernel)
    z = a @ b + bias            # (sums of at most 9 k + 3 < 2^24: exact in fp32)
    np.testing.assert_array_equal(kind.down(pre), kind.values(z))
    np.testing.assert_array_equal(kind.down(c), kind.values(np.maximum(z, 0) + res))


@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("m,n,k,kernel_a,kernel_b", GRADIENTS)
def test_gradient_tiles(rt, kind, m, n, k, kernel_a, kernel_b):
    """each product alone, and both with the column sums"""
    print("case gradients", kind.name, m, n, k, flush=True)
    rng = np.random.default_rng(m + n + k)
    dc, a, b = small_ints(rng, m, n), small_ints(rng, m, k), small_ints(rng, k, n)
    up = [kind.up(rt, x) for x in (dc, a, b)]
    want = [kind.values(x) for x in (dc @ b.T, a.T @ dc, dc.sum(0))]
    da, db, dbias = rt.empty((m, k), kind.numpy), rt.empty((k, n), kind.numpy), rt.empty((n,), kind.numpy)
    rt.matrixMatrixFCActAddGrad(*up, da=da)
    ran(rt, kind, kernel_a)
    rt.matrixMatrixFCActAddGrad(*up, db=db)
    ran(rt, kind, kernel_b)
    for got, value in zip((da, db), want):
        np.testing.assert_array_equal(kind.down(got), value)
    for got in (da, db):
        rt._check(rt.lib.swc_hip_fill_i(got.ptr, 0x7FC07FC0, got.nbytes // 4), "fill")   # (NaN in both types)
    rt.matrixMatrixFCActAddGrad(*up, da=da, db=db, dbias=dbias)
    for got, value in zip((da, db, dbias), want):
        np.testing.assert_array_equal(kind.down(got), value)


# (m, n, k, share of the rows left out, dA's kernel)
LOSSES = [(5444, 12123, 153, 0, BIG + "kk> x"), (5153, 26804, 133, 0.1, BIG + "kk> x"), (4453, 6336, 1800, 0, DEEP + "kk> x1"),
          (1999, 50257, 1024, 0.3, DEEP + "kk> x8"), (1334, 115592, 424, 0.2, DEEP + "kk> x"), (5800, 30000, 1032, 0.3, DEEP + "kk> x2"),
          (6700, 18981, 386, 0.05, ""), (1442, 6274, 5828, 0.2, DEEP + "kk> x1"), (130, 83048, 432, 0.1, ""), (130, 87408, 616, 0, ""),
          (452, 68960, 136, 0.5, ""), (36, 53070, 8, 0.1, ""), (4623, 169, 807, 0.2, ""), (2844, 3584, 67, 0, ""), (7315, 832, 2224, 0, ""),
          (5383, 42048, 384, 0, ""), (542, 8, 6679, 0.1, ""), (2165, 803, 7940, 0.2, ""), (6934, 8, 478, 0, ""), (6496, 53705, 10, 0.3, ""),
          (8535, 18072, 272, 0, ""), (4570, 550, 4494, 0.1, ""), (2209, 577, 7398, 0, ""), (7666, 206, 1669, 0.3, BIG + "kk> x1"),
          (1676, 218, 7006, 0, BIG + "kk> x1"), (1878, 1683, 37, 0.1, ""), (8598, 10923, 129, 0, ""), (429, 83988, 146, 0.1, ""),
          (6869, 3144, 720, 0.1, ""), (6329, 11568, 200, 0, ""), (5254, 182, 3203, 0, ""), (3839, 89, 5380, 0.1, ""), (113, 2824, 7095, 0, ""),
          (657, 27624, 72, 0.2, ""), (262, 87488, 200, 0, ""), (1177, 60288, 72, 0.1, ""), (909, 8472, 72, 0, ""), (1, 42770, 66, 0, "")]


class TwoValued:
    """logits of two values only, 0 for the classes that go with a row's feature and -128 for the others, so that the
    probabilities are a power of two and zero, dz and all that follows small integers.  The first k1 features choose (128 in
    one of them, against 0 or -1 in B); the others come in pairs, the same in a row of A and opposite in a column of B, and
    cancel in the logits but not in the gradients."""

    def __init__(self, m, n, k, share):
        rng = np.random.default_rng(m + n + k)
        k1 = k - k // 4 * 2
        pairs = (k - k1) // 2
        width = 256
        while width > 1 and (width > n // 2 or width > 2 * n // k1 + 1):
            width //= 2
        chosen = np.stack([rng.choice(n, width, replace=False) for _ in range(k1)])      # the classes of a feature
        b = np.empty((k, n), np.float32)
        b[:k1] = -1
        np.put_along_axis(b[:k1], chosen, 0, 1)
        b[k1::2] = rng.integers(-2, 3, (pairs, n))
        b[k1 + 1::2] = -b[k1::2]
        feature = rng.integers(0, k1, m)
        a = np.zeros((m, k), np.float32)
        a[np.arange(m), feature] = 128
        a[:, k1::2] = rng.integers(-2, 3, (m, pairs))
        a[:, k1 + 1::2] = a[:, k1::2]
        sel = np.where(rng.random(m) < 0.7, chosen[feature, rng.integers(0, width, m)], rng.integers(0, n, m)).astype(np.int32)
        out = rng.random(m) < share
        sent = a.copy()
        sent[out] = np.nan
        sel_sent = np.where(out, rng.choice([-1, n, n + 5], m), sel).astype(np.int32)
        grad = (width * rng.integers(1, 3, m)).astype(np.float32)
        self.a, self.b, self.sel, self.grad, self.width = sent, b, sel_sent, grad, width
        self.parts = (a, sel, out, chosen, feature, k1)

    def losses(self):
        """row losses, lse and their mean"""
        a, sel, out, chosen, feature, _ = self.parts
        inside = (chosen[feature] == sel[:, None]).any(1)
        row = np.log(self.width) + np.where(inside, 0.0, 128.0)
        return np.where(out, 0, row), np.where(out, 0, np.log(self.width)), row[~out].mean() if not out.all() else 0.0

    def check_losses(self, row, lse, loss):
        want = self.losses()
        # log and the subtraction of numbers below 134: some roundings of 2^-24 of them
        within(lse, want[1], 4 * U * 8, "lse")
        within(row, want[0], 4 * U * 136, "row loss")
        within(np.reshape(loss, ()), want[2], 8 * U * 136, "loss")

    def check_gradients(self, kind, *got):
        """dA, dB and dbias, every element"""
        a, sel, out, chosen, feature, k1 = self.parts
        b, width, m, n, k = self.b, self.width, self.a.shape[0], self.b.shape[1], self.b.shape[0]
        # dz = g / width at the classes of the row's feature, -g at its own (both at once where it is one of them)
        g = np.where(out, 0, self.grad).astype(np.float64)
        b64, a64 = b.astype(np.float64), np.where(out[:, None], 0, a).astype(np.float64)

        def results(a, b, minus):
            per_feature = np.stack([b[:, c].sum(1) for c in chosen])                    # [feature][k]
            da = (g / width)[:, None] * per_feature[feature] + minus * g[:, None] * b[:, sel].T
            sums, ones = np.zeros((k1, k)), np.zeros(k1)
            np.add.at(sums, feature, (g / width)[:, None] * a)
            np.add.at(ones, feature, g / width)
            db, dbias = np.zeros((n, k)), np.zeros(n)
            for i, c in enumerate(chosen):
                db[c] += sums[i]
                dbias[c] += ones[i]
            np.add.at(db, sel, minus * g[:, None] * a)
            np.add.at(dbias, sel, minus * g)
            return da, db.T, dbias

        exact = results(a64, b64, -1.0)
        if kind is BF:      # (a probability is within 2^-18 of its power of two: rounded to bfloat16, dz is exact)
            bounds = (0.0, 0.0, 0.0)
        else:               # dz within 2^-20 of its parts, and the additions of at most 2 width (m) terms that are not zero
            size = results(np.abs(a64), np.abs(b64), 1.0)
            bounds = [(2.0 ** -20 + 2 * terms * U) * x for x, terms in zip(size, (width, min(m, 4096), min(m, 4096)))]
        for name, x, value, bound in zip(("da", "db", "dbias"), got, exact, bounds):
            if kind is BF:
                np.testing.assert_array_equal(x, kind.values(value), err_msg=name)
            else:
                within(x, value, bound, name)


@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("m,n,k,share,kernel", LOSSES)
def test_loss_tiles(rt, kind, m, n, k, share, kernel):
    print("case loss", kind.name, m, n, k, share, flush=True)
    t = TwoValued(m, n, k, share)
    da_, db_, dsel = kind.up(rt, t.a), kind.up(rt, t.b), rt.upload(t.sel)
    loss, row, lse = rt.matrixFCSoftmaxWithLoss(da_, db_, None, dsel)
    t.check_losses(row.numpy(), lse.numpy(), loss.numpy())
    ga, gb, gbias = (rt.empty(s, kind.numpy) for s in ((m, k), (k, n), (n,)))
    dg = rt.upload(t.grad)
    rt.matrixFCSoftmaxWithLossGrad(da_, db_, None, dsel, lse, dg, da=ga)
    ran(rt, kind, kernel)
    alone = kind.down(ga)
    rt._check(rt.lib.swc_hip_fill_i(ga.ptr, 0x7FC07FC0, ga.nbytes // 4), "fill")
    rt.matrixFCSoftmaxWithLossGrad(da_, db_, None, dsel, lse, dg, da=ga, db=gb, dbias=gbias)
    t.check_gradients(kind, kind.down(ga), kind.down(gb), kind.down(gbias))
    np.testing.assert_array_equal(alone, kind.down(ga))


@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("m,n", [(15, 70), (16, 20000), (17, 900), (17, 5000), (64, 1000), (64, 4200), (65, 300), (255, 3000), (257, 3000)])
def test_few_rows_of_a_loss(rt, kind, m, n):
    """next to where the row statistics' joining and the column sums change their way; a third of the rows left out"""
    print("case few rows", kind.name, m, n, flush=True)
    t = TwoValued(m, n, 40, 0.33)
    a, b, sel = kind.up(rt, t.a), kind.up(rt, t.b), rt.upload(t.sel)
    loss, row, lse = rt.matrixFCSoftmaxWithLoss(a, b, kind.up(rt, np.zeros(n)), sel)
    t.check_losses(row.numpy(), lse.numpy(), loss.numpy())
    da, db, dbias = rt.matrixFCSoftmaxWithLossGrad(a, b, None, sel, lse, rt.upload(t.grad))
    t.check_gradients(kind, kind.down(da), kind.down(db), kind.down(dbias))


@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("pad,first", [(8, 8), (3, 1)])
@pytest.mark.parametrize("m,n,k,share", [(1, 300, 40, 0), (33, 200, 136, 0.2), (300, 1000, 75, 0.3), (700, 2050, 130, 0.1), (4200, 301, 66, 0.3)])
def test_loss_strides_exactly(rt, kind, pad, first, m, n, k, share):
    """operands and gradients in longer rows, off the 16-byte grid, with row gradients, a bias and rows left out: every element,
    and nothing beside the rows"""
    print("case loss strides", kind.name, pad, first, m, n, k, flush=True)
    t = TwoValued(m, n, k, share)
    _da, pa = strided(rt, kind, t.a, k + pad, first)
    _db, pb = strided(rt, kind, t.b, n + pad, first)
    sel, g, bias = rt.upload(t.sel), rt.upload(t.grad), kind.up(rt, np.zeros(n))
    row, lse, loss = rt.empty((m,)), rt.empty((m,)), rt.empty((1,))
    call = lambda name: getattr(rt.lib, "swc_hip_matrixFCSoftmaxWithLoss" + name + kind.suffix())   # noqa: E731
    rt._check(call("")(m, n, k, pa, k + pad, pb, n + pad, bias.ptr, sel.ptr, row.ptr, lse.ptr, loss.ptr), "loss")
    t.check_losses(row.numpy(), lse.numpy(), loss.numpy())
    ga, pga = strided(rt, kind, np.zeros((m, k)), k + 2 * pad, first)
    gb, pgb = strided(rt, kind, np.zeros((k, n)), n + pad, first)
    gbias = rt.empty((n,), kind.numpy)
    rt._check(call("Grad")(m, n, k, pa, k + pad, pb, n + pad, bias.ptr, sel.ptr, lse.ptr, g.ptr, pga, k + 2 * pad, pgb, n + pad,
                           gbias.ptr), "grad")
    (ia, sa, ba), (ib, sb, bb) = rows_of(kind, ga, m, k, k + 2 * pad, first), rows_of(kind, gb, k, n, n + pad, first)
    t.check_gradients(kind, ia, ib, kind.down(gbias))
    for x in (sa, ba, sb, bb):
        assert np.all(np.isnan(x))


@gpu
@pytest.mark.parametrize("kind", KINDS)
def test_empty_operands_through_the_binding(rt, kind):
    """no rows, no columns, no contraction: sums of nothing are zero, and nothing else is written"""
    e = lambda *s: rt.empty(s, kind.numpy)   # noqa: E731
    full = lambda *s: kind.up(rt, np.full(s, 7))   # noqa: E731
    zero = lambda d: np.all(kind.down(d) == 0)   # noqa: E731
    assert rt.matrixMatrixFCActAdd(e(0, 8), full(8, 16), full(16), "gelu").shape == (0, 16)
    assert rt.matrixMatrixFCActAdd(full(5, 8), e(8, 0), e(0), "gelu").shape == (5, 0)
    c, z = full(5, 16), full(5, 16)
    rt.matrixMatrixFCActAdd(e(5, 0), e(0, 16), None, "none", full(5, 16), z, c)
    assert zero(z) and np.all(kind.down(c) == 7)
    _, db, dbias = rt.matrixMatrixFCActAddGrad(e(0, 16), e(0, 8), full(8, 16), e(0, 16), "silu")
    assert zero(db) and zero(dbias)
    da, _, _ = rt.matrixMatrixFCActAddGrad(e(5, 0), full(5, 8), e(8, 0), e(5, 0), "silu")
    assert zero(da)
    _, _, dbias = rt.matrixMatrixFCActAddGrad(full(5, 16), e(5, 0), e(0, 16))
    assert np.all(kind.down(dbias) == 35)
    loss, row, lse = rt.matrixFCSoftmaxWithLoss(e(0, 8), full(8, 16), None, rt.empty((0,), np.int32))
    assert loss.numpy() == 0 and row.shape == lse.shape == (0,)
    _, db, dbias = rt.matrixFCSoftmaxWithLossGrad(e(0, 8), full(8, 16), None, rt.empty((0,), np.int32), rt.empty((0,)))
    assert zero(db) and zero(dbias)
    loss, row, lse = rt.matrixFCSoftmaxWithLoss(full(5, 8), e(8, 0), None, rt.upload(np.zeros(5, np.int32)))
    assert loss.numpy() == 0 and np.all(row.numpy() == 0) and np.all(lse.numpy() == 0)


# -------------------------------------------------------------------------------------------------- values of ReLU
@gpu
@pytest.mark.parametrize("kind", KINDS)
def test_an_inactive_relu_passes_nothing_on(rt, kind):
    """infinities and NaN in the gradient at inactive units (also at a NaN argument) reach nothing, as in reluGrad_f; at an
    active unit they reach its row of dA, its column of dB and its element of dbias, and nothing else"""
    rng = np.random.default_rng(1)
    m, n, k = 75, 200, 136
    dc, a, b, pre = small_ints(rng, m, n), small_ints(rng, m, k), small_ints(rng, k, n), small_ints(rng, m, n)
    a[a == 0], b[b == 0] = 1, 1
    pre[:, 0] = [-1, 0, -0.0] * 25
    pre[7, 3] = np.nan
    off = ~(pre > 0)
    clean = np.where(off, 0, dc).astype(np.float64)
    dc[off] = rng.choice(np.array([np.inf, -np.inf, np.nan, 2], np.float32), off.sum())
    run = lambda: [kind.down(x) for x in rt.matrixMatrixFCActAddGrad(kind.up(rt, dc), kind.up(rt, a), kind.up(rt, b),   # noqa: E731
                                                                      kind.up(rt, pre), "relu")]
    da, db, dbias = run()
    np.testing.assert_array_equal(da, kind.values(clean @ b.T))
    np.testing.assert_array_equal(db, kind.values(a.T @ clean))
    np.testing.assert_array_equal(dbias, kind.values(clean.sum(0)))
    if kind is F32:   # the operator of its own says the same
        np.testing.assert_array_equal(rt.reluGrad(rt.upload(pre), rt.upload(dc)).numpy(), clean)
    row, col = 30, 90
    pre[row, col], dc[row, col], clean[row, col] = 2, np.nan, 0
    da, db, dbias = run()
    assert np.all(np.isnan(da[row])) and np.all(np.isnan(db[:, col])) and np.isnan(dbias[col])
    np.testing.assert_array_equal(np.delete(da, row, 0), np.delete(kind.values(clean @ b.T), row, 0))
    np.testing.assert_array_equal(np.delete(db, col, 1), np.delete(kind.values(a.T @ clean), col, 1))
