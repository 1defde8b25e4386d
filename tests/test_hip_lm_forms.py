"""Operators of language models: forms, sizes and values beside the ones that test_hip_lm_ops.py takes (whose helpers and
tolerances hold here too)."""
import numpy as np
import pytest

from tests.test_hip_lm_ops import BF, F32, KINDS, small_ints

gpu = pytest.mark.gpu


@pytest.fixture(scope="module")
def rt():
    from swcompiler_amd.hip import runtime
    return runtime()


# ------------------------------------------------------------------------------------------------------- gradients
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
