"""so_layer_norm on columns at the ends of the element types: infinities wherever they stand, values whose squares fp32 does not hold, columns without variance.

Statistics and results are those of test_gpu_layer_norm.py, with its tolerances; a column of one value has that value as its mean and no deviation in any order of its sums, so its results are exact."""
import numpy as np
import pytest

import hipabi
from elements import HALF_STEP, SMALLEST, STORAGE, TYPES, U, fetch, place, stored, values
from test_gpu_layer_norm import EPS, check_forward, check_grad, check_statistics, problem, statistics

pytestmark = pytest.mark.gpu

LANES = [-1, 0, 1, 2, 4, 8]          # as the library chooses, in parts, and the lanes a row of the one launch


def forward(ctx, X, gamma, beta, type_, lanes):
    F, B = X.shape
    whole, dX = place(ctx, X, type_, 1, 0)
    out, dY = place(ctx, np.zeros((F, B)), type_, 2, 1, fill=-5.0)
    dG, dB, dM, dR = ctx.array(gamma), ctx.array(beta), ctx.empty((B,)), ctx.empty((B,))
    with ctx.tuning(SPARSEOPS_NORM_LANES=lanes):
        ctx.layer_norm(dX, F, B, dG, dB, EPS, dY, dM, dR, type=type_, x_stride=B + 1, y_stride=B + 2)
    Y, rest = fetch(out, F, B, type_, 2, 1)
    assert np.all(rest == -5.0), "places that are not the result's were written"
    mean, rstd = dM.download().copy(), dR.download().copy()
    for a in (whole, out, dG, dB, dM, dR):
        a.free()
    return Y, mean, rstd


@pytest.mark.parametrize("lanes", LANES)
@pytest.mark.parametrize("B", [1, 5, 40])
def test_columns_of_one_value(ctx, B, lanes):
    """Whatever number of rows a wave or a part has: the mean is the value, no deviation is left, so the results are beta."""
    for F in list(range(1, 70)) + list(range(81, 1100, 97)) + [5000, 8192]:
        beta = np.linspace(-1, 1, F).astype(np.float32)
        X = np.full((F, B), 1000.1, np.float32).astype(np.float64)
        Y, mean, _ = forward(ctx, X, np.ones(F, np.float32), beta, "f32", lanes)
        assert np.array_equal(mean, X[0]), (F, mean)
        assert np.array_equal(Y, np.tile(beta.astype(np.float64)[:, None], (1, B))), F


@pytest.mark.parametrize("B", [1, 5, 40])
def test_columns_of_one_value_in_parts(ctx, B):
    """Whatever number of rows the last part has: no deviation, so the results are beta."""
    for rows in list(range(1, 40)) + list(range(47, 1024, 61)):
        F = 8192 + rows
        beta = np.linspace(-1, 1, F).astype(np.float32)
        X = np.full((F, B), 1000.1, np.float32)
        Y, mean, _ = forward(ctx, X, np.ones(F, np.float32), beta, "f32", -1)
        assert np.array_equal(mean, X[0]), (rows, mean)
        assert np.array_equal(Y, np.tile(beta.astype(np.float64)[:, None], (1, B))), rows


@pytest.mark.parametrize("lanes", LANES)
@pytest.mark.parametrize("type_", ["f32", "bf16"])
@pytest.mark.parametrize("F", [1, 3, 70, 1000, 9000])
def test_values_whose_squares_fp32_does_not_hold(ctx, F, type_, lanes):
    """Columns of one value of 2^64 .. 2^120 have no variance: the results are beta, the statistics the value and 1 / sqrt(eps)."""
    B = 13
    _, _, gamma, beta = problem(F, B, type_)
    value = np.exp2(np.linspace(64, 120, B).round()) * np.where(np.arange(B) % 2, -1.0, 1.0)
    X = np.tile(value, (F, 1))
    Y, mean, rstd = forward(ctx, X, gamma, beta, type_, lanes)
    assert np.array_equal(Y, np.tile(values(stored(beta, type_), type_)[:, None], (1, B)))
    assert np.array_equal(mean.astype(np.float64), value)
    want = 1.0 / np.sqrt(np.float64(np.float32(EPS)))
    assert np.all(np.abs(rstd - want) <= want * 4 * U)          # a root and a quotient


@pytest.mark.parametrize("lanes", LANES)
@pytest.mark.parametrize("type_", ["f32", "bf16"])
@pytest.mark.parametrize("F", [1, 3, 33, 70])
def test_large_values_that_differ(ctx, F, type_, lanes):
    """A mean of 2^66, whose square fp32 does not hold, and deviations of 2^59, the sum of whose squares it does."""
    rng, _, gamma, beta = problem(F, 11, type_)
    X = values(stored(2.0 ** 66 + 2.0 ** 59 * rng.uniform(-2, 2, (F, 11)), type_), type_)
    Y, mean, rstd = forward(ctx, X, gamma, beta, type_, lanes)
    check_forward(Y, X, gamma, beta, type_)
    check_statistics(mean, rstd, X)


@pytest.mark.parametrize("type_", ["f32", "bf16"])
@pytest.mark.parametrize("F,B", [(3, 5), (70, 11), (1100, 40)])
def test_gradient_of_large_values(ctx, F, B, type_):
    """The gradient at such columns: one workgroup's, and in parts."""
    rng, _, gamma, _ = problem(F, B, type_)
    X = values(stored(2.0 ** 66 + 2.0 ** 58 * rng.uniform(-2, 2, (F, B)), type_), type_)
    dY = values(stored(rng.standard_normal((F, B)), type_), type_)
    mean, rstd = (s.astype(np.float32) for s in statistics(X))
    dX, dDy, dDx = (place(ctx, M, type_)[0] for M in (X, dY, np.zeros((F, B))))
    dG, dM, dR, dDg, dDb = ctx.array(gamma), ctx.array(mean), ctx.array(rstd), ctx.empty((F,)), ctx.empty((F,))
    ctx.layer_norm_grad(dX, dDy, F, B, dG, dM, dR, dDx, dDg, dDb, type=type_)
    check_grad(fetch(dDx, F, B, type_)[0], dDg.download(), dDb.download(), X, dY, gamma, mean, rstd, type_)
    for a in (dX, dDy, dDx, dG, dM, dR, dDg, dDb):
        a.free()


@pytest.mark.parametrize("lanes", LANES)
@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("F", [1, 2, 3, 65, 200, 2000, 9000])
def test_not_finite_wherever_it_stands(ctx, F, type_, lanes):
    """One infinity or NaN in a column, in its first, its second, its last or some other row, or several: results and statistics of that column are NaN, the others keep theirs."""
    B = 23
    rng, X, gamma, beta = problem(F, B, type_, seed=11)
    bad = list(range(1, B, 2))
    for i, b in enumerate(bad):
        row = (0, min(1, F - 1), F - 1, int(rng.integers(F)))[i % 4]
        X[row, b] = (np.inf, -np.inf, np.nan)[i % 3]
        if i == len(bad) - 1:
            X[:, b] = np.inf
        if i == len(bad) - 2:
            X[:, b] = np.where(np.arange(F) % 2, np.inf, -np.inf)
    good = [b for b in range(B) if b not in bad]
    Y, mean, rstd = forward(ctx, X, gamma, beta, type_, lanes)
    assert np.isnan(Y[:, bad]).all()
    assert np.isnan(mean[bad]).all(), mean[bad]
    assert np.isnan(rstd[bad]).all(), rstd[bad]
    check_forward(Y[:, good], X[:, good], gamma, beta, type_)
    check_statistics(mean[good], rstd[good], X[:, good])


def test_forced_tiles_that_a_launch_does_not_hold(ctx):
    """2^28 columns are 2^26 workgroups at one lane a row, more threads than a launch has: refused ahead of any work."""
    a = ctx.empty((64,))
    with ctx.tuning(SPARSEOPS_NORM_LANES=1):
        with pytest.raises(hipabi.SoError, match="too large for one launch") as e:
            ctx.layer_norm(a, 1, 1 << 28, None, None, EPS, a)
    assert e.value.status == hipabi.SO_ERR_INVALID
    a.free()


@pytest.mark.parametrize("type_", ["f32", "bf16"])
@pytest.mark.parametrize("F,B", [(300000, 33), (100352, 8), (1000003, 1), (1 << 18, 200)])
def test_very_many_features(ctx, F, B, type_):
    """The features of whole images.  A column's parts are 1024 / lanes rows; 256 / columns threads join up to 48 of them each, one after the other, and one thread what these have, first in
    groups where there are more: so many additions more than test_gpu_layer_norm.py counts, up to the 48 that stand for all there."""
    V = 4 if type_ == "f32" else 8
    lanes = 8 if B > 4 * V else 4 if B > 2 * V else 2 if B > V else 1
    shares, parts, more = 256 // (lanes * V), -(-F * lanes // 1024), 0
    while parts > 48 * shares:
        parts, more = -(-parts // (48 * shares)), more + 48 + shares
    more += 48 + shares
    rng, X, gamma, beta = problem(F, B, type_, seed=5)
    dY = values(stored(0.1 * rng.standard_normal((F, B)), type_), type_)
    dX, dDy, out, dDx = (place(ctx, M, type_)[0] for M in (X, dY, np.zeros((F, B)), np.zeros((F, B))))
    dG, dB, dM, dR, dDg, dDb = ctx.array(gamma), ctx.array(beta), ctx.empty((B,)), ctx.empty((B,)), ctx.empty((F,)), ctx.empty((F,))
    ctx.layer_norm(dX, F, B, dG, dB, EPS, out, dM, dR, type=type_)
    ctx.layer_norm_grad(dX, dDy, F, B, dG, dM, dR, dDx, dDg, dDb, type=type_)
    mean, rstd = statistics(X)
    h = (X - mean) * rstd
    n = (48 + more) * U
    off = n * np.abs(X).max(axis=0)
    g_mean, g_rstd = dM.download().astype(np.float64), dR.download().astype(np.float64)
    assert np.all(np.abs(g_mean - mean) <= off)
    assert np.all(np.abs(g_rstd - rstd) <= rstd * (n + np.square(off * rstd)))
    g = gamma.astype(np.float64)[:, None]
    want = h * g + beta.astype(np.float64)[:, None]
    tol = n * (np.abs(X).max(axis=0) * rstd * np.abs(g) + np.abs(h * g)) + 2 * U * np.abs(want) + HALF_STEP[type_] * np.abs(want) + SMALLEST[type_]
    assert np.all(np.abs(fetch(out, F, B, type_)[0] - want) <= tol)
    h = (X - g_mean) * g_rstd
    dyg = dY * g
    a, b = dyg.mean(axis=0), (dyg * h).mean(axis=0)
    want = g_rstd * (dyg - a - h * b)
    tol = g_rstd * (n * (np.abs(dyg).mean(axis=0) + np.abs(h) * np.abs(dyg * h).mean(axis=0)) + 8 * U * (np.abs(dyg) + np.abs(a) + np.abs(h * b))) + HALF_STEP[type_] * np.abs(want) + SMALLEST[type_]
    assert np.all(np.abs(fetch(dDx, F, B, type_)[0] - want) <= tol)
    assert np.all(np.abs(dDg.download() - (dY * h).sum(axis=1)) <= 48 * U * np.abs(dY * h).sum(axis=1) + 1e-40)
    assert np.all(np.abs(dDb.download() - dY.sum(axis=1)) <= 48 * U * np.abs(dY).sum(axis=1) + 1e-40)
    for t in (dX, dDy, out, dDx, dG, dB, dM, dR, dDg, dDb):
        t.free()


@pytest.mark.parametrize("gradient", [False, True])
def test_time_grows_as_the_features_do(ctx, gradient):
    """Four times the features take about four times as long: what a workgroup joins does not grow with them, which would make it sixteen times."""
    B, times = 32, []
    for F in (1 << 20, 1 << 22):
        dX, dM, dR, dDg = ctx.empty((F, B)), ctx.empty((B,)), ctx.empty((B,)), ctx.empty((F,))
        for a in (dX, dM, dR):
            ctx.fill_zero(a)
        took = []
        for _ in range(4):
            ctx.timer_begin()
            if gradient:
                ctx.layer_norm_grad(dX, dX, F, B, None, dM, dR, dX, dDg, None)
            else:
                ctx.layer_norm(dX, F, B, None, None, EPS, dX, dM, dR)
            took.append(ctx.timer_end())
        times.append(min(took))
        for a in (dX, dM, dR, dDg):
            a.free()
    assert times[1] <= 8 * times[0], times


@pytest.mark.parametrize("lanes", LANES)
@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("F,B", [(257, 40), (2000, 64), (4096, 700), (8192, 33)])
def test_one_feature_that_carries_a_column(ctx, F, B, type_, lanes):
    """A value of 10 to 30000 in one of the first rows or another, beside normal values or zeros: its squares are not taken off each other, so the tolerances are those of any column."""
    rng, _, gamma, beta = problem(F, B, type_)
    for quiet in (0.0, 1e-3, 1.0):
        X = quiet * rng.standard_normal((F, B))
        row = rng.integers(0, F, B)
        row[::2] = rng.integers(0, min(F, 64), row[::2].size)
        X[row, np.arange(B)] = 10 ** rng.uniform(1, 4.4, B)
        X = values(stored(X, type_), type_)
        Y, mean, rstd = forward(ctx, X, gamma, beta, type_, lanes)
        check_statistics(mean, rstd, X)
        check_forward(Y, X, gamma, beta, type_)


@pytest.mark.parametrize("type_,F,B", [("f32", 3300007, 1), ("bf16", 1700003, 5), ("f32", 900001, 7), ("f32", 210001, 12), ("f16", 4800011, 33)])
def test_groups_of_parts(ctx, type_, F, B):
    """Groups of parts for every number of columns a tile, the last two times over (37501 parts, 196 groups of 192, 2): rows that repeat every 1009, whose statistics are those of so many times
    each.  Tolerances as in test_very_many_features, of 2 (48 + 64) additions and the 48 there."""
    P = 1009
    rng = np.random.default_rng(F)
    base = values(stored(rng.standard_normal((P, B)) + 0.5, type_), type_)
    often = np.bincount(np.arange(F) % P, minlength=P).astype(np.float64)[:, None]
    whole = np.arange(F) % P
    gamma, dY = (1 + 0.2 * rng.standard_normal(P)).astype(np.float32), values(stored(0.1 * rng.standard_normal((P, B)), type_), type_)
    dX, dDy = ctx.array(stored(base, type_)[whole], STORAGE[type_]), ctx.array(stored(dY, type_)[whole], STORAGE[type_])
    out, dDx = ctx.empty((F, B), STORAGE[type_]), ctx.empty((F, B), STORAGE[type_])
    dG, dM, dR, dDg, dDb = ctx.array(gamma[whole]), ctx.empty((B,)), ctx.empty((B,)), ctx.empty((F,)), ctx.empty((F,))
    ctx.layer_norm(dX, F, B, dG, None, EPS, out, dM, dR, type=type_)
    ctx.layer_norm_grad(dX, dDy, F, B, dG, dM, dR, dDx, dDg, dDb, type=type_)
    n = U * (48 + 2 * (48 + 64))
    mean = (base * often).sum(axis=0) / F
    rstd = 1.0 / np.sqrt((np.square(base - mean) * often).sum(axis=0) / F + np.float64(np.float32(EPS)))
    off = n * np.abs(base).max(axis=0)
    g_mean, g_rstd = dM.download().astype(np.float64), dR.download().astype(np.float64)
    assert np.all(np.abs(g_mean - mean) <= off)
    assert np.all(np.abs(g_rstd - rstd) <= rstd * (n + np.square(off * rstd)))

    def check(array, want, tol):
        """A row of every repetition, most of them taken together: the largest and the smallest of each."""
        got = values(array.download(), type_) if array.shape == (F, B) else array.download().astype(np.float64).reshape(F, 1)
        low, high = got[:P].copy(), got[:P].copy()
        for at in range(P, F, P):
            part = got[at:at + P]
            np.minimum(low[:len(part)], part, out=low[:len(part)])
            np.maximum(high[:len(part)], part, out=high[:len(part)])
        assert np.all(np.abs(low - want) <= tol) and np.all(np.abs(high - want) <= tol)

    h, g = (base - mean) * rstd, gamma.astype(np.float64)[:, None]
    check(out, h * g, n * (np.abs(base).max(axis=0) * rstd * np.abs(g) + np.abs(h * g)) + (2 * U + HALF_STEP[type_]) * np.abs(h * g) + SMALLEST[type_])
    h = (base - g_mean) * g_rstd
    dyg = dY * g
    a, b = (dyg * often).sum(axis=0) / F, (dyg * h * often).sum(axis=0) / F
    want = g_rstd * (dyg - a - h * b)
    mags = (np.abs(dyg) * often).sum(axis=0) / F + np.abs(h) * (np.abs(dyg * h) * often).sum(axis=0) / F
    check(dDx, want, g_rstd * (n * mags + 8 * U * (np.abs(dyg) + np.abs(a) + np.abs(h * b))) + HALF_STEP[type_] * np.abs(want) + SMALLEST[type_])
    check(dDg, (dY * h).sum(axis=1, keepdims=True), 48 * U * np.abs(dY * h).sum(axis=1, keepdims=True) + 1e-40)
    check(dDb, dY.sum(axis=1, keepdims=True), 48 * U * np.abs(dY).sum(axis=1, keepdims=True) + 1e-40)
    for t in (dX, dDy, out, dDx, dG, dM, dR, dDg, dDb):
        t.free()
