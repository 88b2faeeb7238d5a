"""so_layer_norm on columns at the ends of the element types: columns without variance.

Statistics and results are those of test_gpu_layer_norm.py, with its tolerances; a column of one value has that value as its mean and no deviation in any order of its sums, so its results are exact."""
import numpy as np
import pytest

from elements import fetch, place
from test_gpu_layer_norm import EPS

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
