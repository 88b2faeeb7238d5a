"""4-bit products beyond test_gpu_mxfp4.py: blocks that are not numbers through every activation."""
import numpy as np
import pytest

import mx_reference as mx
from elements import TYPES, fetch, place, stored, values
from test_gpu_mxfp4 import FORMS, activated, product_tolerance

pytestmark = pytest.mark.gpu

ACTS = ["none", "relu", "sigmoid", "tanh"]


def handle_of(ctx, codes, scales, n):
    W = ctx.mxfp4(ctx.array(codes, np.uint8), ctx.array(scales, np.uint8), codes.shape[0], n)
    return W, mx.dequantize(codes, scales, n)


def quantized(X):
    return mx.dequantize(*mx.quantize(np.ascontiguousarray(X.T)), X.shape[0]).T


@pytest.mark.parametrize("form", range(1, len(FORMS) + 1))
@pytest.mark.parametrize("act", ACTS)
def test_not_a_number_through_every_activation(ctx, act, form):
    """A block of W that is not a number makes its row of Y NaN, one of X its column, after the activation too; all else is as it would be."""
    rng = np.random.default_rng(40 + form)
    m, n, C = 70, 500, 45
    codes, scales = mx.quantize(rng.standard_normal((m, n)) / np.sqrt(n))
    scales[11, 3] = scales[69, 15] = 255
    handle, W = handle_of(ctx, codes, scales, n)
    bias = rng.standard_normal(m).astype(np.float32)
    for type_ in TYPES:
        X = values(stored(rng.standard_normal((n, C)), type_), type_)
        X[499, 7], X[0, 44], X[33, 20] = np.nan, np.inf, -np.inf
        bad = np.zeros((m, C), bool)
        bad[[11, 69]], bad[:, [7, 20, 44]] = True, True
        whole, dX = place(ctx, X, type_, 3, 1)
        out, dY = place(ctx, np.zeros((m, C)), type_, 1, 0, fill=-5.0)
        dB = ctx.array(bias)
        with ctx.tuning(SPARSEOPS_MXFP4_MATMUL=form):
            ctx.mxfp4_matmul(handle, dX, C, dB, dY, act, type=type_, x_stride=C + 3, y_stride=C + 1)
        Y, rest = fetch(out, m, C, type_, 1, 0)
        assert np.array_equal(np.isnan(Y), bad)
        assert np.all(rest == -5.0), "places that are not the result's were written"
        Wf, Xf = np.where(bad.all(axis=1)[:, None], 0.0, W), np.where(bad.all(axis=0), 0.0, X)
        Xq = quantized(Xf)
        want = activated(Wf @ Xq + bias.astype(np.float64)[:, None], act)
        assert np.all((np.abs(Y - want) <= product_tolerance(Wf, Xq, bias, want, act, type_)) | bad)
        for a in (whole, out, dB):
            a.free()
    handle.free()
