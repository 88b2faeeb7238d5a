"""Calls of the layer norm and the 4-bit operators that their documentation allows, in combinations: arguments left out, in place inside longer rows, arrays at any byte, one call's result
as the next one's input without a wait between them.  Results are those of test_gpu_layer_norm.py and test_gpu_mxfp4.py, with their tolerances."""
import ctypes as ct
import itertools

import numpy as np
import pytest

import hipabi
import mx_reference as mx
from elements import TYPES, fetch, place, stored, values
from test_gpu_layer_norm import EPS, check_forward, check_grad, check_statistics, problem, statistics
from test_gpu_mxfp4 import product_tolerance, weights

pytestmark = pytest.mark.gpu

# one workgroup, all features in one of several, in parts
SIZES = [(60, 3), (300, 40), (300, 9001), (2049, 65)]


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("F,B", SIZES)
def test_forward_with_arguments_left_out(ctx, F, B, type_):
    _, X, gamma, beta = problem(F, B, type_, seed=21)
    dX, out = place(ctx, X, type_)[0], place(ctx, np.zeros((F, B)), type_)[0]
    dG, dB = ctx.array(gamma), ctx.array(beta)
    for g, b, m, r in itertools.product((False, True), repeat=4):
        dM, dR = ctx.array(np.full(B, -5.0, np.float32)), ctx.array(np.full(B, -5.0, np.float32))
        ctx.layer_norm(dX, F, B, dG if g else None, dB if b else None, EPS, out, dM if m else None, dR if r else None, type=type_)
        check_forward(fetch(out, F, B, type_)[0], X, gamma if g else np.ones(F, np.float32), beta if b else np.zeros(F, np.float32), type_)
        mean, rstd = statistics(X)
        check_statistics(dM.download() if m else mean, dR.download() if r else rstd, X)
        assert m or np.all(dM.download() == -5.0)
        assert r or np.all(dR.download() == -5.0)
        dM.free()
        dR.free()
    for a in (dX, out, dG, dB):
        a.free()


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("F,B", SIZES)
def test_gradient_with_arguments_left_out(ctx, F, B, type_):
    rng, X, gamma, _ = problem(F, B, type_, seed=22)
    dY = values(stored(0.1 * rng.standard_normal((F, B)), type_), type_)
    mean, rstd = (s.astype(np.float32) for s in statistics(X))
    dX, dDy, out = (place(ctx, M, type_)[0] for M in (X, dY, np.zeros((F, B))))
    dG, dM, dR = ctx.array(gamma), ctx.array(mean), ctx.array(rstd)
    for g, x, dg, db in itertools.product((False, True), repeat=4):
        dDg, dDb = ctx.array(np.full(F, -5.0, np.float32)), ctx.array(np.full(F, -5.0, np.float32))
        out.upload(stored(np.full((F, B), -5.0), type_).reshape(out.shape))
        ctx.layer_norm_grad(dX, dDy, F, B, dG if g else None, dM, dR, out if x else None, dDg if dg else None, dDb if db else None, type=type_)
        got = fetch(out, F, B, type_)[0]
        check_grad(got if x else None, dDg.download() if dg else None, dDb.download() if db else None, X, dY, gamma if g else np.ones(F, np.float32), mean, rstd, type_)
        assert x or np.all(got == -5.0)
        assert dg or np.all(dDg.download() == -5.0)
        assert db or np.all(dDb.download() == -5.0)
        dDg.free()
        dDb.free()
    for a in (dX, dDy, out, dG, dM, dR):
        a.free()


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("F,B", SIZES + [(1, 70), (3, 33), (4000, 130), (9000, 20)])
def test_in_place_inside_longer_rows(ctx, F, B, type_):
    """A row's last columns are read together with the places behind them, which other workgroups may be writing."""
    rng, X, gamma, beta = problem(F, B, type_, seed=23)
    dY = values(stored(0.1 * rng.standard_normal((F, B)), type_), type_)
    dG, dB = ctx.array(gamma), ctx.array(beta)
    mean, rstd = (s.astype(np.float32) for s in statistics(X))
    dM, dR, dDg, dDb = ctx.array(mean), ctx.array(rstd), ctx.empty((F,)), ctx.empty((F,))
    for pad, shift in ((0, 0), (1, 1), (5, 2)):
        whole, dX = place(ctx, X, type_, pad, shift, fill=-5.0)
        ctx.layer_norm(dX, F, B, dG, dB, EPS, dX, type=type_, x_stride=B + pad, y_stride=B + pad)
        Y, rest = fetch(whole, F, B, type_, pad, shift)
        check_forward(Y, X, gamma, beta, type_)
        assert np.all(rest == -5.0)
        whole.free()
        for target in range(2):
            whole, dX = place(ctx, X, type_, pad, shift, fill=-5.0)
            whole2, dDy = place(ctx, dY, type_, pad, shift, fill=-5.0)
            ctx.layer_norm_grad(dX, dDy, F, B, dG, dM, dR, (dX, dDy)[target], dDg, dDb, type=type_, x_stride=B + pad, dy_stride=B + pad, dx_stride=B + pad)
            got, rest = fetch((whole, whole2)[target], F, B, type_, pad, shift)
            check_grad(got, dDg.download(), dDb.download(), X, dY, gamma, mean, rstd, type_)
            kept, rest2 = fetch((whole2, whole)[target], F, B, type_, pad, shift)
            assert np.array_equal(kept, (dY, X)[target]) and np.all(rest == -5.0) and np.all(rest2 == -5.0)
            whole.free()
            whole2.free()
    for a in (dG, dB, dM, dR, dDg, dDb):
        a.free()


@pytest.mark.parametrize("shift", [1, 2, 3, 7])
def test_scales_at_any_byte(ctx, shift):
    rng = np.random.default_rng(shift)
    rows, cols = 37, 333
    X = rng.standard_normal((rows, cols)).astype(np.float32)
    codes, scales = mx.quantize(X.astype(np.float64))
    dX, dC, held, dY = ctx.array(X), ctx.empty(codes.shape, np.uint8), ctx.array(np.full(scales.size + 16, 9, np.uint8), np.uint8), ctx.empty((rows, cols))
    dS = held.offset(shift)
    ctx.mxfp4_quantize(dX, rows, cols, dC, dS)
    got = held.download()
    assert np.array_equal(dC.download(), codes) and np.array_equal(got[shift:shift + scales.size], scales.ravel())
    assert np.all(got[:shift] == 9) and np.all(got[shift + scales.size:] == 9)
    ctx.mxfp4_dequantize(dC, dS, rows, cols, dY)
    want = mx.dequantize(codes, scales, cols)
    assert np.array_equal(dY.download(), want.astype(np.float32))
    W = ctx.mxfp4(dC, dS, rows, cols)
    x = rng.standard_normal(cols).astype(np.float32)
    dy = ctx.empty((rows,))
    ctx.mxfp4_matvec(W, ctx.array(x), None, dy)
    assert np.all(np.abs(dy.download() - want @ x) <= 2.0 ** -24 * 80 * (np.abs(want) @ np.abs(x)))
    W.free()


@pytest.mark.parametrize("type_", TYPES)
def test_from_values_to_a_product_without_a_wait(ctx, type_):
    """Quantised, laid out and multiplied, the codes overwritten as soon as the handle is there."""
    rng = np.random.default_rng(31)
    m, n, C = 500, 1100, 130
    Wv = values(stored(rng.standard_normal((m, n)) / np.sqrt(n), type_), type_)
    codes, scales = mx.quantize(Wv)
    dW, dC, dS = place(ctx, Wv, type_)[0], ctx.empty(codes.shape, np.uint8), ctx.empty(scales.shape, np.uint8)
    X = values(stored(rng.standard_normal((n, C)), type_), type_)
    dX, dY = place(ctx, X, type_)[0], place(ctx, np.zeros((m, C)), type_)[0]
    ctx.mxfp4_quantize(dW, m, n, dC, dS, type=type_)
    handle = ctx.mxfp4(dC, dS, m, n)
    ctx.fill_zero(dC)
    ctx.mxfp4_matmul(handle, dX, C, None, dY, type=type_)
    W, Xq = mx.dequantize(codes, scales, n), mx.dequantize(*mx.quantize(np.ascontiguousarray(X.T)), n).T
    want = W @ Xq
    assert np.all(np.abs(fetch(dY, m, C, type_)[0] - want) <= product_tolerance(W, Xq, None, want, "none", type_))
    rows, cols = ct.c_uint32(), ct.c_uint32()
    assert ctx.lib.so_mxfp4_dims(handle.h, ct.byref(rows), ct.byref(cols)) == hipabi.SO_OK and (rows.value, cols.value) == (m, n)
    assert ctx.lib.so_mxfp4_dims(handle.h, None, None) == hipabi.SO_OK
    handle.free()
    for a in (dW, dC, dS, dX, dY):
        a.free()


def test_both_operators_and_sparse_products_share_a_workspace(ctx):
    """Sums of a layer norm in parts, codes of a product's input and the sparse product's own use of the context's workspace, one behind the other, twice with the same bits."""
    rng = np.random.default_rng(17)
    m, n, C = 2048, 2048, 40
    dense = rng.standard_normal((m, n)).astype(np.float32) * (rng.random((m, n)) < 0.1)
    nnz = (dense != 0).sum(axis=1).astype(np.uint32)
    r = int(nnz.max())
    Wd, idx = np.zeros((m, r), np.float32), np.zeros((m, r), np.uint32)
    for i in range(m):
        at = np.flatnonzero(dense[i])
        Wd[i, :at.size], idx[i, :at.size] = dense[i, at], at
    E = ctx.upload_ellpack(Wd, idx, nnz, m, n, r, hipabi.LAYOUT_ROW | hipabi.LAYOUT_RBM)
    handle, W = weights(ctx, rng, m, n)
    X = rng.standard_normal((n, C)).astype(np.float32)
    dX, dN, dS, dM = ctx.array(X), ctx.empty((n, C)), ctx.empty((m, C)), ctx.empty((m, C))
    results = []
    with ctx.tuning(SPARSEOPS_NORM_LANES=0):
        for _ in range(2):
            ctx.layer_norm(dX, n, C, None, None, EPS, dN)
            ctx.matmul(E, dN, C, None, dS)
            ctx.mxfp4_matmul(handle, dN, C, None, dM)
            ctx.matmul(E, dN, C, None, dS)
            results.append([a.download().copy() for a in (dN, dS, dM)])
    for a, b in zip(*results):
        assert np.array_equal(a.view(np.uint32), b.view(np.uint32))
    N = results[0][0].astype(np.float64)
    check_forward(N, X.astype(np.float64), np.ones(n, np.float32), np.zeros(n, np.float32), "f32")
    want = dense.astype(np.float64) @ N
    assert np.abs(results[0][1] - want).max() <= 1e-5 * np.abs(want).max()
    Nq = mx.dequantize(*mx.quantize(np.ascontiguousarray(N.T)), n).T
    assert np.all(np.abs(results[0][2] - W @ Nq) <= product_tolerance(W, Nq, None, W @ Nq, "none", "f32"))
    handle.free()
    E.free()
