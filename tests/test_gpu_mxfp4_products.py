"""4-bit products beyond test_gpu_mxfp4.py: blocks that are not numbers through every activation, blocks of very different size along the contraction, sums that fp32 holds exactly."""
import numpy as np
import pytest

import mx_reference as mx
from elements import TYPES, U, fetch, place, stored, values
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


@pytest.mark.parametrize("form", range(1, len(FORMS) + 1))
@pytest.mark.parametrize("m,n,C", [(40, 100, 20), (130, 1400, 70), (300, 4133, 40)])
def test_blocks_of_very_different_size(ctx, m, n, C, form):
    """Every block of W and of X has a power of two of its own, 2^-20 .. 2^20.  A matrix instruction adds four blocks to what is there, four additions of which each is off by at most a
    step (twice u) of the magnitudes added so far: 2 u for each block of a row, as product_tolerance has it."""
    rng = np.random.default_rng(m + n + C)
    blocks = -(-n // 32)
    spread = lambda shape, axis: np.repeat(np.exp2(rng.integers(-20, 21, shape)), 32, axis=axis)
    codes, scales = mx.quantize(rng.standard_normal((m, n)) * spread((m, blocks), 1)[:, :n])
    handle, W = handle_of(ctx, codes, scales, n)
    for type_ in ("f32", "bf16"):
        X = values(stored(rng.standard_normal((n, C)) * spread((blocks, C), 0)[:n], type_), type_)
        Xq = quantized(X)
        want = W @ Xq
        whole, dX = place(ctx, X, type_, 1, 0)
        out, dY = place(ctx, np.zeros((m, C)), type_, 0, 0)
        with ctx.tuning(SPARSEOPS_MXFP4_MATMUL=form):
            ctx.mxfp4_matmul(handle, dX, C, None, dY, type=type_, x_stride=C + 1)
        Y, _ = fetch(out, m, C, type_)
        tol = product_tolerance(W, Xq, None, want, "none", type_)
        assert np.all(np.abs(Y - want) <= tol), np.max(np.abs(Y - want) / tol)
        whole.free()
        out.free()
    handle.free()


@pytest.mark.parametrize("m,n", [(40, 100), (33, 4133), (70, 40000)])
def test_matvec_over_blocks_of_very_different_size(ctx, m, n):
    """As test_matvec: a block is a chain of 32 additions, a row's blocks and the waves' sums a few dozen more."""
    rng = np.random.default_rng(m + n)
    blocks = -(-n // 32)
    scale = np.repeat(np.exp2(rng.integers(-20, 21, (m, blocks))), 32, axis=1)[:, :n]
    codes, scales = mx.quantize(rng.standard_normal((m, n)) * scale)
    handle, W = handle_of(ctx, codes, scales, n)
    x = (rng.standard_normal(n) * np.repeat(np.exp2(rng.integers(-20, 21, blocks)), 32)[:n]).astype(np.float32)
    dx, dy = ctx.array(x), ctx.empty((m,))
    ctx.mxfp4_matvec(handle, dx, None, dy)
    want = W @ x.astype(np.float64)
    tol = U * (64 + n // 32) * (np.abs(W) @ np.abs(x.astype(np.float64)))
    assert np.all(np.abs(dy.download() - want) <= tol), np.max(np.abs(dy.download() - want) / tol)
    for a in (handle, dx, dy):
        a.free()


def exact_operands(rng, m, n, C, largest):
    """Codes up to `largest` with scales 2^-2 .. 2^2, neighbouring blocks of the first half cancelling each other, and X of such values, its blocks' largest entry at 4 or 6 of their scale so
    that it is kept as it is."""
    blocks = n // 32
    grid = mx.GRID[:largest + 1]

    def draw(rows):
        v = rng.choice(grid, (rows, blocks, 32)) * rng.choice([-1.0, 1.0], (rows, blocks, 32))
        e = rng.integers(-2, 3, (rows, blocks))
        return v, e

    v, e = draw(m)
    u, f = draw(C)
    for b in range(0, blocks // 2 - 1, 2):
        v[:, b + 1], e[:, b + 1], u[:, b + 1], f[:, b + 1] = -v[:, b], e[:, b], u[:, b], f[:, b]
    code = np.array([np.abs(mx.GRID - a).argmin() for a in np.abs(v).ravel()], np.uint8).reshape(v.shape) + 8 * np.signbit(v).astype(np.uint8)
    codes, scales = (code[..., 0::2] | code[..., 1::2] << 4).astype(np.uint8), (e + 127).astype(np.uint8)
    return codes, scales, (u * np.exp2(f)[..., None]).reshape(C, n).T


@pytest.mark.parametrize("form", range(0, len(FORMS) + 1))          # the last: the matvec
@pytest.mark.parametrize("n,largest", [(256, 7), (2048, 2), (32, 7)])
def test_sums_that_fp32_holds_are_exact(ctx, n, largest, form):
    """All products are multiples of 2^-2 2^-2 2^-2 = 2^-6, and the magnitudes of a row add up to less than 2^24 of these (256: 8 blocks of 32 * 36 * 2^4 = 2^17.2; 2048: 64 of 32 * 2^4 = 2^15), so
    that every partial sum in any order is a number of fp32 and nothing is rounded, with large blocks that cancel and small ones that remain."""
    rng = np.random.default_rng(n + largest)
    m, C = 75, 50
    codes, scales, X = exact_operands(rng, m, n, C, largest)
    handle, W = handle_of(ctx, codes, scales, n)
    Xq = quantized(X)
    mag = np.abs(W) @ np.abs(Xq)
    assert mag.max() < 2.0 ** 18 and np.array_equal(np.floor(X * 16), X * 16)
    want = W @ Xq
    dX, dY = ctx.array(X.astype(np.float32)), ctx.empty((m, C))
    if form == len(FORMS):
        dy = ctx.empty((m,))
        for c in (0, 7):
            dx = ctx.array(X[:, c].astype(np.float32))
            ctx.mxfp4_matvec(handle, dx, None, dy)
            assert np.array_equal(dy.download().astype(np.float64), W @ X[:, c])
    else:
        with ctx.tuning(SPARSEOPS_MXFP4_MATMUL=form + 1):
            ctx.mxfp4_matmul(handle, dX, C, None, dY)
        assert ctx.last_kernel() == FORMS[form]
        assert np.array_equal(dY.download().astype(np.float64), want)
    handle.free()
