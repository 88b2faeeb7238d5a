"""Microscaled 4-bit floating point: quantisation and its way back bit for bit, products against float64 on the same stored values."""
import numpy as np
import pytest

import hipabi
import mx_reference as mx
from elements import HALF_STEP, SMALLEST, STORAGE, TYPES, U, fetch, fetch_apart, place, place_apart, stored, values

pytestmark = pytest.mark.gpu


def wide_values(rng, rows, cols, type_):
    """Values of very different blocks: many binades, exact ties, zeros of both signs, subnormal numbers."""
    X = rng.standard_normal((rows, cols)) * np.exp2(rng.integers(-6, 7, (rows, 1)))
    ties = rng.choice([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0, 0.0, -0.0, 6.0], (rows, cols)) * rng.choice([-1.0, 1.0], (rows, cols))
    X = np.where(rng.random((rows, 1)) < 0.4, ties, X)
    if rows > 3:
        X[1] = 0.0
        X[2] = X[2] * 2.0 ** (-130 if type_ != "f16" else -18)
        X[3] = X[3] * 2.0 ** (110 if type_ != "f16" else 6)
    return values(stored(X, type_), type_)


SHAPES = [(1, 1), (1, 31), (3, 32), (5, 33), (4, 64), (7, 100), (33, 257), (100, 1000), (17, 4096), (300, 2049), (1025, 96)]


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_quantize_and_back(ctx, rows, cols, type_):
    rng = np.random.default_rng(rows * 10000 + cols)
    X = wide_values(rng, rows, cols, type_)
    codes, scales = mx.quantize(X)
    blocks = codes.shape[1]
    for pad, shift in ((0, 0), (5, 1), (8, 3)):
        whole, dX = place(ctx, X, type_, pad, shift)
        dC, dS = ctx.empty((rows, blocks, 16), np.uint8), ctx.empty((rows, blocks), np.uint8)
        ctx.mxfp4_quantize(dX, rows, cols, dC, dS, type=type_, x_stride=cols + pad)
        assert np.array_equal(dS.download(), scales)
        assert np.array_equal(dC.download(), codes)
        for back in TYPES:
            out, dY = place(ctx, np.zeros((rows, cols)), back, pad, shift, fill=-5.0)
            ctx.mxfp4_dequantize(dC, dS, rows, cols, dY, type=back, y_stride=cols + pad)
            Y, rest = fetch(out, rows, cols, back, pad, shift)
            want = values(stored(mx.dequantize(codes, scales, cols), back), back)
            assert np.array_equal(Y, want) and np.all(rest == -5.0)
            out.free()
        for a in (whole, dC, dS):
            a.free()


@pytest.mark.parametrize("type_", ["f16", "bf16"])
@pytest.mark.parametrize("apart", [1, 8, 64, 512, 2048])
def test_quantize_every_16_bit_pattern(ctx, type_, apart):
    """Blocks of 32 patterns `apart` from each other: infinities and NaN, subnormal numbers, every mantissa beside a largest one of its own binade and of others."""
    bits = np.arange(65536, dtype=np.uint16).reshape(-1, 32, apart).transpose(0, 2, 1).reshape(2048, 32)
    array = np.ascontiguousarray(bits).view(STORAGE[type_])
    with np.errstate(invalid="ignore"):
        codes, scales = mx.quantize(values(array, type_))
    dX, dC, dS = ctx.array(array, STORAGE[type_]), ctx.empty((2048, 1, 16), np.uint8), ctx.empty((2048, 1), np.uint8)
    ctx.mxfp4_quantize(dX, 2048, 32, dC, dS, type=type_)
    assert np.array_equal(dS.download(), scales)
    assert np.array_equal(dC.download(), codes)


def test_every_code_and_scale_and_blocks_that_are_not_numbers(ctx):
    codes = np.tile((np.arange(256, dtype=np.uint8)).reshape(1, 16, 16), (256, 1, 1))
    scales = np.repeat(np.arange(256, dtype=np.uint8)[:, None], 16, axis=1)
    dC, dS, dY = ctx.array(codes, np.uint8), ctx.array(scales, np.uint8), ctx.empty((256, 512))
    ctx.mxfp4_dequantize(dC, dS, 256, 512, dY)
    with np.errstate(over="ignore"):
        want = mx.dequantize(codes, scales, 512).astype(np.float32)
    assert np.array_equal(dY.download(), want, equal_nan=True)

    X = np.random.default_rng(0).standard_normal((6, 96)).astype(np.float32)
    X[0, 3], X[1, 40], X[2, 95], X[3, 0] = np.nan, np.inf, -np.inf, 3.4e38
    codes, scales = mx.quantize(X.astype(np.float64))
    assert scales[0, 0] == scales[1, 1] == scales[2, 2] == 255 and scales[3, 0] == 252
    dC, dS = ctx.empty((6, 3, 16), np.uint8), ctx.empty((6, 3), np.uint8)
    ctx.mxfp4_quantize(ctx.array(X), 6, 96, dC, dS)
    assert np.array_equal(dC.download(), codes) and np.array_equal(dS.download(), scales)
    dY = ctx.empty((6, 96))
    ctx.mxfp4_dequantize(dC, dS, 6, 96, dY)
    assert np.array_equal(dY.download(), mx.dequantize(codes, scales, 96).astype(np.float32), equal_nan=True)


def weights(ctx, rng, m, n):
    codes, scales = mx.quantize((rng.standard_normal((m, n)) * np.exp2(rng.integers(-3, 4, (m, 1))) / np.sqrt(n)).astype(np.float32).astype(np.float64))
    W = ctx.mxfp4(ctx.array(codes, np.uint8), ctx.array(scales, np.uint8), m, n)
    ctx.sync()
    return W, mx.dequantize(codes, scales, n)


def activated(Z, act):
    return {"none": Z, "relu": np.maximum(Z, 0), "sigmoid": 1 / (1 + np.exp(-Z)), "tanh": np.tanh(Z)}[act]


def product_tolerance(W, Xq, bias, want, act, type_):
    """A row's blocks are added in fp32 one after the other, two to an instruction: at most a rounding (taken as twice u) for each block and 16 more of joins, of the sum of the
    products' magnitudes, and the bias.  No activation makes a difference larger; its own result is within 4 roundings.  Then half a step of the result's type."""
    blocks = -(-W.shape[1] // 32)
    mag = np.abs(W) @ np.abs(Xq) + (0 if bias is None else np.abs(bias)[:, None])
    return 2 * U * (blocks + 16) * mag + (0 if act in ("none", "relu") else 4 * 2 * U) + HALF_STEP[type_] * np.abs(want) + SMALLEST[type_]


PRODUCTS = [(1, 1, 1), (3, 31, 2), (32, 32, 32), (33, 65, 33), (10, 4096, 64), (257, 255, 1), (64, 256, 16), (100, 1000, 101), (1000, 300, 7), (513, 784, 256), (2100, 520, 600),
            (31, 8200, 40), (4100, 256, 65), (300, 3333, 1500)]


@pytest.mark.parametrize("type_,act", [("f32", "none"), ("f32", "relu"), ("f32", "sigmoid"), ("f32", "tanh"), ("f16", "relu"), ("f16", "none"), ("bf16", "none"), ("bf16", "tanh")])
@pytest.mark.parametrize("m,n,C", PRODUCTS)
def test_matmul(ctx, m, n, C, type_, act):
    rng = np.random.default_rng(m + 7 * n + 13 * C)
    handle, W = weights(ctx, rng, m, n)
    X = values(stored(rng.standard_normal((n, C)) * np.exp2(rng.integers(-2, 3, (1, C))), type_), type_)
    Xq = mx.dequantize(*mx.quantize(np.ascontiguousarray(X.T)), n).T
    for pad, shift, ypad, with_bias in ((0, 0, 0, True), (3, 1, 5, False)):
        bias = rng.standard_normal(m).astype(np.float32) if with_bias else None
        want = activated(W @ Xq + (0 if bias is None else bias.astype(np.float64)[:, None]), act)
        whole, dX = place(ctx, X, type_, pad, shift)
        out, dY = place(ctx, np.zeros((m, C)), type_, ypad, shift, fill=-5.0)
        dB = None if bias is None else ctx.array(bias)
        ctx.mxfp4_matmul(handle, dX, C, dB, dY, act, type=type_, x_stride=C + pad, y_stride=C + ypad)
        Y, rest = fetch(out, m, C, type_, ypad, shift)
        tol = product_tolerance(W, Xq, bias, want, act, type_)
        assert np.all(np.abs(Y - want) <= tol), np.max(np.abs(Y - want) / tol)
        assert np.all(rest == -5.0), "places that are not the result's were written"
        whole.free()
        out.free()
    handle.free()


FORMS = ["mx-16x16", "mx-32x16", "mx-32x32", "mx-64x32", "mx-64x64", "mx-64x64-four", "mx-128x128", "mx-256x256"]


@pytest.mark.parametrize("form", range(1, len(FORMS) + 1))
@pytest.mark.parametrize("m,n,C", [(1, 40, 1), (70, 256, 33), (300, 257, 300), (257, 600, 17), (40, 1300, 530), (530, 2500, 65)])
def test_matmul_on_every_tile(ctx, m, n, C, form):
    """Each kernel form where another would be chosen: tiles that end inside the matrix, one to ten units of the contraction."""
    rng = np.random.default_rng(m + 7 * n + 13 * C)
    handle, W = weights(ctx, rng, m, n)
    for type_ in ("f32", "bf16"):
        X = values(stored(rng.standard_normal((n, C)), type_), type_)
        Xq = mx.dequantize(*mx.quantize(np.ascontiguousarray(X.T)), n).T
        bias = rng.standard_normal(m).astype(np.float32)
        want = activated(W @ Xq + bias.astype(np.float64)[:, None], "relu")
        whole, dX = place(ctx, X, type_, 1, 0)
        out, dY = place(ctx, np.zeros((m, C)), type_, 2, 1, fill=-5.0)
        with ctx.tuning(SPARSEOPS_MXFP4_MATMUL=form):
            ctx.mxfp4_matmul(handle, dX, C, ctx.array(bias), dY, "relu", type=type_, x_stride=C + 1, y_stride=C + 2)
        assert ctx.last_kernel() == FORMS[form - 1]
        Y, rest = fetch(out, m, C, type_, 2, 1)
        assert np.all(np.abs(Y - want) <= product_tolerance(W, Xq, bias, want, "relu", type_))
        assert np.all(rest == -5.0), "places that are not the result's were written"
        whole.free()
        out.free()
    handle.free()


@pytest.mark.parametrize("m,n", [(1, 1), (5, 31), (32, 32), (33, 1000), (1024, 1024), (1000, 8193), (70, 20000), (17000, 300), (40000, 40)])
def test_matvec(ctx, m, n):
    """x is fp32 and stays so: a block is a chain of 32 additions, its waves' and chunks' sums a few dozen more."""
    rng = np.random.default_rng(m + n)
    handle, W = weights(ctx, rng, m, n)
    x = rng.standard_normal(n).astype(np.float32)
    for bias in (None, rng.standard_normal(m).astype(np.float32)):
        dy = ctx.array(np.full(m + 3, -5.0, np.float32))
        whole = ctx.array(np.concatenate([[9.0], x]).astype(np.float32))
        ctx.mxfp4_matvec(handle, whole.offset(1), None if bias is None else ctx.array(bias), dy)
        got = dy.download().astype(np.float64)
        want = W @ x.astype(np.float64) + (0 if bias is None else bias)
        tol = U * ((64 + n // 32) * (np.abs(W) @ np.abs(x)) + (0 if bias is None else 2 * np.abs(bias)))
        assert np.all(np.abs(got[:m] - want) <= tol), np.max(np.abs(got[:m] - want) / tol)
        assert np.all(got[m:] == -5.0)
    handle.free()


def test_not_a_number_stays_in_its_row_and_column(ctx):
    rng = np.random.default_rng(4)
    m, n, C = 70, 500, 45
    codes, scales = mx.quantize(rng.standard_normal((m, n)))
    scales[11, 3] = 255
    W = ctx.mxfp4(ctx.array(codes, np.uint8), ctx.array(scales, np.uint8), m, n)
    X = rng.standard_normal((n, C)).astype(np.float32)
    X[499, 7], X[0, 44] = np.nan, np.inf
    dY = ctx.empty((m, C))
    ctx.mxfp4_matmul(W, ctx.array(X), C, None, dY)
    bad = np.zeros((m, C), bool)
    bad[11], bad[:, 7], bad[:, 44] = True, True, True
    assert np.array_equal(np.isnan(dY.download()), bad)
    dy = ctx.empty((m,))
    ctx.mxfp4_matvec(W, ctx.array(X[:, 0].copy()), None, dy)
    assert np.array_equal(np.isnan(dy.download()), np.arange(m) == 11)
    W.free()


def test_scales_at_the_ends(ctx):
    """Tiny and huge blocks: products that fp32 holds only as subnormal numbers, or not at all."""
    m, n, C = 32, 64, 32
    codes = np.full((m, 2, 16), 0x22, np.uint8)                       # ones
    for s_w, x in ((0, 1.0), (1, 2.0 ** -10), (250, 2.0 ** -100), (254, 4.0)):
        scales = np.full((m, 2), s_w, np.uint8)
        W = ctx.mxfp4(ctx.array(codes, np.uint8), ctx.array(scales, np.uint8), m, n)
        dY = ctx.empty((m, C))
        ctx.mxfp4_matmul(W, ctx.array(np.full((n, C), x, np.float32)), C, None, dY)
        with np.errstate(over="ignore"):
            want = np.float32(64 * x * 2.0 ** (s_w - 127))
        assert np.array_equal(dY.download(), np.full((m, C), want, np.float32)), (s_w, x)
        dy = ctx.empty((m,))
        ctx.mxfp4_matvec(W, ctx.array(np.full(n, x, np.float32)), None, dy)
        assert np.array_equal(dy.download(), np.full(m, want, np.float32)), (s_w, x)
        W.free()


def test_the_same_bits_every_time_and_across_states(ctx):
    """A second product in between uses the same workspace."""
    rng = np.random.default_rng(8)
    first, _ = weights(ctx, rng, 700, 900)
    second, _ = weights(ctx, rng, 900, 2000)
    dX, dX2 = ctx.array(rng.standard_normal((900, 130)).astype(np.float32)), ctx.array(rng.standard_normal((2000, 300)).astype(np.float32))
    dY, dY2, dZ = ctx.empty((700, 130)), ctx.empty((900, 300)), ctx.empty((700, 130))
    ctx.mxfp4_matmul(first, dX, 130, None, dY)
    ctx.mxfp4_matmul(second, dX2, 300, None, dY2)
    ctx.mxfp4_matmul(first, dX, 130, None, dZ)
    assert np.array_equal(dY.download().view(np.uint32), dZ.download().view(np.uint32))
    first.free()
    second.free()


def test_one_matrix_from_two_contexts(ctx):
    """A matrix made by one context is ready for another's stream at once; the two multiply without waiting for each other, each in its own workspace."""
    rng = np.random.default_rng(21)
    other = hipabi.Context()
    try:
        handle, W = weights(ctx, rng, 1500, 2000)
        X = rng.standard_normal((2, 2000, 300)).astype(np.float32)
        ins, outs = [c.array(x) for c, x in zip((ctx, other), X)], [c.empty((1500, 300)) for c in (ctx, other)]
        for _ in range(3):
            for c, dX, dY in zip((ctx, other), ins, outs):
                c.mxfp4_matmul(handle, dX, 300, None, dY)
        for x, dY in zip(X, outs):
            Xq = mx.dequantize(*mx.quantize(np.ascontiguousarray(x.T.astype(np.float64))), 2000).T
            want = W @ Xq
            assert np.all(np.abs(dY.download() - want) <= product_tolerance(W, Xq, None, want, "none", "f32"))
        ctx.sync()
        other.sync()
        handle.free()
        for a in ins + outs:
            a.free()
    finally:
        other.close()


def test_offsets_beyond_32_bits(ctx):
    """Rows 2^30 + 5 elements apart, the last ones beyond 2^32 elements: quantisation, its way back, the input and the output of a product."""
    rng = np.random.default_rng(15)
    rows, cols, apart = 6, 70, 2 ** 30 + 5
    X = values(stored(rng.standard_normal((rows, cols)), "f16"), "f16")
    dX, dY = place_apart(ctx, X, "f16", apart), ctx.empty(((rows - 1) * apart + cols,), np.float16)
    codes, scales = mx.quantize(X)
    dC, dS = ctx.empty(codes.shape, np.uint8), ctx.empty(scales.shape, np.uint8)
    ctx.mxfp4_quantize(dX, rows, cols, dC, dS, type="f16", x_stride=apart)
    assert np.array_equal(dC.download(), codes) and np.array_equal(dS.download(), scales)
    ctx.mxfp4_dequantize(dC, dS, rows, cols, dY, type="f16", y_stride=apart)
    assert np.array_equal(fetch_apart(ctx, dY, rows, cols, "f16", apart), mx.dequantize(codes, scales, cols))
    handle, W = weights(ctx, rng, rows, rows)
    ctx.mxfp4_matmul(handle, dX, cols, None, dY, type="f16", x_stride=apart, y_stride=apart)
    Xq = mx.dequantize(*mx.quantize(np.ascontiguousarray(X.T)), rows).T
    want = W @ Xq
    assert np.all(np.abs(fetch_apart(ctx, dY, rows, cols, "f16", apart) - want) <= product_tolerance(W, Xq, None, want, "none", "f16"))
    for a in (handle, dX, dY):
        a.free()


def test_empty_calls_and_refusals(ctx):
    a, b, c = ctx.empty((64, 64)), ctx.empty((64, 2, 16), np.uint8), ctx.empty((64, 2), np.uint8)
    ctx.mxfp4_quantize(None, 0, 5, None, None)
    ctx.mxfp4_quantize(None, 5, 0, None, None)
    ctx.mxfp4_dequantize(None, None, 0, 5, None)
    ctx.mxfp4_quantize(a, 64, 64, b, c)
    W = ctx.mxfp4(b, c, 64, 64)
    ctx.mxfp4_matmul(W, None, 0, None, None)

    def refused(match, call):
        with pytest.raises(hipabi.SoError, match=match) as e:
            call()
        assert e.value.status == hipabi.SO_ERR_INVALID

    refused("null array", lambda: ctx.mxfp4_quantize(None, 64, 64, b, c))
    refused("null array", lambda: ctx.mxfp4_quantize(a, 64, 64, b, None))
    refused("stride", lambda: ctx.mxfp4_quantize(a, 64, 64, b, c, x_stride=63))
    refused("aligned", lambda: ctx.mxfp4_quantize(a, 8, 64, b.offset(4), c))
    refused("null array", lambda: ctx.mxfp4_dequantize(b, None, 64, 64, a))
    refused("stride", lambda: ctx.mxfp4_dequantize(b, c, 64, 64, a, y_stride=1))
    refused("aligned", lambda: ctx.mxfp4_dequantize(b.offset(8), c, 8, 64, a))
    refused("empty", lambda: ctx.mxfp4(b, c, 0, 64))
    refused("empty", lambda: ctx.mxfp4(b, c, 64, 0))
    refused("null array", lambda: ctx.mxfp4(None, c, 64, 64))
    refused("aligned", lambda: ctx.mxfp4(b.offset(1), c, 8, 64))
    refused("too large", lambda: ctx.mxfp4(b, c, 64, 0xffffffff))
    refused("null or aliased", lambda: ctx.mxfp4_matmul(W, None, 4, None, a))
    refused("null or aliased", lambda: ctx.mxfp4_matmul(W, a, 4, None, a))
    refused("stride", lambda: ctx.mxfp4_matmul(W, a, 4, None, ctx.empty((64, 4)), x_stride=3))
    refused("too large for one launch", lambda: ctx.mxfp4(b, c, 0xffffffe0, 1 << 20))
    refused("too large for one launch", lambda: ctx.mxfp4_matmul(W, a, 0xffffffff, None, ctx.empty((64, 4))))
    refused("null or aliased", lambda: ctx.mxfp4_matvec(W, None, None, a))
    lib = ctx.lib
    assert lib.so_mxfp4_quantize(ctx.h, 7, a.ptr, 64, 64, 64, b.ptr, c.ptr) == hipabi.SO_ERR_INVALID
    assert lib.so_mxfp4_dequantize(ctx.h, b.ptr, c.ptr, 64, 64, 3, a.ptr, 64) == hipabi.SO_ERR_INVALID
    assert lib.so_mxfp4_matmul(ctx.h, W.h, 9, a.ptr, 64, 4, None, b.ptr, 64, 0) == hipabi.SO_ERR_INVALID
    assert lib.so_mxfp4_matmul(ctx.h, W.h, 0, a.ptr, 64, 4, None, b.ptr, 64, 4) == hipabi.SO_ERR_INVALID
    ctx.graph_begin()
    try:
        refused("recorded", W.free)
        refused("recorded", lambda: ctx.mxfp4(b, c, 64, 64))
    finally:
        ctx.graph_free(ctx.graph_end())
    W.free()


def test_recorded_and_replayed():
    """Products of two shapes and a quantisation in two graphs of one context, which share its workspace; replayed in turn, with eager calls between."""
    rng = np.random.default_rng(6)
    fresh = hipabi.Context()
    try:
        held = []
        for m, n, C, type_ in ((300, 700, 90, "f32"), (900, 1500, 300, "bf16")):
            W, _ = weights(fresh, rng, m, n)
            dX, dY = place(fresh, rng.standard_normal((n, C)), type_)[0], place(fresh, np.zeros((m, C)), type_)[0]
            dx, dy = fresh.array(rng.standard_normal(n).astype(np.float32)), fresh.empty((m,))
            if not held:
                fresh.graph_begin()
                try:
                    with pytest.raises(hipabi.SoError, match="so_mxfp4_matmul_reserve"):
                        fresh.mxfp4_matmul(W, dX, C, None, dY, type=type_)
                    with pytest.raises(hipabi.SoError, match="recorded"):
                        fresh.mxfp4_matmul_reserve(W, C)
                finally:
                    fresh.graph_free(fresh.graph_end())
            fresh.mxfp4_matmul_reserve(W, C)

            def calls(W=W, dX=dX, dY=dY, C=C, type_=type_, dx=dx, dy=dy):
                fresh.mxfp4_matmul(W, dX, C, None, dY, type=type_)
                fresh.mxfp4_matvec(W, dx, None, dy)

            fresh.graph_begin()
            calls()
            held.append((fresh.graph_end(), calls, dX, (dY, dy), n, C, type_, W))
        for _ in range(3):
            for graph, calls, dX, outs, n, C, type_, _W in held:
                dX.upload(stored(rng.standard_normal((n, C)), type_))
                calls()
                want = [o.download().copy() for o in outs]
                for o in outs:
                    fresh.fill_zero(o)
                fresh.graph_launch(graph)
                for o, w in zip(outs, want):
                    assert np.array_equal(o.download().view(np.uint8), w.view(np.uint8))
        for graph, *_rest, W in held:
            fresh.graph_free(graph)
            W.free()
    finally:
        fresh.close()


def test_a_block_of_layers(ctx):
    """Layer norm into a product, its activation into a product, the sum with the way past: the operators as a network uses them, on fp32 [features x batch], step by step against
    float64 on the values that the step before left, since a rounding to four bits may go either way at a border."""
    rng = np.random.default_rng(12)
    F, H, B = 384, 1000, 50
    up, Wu = weights(ctx, rng, H, F)
    down, Wd = weights(ctx, rng, F, H)
    X = rng.standard_normal((F, B)).astype(np.float32)
    gamma, beta = (1 + 0.1 * rng.standard_normal(F)).astype(np.float32), (0.1 * rng.standard_normal(F)).astype(np.float32)
    bias = rng.standard_normal(H).astype(np.float32)
    dX, dG, dBe, dBi = ctx.array(X), ctx.array(gamma), ctx.array(beta), ctx.array(bias)
    dN, dH, dO, dS = ctx.empty((F, B)), ctx.empty((H, B)), ctx.empty((F, B)), ctx.empty((F, B))
    ctx.layer_norm(dX, F, B, dG, dBe, 1e-5, dN)
    ctx.mxfp4_matmul(up, dN, B, dBi, dH, "relu")
    ctx.mxfp4_matmul(down, dH, B, None, dO)
    ctx.add(dO, dX, F * B, dS)
    N, Hid, O = (a.download().astype(np.float64) for a in (dN, dH, dO))
    X64 = X.astype(np.float64)
    h = (X64 - X64.mean(0)) / np.sqrt(X64.var(0) + np.float64(np.float32(1e-5)))
    assert np.abs(N - (h * gamma[:, None] + beta[:, None])).max() <= U * 48 * (np.abs(X64).max() / X64.std(0).min() + np.abs(h).max()) * 1.5
    for Wt, inp, out, bi, act in ((Wu, N, Hid, bias, "relu"), (Wd, Hid, O, None, "none")):
        Xq = mx.dequantize(*mx.quantize(np.ascontiguousarray(inp.T)), inp.shape[0]).T
        want = activated(Wt @ Xq + (0 if bi is None else bi.astype(np.float64)[:, None]), act)
        assert np.all(np.abs(out - want) <= product_tolerance(Wt, Xq, bi, want, act, "f32"))
    assert np.array_equal(dS.download(), dO.download() + X)
    up.free()
    down.free()
