"""so_layer_norm and so_layer_norm_grad against the formulas in float64.

Tolerances, u = 2^-24.  A thread adds the values it holds and the workgroup's joins of them are trees; no fp32 sum here runs through more than 40 additions one after the other, so a mean is off by at most 40 u of the mean
magnitude, and so is the sum of squares behind rstd; the elementwise formula adds 8 roundings at most.  A 16-bit result is rounded once more, by half a step."""
import numpy as np
import pytest

import hipabi
from elements import HALF_STEP, SMALLEST, TYPES, U, fetch, fetch_apart, place, place_apart, stored, values

pytestmark = pytest.mark.gpu

EPS = 1e-5
SHAPES = [(1, 1), (1, 6), (7, 1), (64, 3), (97, 13), (257, 9), (1000, 33), (2049, 65), (4096, 1), (5000, 2), (301, 700), (8200, 17), (784, 64), (4099, 40), (128, 2500), (16384, 5), (16385, 3), (20000, 12)]


def problem(F, B, type_, seed=0, mean=0.5):
    rng = np.random.default_rng(1000 * F + B + seed)
    X = values(stored(rng.standard_normal((F, B)) + mean * rng.standard_normal((1, B)), type_), type_)
    return rng, X, (1 + 0.2 * rng.standard_normal(F)).astype(np.float32), (0.3 * rng.standard_normal(F)).astype(np.float32)


def statistics(X, eps=EPS):
    mean = X.mean(axis=0)
    return mean, 1.0 / np.sqrt(np.square(X - mean).mean(axis=0) + np.float64(np.float32(eps)))


def check_forward(Y, X, gamma, beta, type_, eps=EPS):
    mean, rstd = statistics(X, eps)
    h = (X - mean) * rstd
    g, b = gamma.astype(np.float64)[:, None], beta.astype(np.float64)[:, None]
    want = h * g + b
    tol = U * (48 * np.abs(X).max(axis=0) * rstd * np.abs(g) + 48 * np.abs(h * g) + 2 * np.abs(b)) + HALF_STEP[type_] * np.abs(want) + SMALLEST[type_]
    assert np.all(np.abs(Y - want) <= tol), np.max(np.abs(Y - want) / tol)


def check_statistics(mean, rstd, X, eps=EPS):
    want_mean, want_rstd = statistics(X, eps)
    off = 48 * U * np.abs(X).max(axis=0)
    assert np.all(np.abs(mean - want_mean) <= off)
    # the mean that the deviations are taken from may be off too: its square adds to the variance
    assert np.all(np.abs(rstd - want_rstd) <= want_rstd * (48 * U + np.square(off * want_rstd)))


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("F,B", SHAPES)
def test_forward(ctx, F, B, type_):
    rng, X, gamma, beta = problem(F, B, type_)
    for pad, shift, ypad in ((0, 0, 0), (3, 1, 5), (8, 0, 1)):
        whole, dX = place(ctx, X, type_, pad, shift)
        out, dY = place(ctx, np.zeros((F, B)), type_, ypad, shift, fill=-5.0)
        dG, dB, dM, dR = ctx.array(gamma), ctx.array(beta), ctx.empty((B,)), ctx.empty((B,))
        ctx.layer_norm(dX, F, B, dG, dB, EPS, dY, dM, dR, type=type_, x_stride=B + pad, y_stride=B + ypad)
        Y, rest = fetch(out, F, B, type_, ypad, shift)
        check_forward(Y, X, gamma, beta, type_)
        check_statistics(dM.download(), dR.download(), X)
        assert np.all(rest == -5.0), "places that are not the result's were written"
        for a in (whole, out, dG, dB, dM, dR):
            a.free()


@pytest.mark.parametrize("lanes", [0, 1, 2, 4, 8])
@pytest.mark.parametrize("F,B", [(1, 1), (70, 9), (600, 40), (2049, 65), (4000, 130), (9000, 20)])
def test_forward_however_it_is_cut(ctx, F, B, lanes):
    """Every number of lanes a row of the kernel that holds all features, and the two kernels that share them out."""
    for type_ in ("f32", "bf16"):
        _, X, gamma, beta = problem(F, B, type_, seed=2)
        whole, dX = place(ctx, X, type_, 3, 1)
        out, dY = place(ctx, np.zeros((F, B)), type_, 2, 1, fill=-5.0)
        dM, dR = ctx.empty((B,)), ctx.empty((B,))
        with ctx.tuning(SPARSEOPS_NORM_LANES=lanes):
            ctx.layer_norm(dX, F, B, ctx.array(gamma), ctx.array(beta), EPS, dY, dM, dR, type=type_, x_stride=B + 3, y_stride=B + 2)
        Y, rest = fetch(out, F, B, type_, 2, 1)
        check_forward(Y, X, gamma, beta, type_)
        check_statistics(dM.download(), dR.download(), X)
        assert np.all(rest == -5.0), "places that are not the result's were written"


def check_grad(dx, dgamma, dbeta, X, dY, gamma, mean, rstd, type_):
    mean, rstd = mean.astype(np.float64), rstd.astype(np.float64)
    g = dY * gamma.astype(np.float64)[:, None]
    h = (X - mean) * rstd
    a, b = g.mean(axis=0), (g * h).mean(axis=0)
    if dx is not None:
        want = rstd * (g - a - h * b)
        tol = rstd * U * (48 * (np.abs(g).mean(axis=0) + np.abs(h) * np.abs(g * h).mean(axis=0)) + 8 * (np.abs(g) + np.abs(a) + np.abs(h * b)))
        tol = tol + HALF_STEP[type_] * np.abs(want) + SMALLEST[type_]
        assert np.all(np.abs(dx - want) <= tol), np.max(np.abs(dx - want) / tol)
    if dgamma is not None:
        assert np.all(np.abs(dgamma - (dY * h).sum(axis=1)) <= U * (48 * np.abs(dY * h).sum(axis=1)) + 1e-40)
    if dbeta is not None:
        assert np.all(np.abs(dbeta - dY.sum(axis=1)) <= U * 48 * np.abs(dY).sum(axis=1) + 1e-40)


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("F,B", SHAPES)
def test_gradient(ctx, F, B, type_):
    rng, X, gamma, _ = problem(F, B, type_, seed=7)
    dY = values(stored(0.1 * rng.standard_normal((F, B)), type_), type_)
    mean, rstd = (s.astype(np.float32) for s in statistics(X))
    for pad, shift, ypad, xpad in ((0, 0, 0, 0), (3, 1, 5, 2), (8, 0, 1, 0)):
        whole, dX = place(ctx, X, type_, pad, shift)
        whole2, dDy = place(ctx, dY, type_, ypad, shift)
        out, dDx = place(ctx, np.zeros((F, B)), type_, xpad, shift, fill=-5.0)
        dG, dM, dR, dDg, dDb = ctx.array(gamma), ctx.array(mean), ctx.array(rstd), ctx.empty((F,)), ctx.empty((F,))
        ctx.layer_norm_grad(dX, dDy, F, B, dG, dM, dR, dDx, dDg, dDb, type=type_, x_stride=B + pad, dy_stride=B + ypad, dx_stride=B + xpad)
        dx, rest = fetch(out, F, B, type_, xpad, shift)
        check_grad(dx, dDg.download(), dDb.download(), X, dY, gamma, mean, rstd, type_)
        assert np.all(rest == -5.0), "places that are not the result's were written"
        for a in (whole, whole2, out, dG, dM, dR, dDg, dDb):
            a.free()


@pytest.mark.parametrize("lanes", [0, 1, 2, 4, 8])
@pytest.mark.parametrize("F,B", [(1, 1), (70, 9), (600, 40), (2049, 65), (4000, 130), (8100, 20), (9000, 3), (300, 9001), (1100, 5003)])
def test_gradient_however_it_is_cut(ctx, F, B, lanes):
    """Every number of lanes a row of the kernel that holds all features for a batch of one tile, and the two kernels that share the features out."""
    for type_ in ("f32", "bf16"):
        rng, X, gamma, _ = problem(F, B, type_, seed=9)
        dY = values(stored(0.1 * rng.standard_normal((F, B)), type_), type_)
        mean, rstd = (s.astype(np.float32) for s in statistics(X))
        whole, dX = place(ctx, X, type_, 3, 1)
        whole2, dDy = place(ctx, dY, type_, 1, 0)
        out, dDx = place(ctx, np.zeros((F, B)), type_, 2, 1, fill=-5.0)
        dDg, dDb = ctx.empty((F,)), ctx.empty((F,))
        with ctx.tuning(SPARSEOPS_NORM_LANES=lanes):
            ctx.layer_norm_grad(dX, dDy, F, B, ctx.array(gamma), ctx.array(mean), ctx.array(rstd), dDx, dDg, dDb, type=type_, x_stride=B + 3, dy_stride=B + 1, dx_stride=B + 2)
        dx, rest = fetch(out, F, B, type_, 2, 1)
        check_grad(dx, dDg.download(), dDb.download(), X, dY, gamma, mean, rstd, type_)
        assert np.all(rest == -5.0), "places that are not the result's were written"
        for a in (whole, whole2, out):
            a.free()


def test_gradient_is_that_of_the_forward_pass(ctx):
    """Central differences of sum(Y * dY) along X, gamma and beta, from the kernel's own forward pass in fp32: with steps of 2^-6 the third derivative and the roundings of the
    sum are below the bound of one part in a hundred of the gradient's largest entry."""
    F, B = 40, 5
    rng, X, gamma, beta = problem(F, B, "f32", seed=3)
    dY = rng.standard_normal((F, B)).astype(np.float32)
    dG, dBe, dM, dR, out = ctx.array(gamma), ctx.array(beta), ctx.empty((B,)), ctx.empty((B,)), ctx.empty((F, B))

    def loss(X, gamma, beta):
        a, g, b = ctx.array(X), ctx.array(gamma), ctx.array(beta)
        ctx.layer_norm(a, F, B, g, b, EPS, out)
        y = out.download().astype(np.float64)
        for t in (a, g, b):
            t.free()
        return float((y * dY).sum())

    dX = ctx.array(X.astype(np.float32))
    ctx.layer_norm(dX, F, B, dG, dBe, EPS, out, dM, dR)
    dDy, dDx, dDg, dDb = ctx.array(dY), ctx.empty((F, B)), ctx.empty((F,)), ctx.empty((F,))
    ctx.layer_norm_grad(dX, dDy, F, B, dG, dM, dR, dDx, dDg, dDb)
    got = {"X": dDx.download().ravel(), "gamma": dDg.download(), "beta": dDb.download()}
    step = 2.0 ** -6
    for name, size in (("X", F * B), ("gamma", F), ("beta", F)):
        scale = np.abs(got[name]).max()
        for i in range(0, size, 7):
            sides = []
            for sign in (1, -1):
                args = {"X": X.astype(np.float32).copy(), "gamma": gamma.copy(), "beta": beta.copy()}
                args[name].reshape(-1)[i] += np.float32(sign * step)
                sides.append(loss(**args))
            assert abs((sides[0] - sides[1]) / (2 * step) - got[name][i]) <= 1e-2 * scale, (name, i)


def test_without_parameters_and_in_place(ctx):
    F, B = 333, 70
    _, X, gamma, beta = problem(F, B, "f32")
    ones, zeros = np.ones(F, np.float32), np.zeros(F, np.float32)
    dX = ctx.array(X)
    ctx.layer_norm(dX, F, B, None, None, EPS, dX)
    check_forward(dX.download().astype(np.float64), X, ones, zeros, "f32")
    rng = np.random.default_rng(1)
    dY = rng.standard_normal((F, B)).astype(np.float32)
    mean, rstd = (s.astype(np.float32) for s in statistics(X))
    dM, dR = ctx.array(mean), ctx.array(rstd)
    for target in ("x", "dy", "none"):
        dX, dDy = ctx.array(X), ctx.array(dY)
        dDg = ctx.empty((F,))
        dDx = {"x": dX, "dy": dDy, "none": None}[target]
        ctx.layer_norm_grad(dX, dDy, F, B, None, dM, dR, dDx, dDg, None)
        check_grad(None if dDx is None else dDx.download().astype(np.float64), dDg.download(), None, X, dY.astype(np.float64), ones, mean, rstd, "f32")
    dX, dDy, dDx = ctx.array(X), ctx.array(dY), ctx.empty((F, B))
    ctx.layer_norm_grad(dX, dDy, F, B, None, dM, dR, dDx, None, None)          # the input's gradient alone
    check_grad(dDx.download().astype(np.float64), None, None, X, dY.astype(np.float64), ones, mean, rstd, "f32")
    ctx.layer_norm_grad(dX, dDy, F, B, None, dM, dR, None, None, None)          # nothing asked for


def test_columns_far_from_zero_constant_and_not_finite(ctx):
    F, B = 2000, 37
    _, X, gamma, beta = problem(F, B, "f32")
    X[:, 5] = X[:, 5] + 3000.0          # a mean of a thousand deviations
    X[:, 6] = 2.5                       # no variance
    X[:, 7] = 0.0
    X = X.astype(np.float32).astype(np.float64)
    bad = X.copy()
    bad[11, 8], bad[1999, 9], bad[0, 10] = np.inf, np.nan, -np.inf
    dX, dY, dG, dBe, dM, dR = ctx.array(bad), ctx.empty((F, B)), ctx.array(gamma), ctx.array(beta), ctx.empty((B,)), ctx.empty((B,))
    ctx.layer_norm(dX, F, B, dG, dBe, EPS, dY, dM, dR)
    Y, rstd = dY.download().astype(np.float64), dR.download()
    assert np.all(np.isnan(Y[:, 8:11])) and np.all(np.isnan(rstd[8:11]))
    rest = [b for b in range(B) if b not in (8, 9, 10)]
    check_forward(Y[:, rest], X[:, rest], gamma, beta, "f32")
    check_statistics(dM.download()[rest], rstd[rest], X[:, rest])
    assert np.array_equal(Y[:, 6], beta.astype(np.float64)) and np.array_equal(Y[:, 7], beta.astype(np.float64))


@pytest.mark.parametrize("lanes", [-1, 0])
def test_offsets_beyond_32_bits(ctx, lanes):
    """Rows 2^30 + 5 elements apart: the last ones begin beyond 2^32 elements."""
    F, B, apart = 6, 70, 2 ** 30 + 5
    _, X, gamma, beta = problem(F, B, "f16", seed=4)
    dX, dY, dM, dR = place_apart(ctx, X, "f16", apart), ctx.empty(((F - 1) * apart + B,), np.float16), ctx.empty((B,)), ctx.empty((B,))
    dG, dB, dg, db = ctx.array(gamma), ctx.array(beta), ctx.empty((F,)), ctx.empty((F,))
    with ctx.tuning(SPARSEOPS_NORM_LANES=lanes):
        ctx.layer_norm(dX, F, B, dG, dB, EPS, dY, dM, dR, type="f16", x_stride=apart, y_stride=apart)
        check_forward(fetch_apart(ctx, dY, F, B, "f16", apart), X, gamma, beta, "f16")
        # the gradient of the sum of all results: none for X, the normalised rows' sums for gamma, B for beta
        ones = place_apart(ctx, np.ones((F, B)), "f16", apart)
        ctx.layer_norm_grad(dX, ones, F, B, None, dM, dR, dY, dg, db, type="f16", x_stride=apart, dy_stride=apart, dx_stride=apart)
    mean, rstd = statistics(X)
    h = (X - mean) * rstd
    bound = U * 64 * (np.abs(X).max(axis=0) * rstd)                    # of h; g and its mean are exact here
    assert np.all(np.abs(fetch_apart(ctx, dY, F, B, "f16", apart)) <= rstd * (1 + np.abs(h)) * bound + SMALLEST["f16"])
    assert np.all(np.abs(dg.download() - h.sum(axis=1)) <= bound.sum() + U * 16 * np.abs(h).sum(axis=1))
    assert np.array_equal(db.download(), np.full(F, B, np.float32))
    for a in (dX, dY, ones):
        a.free()


def test_no_columns_and_refusals(ctx):
    F, B = 10, 4
    dX, dY, dF, dB = ctx.empty((F, B)), ctx.empty((F, B)), ctx.array(np.full(F, 3.0, np.float32)), ctx.array(np.full(F, 3.0, np.float32))
    st = ctx.empty((B,))
    ctx.layer_norm(None, F, 0, None, None, EPS, None)
    ctx.layer_norm_grad(None, None, F, 0, None, None, None, None, dF, dB)
    assert not dF.download().any() and not dB.download().any()

    def refused(match, call):
        with pytest.raises(hipabi.SoError, match=match) as e:
            call()
        assert e.value.status == hipabi.SO_ERR_INVALID

    refused("no features", lambda: ctx.layer_norm(dX, 0, B, None, None, EPS, dY))
    refused("null tensor", lambda: ctx.layer_norm(None, F, B, None, None, EPS, dY))
    refused("null tensor", lambda: ctx.layer_norm(dX, F, B, None, None, EPS, None))
    refused("stride", lambda: ctx.layer_norm(dX, F, B, None, None, EPS, dY, x_stride=B - 1))
    refused("stride", lambda: ctx.layer_norm(dX, F, B, None, None, EPS, dY, y_stride=B - 1))
    refused("one stride", lambda: ctx.layer_norm(dX, F, B - 1, None, None, EPS, dX, y_stride=B))
    refused("eps", lambda: ctx.layer_norm(dX, F, B, None, None, -1.0, dY))
    refused("eps", lambda: ctx.layer_norm(dX, F, B, None, None, float("nan"), dY))
    refused("too large for one launch", lambda: ctx.layer_norm(dX, 1, 0xffffffff, None, None, EPS, dY))
    refused("too large for one launch", lambda: ctx.layer_norm_grad(dX, dY, 0x7fffffff, 100, None, st, st, dX, None, None))
    refused("too large for one launch", lambda: ctx.layer_norm_reserve(1, 0xffffffff))
    refused("no features", lambda: ctx.layer_norm_grad(dX, dY, 0, B, None, st, st, dX, None, None))
    refused("both statistics", lambda: ctx.layer_norm(dX, F, B, None, None, EPS, dY, st, st))
    wide, other = ctx.empty((F,)), ctx.empty((F,))
    for args in ((wide, wide, other), (wide, other, wide), (wide, other, other)):
        refused("aliased", lambda: ctx.layer_norm_grad(dX, dY, F, B, args[0], st, st, dX, args[1], args[2]))
    refused("null tensor", lambda: ctx.layer_norm_grad(dX, None, F, B, None, st, st, dX, None, None))
    refused("null tensor", lambda: ctx.layer_norm_grad(dX, dY, F, B, None, None, st, dX, None, None))
    refused("stride", lambda: ctx.layer_norm_grad(dX, dY, F, B, None, st, st, dX, None, None, dy_stride=1))
    refused("one stride", lambda: ctx.layer_norm_grad(dX, dY, F, B - 1, None, st, st, dX, None, None, dx_stride=B))
    assert ctx.lib.so_layer_norm(ctx.h, 3, F, B, dX.ptr, B, None, None, EPS, dY.ptr, B, None, None) == hipabi.SO_ERR_INVALID
    assert ctx.lib.so_layer_norm_grad(ctx.h, -1, F, B, dX.ptr, B, dY.ptr, B, None, st.ptr, st.ptr, dX.ptr, B, None, None) == hipabi.SO_ERR_INVALID


def test_recorded_and_replayed(ctx):
    """Two graphs of different shapes on one context, replayed in turn with eager work between them: the same bits as eager calls, with new inputs too."""
    rng = np.random.default_rng(5)
    shapes = ((500, 30, "f32"), (1300, 90, "bf16"))
    held = []
    fresh = hipabi.Context()
    try:
        with pytest.raises(hipabi.SoError, match="so_layer_norm_reserve"):
            a = fresh.empty((20000, 8))
            fresh.graph_begin()
            try:
                fresh.layer_norm(a, 20000, 8, None, None, EPS, a)
            finally:
                fresh.graph_free(fresh.graph_end())
        for F, B, type_ in shapes:
            fresh.layer_norm_reserve(F, B, type=type_)
            dX = place(fresh, rng.standard_normal((F, B)), type_)[0]
            dDy = place(fresh, rng.standard_normal((F, B)), type_)[0]
            outs = [place(fresh, np.zeros((F, B)), type_)[0] for _ in range(2)] + [fresh.empty((n,)) for n in (B, B, F, F)]

            def calls(F=F, B=B, type_=type_, dX=dX, dDy=dDy, o=outs):
                fresh.layer_norm(dX, F, B, None, None, EPS, o[0], o[2], o[3], type=type_)
                fresh.layer_norm_grad(dX, dDy, F, B, None, o[2], o[3], o[1], o[4], o[5], type=type_)

            fresh.graph_begin()
            calls()
            held.append((fresh.graph_end(), calls, outs, dX, F, B, type_))
        for _ in range(3):
            for graph, calls, outs, dX, F, B, type_ in held:
                dX.upload(stored(rng.standard_normal((F, B)), type_))
                calls()
                want = [o.download().copy() for o in outs]
                for o in outs:
                    fresh.fill_zero(o)
                fresh.graph_launch(graph)
                for o, w in zip(outs, want):
                    assert np.array_equal(o.download().view(np.uint8), w.view(np.uint8))
        for graph, *_ in held:
            fresh.graph_free(graph)
    finally:
        fresh.close()
