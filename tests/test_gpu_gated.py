"""so_gated and so_gated_grad against the formulas in float64 (tests/gated_reference.py derives the tolerances).  What lies between and around the operands' rows is NaN, so that a value read
from there shows."""
import numpy as np
import pytest

import hipabi
from elements import STORAGE, TYPES, fetch, fetch_apart, place, place_apart, stored, values
from gated_reference import ACTS, backward, check, forward, gate
from hipabi import SO_ERR_INVALID

pytestmark = pytest.mark.gpu

# (m, n, B): one of everything, sizes around the tiles', a contraction that ends inside a group, no size a multiple of anything, one token to many
SHAPES = [(1, 1, 1), (1, 5, 3), (7, 1, 1), (33, 70, 1), (64, 64, 64), (65, 129, 17), (130, 100, 2), (257, 300, 70), (40, 1000, 24), (128, 64, 256), (300, 333, 140), (20, 4133, 9), (515, 263, 600),
          (16, 40, 8), (1000, 515, 1), (300, 9000, 1), (200, 520, 33), (513, 72, 129), (600, 320, 520)]
PLACES = [(0, 0), (3, 1), (8, 0)]          # places between the rows, elements ahead of the first


class Arrays:
    """Device arrays of a test, freed together."""

    def __init__(self, ctx, type_):
        self.ctx, self.type, self.all = ctx, type_, []

    def put(self, matrix, pad=0, shift=0, fill=np.nan):
        whole, at = place(self.ctx, matrix, self.type, pad, shift, fill)
        self.all.append(whole)
        return whole, at

    def free(self):
        for a in self.all:
            a.free()


def draw(rng, type_, *shape, size=1.0):
    return values(stored(size * rng.standard_normal(shape), type_), type_)


def weights(rng, type_, m, n):
    return draw(rng, type_, m, n, size=n ** -0.5)


def run_forward(ctx, rng, m, n, B, type_, act, pad=0, shift=0, wpad=0, add=(True, True), save=(True, True)):
    Wg, Wu, X = weights(rng, type_, m, n), weights(rng, type_, m, n), draw(rng, type_, n, B)
    G0, U0 = draw(rng, type_, m, B, size=0.5), draw(rng, type_, m, B, size=0.5)
    a = Arrays(ctx, type_)
    dWg, dWu, dX = a.put(Wg, wpad, shift)[1], a.put(Wu, wpad, shift)[1], a.put(X, pad, shift)[1]
    dG0, dU0 = (a.put(v, pad + 1, shift)[1] if on else None for v, on in zip((G0, U0), add))
    outs = {k: a.put(np.zeros((m, B)), p, shift, fill=-5.0) for k, p in (("H", pad), ("G", pad + 2), ("U", pad + 2))}
    ctx.gated(dWg, dWu, m, n, dX, B, act, outs["H"][1], *(outs[k][1] if on else None for k, on in zip("GU", save)), dG0, dU0, type=type_, w_stride=n + wpad, x_stride=B + pad, h_stride=B + pad,
              g_stride=B + pad + 2, g0_stride=B + pad + 1)
    want = forward(Wg, Wu, X, act, type_, G0 if add[0] else None, U0 if add[1] else None)
    for name, p, on in (("H", pad, True), ("G", pad + 2, save[0]), ("U", pad + 2, save[1])):
        got, rest = fetch(outs[name][0], m, B, type_, p, shift)
        if on:
            check(got, want[name], name)
        else:
            assert not got.any()
        assert np.all(rest == -5.0), "places that are not the result's were written"
    a.free()


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("m,n,B", SHAPES)
def test_forward(ctx, m, n, B, type_):
    rng = np.random.default_rng(m + 1000 * n + B)
    for i, (pad, shift) in enumerate(PLACES):
        run_forward(ctx, rng, m, n, B, type_, ACTS[(m + n + B + i) % len(ACTS)], pad, shift, wpad=(0, 5, 8)[i])


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("m,n,B", [(70, 75, 3), (66, 261, 21), (130, 517, 129), (301, 131, 267), (517, 1029, 35)])
def test_rows_that_are_aligned_and_end_inside_a_group(ctx, m, n, B, type_):
    """Every row begins at a multiple of 16 bytes, and ends at none; the last one is the end of its array."""
    rng = np.random.default_rng(m + n + B)
    up = lambda v: -v % 8
    for make in (lambda pad, wpad: run_forward(ctx, rng, m, n, B, type_, "silu", pad, 0, wpad), lambda pad, wpad: run_backward(ctx, rng, m, n, B, type_, "silu", pad, 0, wpad)):
        make(up(B), up(n))
        make(up(B), 0)
        make(0, up(n))


FORMS = ["gated-32x32", "gated-32x64", "gated-64x64", "gated-64x128", "gated-128x128", "gated-256x256"]


@pytest.mark.parametrize("form", range(1, 7))
@pytest.mark.parametrize("m,n,B", [(40, 24, 16), (70, 72, 40), (150, 264, 72), (300, 520, 264), (280, 1032, 328), (96, 4096, 48), (520, 2056, 40)])
def test_every_tile(ctx, m, n, B, form):
    """Each tile of the result on contractions of less than one step of its ring, a few, and many, with and without a last one that is not whole; both ways that operands go to LDS."""
    rng = np.random.default_rng(form + m + n + B)
    for type_ in TYPES:
        with ctx.tuning(SPARSEOPS_GATED_TILE=form):
            run_forward(ctx, rng, m, n, B, type_, "silu", pad=8, wpad=0)
            assert ctx.last_kernel() == FORMS[min(form, 6 if type_ != "f32" else 5) - 1]
            run_backward(ctx, rng, m, n, B, type_, "silu", pad=8, wpad=8)
            run_forward(ctx, rng, m, n, B, type_, "gelu", pad=3, wpad=5)
            run_backward(ctx, rng, m, n, B, type_, "gelu", pad=3, wpad=5)


@pytest.mark.parametrize("act", ACTS)
def test_forward_of_every_activation(ctx, act):
    rng = np.random.default_rng(5)
    for type_ in TYPES:
        for m, n, B in ((50, 90, 1), (50, 90, 20), (150, 90, 200)):
            for add, save in (((True, False), (False, True)), ((False, True), (True, False)), ((False, False), (False, False))):
                run_forward(ctx, rng, m, n, B, type_, act, add=add, save=save)


@pytest.mark.parametrize("type_", TYPES)
def test_large_sums_through_every_activation(ctx, type_):
    """Sums from the activations' middle to where they are flat and beyond the range of the exponential: 0.01 to 30000 in size."""
    rng = np.random.default_rng(6)
    m, n, B = 60, 64, 40
    for act in ACTS:
        for B_ in (1, B):
            Wg, Wu, X = weights(rng, type_, m, n), weights(rng, type_, m, n) / 64, draw(rng, type_, n, B_)
            Wg, Wu = values(stored(Wg * np.logspace(-2, 4, m)[:, None], type_), type_), values(stored(Wu, type_), type_)
            a = Arrays(ctx, type_)
            H, dH = a.put(np.zeros((m, B_)))
            ctx.gated(a.put(Wg)[1], a.put(Wu)[1], m, n, a.put(X)[1], B_, act, dH, type=type_)
            want, tol = forward(Wg, Wu, X, act, type_)["H"]
            # an error of the argument goes in with the slope, 1.2 at most, and in the flat parts the sums' own error exceeds the tails': what is left out there is below it
            check(fetch(H, m, B_, type_)[0], (want, tol), act)
            a.free()


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("m,n,B", [(70, 100, 1), (70, 100, 30), (300, 200, 300), (257, 97, 129)])
def test_what_is_not_a_number_stays_where_it_is(ctx, m, n, B, type_):
    """NaN in a column of X makes that column of H NaN, one in a row of a projection that row, in G0 its entry; everything else has the same bits as without."""
    rng = np.random.default_rng(m + B)
    for act in ("relu", "silu", "gelu"):
        Wg, Wu, X, G0 = weights(rng, type_, m, n), weights(rng, type_, m, n), draw(rng, type_, n, B), draw(rng, type_, m, B)
        bad = np.zeros((m, B), bool)
        outs = []
        for marked in (False, True):
            if marked:
                Wg[m // 2, n - 1] = np.nan
                Wu[m - 1, 0] = np.nan
                G0[1, B - 1] = np.nan
                bad[[m // 2, m - 1]], bad[1, B - 1] = True, True
                if B > 1:
                    X[n - 1, B // 2] = np.nan
                    bad[:, B // 2] = True
            a = Arrays(ctx, type_)
            H, dH = a.put(np.zeros((m, B)))
            ctx.gated(a.put(Wg)[1], a.put(Wu)[1], m, n, a.put(X)[1], B, act, dH, dG0=a.put(G0)[1], type=type_)
            outs.append(fetch(H, m, B, type_)[0])
            a.free()
        assert np.array_equal(np.isnan(outs[1]), bad)
        assert np.array_equal(outs[0][~bad], outs[1][~bad])


def test_in_place_and_twice_the_same_bits(ctx):
    rng = np.random.default_rng(8)
    for type_ in TYPES:
        for m, n, B in ((90, 130, 1), (90, 130, 12), (333, 257, 190)):
            Wg, Wu, X, G0, U0 = weights(rng, type_, m, n), weights(rng, type_, m, n), draw(rng, type_, n, B), draw(rng, type_, m, B), draw(rng, type_, m, B)
            a = Arrays(ctx, type_)
            dWg, dWu, dX, dG0, dU0 = (a.put(v)[1] for v in (Wg, Wu, X, G0, U0))
            outs = [a.put(np.zeros((m, B))) for _ in range(4)]
            ctx.gated(dWg, dWu, m, n, dX, B, "gelu", outs[0][1], outs[1][1], outs[2][1], dG0, dU0, type=type_)
            ctx.gated(dWg, dWu, m, n, dX, B, "gelu", outs[3][1], dG0, dU0, dG0, dU0, type=type_)
            same = lambda p, q: np.array_equal(p.download().view(np.uint8), q.download().view(np.uint8))
            assert same(outs[0][0], outs[3][0]) and same(outs[1][0], a.all[3]) and same(outs[2][0], a.all[4])
            a.free()


def run_backward(ctx, rng, m, n, B, type_, act, pad=0, shift=0, wpad=0, wanted=("dX", "dWg", "dWu", "dG", "dU")):
    Wg, Wu, X = weights(rng, type_, m, n), weights(rng, type_, m, n), draw(rng, type_, n, B)
    G, S, dH = draw(rng, type_, m, B, size=1.5), draw(rng, type_, m, B), draw(rng, type_, m, B, size=0.1)
    a = Arrays(ctx, type_)
    dWg, dWu, dX = a.put(Wg, wpad, shift)[1], a.put(Wu, wpad, shift)[1], a.put(X, pad, shift)[1]
    dG, dS, dDh = a.put(G, pad + 1, shift)[1], a.put(S, pad + 1, shift)[1], a.put(dH, pad, shift)[1]
    places = {"dX": (n, B, pad + 2), "dWg": (m, n, wpad + 1), "dWu": (m, n, wpad + 1), "dG": (m, B, pad), "dU": (m, B, pad)}
    outs = {k: a.put(np.zeros((r, c)), p, shift, fill=-5.0) for k, (r, c, p) in places.items()}
    ctx.gated_grad(dWg, dWu, m, n, dX, B, act, dG, dS, dDh, *(outs[k][1] if k in wanted else None for k in ("dX", "dWg", "dWu", "dG", "dU")), type=type_, w_stride=n + wpad, x_stride=B + pad,
                   g_stride=B + pad + 1, dh_stride=B + pad, dx_stride=B + pad + 2, dw_stride=n + wpad + 1, dg_stride=B + pad)
    want = backward(Wg, Wu, X, act, G, S, dH, type_)
    for name, (r, c, p) in places.items():
        got, rest = fetch(outs[name][0], r, c, type_, p, shift)
        if name in wanted:
            check(got, want[name], name)
        else:
            assert not got.any()
        assert np.all(rest == -5.0), "places that are not the result's were written"
    a.free()


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("m,n,B", SHAPES)
def test_backward(ctx, m, n, B, type_):
    rng = np.random.default_rng(m + 1000 * n + B + 1)
    for i, (pad, shift) in enumerate(PLACES):
        run_backward(ctx, rng, m, n, B, type_, ACTS[(m + n + B + i) % len(ACTS)], pad, shift, wpad=(0, 5, 8)[i])


@pytest.mark.parametrize("act", ACTS)
def test_backward_of_every_activation(ctx, act):
    rng = np.random.default_rng(9)
    for type_ in TYPES:
        for m, n, B in ((50, 90, 1), (50, 90, 20), (150, 90, 200)):
            run_backward(ctx, rng, m, n, B, type_, act)


@pytest.mark.parametrize("wanted", [("dX",), ("dWg",), ("dWu",), ("dG",), ("dU",), ("dX", "dG"), ("dWu", "dU"), ("dWg", "dU"), ("dX", "dWg", "dWu"), ("dG", "dU"), ()])
def test_any_result_may_be_left_out(ctx, wanted):
    rng = np.random.default_rng(10)
    for type_ in ("f32", "bf16"):
        run_backward(ctx, rng, 75, 140, 33, type_, "silu", pad=1, wpad=3, wanted=wanted)
        run_backward(ctx, rng, 80, 144, 40, type_, "silu", wanted=wanted)


def test_gradients_in_place(ctx):
    """dG and dU over the saved sums, or one of them over the gradient of H: the bits of the call into arrays of their own."""
    rng = np.random.default_rng(11)
    for type_ in TYPES:
        for m, n, B in ((40, 66, 30), (72, 64, 64)):
            Wg, Wu, X = weights(rng, type_, m, n), weights(rng, type_, m, n), draw(rng, type_, n, B)
            G, S, D = draw(rng, type_, m, B), draw(rng, type_, m, B), draw(rng, type_, m, B)
            seen = []
            for case in range(4):
                a = Arrays(ctx, type_)
                dWg, dWu, dX, dG, dS, dD = (a.put(v)[1] for v in (Wg, Wu, X, G, S, D))
                res = [a.put(np.zeros(s))[0] for s in ((n, B), (m, n), (m, n), (m, B), (m, B))]
                g, u = [(res[3], res[4]), (dG, dS), (dS, dG), (dD, dS)][case]
                ctx.gated_grad(dWg, dWu, m, n, dX, B, "gelu", dG, dS, dD, res[0], res[1], res[2], g, u, type=type_)
                shape = (m, B)
                ctx.sync()
                whole = {0: (res[3], res[4]), 1: (a.all[3], a.all[4]), 2: (a.all[4], a.all[3]), 3: (a.all[5], a.all[4])}[case]
                seen.append([x.download().copy() for x in (res[0], res[1], res[2]) + whole])
                assert seen[-1][3].shape[0] == shape[0] * shape[1]
                a.free()
            for other in seen[1:]:
                for x, y in zip(seen[0], other):
                    assert np.array_equal(x.view(np.uint8), y.view(np.uint8))


def test_gradient_against_differences(ctx):
    """The sum of D * H: its gradient along a random half of the gradient's own entries, from so_gated_grad, and differences of the formula in float64.  fp32 sums of at most 260 products are off by
    2 u (260 + 16) = 3.3e-5 of their magnitudes, which are some ten times the sums: less than 1e-3 of the gradient's norm; the differences to 1e-6."""
    rng = np.random.default_rng(12)
    m, n, B = 130, 70, 50
    for act in ACTS:
        Wg, Wu, X, D = weights(rng, "f32", m, n), weights(rng, "f32", m, n), draw(rng, "f32", n, B), draw(rng, "f32", m, B)
        loss = lambda Wg, Wu, X: float((D * gate(Wg @ X, act)[0] * (Wu @ X)).sum())
        a = Arrays(ctx, "f32")
        dWg, dWu, dX, dD = (a.put(v)[1] for v in (Wg, Wu, X, D))
        H, G, S, gX, gWg, gWu = (a.put(np.zeros(s))[0] for s in ((m, B), (m, B), (m, B), (n, B), (m, n), (m, n)))
        ctx.gated(dWg, dWu, m, n, dX, B, act, H, G, S)
        ctx.gated_grad(dWg, dWu, m, n, dX, B, act, G, S, dD, gX, gWg, gWu)
        for at, grad in enumerate((gWg, gWu, gX)):
            got = grad.download().astype(np.float64).reshape((Wg, Wu, X)[at].shape)
            along = got * (rng.random(got.shape) < 0.5)
            moved = lambda s: [v + (s * along if i == at else 0.0) for i, v in enumerate((Wg, Wu, X))]
            step = 1e-7 if act == "relu" else 1e-5
            difference = (loss(*moved(step)) - loss(*moved(-step))) / (2 * step)
            assert abs(float((got * along).sum()) - difference) <= 1e-3 * np.linalg.norm(got) * np.linalg.norm(along), (act, at)
        a.free()


def test_empty_sizes(ctx):
    a = Arrays(ctx, "f32")
    one = a.put(np.ones((4, 4)))[0]
    out, w = a.put(np.full((4, 4), 3.0))[0], a.put(np.full((4, 4), 3.0))[0]
    ctx.gated(one, one, 0, 4, one, 4, "silu", out)
    ctx.gated(one, one, 4, 4, one, 0, "silu", out)
    assert np.all(out.download() == 3.0)
    ctx.gated_grad(one, one, 4, 4, None, 0, "silu", None, None, None, None, out, w)      # no columns: the weights' gradients are zeros
    assert not out.download().any() and not w.download().any()
    out.upload(np.full(out.shape, 3.0))
    ctx.gated_grad(None, None, 0, 4, None, 4, "silu", None, None, None, out)             # no rows: nor has X one
    assert not out.download().any()
    a.free()


def test_offsets_beyond_32_bits(ctx):
    """Rows of the weights, of X and of the results 2^28 + 1 elements apart, twenty of them."""
    rng = np.random.default_rng(13)
    far = 2 ** 28 + 1
    m, n, B = 12, 20, 3
    for type_ in ("bf16",):
        Wg, X = weights(rng, type_, m, n), draw(rng, type_, n, B)
        dW, dX, dH = place_apart(ctx, Wg, type_, far), place_apart(ctx, X, type_, far), place_apart(ctx, np.zeros((m, B)), type_, far)
        a = Arrays(ctx, type_)
        G = a.put(np.zeros((m, B)))[0]
        ctx.gated(dW, dW, m, n, dX, B, "gelu", dH, G, type=type_, w_stride=far, x_stride=far, h_stride=far)
        want = forward(Wg, Wg, X, "gelu", type_)
        check(fetch_apart(ctx, dH, m, B, type_, far), want["H"])
        got = fetch(G, m, B, type_)[0]
        check(got, want["G"])
        D = draw(rng, type_, m, B)
        dD = place_apart(ctx, D, type_, far)
        gX = a.put(np.zeros((n, B)))[0]
        gW = a.put(np.zeros((m, n)))[0]
        ctx.gated_grad(dW, dW, m, n, dX, B, "gelu", G, G, dD, gX, gW, None, type=type_, w_stride=far, x_stride=far, dh_stride=far)
        back = backward(Wg, Wg, X, "gelu", got, got, D, type_)
        check(fetch(gX, n, B, type_)[0], back["dX"])
        check(fetch(gW, m, n, type_)[0], back["dWg"])
        a.free()
        for x in (dW, dX, dH, dD):
            x.free()


def test_refusals(ctx):
    a = Arrays(ctx, "f32")
    W, X, H, G, S, D = (a.put(np.ones((8, 8)))[0] for _ in range(6))
    out = a.put(np.full((8, 8), 3.0))[0]

    def refused(call, text):
        with pytest.raises(hipabi.SoError) as e:
            call()
        assert e.value.status == SO_ERR_INVALID and text in str(e.value), e.value

    lib, h = ctx.lib, ctx.h
    refused(lambda: ctx._ck(lib.so_gated(h, 7, 8, 8, 8, W.ptr, W.ptr, 8, X.ptr, 8, 4, None, None, 8, out.ptr, 8, None, None, 8)), "element type")
    refused(lambda: ctx._ck(lib.so_gated(h, 0, 8, 8, 8, W.ptr, W.ptr, 8, X.ptr, 8, 7, None, None, 8, out.ptr, 8, None, None, 8)), "activation")
    refused(lambda: ctx._ck(lib.so_gated(h, 0, 8, 8, 8, W.ptr, W.ptr, 8, X.ptr, 8, -1, None, None, 8, out.ptr, 8, None, None, 8)), "activation")
    refused(lambda: ctx.gated(W, W, 8, 0, X, 8, "silu", out), "no input features")
    for args in ((None, W, X, out), (W, None, X, out), (W, W, None, out), (W, W, X, None)):
        refused(lambda: ctx.gated(args[0], args[1], 8, 8, args[2], 8, "silu", args[3]), "null")
    for stride in ("w_stride", "x_stride", "h_stride"):
        refused(lambda: ctx.gated(W, W, 8, 8, X, 8, "silu", out, **{stride: 7}), "stride")
    refused(lambda: ctx.gated(W, W, 8, 8, X, 8, "silu", out, G, g_stride=7), "stride")
    refused(lambda: ctx.gated(W, W, 8, 8, X, 8, "silu", out, None, None, None, G, g0_stride=7), "stride")
    refused(lambda: ctx.gated(W, W, 4, 8, X, 4, "silu", out, G, None, G, g_stride=4, g0_stride=8), "one stride")
    refused(lambda: ctx.gated(W, W, 8, 8, X, 8, "silu", X), "is an input")
    refused(lambda: ctx.gated(W, W, 8, 8, X, 8, "silu", G, None, None, G), "is an input")
    refused(lambda: ctx.gated(W, W, 8, 8, X, 8, "silu", out, G, None, None, G), "is an input")
    refused(lambda: ctx.gated(W, W, 8, 8, X, 8, "silu", out, G, G), "two results")
    refused(lambda: ctx.gated(W, W, 8, 8, X, 8, "silu", out, out), "two results")
    refused(lambda: ctx.gated_grad(W, W, 8, 0, X, 8, "silu", G, S, D, out), "no input features")
    for args in ((None, S, D), (G, None, D), (G, S, None)):
        refused(lambda: ctx.gated_grad(W, W, 8, 8, X, 8, "silu", *args, out), "null")
    refused(lambda: ctx.gated_grad(None, W, 8, 8, X, 8, "silu", G, S, D, out), "null weights")
    refused(lambda: ctx.gated_grad(W, W, 8, 8, None, 8, "silu", G, S, D, None, out), "null input")
    for stride in ("w_stride", "g_stride", "dh_stride", "dx_stride"):
        refused(lambda: ctx.gated_grad(W, W, 8, 8, X, 8, "silu", G, S, D, out, **{stride: 7}), "stride")
    for stride in ("x_stride", "dw_stride"):
        refused(lambda: ctx.gated_grad(W, W, 8, 8, X, 8, "silu", G, S, D, None, out, **{stride: 7}), "stride")
    refused(lambda: ctx.gated_grad(W, W, 8, 8, X, 8, "silu", G, S, D, None, None, None, out, dg_stride=7), "stride")
    refused(lambda: ctx.gated_grad(W, W, 8, 8, X, 8, "silu", G, S, D, X), "is an input")
    refused(lambda: ctx.gated_grad(W, W, 8, 8, X, 8, "silu", G, S, D, None, G), "is an input")
    refused(lambda: ctx.gated_grad(W, W, 4, 8, X, 4, "silu", G, S, D, None, None, None, G, g_stride=8, dg_stride=4), "two strides")
    refused(lambda: ctx.gated_grad(W, W, 8, 8, X, 8, "silu", G, S, D, out, out), "two results")
    refused(lambda: ctx._ck(lib.so_gated_reserve(h, 3, 8, 8, 8)), "element type")
    assert np.all(out.download() == 3.0)
    a.free()


@pytest.mark.parametrize("type_,m,n,B", [("f32", 300, 130, 70), ("bf16", 520, 256, 300), ("f16", 90, 77, 33), ("bf16", 2000, 512, 1), ("bf16", 200, 128, 16)])
def test_recorded_ahead_of_the_first_launch(type_, m, n, B):
    """Both recorded on a fresh context behind their reserve, replayed with new inputs as often as they are called: the same bits."""
    rng = np.random.default_rng(m)
    ctx = hipabi.Context()
    try:
        a = Arrays(ctx, type_)
        Wg, Wu, X, D = (a.put(v)[0] for v in (weights(rng, type_, m, n), weights(rng, type_, m, n), np.zeros((n, B)), draw(rng, type_, m, B)))
        H, G, S, gX, gWg, gWu = outs = [a.put(np.zeros(s))[0] for s in ((m, B), (m, B), (m, B), (n, B), (m, n), (m, n))]
        ctx.gated_reserve(m, n, B, type=type_)

        def calls():
            ctx.gated(Wg, Wu, m, n, X, B, "silu", H, G, S, type=type_)
            ctx.gated_grad(Wg, Wu, m, n, X, B, "silu", G, S, D, gX, gWg, gWu, type=type_)

        ctx.graph_begin()
        try:
            calls()
        finally:
            graph = ctx.graph_end()
        for _ in range(3):
            X.upload(stored(rng.standard_normal(n * B), type_))
            ctx.graph_launch(graph)
            got = [o.download().copy() for o in outs]
            for o in outs:
                o.upload(np.zeros(o.shape, o.dtype))
            calls()
            for o, g in zip(outs, got):
                assert np.array_equal(o.download().view(np.uint8), g.view(np.uint8)) and g.any()
        ctx.graph_free(graph)
    finally:
        ctx.close()


def test_a_workspace_that_must_grow_is_refused_while_recording():
    ctx = hipabi.Context()
    try:
        a = Arrays(ctx, "f32")
        W, X, G, S, D, out = (a.put(np.ones((64, 64)))[0] for _ in range(6))
        ctx.graph_begin()
        try:
            with pytest.raises(hipabi.SoError, match="so_gated_reserve"):
                ctx.gated_grad(W, W, 64, 64, X, 64, "silu", G, S, D, out)
        finally:
            ctx.graph_free(ctx.graph_end())
        ctx.gated_grad(W, W, 64, 64, X, 64, "silu", G, S, D, out)
        assert out.download().any()
    finally:
        ctx.close()


def test_two_contexts_at_once():
    rng = np.random.default_rng(14)
    m, n, B, type_ = 300, 200, 150, "bf16"
    each = []
    contexts = [hipabi.Context() for _ in range(2)]
    try:
        for ctx in contexts:
            Wg, Wu, X, D = weights(rng, type_, m, n), weights(rng, type_, m, n), draw(rng, type_, n, B), draw(rng, type_, m, B)
            a = Arrays(ctx, type_)
            devs = [a.put(v)[0] for v in (Wg, Wu, X, D)]
            outs = [a.put(np.zeros(s))[0] for s in ((m, B), (m, B), (m, B), (n, B), (m, n), (m, n))]
            each.append((ctx, (Wg, Wu, X, D), devs, outs))
        for _ in range(5):
            for ctx, _, (Wg, Wu, X, D), (H, G, S, gX, gWg, gWu) in each:
                ctx.gated(Wg, Wu, m, n, X, B, "silu", H, G, S, type=type_)
                ctx.gated_grad(Wg, Wu, m, n, X, B, "silu", G, S, D, gX, gWg, gWu, type=type_)
        for _, (Wg, Wu, X, D), _, (H, G, S, gX, gWg, gWu) in each:
            check(fetch(H, m, B, type_)[0], forward(Wg, Wu, X, "silu", type_)["H"])
            back = backward(Wg, Wu, X, "silu", fetch(G, m, B, type_)[0], fetch(S, m, B, type_)[0], D, type_)
            check(fetch(gX, n, B, type_)[0], back["dX"])
            check(fetch(gWg, m, n, type_)[0], back["dWg"])
            check(fetch(gWu, m, n, type_)[0], back["dWu"])
    finally:
        for ctx in contexts:
            ctx.close()


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("m,n,B", [(24, 6000, 40), (16, 9001, 2), (2500, 33, 20), (33, 50, 5000), (30, 40, 3001), (700, 16, 9), (12, 700, 70)])
def test_long_contractions_over_few_tiles(ctx, m, n, B, type_):
    """A result of few tiles is made in pieces of its contraction, of n, m or B terms, which another kernel adds up: twice with the same bits."""
    rng = np.random.default_rng(m + n + B + 2)
    for pad, shift, wpad in ((0, 0, 0), (3, 1, 5), (8 - B % 8, 0, 8 - n % 8)):
        run_forward(ctx, rng, m, n, B, type_, "silu", pad, shift, wpad)
        run_backward(ctx, rng, m, n, B, type_, "gelu_tanh", pad, shift, wpad)
    a = Arrays(ctx, type_)
    Wg, Wu, X, D = (a.put(v)[0] for v in (weights(rng, type_, m, n), weights(rng, type_, m, n), draw(rng, type_, n, B), draw(rng, type_, m, B)))
    outs = [a.put(np.zeros(s))[0] for s in ((m, B), (m, B), (m, B), (n, B), (m, n), (m, n))]
    seen = []
    for _ in range(2):
        ctx.gated(Wg, Wu, m, n, X, B, "silu", *outs[:3], type=type_)
        ctx.gated_grad(Wg, Wu, m, n, X, B, "silu", outs[1], outs[2], D, *outs[3:], type=type_)
        seen.append([o.download().view(np.uint8).copy() for o in outs])
    for first, second in zip(*seen):
        assert np.array_equal(first, second)
    a.free()


@pytest.mark.parametrize("type_", TYPES)
def test_what_is_not_a_number_stays_where_it_is_in_pieces(ctx, type_):
    rng = np.random.default_rng(18)
    m, n, B = 40, 5000, 30
    Wg, Wu, X = weights(rng, type_, m, n), weights(rng, type_, m, n), draw(rng, type_, n, B)
    Wg[3, 4999], Wu[39, 0], X[2500, 7] = np.nan, np.inf, np.nan
    a = Arrays(ctx, type_)
    outs = [a.put(np.zeros((m, B)), 1)[0] for _ in range(3)]
    ctx.gated(a.put(Wg)[0], a.put(Wu)[0], m, n, a.put(X)[0], B, "silu", *outs, type=type_, h_stride=B + 1, g_stride=B + 1)
    bad = np.zeros((m, B), bool)
    bad[3], bad[39], bad[:, 7] = True, True, True
    H = fetch(outs[0], m, B, type_, 1)[0]
    assert np.array_equal(~np.isfinite(H), bad)
    a.free()


@pytest.mark.parametrize("type_", TYPES)
def test_millions_of_columns(ctx, type_):
    """Rows so long that offsets inside a tile pass 31 bits.  All but 1000 columns of dH are zero, and adding a zero is exact: the weights' gradients are sums of 1000 terms."""
    rng = np.random.default_rng(20)
    m, n, B = 3, 2, 4_300_001
    Wg, Wu, X = weights(rng, type_, m, n), weights(rng, type_, m, n), draw(rng, type_, n, B)
    dH = np.zeros((m, B))
    some = np.unique(np.append(rng.integers(0, B, 1000), [0, B - 1]))
    dH[:, some] = draw(rng, type_, m, some.size)
    a = Arrays(ctx, type_)
    dWg, dWu, dX, dDh = (a.put(v)[0] for v in (Wg, Wu, X, dH))
    H, G, S, gX, gWg, gWu = (a.put(np.zeros(s))[0] for s in ((m, B), (m, B), (m, B), (n, B), (m, n), (m, n)))
    ctx.gated(dWg, dWu, m, n, dX, B, "silu", H, G, S, type=type_)
    ctx.gated_grad(dWg, dWu, m, n, dX, B, "silu", G, S, dDh, gX, gWg, gWu, type=type_)
    want = forward(Wg, Wu, X, "silu", type_)
    check(fetch(H, m, B, type_)[0], want["H"])
    vG, vS = fetch(G, m, B, type_)[0], fetch(S, m, B, type_)[0]
    got = fetch(gX, n, B, type_)[0]
    rest = np.ones(B, bool)
    rest[some] = False
    assert not got[:, rest].any()
    back = backward(Wg, Wu, X[:, some], "silu", vG[:, some], vS[:, some], dH[:, some], type_)
    check(got[:, some], back["dX"])
    check(fetch(gWg, m, n, type_)[0], back["dWg"])
    check(fetch(gWu, m, n, type_)[0], back["dWu"])
    a.free()
