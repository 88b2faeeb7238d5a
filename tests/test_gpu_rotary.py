"""so_head_rotary and so_head_rotary_grad against the formulas in float64.  What lies between and around the operands' rows is NaN, so that a value read from there shows.

Tolerances, u = 2^-24.  A sum over the features of a head runs through fewer than 40 additions one after the other (8 of a thread, 8 of a wave's lanes and waves, and what the squares and products add), so that
it is off by at most 40 u of its magnitudes.  A cosine and a sine are off by 4 u of 1: the angle is exact to less than u of a turn, times 2 pi, and the function adds a step.  Then there are at most 8
elementwise operations."""
import numpy as np
import pytest

import hipabi
from elements import HALF_STEP, SMALLEST, TYPES, U, fetch, fetch_apart, place, place_apart, stored, values
from hipabi import SO_ERR_INVALID
from test_gpu_gated import PLACES, Arrays, draw

pytestmark = pytest.mark.gpu

EPS = 1e-6
TRIG = 10 * U                 # 2 pi u of the angle and a step of the function, for the cosine and the sine each
# (heads_q, heads_k, D, rot, B)
SHAPES = [(1, 0, 1, 0, 1), (0, 1, 2, 2, 3), (1, 1, 3, 2, 7), (2, 1, 16, 16, 1), (4, 2, 64, 64, 8), (3, 1, 80, 50, 9), (2, 2, 128, 128, 17), (5, 1, 33, 8, 40), (8, 8, 128, 64, 1), (1, 3, 256, 256, 70),
          (2, 1, 130, 130, 33), (2, 1, 511, 500, 21), (1, 1, 512, 512, 130), (1, 2, 300, 128, 1), (7, 1, 96, 96, 200), (3, 2, 64, 32, 1030), (40, 8, 64, 64, 2000)]


def inputs(rng, q, k, D, rot, B, type_):
    X = draw(rng, type_, (q + k) * D, B)
    pos = (rng.integers(0, 2 ** 20) + np.arange(B)).astype(np.int32)
    pos[rng.integers(0, B)] = rng.choice([0, -5, 2 ** 31 - 1, -2 ** 31])
    freq = (10000.0 ** (-np.arange(rot // 2) / max(rot // 2, 1)) * rng.uniform(0.5, 1.0, rot // 2)).astype(np.float32)
    return X, pos, freq, (1 + 0.2 * rng.standard_normal(D)).astype(np.float32), (1 + 0.2 * rng.standard_normal(D)).astype(np.float32)


def turned(x, pos, freq, rot, layout, amplitude, back=False):
    """x [heads, D, B], the first rot features of every head turned; and the magnitudes that went into each entry."""
    turns = freq.astype(np.float64)[:, None] * pos.astype(np.float64)[None, :]
    c, s = amplitude * np.cos(turns), amplitude * np.sin(turns) * (-1 if back else 1)
    i = np.arange(rot // 2)
    first, second = (i, i + rot // 2) if layout == "halves" else (2 * i, 2 * i + 1)
    out, mag = x.copy(), np.abs(x)
    a, b = x[:, first], x[:, second]
    out[:, first], out[:, second] = a * c - b * s, b * c + a * s
    mag[:, first] = mag[:, second] = (np.abs(a) + np.abs(b)) * abs(amplitude)
    return out, mag


def gains_of(q, k, gain_q, gain_k):
    D = gain_q.size
    return np.concatenate([np.broadcast_to(gain_q.astype(np.float64), (q, D)), np.broadcast_to(gain_k.astype(np.float64), (k, D))])[:, :, None]


def forward(X, q, k, D, pos, freq, rot, layout, amplitude, norm, gain_q, gain_k, type_, eps=EPS):
    """-> (Y, its tolerance, rstd)"""
    x = X.reshape(q + k, D, -1)
    r = None
    if norm:
        r = 1.0 / np.sqrt(np.square(x).mean(axis=1) + np.float64(np.float32(eps)))
        x = x * r[:, None] * gains_of(q, k, gain_q, gain_k)
    amplitude = np.float64(np.float32(amplitude))
    y, mag = turned(x, pos, freq, rot, layout, amplitude)
    off = mag * (TRIG + U * (40 + 8))
    tol = off + HALF_STEP[type_] * (np.abs(y) + off) + SMALLEST[type_]
    if not norm:
        tol[:, rot:] = 0.0                                     # what is not touched
    return y.reshape(X.shape), tol.reshape(X.shape), r


def run_forward(ctx, rng, q, k, D, rot, B, type_, layout, norm, amplitude=1.1, pad=0, shift=0, in_place=False, gains=True):
    X, pos, freq, gain_q, gain_k = inputs(rng, q, k, D, rot, B, type_)
    rows = (q + k) * D
    a = Arrays(ctx, type_)
    whole, dX = a.put(X, pad, shift, fill=-5.0 if in_place else np.nan)
    out, dY = (whole, dX) if in_place else a.put(np.zeros((rows, B)), pad + 1, shift, fill=-5.0)
    ypad = pad if in_place else pad + 1
    dPos, dFreq = ctx.array(pos, np.int32), ctx.array(freq if rot else np.zeros(1))
    dR, dGq, dGk = ctx.array(np.full((q + k, B), -7.0)), ctx.array(gain_q), ctx.array(gain_k)
    ctx.head_rotary(dX, q, k, D, B, dPos if rot else None, dFreq if rot else None, rot, dY, layout, amplitude, norm, EPS, dGq if gains else None, dGk if gains else None, dR, type=type_,
                    x_stride=B + pad, y_stride=B + ypad)
    got, rest = fetch(out, rows, B, type_, ypad, shift)
    ones = np.ones(D, np.float32)
    want, tol, r = forward(X, q, k, D, pos, freq, rot, layout, amplitude, norm, gain_q if gains else ones, gain_k if gains else ones, type_)
    assert np.all(np.abs(got - want) <= tol), np.nanmax(np.abs(got - want) / np.maximum(tol, 1e-300))
    assert np.all(rest == -5.0), "places that are not the result's were written"
    if norm:
        assert np.all(np.abs(dR.download() - r) <= 44 * U * r)
    else:
        assert np.all(dR.download() == -7.0)
    a.free()
    for x in (dPos, dFreq, dR, dGq, dGk):
        x.free()


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("q,k,D,rot,B", SHAPES)
def test_forward(ctx, q, k, D, rot, B, type_):
    rng = np.random.default_rng(q + 10 * k + D + rot + B)
    for i, (pad, shift) in enumerate(PLACES):
        for norm in (False, True):
            run_forward(ctx, rng, q, k, D, rot, B, type_, ("halves", "pairs")[(i + norm) % 2], norm, pad=pad, shift=shift, in_place=i == 2, gains=i != 1)


def backward(X, dY, q, k, D, pos, freq, rot, layout, amplitude, norm, gain_q, gain_k, rstd, type_):
    """-> {name: (value, tolerance)}; rstd is what the call was given"""
    amplitude = np.float64(np.float32(amplitude))
    g, mag = turned(dY.reshape(q + k, D, -1), pos, freq, rot, layout, amplitude, back=True)
    g_off = mag * (TRIG + 4 * U)
    if not norm:
        tol = g_off + HALF_STEP[type_] * (np.abs(g) + g_off) + SMALLEST[type_]
        tol[:, rot:] = 0.0
        return {"dX": (g.reshape(X.shape), tol.reshape(X.shape))}
    gain, r = gains_of(q, k, gain_q, gain_k), rstd.astype(np.float64)[:, None]
    h = X.reshape(q + k, D, -1) * r
    inner = (g * gain * h).mean(axis=1, keepdims=True)
    inner_off = (g_off * np.abs(gain * h)).mean(axis=1, keepdims=True) + 48 * U * (mag * np.abs(gain * h)).mean(axis=1, keepdims=True)
    dX = r * (g * gain - h * inner)
    off = r * (g_off * np.abs(gain) + np.abs(h) * inner_off + 8 * U * (np.abs(g * gain) + np.abs(h * inner)))
    each, each_off = (g * h).sum(axis=2), (g_off * np.abs(h)).sum(axis=2)
    # a gain's gradient: a thread adds its columns' and heads' one after the other, then lanes, then shares of workgroups; fewer than B + heads additions in all
    each_off = each_off + 2 * U * (X.shape[1] + q + k + 16) * (mag * np.abs(h)).sum(axis=2)
    tol = off + HALF_STEP[type_] * (np.abs(dX) + off) + SMALLEST[type_]
    return {"dX": (dX.reshape(X.shape), tol.reshape(X.shape)), "dq": (each[:q].sum(axis=0), each_off[:q].sum(axis=0)), "dk": (each[q:].sum(axis=0), each_off[q:].sum(axis=0))}


def run_backward(ctx, rng, q, k, D, rot, B, type_, layout, norm, amplitude=0.9, pad=0, shift=0, in_place=None, gains=True, wanted=("dX", "dq", "dk")):
    X, pos, freq, gain_q, gain_k = inputs(rng, q, k, D, rot, B, type_)
    rows = (q + k) * D
    dY = draw(rng, type_, rows, B, size=0.1)
    rstd = (1.0 / np.sqrt(np.square(X.reshape(q + k, D, B)).mean(axis=1) + EPS)).astype(np.float32)
    a = Arrays(ctx, type_)
    pads = {"X": pad, "dY": pad + 2}
    x_whole, dX = a.put(X, pads["X"], shift, fill=-5.0 if in_place == "X" else np.nan)
    d_whole, dDy = a.put(dY, pads["dY"], shift, fill=-5.0 if in_place == "dY" else np.nan)
    if in_place:
        (out, dDx), opad = {"X": (x_whole, dX), "dY": (d_whole, dDy)}[in_place], pads[in_place]
    else:
        (out, dDx), opad = a.put(np.zeros((rows, B)), pad + 1, shift, fill=-5.0), pad + 1
    others = [ctx.array(pos, np.int32), ctx.array(freq if rot else np.zeros(1)), ctx.array(rstd), ctx.array(gain_q), ctx.array(gain_k), ctx.array(np.full(D, -7.0)), ctx.array(np.full(D, -7.0))]
    dPos, dFreq, dR, dGq, dGk, dQ, dK = others
    ctx.head_rotary_grad(dX, dDy, q, k, D, B, dPos, dFreq, rot, dDx if "dX" in wanted else None, layout, amplitude, norm, dGq if gains else None, dGk if gains else None, dR,
                         dQ if "dq" in wanted else None, dK if "dk" in wanted else None, type=type_, x_stride=B + pads["X"], dy_stride=B + pads["dY"], dx_stride=B + opad)
    ones = np.ones(D, np.float32)
    want = backward(X, dY, q, k, D, pos, freq, rot, layout, amplitude, norm, gain_q if gains else ones, gain_k if gains else ones, rstd, type_)
    got, rest = fetch(out, rows, B, type_, opad, shift)
    results = {"dX": got, "dq": dQ.download().astype(np.float64), "dk": dK.download().astype(np.float64)}
    for name, result in results.items():
        if name in wanted and name in want:
            value, tol = want[name]
            assert np.all(np.abs(result - value) <= tol), (name, np.nanmax(np.abs(result - value) / np.maximum(tol, 1e-300)))
        elif name != "dX":
            assert np.all(result == -7.0)
        else:
            assert not result.any()
    assert np.all(rest == -5.0), "places that are not the result's were written"
    a.free()
    for x in others:
        x.free()


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("q,k,D,rot,B", SHAPES)
def test_backward(ctx, q, k, D, rot, B, type_):
    rng = np.random.default_rng(q + 10 * k + D + rot + B + 1)
    for i, (pad, shift) in enumerate(PLACES):
        for norm in (False, True):
            run_backward(ctx, rng, q, k, D, rot, B, type_, ("pairs", "halves")[(i + norm) % 2], norm, pad=pad, shift=shift, in_place=(None, "X" if norm else "dY", "dY")[i], gains=i != 1)


@pytest.mark.parametrize("wanted", [("dX",), ("dq",), ("dk",), ("dq", "dk"), ("dX", "dk"), ()])
def test_any_result_may_be_left_out(ctx, wanted):
    rng = np.random.default_rng(2)
    for B in (1, 50):
        run_backward(ctx, rng, 3, 2, 48, 32, B, "bf16", "halves", True, wanted=wanted)


def test_gradient_against_differences(ctx):
    """The sum of D * Y along directions of X and of the gains: fp32 and bf16 apart, the differences of the formula in float64 are exact to 1e-7 of the scale, the fp32 gradient to 1e-4."""
    rng = np.random.default_rng(3)
    q, k, D, rot, B = 3, 2, 24, 16, 30
    for layout in ("halves", "pairs"):
        X, pos, freq, gq, gk = inputs(rng, q, k, D, rot, B, "f32")
        pos = np.arange(B, dtype=np.int32)
        C = draw(rng, "f32", (q + k) * D, B)
        loss = lambda X, gq, gk: float((C * forward(X, q, k, D, pos, freq, rot, layout, 1.0, True, gq, gk, "f32")[0]).sum())
        a = Arrays(ctx, "f32")
        dX, dC, dY, dDx = a.put(X)[0], a.put(C)[0], a.put(np.zeros(X.shape))[0], a.put(np.zeros(X.shape))[0]
        dPos, dFreq, dR, dGq, dGk, dQ, dK = ctx.array(pos, np.int32), ctx.array(freq), ctx.empty((q + k, B)), ctx.array(gq), ctx.array(gk), ctx.empty((D,)), ctx.empty((D,))
        ctx.head_rotary(dX, q, k, D, B, dPos, dFreq, rot, dY, layout, 1.0, True, EPS, dGq, dGk, dR)
        ctx.head_rotary_grad(dX, dC, q, k, D, B, dPos, dFreq, rot, dDx, layout, 1.0, True, dGq, dGk, dR, dQ, dK)
        for at, grad in enumerate((dDx, dQ, dK)):
            got = grad.download().astype(np.float64).reshape((X, gq, gk)[at].shape)
            along = got * (rng.random(got.shape) < 0.5)
            moved = lambda s: [v + (s * along if i == at else 0.0) for i, v in enumerate((X, gq.astype(np.float64), gk.astype(np.float64)))]
            difference = (loss(*moved(1e-5)) - loss(*moved(-1e-5))) / 2e-5
            assert abs(float((got * along).sum()) - difference) <= 1e-4 * np.linalg.norm(got) * np.linalg.norm(along), (layout, at)
        a.free()


@pytest.mark.parametrize("type_", TYPES)
def test_what_is_not_a_number_stays_where_it_is(ctx, type_):
    """NaN in a head of a column: with a norm that head of that column, without one the pair that it is turned with; everything else has the same bits."""
    rng = np.random.default_rng(4)
    q, k, D, rot = 3, 1, 64, 32
    for B in (1, 21, 70):
        X, pos, freq, gq, gk = inputs(rng, q, k, D, rot, B, type_)
        for norm in (False, True):
            seen = []
            for marked in (False, True):
                V = X.copy()
                if marked:
                    V[2 * D + 3, B - 1] = np.nan
                a = Arrays(ctx, type_)
                out, dY = a.put(np.zeros(X.shape))
                ctx.head_rotary(a.put(V)[1], q, k, D, B, ctx.array(pos, np.int32), ctx.array(freq), rot, dY, "halves", 1.0, norm, EPS, type=type_)
                seen.append(fetch(out, *X.shape, type_)[0])
                a.free()
            bad = np.zeros(X.shape, bool)
            bad[2 * D:3 * D, B - 1] = norm
            bad[[2 * D + 3, 2 * D + 3 + rot // 2], B - 1] = True
            assert np.array_equal(np.isnan(seen[1]), bad)
            assert np.array_equal(seen[0][~bad], seen[1][~bad])


def test_extremes(ctx):
    """A head of zeros with and without eps's help, and values whose squares leave fp32: a head beyond 2^64 has an infinite sum and becomes zeros, as the formula in fp32 has it."""
    D, B = 32, 3
    X = np.zeros((D, B), np.float32)
    X[:, 1], X[:, 2] = 1e-12, 3e25
    dX, dY, dR = ctx.array(X), ctx.empty((D, B)), ctx.empty((1, B))
    ctx.head_rotary(dX, 1, 0, D, B, None, None, 0, dY, "halves", 1.0, True, 1e-6, None, None, dR)
    Y = dY.download()
    assert not Y[:, 0].any() and np.allclose(Y[:, 1], 1e-9, rtol=1e-6, atol=0) and not Y[:, 2].any()
    assert np.allclose(dR.download()[0, :2], 1000.0, rtol=1e-6) and dR.download()[0, 2] == 0.0


def test_rows_far_apart(ctx):
    rng = np.random.default_rng(5)
    far, type_ = 2 ** 28 + 3, "bf16"
    q, k, D, rot, B = 2, 1, 6, 4, 5
    X, pos, freq, gq, gk = inputs(rng, q, k, D, rot, B, type_)
    rows = (q + k) * D
    dX, dY = place_apart(ctx, X, type_, far), place_apart(ctx, np.zeros((rows, B)), type_, far)
    dPos, dFreq, dGq, dGk, dR = ctx.array(pos, np.int32), ctx.array(freq), ctx.array(gq), ctx.array(gk), ctx.empty((q + k, B))
    ctx.head_rotary(dX, q, k, D, B, dPos, dFreq, rot, dY, "pairs", 1.0, True, EPS, dGq, dGk, dR, type=type_, x_stride=far, y_stride=far)
    want, tol, _ = forward(X, q, k, D, pos, freq, rot, "pairs", 1.0, True, gq, gk, type_)
    got = fetch_apart(ctx, dY, rows, B, type_, far)
    assert np.all(np.abs(got - want) <= tol)
    ctx.head_rotary_grad(dX, dY, q, k, D, B, dPos, dFreq, rot, dX, "pairs", 1.0, True, dGq, dGk, dR, type=type_, x_stride=far, dy_stride=far, dx_stride=far)
    value, tol = backward(X, got, q, k, D, pos, freq, rot, "pairs", 1.0, True, gq, gk, dR.download(), type_)["dX"]
    assert np.all(np.abs(fetch_apart(ctx, dX, rows, B, type_, far) - value) <= tol)
    dX.free()
    dY.free()


def test_refusals_and_empty_sizes(ctx):
    a = Arrays(ctx, "f32")
    X, D_ = (a.put(np.ones((16, 8)))[0] for _ in range(2))
    Y = a.put(np.full((16, 8), 3.0))[0]
    pos, freq, R, gq, gk = ctx.array(np.zeros(8), np.int32), ctx.array(np.ones(4)), ctx.array(np.ones((2, 8))), ctx.array(np.full(8, 2.0)), ctx.array(np.full(8, 2.0))
    base = dict(X=X, q=1, k=1, D=8, B=8, pos=pos, freq=freq, rot=8, Y=Y)

    def fwd(norm=False, eps=EPS, dRstd=None, layout="halves", **k):
        v = {**base, **{n: k.pop(n) for n in list(k) if n in base}}
        ctx.head_rotary(v["X"], v["q"], v["k"], v["D"], v["B"], v["pos"], v["freq"], v["rot"], v["Y"], layout, 1.0, norm, eps, None, None, dRstd, **k)

    def bwd(norm=True, dRstd=R, dDgainQ=None, dDgainK=None, dY=D_, **k):
        v = {**base, **{n: k.pop(n) for n in list(k) if n in base}}
        ctx.head_rotary_grad(v["X"], dY, v["q"], v["k"], v["D"], v["B"], v["pos"], v["freq"], v["rot"], v["Y"], "halves", 1.0, norm, gq, gk, dRstd, dDgainQ, dDgainK, **k)

    def refused(call, text, **k):
        with pytest.raises(hipabi.SoError) as e:
            call(**k)
        assert e.value.status == SO_ERR_INVALID and text in str(e.value), e.value

    for call in (fwd, bwd):
        refused(call, "even number", rot=7)
        refused(call, "even number", rot=10)
        refused(call, "features a head", D=0, rot=0)
        refused(call, "features a head", D=513)
        refused(call, "heads", q=2 ** 31, k=2 ** 31)
        refused(call, "null positions", pos=None)
        refused(call, "null positions", freq=None)
        refused(call, "null", X=None)
        refused(call, "stride", x_stride=7)
    refused(fwd, "null", Y=None)
    refused(fwd, "stride", y_stride=7)
    refused(fwd, "one stride", Y=X, B=4, x_stride=8, y_stride=4)
    refused(fwd, "eps", norm=True, eps=-1.0)
    refused(fwd, "eps", norm=True, eps=float("nan"))
    refused(fwd, "both results", norm=True, dRstd=Y)
    refused(bwd, "null factors", dRstd=None)
    refused(bwd, "null", dY=None)
    refused(bwd, "stride", dy_stride=7)
    refused(bwd, "stride", dx_stride=7)
    refused(bwd, "two results", dDgainQ=gq, dDgainK=gq)
    refused(bwd, "two results", dDgainQ=Y)
    refused(bwd, "is an input", dDgainQ=gq)
    with pytest.raises(hipabi.SoError, match="layout"):
        ctx._ck(ctx.lib.so_head_rotary(ctx.h, 0, 1, 1, 8, 8, X.ptr, 8, 0, None, None, 0.0, pos.ptr, freq.ptr, 8, 1.0, 2, Y.ptr, 8, None))
    with pytest.raises(hipabi.SoError, match="element type"):
        ctx.head_rotary_reserve(1, 1, 8, 8, type="f32") or ctx._ck(ctx.lib.so_head_rotary_reserve(ctx.h, 9, 1, 1, 8, 8))
    fwd(q=0, k=0)
    fwd(B=0)
    bwd(B=0)
    assert np.all(Y.download() == 3.0)
    zeros = ctx.array(np.full(8, 5.0))
    bwd(B=0, dDgainQ=zeros)                                    # no columns: the gains' gradients are zeros
    assert not zeros.download().any()
    zeros.upload(np.full(8, 5.0))
    bwd(k=0, dDgainK=zeros)                                    # no keys
    assert not zeros.download().any()
    a.free()


@pytest.mark.parametrize("type_,q,k,D,rot,B", [("f32", 3, 2, 64, 64, 90), ("bf16", 4, 1, 128, 64, 300), ("f16", 2, 2, 80, 40, 1)])
def test_recorded_ahead_of_the_first_launch(type_, q, k, D, rot, B):
    """Recorded on a fresh context behind the reserve, replayed with new values and positions: the bits of eager calls."""
    rng = np.random.default_rng(D)
    ctx = hipabi.Context()
    try:
        X, pos, freq, gq, gk = inputs(rng, q, k, D, rot, B, type_)
        a = Arrays(ctx, type_)
        dX, dD, dY, dDx = (a.put(v)[0] for v in (X, draw(rng, type_, *X.shape), np.zeros(X.shape), np.zeros(X.shape)))
        dPos, dFreq, dR, dGq, dGk, dQ, dK = ctx.array(pos, np.int32), ctx.array(freq), ctx.empty((q + k, B)), ctx.array(gq), ctx.array(gk), ctx.empty((D,)), ctx.empty((D,))
        ctx.head_rotary_reserve(q, k, D, B, type=type_)

        def calls():
            ctx.head_rotary(dX, q, k, D, B, dPos, dFreq, rot, dY, "halves", 1.0, True, EPS, dGq, dGk, dR, type=type_)
            ctx.head_rotary_grad(dX, dD, q, k, D, B, dPos, dFreq, rot, dDx, "halves", 1.0, True, dGq, dGk, dR, dQ, dK, type=type_)

        ctx.graph_begin()
        try:
            calls()
        finally:
            graph = ctx.graph_end()
        outs = (dY, dR, dDx, dQ, dK)
        for _ in range(3):
            dX.upload(stored(rng.standard_normal(X.size), type_))
            dPos.upload(rng.integers(0, 1 << 20, B).astype(np.int32))
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


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("q,k,D,rot,B", [(3, 2, 32, 32, 4161), (1, 1, 16, 8, 8300), (2, 0, 130, 20, 4200), (0, 1, 300, 300, 4100)])
def test_many_tiles_of_columns(ctx, q, k, D, rot, B, type_):
    rng = np.random.default_rng(B + D)
    for pad, shift in ((0, 0), (3, 1), (128 - B % 64, 0)):
        run_forward(ctx, rng, q, k, D, rot, B, type_, "halves", pad != 3, pad=pad, shift=shift)
        run_backward(ctx, rng, q, k, D, rot, B, type_, "pairs", pad != 3, pad=pad, shift=shift, in_place=(None, "X", "dY")[pad % 3])
