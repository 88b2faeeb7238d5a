"""Features of a head that so_head_rotary does not turn: those behind `rot`, which without a norm stay the bits that they are, whatever lies beside them, and with one are scaled each for itself."""
import numpy as np
import pytest

import hipabi
from elements import TYPES, fetch, stored
from test_gpu_gated import Arrays, draw
from test_gpu_rotary import EPS, inputs

pytestmark = pytest.mark.gpu

Q, K = 2, 1
CASES = [(64, 32, 21), (64, 0, 70), (33, 8, 9), (130, 2, 300), (300, 100, 40), (16, 6, 1)]      # D, rot, B


def mark(X, D, rot, rng):
    """An infinity, a NaN and a negative zero, each in every third of the features behind `rot`, the others as they are; -> where they are."""
    V = X.copy()
    where = np.zeros(X.shape, bool)
    for head in range(Q + K):
        some = head * D + rot + np.arange((head + 1) % 2, D - rot, 2)      # no neighbour of one is another
        for value, rows in zip((np.inf, np.nan, -0.0, -np.inf), (some[i::4] for i in range(4))):
            V[rows, -1] = value
            where[rows, -1] = True
    return V, where


def turn(ctx, type_, V, D, rot, B, layout, norm, seed, grad=False, in_place=False):
    rng = np.random.default_rng(seed)
    _, pos, freq, _, _ = inputs(rng, Q, K, D, rot, B, type_)
    a = Arrays(ctx, type_)
    dX = a.put(V)[0]
    out = dX if in_place else a.put(np.zeros(V.shape))[0]
    dPos, dFreq = ctx.array(pos, np.int32), ctx.array(freq if rot else np.zeros(1))
    if grad:
        ctx.head_rotary_grad(None, dX, Q, K, D, B, dPos, dFreq, rot, out, layout, 1.1, False, type=type_)
    else:
        ctx.head_rotary(dX, Q, K, D, B, dPos, dFreq, rot, out, layout, 1.1, norm, EPS, type=type_)
    bits = out.download().copy()
    a.free()
    dPos.free()
    dFreq.free()
    return bits.reshape(V.shape)


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("layout", ["halves", "pairs"])
@pytest.mark.parametrize("D,rot,B", CASES)
def test_without_a_norm_they_keep_their_bits(ctx, D, rot, B, layout, type_):
    rng = np.random.default_rng(D + rot)
    X = draw(rng, type_, (Q + K) * D, B)
    V, where = mark(X, D, rot, rng)
    rest = np.zeros(V.shape, bool).reshape(Q + K, D, B)
    rest[:, rot:] = True
    rest = rest.reshape(V.shape)
    bits = lambda x: x.view(np.uint32 if type_ == "f32" else np.uint16)
    want = bits(stored(V, type_))
    for grad in (False, True):
        for in_place in (False, True):
            got, clean = (bits(turn(ctx, type_, v, D, rot, B, layout, False, 7, grad, in_place)) for v in (V, X))
            nan = np.isnan(V)
            assert np.array_equal(got[rest & ~nan], want[rest & ~nan])
            floats = turn(ctx, type_, V, D, rot, B, layout, False, 7, grad, in_place)
            assert np.all(np.isnan(floats[nan]) if type_ != "bf16" else (floats[nan] & 0x7fff) > 0x7f80)
            assert np.array_equal(got[~rest], clean[~rest])


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("layout", ["halves", "pairs"])
@pytest.mark.parametrize("D,rot,B", CASES)
def test_with_a_norm_each_is_scaled_for_itself(ctx, D, rot, B, layout, type_):
    """An infinity makes its head's factor of that column 0: it becomes NaN itself, all other features zeros."""
    rng = np.random.default_rng(D + rot + 1)
    X = draw(rng, type_, (Q + K) * D, B)
    V = X.copy()
    row = D + rot + (D - rot) // 2
    V[row, -1] = -np.inf
    a = Arrays(ctx, type_)
    out = a.put(np.zeros(V.shape))[0]
    _, pos, freq, gq, gk = inputs(rng, Q, K, D, rot, B, type_)
    dPos, dFreq, dGq, dGk = ctx.array(pos, np.int32), ctx.array(freq if rot else np.zeros(1)), ctx.array(gq), ctx.array(gk)
    ctx.head_rotary(a.put(V)[0], Q, K, D, B, dPos, dFreq, rot, out, layout, 1.0, True, EPS, dGq, dGk, type=type_)
    got = fetch(out, *V.shape, type_)[0]
    head = got[D:2 * D, -1]
    assert np.array_equal(np.isnan(head), np.arange(D) == row - D) and not np.any(head[~np.isnan(head)])
    got[D:2 * D, -1] = 0.0
    assert np.isfinite(got).all()
    a.free()
    for x in (dPos, dFreq, dGq, dGk):
        x.free()


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("layout", ["halves", "pairs"])
@pytest.mark.parametrize("D,rot,B", CASES)
def test_gains_of_their_neighbours(ctx, D, rot, B, layout, type_):
    """With a norm an infinite entry of dY behind `rot` reaches its own gain's gradient and, by the head's sum, that column of dX, as an infinity of the other entries' own sign; no other gain's gradient."""
    rng = np.random.default_rng(D + rot + 2)
    X, pos, freq, gq, gk = inputs(rng, Q, K, D, rot, B, type_)
    dY = draw(rng, type_, (Q + K) * D, B, size=0.1)
    row = D + rot + (D - rot) // 2
    dPos, dFreq, dGq, dGk = ctx.array(pos, np.int32), ctx.array(freq if rot else np.zeros(1)), ctx.array(gq), ctx.array(gk)
    rstd = (1.0 / np.sqrt(np.square(X.reshape(Q + K, D, B)).mean(axis=1) + EPS)).astype(np.float32)
    dR = ctx.array(rstd)
    seen = []
    for marked in (False, True):
        if marked:
            dY = dY.copy()
            dY[row, -1] = np.inf
        a = Arrays(ctx, type_)
        out = a.put(np.zeros(X.shape))[0]
        oq, ok = ctx.empty((D,)), ctx.empty((D,))
        ctx.head_rotary_grad(a.put(X)[0], a.put(dY)[0], Q, K, D, B, dPos, dFreq, rot, out, layout, 1.0, True, dGq, dGk, dR, oq, ok, type=type_)
        seen.append((fetch(out, *X.shape, type_)[0], oq.download().copy(), ok.download().copy()))
        a.free()
        oq.free()
        ok.free()
    (dx0, q0, k0), (dx1, q1, k1) = seen
    other = np.arange(D) != row - D
    assert np.array_equal(q0[other], q1[other]) and np.array_equal(k0, k1) and not np.isfinite(q1[row - D])
    column = dx1[D:2 * D, -1]
    sign = -np.sign(X[D:2 * D, -1]) * np.sign(X[row, -1]) * np.sign(gq[row - D])
    assert np.array_equal(column[other], np.where(sign[other] < 0, -np.inf, np.inf))
    dx1[D:2 * D, -1] = dx0[D:2 * D, -1]
    assert np.array_equal(dx0, dx1)
    for x in (dPos, dFreq, dGq, dGk, dR):
        x.free()


@pytest.mark.parametrize("D,B", [(33, 40), (129, 9), (257, 300)])
def test_one_reserve_for_every_number_of_turned_features(D, B):
    """Of heads with an odd number of features: the gradient recorded behind one reserve, whatever is turned."""
    rng = np.random.default_rng(D)
    for rot in (0, 2, D - 1):
        ctx = hipabi.Context()
        try:
            X, pos, freq, gq, gk = inputs(rng, Q, K, D, rot, B, "bf16")
            a = Arrays(ctx, "bf16")
            dX, out = a.put(X)[0], a.put(np.zeros(X.shape))[0]
            dPos, dFreq, dR, oq, ok = ctx.array(pos, np.int32), ctx.array(freq if rot else np.zeros(1)), ctx.array(np.ones((Q + K, B))), ctx.empty((D,)), ctx.empty((D,))
            call = lambda: ctx.head_rotary_grad(dX, dX, Q, K, D, B, dPos, dFreq, rot, out, "pairs", 1.0, True, None, None, dR, oq, ok, type="bf16")
            ctx.head_rotary_reserve(Q, K, D, B, type="bf16")
            ctx.graph_begin()
            try:
                call()
            finally:
                graph = ctx.graph_end()
            seen = []
            for again in (lambda: ctx.graph_launch(graph), call, lambda: ctx.graph_launch(graph)):
                again()
                seen.append([o.download().copy() for o in (out, oq, ok)])
            for other in seen[1:]:
                assert all(np.array_equal(x, y) for x, y in zip(seen[0], other))
            assert seen[0][1].any() and seen[0][0].any()
            ctx.graph_free(graph)
        finally:
            ctx.close()
