"""so_adapters against the formula in float64.  What lies between and around the operands' rows is NaN, so that a value read from there shows.

Tolerances, u = 2^-24.  A_a x is a sum of n products in fp32, off by at most 2 u (n + 16) of their magnitudes (n + 16 additions of a step each, which a matrix instruction may cut off); of the 16-bit types it
goes into the second product as two numbers of that type, which hold it to 2^-16.  That product is a sum of `rank` of them (twice as many for 16 bits), and the scale and the base are one operation each; a
16-bit result is rounded once more, by half a step."""
import numpy as np
import pytest

import hipabi
from elements import HALF_STEP, SMALLEST, TYPES, U, fetch, fetch_apart, place, place_apart, stored, values
from hipabi import SO_ERR_INVALID
from test_gpu_gated import PLACES, Arrays, draw

pytestmark = pytest.mark.gpu

# (m, n, C, count, rank)
SHAPES = [(1, 1, 1, 1, 1), (5, 7, 3, 2, 1), (64, 64, 64, 4, 8), (70, 130, 1, 3, 16), (33, 300, 17, 40, 5), (257, 129, 70, 5, 10), (130, 515, 200, 7, 33), (300, 96, 40, 2, 64), (90, 1100, 24, 9, 100),
          (48, 40, 30, 3, 256), (1000, 70, 65, 3, 16), (64, 4133, 20, 6, 4), (520, 264, 600, 3, 16), (264, 1032, 1030, 4, 24), (16, 64, 5, 70, 8)]


def problem(rng, m, n, C, count, rank, type_):
    A, B = draw(rng, type_, count, rank, n, size=n ** -0.5), draw(rng, type_, count, m, rank, size=rank ** -0.5)
    return A, B, (0.5 + rng.random(count)).astype(np.float32), draw(rng, type_, n, C), draw(rng, type_, m, C)


def check(got, A, B, scale, which, X, base, type_):
    count, m, rank = B.shape
    n = X.shape[0]
    want = np.zeros((m, X.shape[1])) if base is None else base.copy()
    off = np.zeros_like(want)
    for a in np.unique(which):
        if not 0 <= a < count:
            continue
        c = which == a
        s = 1.0 if scale is None else np.float64(scale[a])
        T, T_off = A[a] @ X[:, c], 2 * U * (n + 16) * (np.abs(A[a]) @ np.abs(X[:, c]))
        if type_ != "f32":
            T_off = T_off + 2.0 ** -16 * np.abs(T)
        D, mag = s * (B[a] @ T), np.abs(s) * (np.abs(B[a]) @ (np.abs(T) + T_off))
        off[:, c] = np.abs(s) * (np.abs(B[a]) @ T_off) + 2 * U * (2 * rank + 16) * mag + U * (np.abs(want[:, c]) + np.abs(D))
        want[:, c] += D
    tol = off + HALF_STEP[type_] * (np.abs(want) + off) + SMALLEST[type_]
    untouched = ~((which >= 0) & (which < count))
    assert np.array_equal(got[:, untouched], want[:, untouched])
    assert np.all(np.abs(got - want) <= tol), (np.nanmax(np.abs(got - want) / tol), int(np.isnan(got).sum()))


def run(ctx, A, B, scale, which, X, base, type_, pad=0, shift=0, in_place=False):
    """-> the result's values"""
    count, m, rank = B.shape
    n, C = X.shape
    a = Arrays(ctx, type_)
    dA, dB, dX = a.put(A.reshape(-1, n), 0, shift)[1], a.put(B.reshape(-1, rank), 0, shift)[1], a.put(X, pad, shift)[1]
    dS = None if scale is None else ctx.array(scale)
    dW = ctx.array(which, np.int32)
    out, dY = a.put(np.zeros((m, C)) if not in_place else base, pad + 2, shift, fill=-5.0)
    dBase = None if base is None else dY if in_place else a.put(base, pad + 1, shift)[1]
    ctx.adapters(dA, dB, dS, count, rank, dW, m, n, dX, C, dBase, dY, type=type_, x_stride=C + pad, base_stride=C + pad + (2 if in_place else 1), y_stride=C + pad + 2)
    got, rest = fetch(out, m, C, type_, pad + 2, shift)
    assert np.all(rest == -5.0), "places that are not the result's were written"
    a.free()
    dW.free()
    if dS:
        dS.free()
    return got


def requests(rng, C, count):
    """Runs of columns with one adapter, some without, some with a number that no adapter has."""
    numbers = rng.integers(-1, count + 1, C)
    start = rng.random(C) < rng.choice([0.02, 0.3, 1.0])
    start[0] = True
    return numbers[np.maximum.accumulate(np.where(start, np.arange(C), 0))].astype(np.int32)


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("m,n,C,count,rank", SHAPES)
def test_against_the_formula(ctx, m, n, C, count, rank, type_):
    rng = np.random.default_rng(m + n + C + rank)
    for i, (pad, shift) in enumerate(PLACES):
        A, B, scale, X, base = problem(rng, m, n, C, count, rank, type_)
        which = requests(rng, C, count)
        which[0] = i % count
        base = None if i == 1 else base
        scale = None if i == 2 else scale
        check(run(ctx, A, B, scale, which, X, base, type_, pad, shift, in_place=i == 2), A, B, scale, which, X, base, type_)


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("C", [1, 16, 33, 64, 65, 130, 257])
def test_however_the_columns_are_shared(ctx, C, type_):
    """One adapter for all, one for each, in turn, all but one without, numbers far out of range."""
    rng = np.random.default_rng(C)
    m, n, count, rank = 80, 72, 300, 12
    A, B, scale, X, base = problem(rng, m, n, C, count, rank, type_)
    alone = np.full(C, -1)
    alone[C // 2] = 7
    for which in (np.full(C, 3), rng.permutation(count)[:C], np.arange(C) % 5, np.arange(C) % 2 * 9, alone, np.full(C, -1), rng.choice([-2 ** 31, -7, count, 2 ** 31 - 1, 0], C)):
        check(run(ctx, A, B, scale, which.astype(np.int32), X, base, type_), A, B, scale, which, X, base, type_)


@pytest.mark.parametrize("type_", TYPES)
def test_a_column_does_not_depend_on_the_others(ctx, type_):
    """A column's result has the same bits whatever its neighbours' adapters and values are, NaN and infinities among them."""
    rng = np.random.default_rng(3)
    for m, n, C, count, rank in ((70, 140, 50, 6, 9), (130, 300, 200, 4, 16), (40, 64, 70, 3, 40)):
        A, B, scale, X, base = problem(rng, m, n, C, count, rank, type_)
        which = rng.integers(0, count - 1, C).astype(np.int32)
        mine = rng.random(C) < 0.4
        mine[0] = True
        first = run(ctx, A, B, scale, which, X, base, type_)
        A2, B2, X2, base2, which2 = A.copy(), B.copy(), X.copy(), base.copy(), which.copy()
        which2[~mine] = rng.integers(-1, count + 1, int((~mine).sum()))
        A2[count - 1], B2[count - 1] = np.nan, np.inf
        X2[:, ~mine], base2[:, ~mine] = rng.choice([np.nan, np.inf, -np.inf, 1.0], (n, int((~mine).sum()))), np.nan
        second = run(ctx, A2, B2, scale, which2, X2, base2, type_)
        assert np.array_equal(first[:, mine], second[:, mine])


@pytest.mark.parametrize("type_", TYPES)
def test_what_is_not_a_number_stays_where_it_is(ctx, type_):
    """NaN in a column of X, or in a row of an adapter's A, marks the columns that read it, one in a row of its B that row of its columns, one in base its entry."""
    rng = np.random.default_rng(4)
    m, n, C, count, rank = 75, 133, 90, 4, 10
    A, B, scale, X, base = problem(rng, m, n, C, count, rank, type_)
    which = (np.arange(C) // 10 % (count + 1)).astype(np.int32)
    A[1, rank - 1, n - 1], B[2, m - 1, 0], X[n - 1, 5], X[0, 45], base[3, 89] = np.nan, np.nan, np.nan, np.nan, np.nan
    bad = np.zeros((m, C), bool)
    bad[:, which == 1], bad[m - 1, which == 2], bad[:, 5], bad[3, 89] = True, True, True, True      # column 45 has no adapter
    assert which[45] == count
    assert np.array_equal(np.isnan(run(ctx, A, B, scale, which, X, base, type_)), bad)


def test_values_beyond_the_types_range(ctx):
    """A x far beyond what fp16 holds, and far below it, where the result is not: sums are kept in fp32."""
    rng = np.random.default_rng(5)
    for type_ in ("f16", "bf16"):
        for size in (300.0, 2.0 ** -12):
            m, n, C, count, rank = 40, 256, 20, 3, 8
            A, B, scale, X, base = problem(rng, m, n, C, count, rank, type_)
            A, X, B = values(stored(A * 16 * size, type_), type_), values(stored(X * size, type_), type_), values(stored(B / 4096 if size > 1 else B * 1024, type_), type_)
            which = (np.arange(C) % count).astype(np.int32)
            check(run(ctx, A, B, scale, which, X, base, type_), A, B, scale, which, X, base, type_)


def test_adapters_beyond_32_bits(ctx):
    """The last of 34 adapters begins 2^32 entries and more into A: only the used ones are written."""
    rng = np.random.default_rng(6)
    n, rank, count, m, C, type_ = 1 << 20, 128, 34, 24, 5, "bf16"
    whole = ctx.empty((count * rank * n,), np.uint16)
    A = draw(rng, type_, 1, rank, 64, size=0.2)
    line = np.zeros((rank, n), np.uint16)
    line[:, -64:] = stored(A[0], type_)
    at = whole.offset((count - 1) * rank * n)
    ctx._ck(ctx.lib.so_h2d(ctx.h, at.ptr, line.ctypes.data, line.nbytes))
    X = np.zeros((n, C))
    X[-64:] = draw(rng, type_, 64, C)
    B, base = draw(rng, type_, count, m, rank, size=0.1), draw(rng, type_, m, C)
    a = Arrays(ctx, type_)
    dX, dB, dBase, Y = a.put(X)[0], a.put(B.reshape(-1, rank))[0], a.put(base)[0], a.put(np.zeros((m, C)))[0]
    which = np.full(C, count - 1, np.int32)
    ctx.adapters(whole, dB, None, count, rank, ctx.array(which, np.int32), m, n, dX, C, dBase, Y, type=type_)
    check(fetch(Y, m, C, type_)[0], np.concatenate([np.zeros((count - 1, rank, 64)), A]), B, None, which, X[-64:], base, type_)
    a.free()
    whole.free()


def test_rows_far_apart(ctx):
    rng = np.random.default_rng(7)
    far, type_ = 2 ** 28 + 3, "f16"
    m, n, C, count, rank = 12, 20, 3, 2, 4
    A, B, scale, X, base = problem(rng, m, n, C, count, rank, type_)
    which = np.array([1, -1, 0], np.int32)
    dX, dY = place_apart(ctx, X, type_, far), place_apart(ctx, base, type_, far)
    a = Arrays(ctx, type_)
    ctx.adapters(a.put(A.reshape(-1, n))[0], a.put(B.reshape(-1, rank))[0], ctx.array(scale), count, rank, ctx.array(which, np.int32), m, n, dX, C, dY, dY, type=type_, x_stride=far, base_stride=far,
                 y_stride=far)
    check(fetch_apart(ctx, dY, m, C, type_, far), A, B, scale, which, X, base, type_)
    a.free()
    dX.free()
    dY.free()


def test_empty_sizes_and_refusals(ctx):
    a = Arrays(ctx, "f32")
    A, B, X, base = (a.put(np.ones((8, 8)))[0] for _ in range(4))
    Y = a.put(np.full((8, 8), 3.0))[0]
    which = ctx.array(np.zeros(8), np.int32)
    call = lambda **k: ctx.adapters(*(k.get(v, d) for v, d in (("A", A), ("B", B), ("scale", None), ("count", 1), ("rank", 8), ("which", which), ("m", 8), ("n", 8), ("X", X), ("C", 8), ("base", base),
                                                              ("Y", Y))), **{v: k[v] for v in ("x_stride", "base_stride", "y_stride") if v in k})
    call(m=0)
    call(C=0)
    assert np.all(Y.download() == 3.0)

    def refused(text, **k):
        with pytest.raises(hipabi.SoError) as e:
            call(**k)
        assert e.value.status == SO_ERR_INVALID and text in str(e.value), e.value

    for name in ("A", "B", "which", "X", "Y"):
        refused("null", **{name: None})
    for name in ("x_stride", "base_stride", "y_stride"):
        refused("stride", **{name: 7})
    refused("rank", rank=0)
    refused("rank", rank=257)
    refused("no input features", n=0)
    refused("is an input", Y=X)
    refused("is an input", Y=A)
    refused("is an input", Y=B)
    refused("one stride", base=Y, base_stride=8, y_stride=9, m=4, C=4)
    with pytest.raises(hipabi.SoError, match="element type"):
        ctx._ck(ctx.lib.so_adapters(ctx.h, 3, 8, 8, 8, 1, 8, A.ptr, B.ptr, None, which.ptr, X.ptr, 8, base.ptr, 8, Y.ptr, 8))
    with pytest.raises(hipabi.SoError, match="rank"):
        ctx.adapters_reserve(8, 8, 8, 0)
    assert np.all(Y.download() == 3.0)
    call(count=0, A=None, B=None)                              # no adapters at all: the base
    assert np.all(Y.download() == 1.0)
    call(count=0, A=None, B=None, base=None)
    assert not Y.download().any()
    a.free()


@pytest.mark.parametrize("type_,m,n,C,rank", [("f32", 100, 130, 70, 6), ("bf16", 520, 256, 300, 16), ("f16", 90, 77, 1, 40)])
def test_recorded_ahead_of_the_first_launch(type_, m, n, C, rank):
    """Recorded on a fresh context behind the reserve, replayed with new columns and new requests."""
    rng = np.random.default_rng(m)
    ctx = hipabi.Context()
    try:
        count = 5
        A, B, scale, X, base = problem(rng, m, n, C, count, rank, type_)
        a = Arrays(ctx, type_)
        dA, dB, dX, dBase, Y = (a.put(v)[0] for v in (A.reshape(-1, n), B.reshape(-1, rank), X, base, np.zeros((m, C))))
        which = ctx.array(np.zeros(C), np.int32)
        ctx.adapters_reserve(m, n, C, rank, type=type_)
        calls = lambda: ctx.adapters(dA, dB, None, count, rank, which, m, n, dX, C, dBase, Y, type=type_)
        ctx.graph_begin()
        try:
            calls()
        finally:
            graph = ctx.graph_end()
        for _ in range(4):
            X, w = draw(rng, type_, n, C), rng.integers(-1, count, C).astype(np.int32)
            dX.upload(stored(X, type_).ravel())
            which.upload(w)
            ctx.graph_launch(graph)
            got = Y.download().copy()
            Y.upload(np.zeros(Y.shape, Y.dtype))
            calls()
            assert np.array_equal(Y.download(), got)
            check(values(got, type_).reshape(m, C), A, B, None, w, X, base, type_)
        ctx.graph_free(graph)
    finally:
        ctx.close()


def test_a_workspace_that_must_grow_is_refused_while_recording():
    ctx = hipabi.Context()
    try:
        a = Arrays(ctx, "f32")
        A, B, X, base, Y = (a.put(np.ones((64, 64)))[0] for _ in range(5))
        which = ctx.array(np.zeros(64), np.int32)
        ctx.graph_begin()
        try:
            with pytest.raises(hipabi.SoError, match="so_adapters_reserve"):
                ctx.adapters(A, B, None, 1, 64, which, 64, 64, X, 64, base, Y)
        finally:
            ctx.graph_free(ctx.graph_end())
        ctx.adapters(A, B, None, 1, 64, which, 64, 64, X, 64, base, Y)
        assert np.all(Y.download() == 64.0 * 64.0 + 1.0)
    finally:
        ctx.close()


# a last tile of columns of every kind, ranks that end inside a run of products and a group, adapters and rows to the end of their arrays
@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("m,n,C,count,rank", [(70, 40, 256, 3, 1), (33, 72, 257, 4, 3), (100, 130, 320, 5, 10), (17, 64, 383, 2, 33), (65, 33, 449, 3, 100), (40, 200, 300, 6, 4), (130, 24, 511, 2, 256),
                                              (3, 5, 290, 2, 7), (1, 1, 260, 1, 1), (40, 48, 4161, 5, 6), (20, 33, 4500, 3, 17), (70, 24, 8192, 4, 16)])
def test_many_columns(ctx, m, n, C, count, rank, type_):
    rng = np.random.default_rng(C + rank)
    A, B, scale, X, base = problem(rng, m, n, C, count, rank, type_)
    for i, (pad, shift) in enumerate(PLACES):
        for which in (requests(rng, C, count), rng.integers(-1, count + 1, C).astype(np.int32), np.full(C, count - 1, np.int32)):
            check(run(ctx, A, B, scale if i else None, which, X, base if i != 1 else None, type_, pad, shift, in_place=i == 2), A, B, scale if i else None, which, X, base if i != 1 else None, type_)


@pytest.mark.parametrize("type_", TYPES)
def test_sixty_four_adapters_in_every_tile_of_many_columns(ctx, type_):
    rng = np.random.default_rng(12)
    m, n, C, count, rank = 90, 100, 330, 64, 6
    A, B, scale, X, base = problem(rng, m, n, C, count, rank, type_)
    which = np.concatenate([rng.permutation(count) for _ in range(6)])[:C].astype(np.int32)
    check(run(ctx, A, B, scale, which, X, base, type_), A, B, scale, which, X, base, type_)


@pytest.mark.parametrize("type_", TYPES)
def test_a_column_of_many_does_not_depend_on_the_others(ctx, type_):
    rng = np.random.default_rng(13)
    m, n, C, count, rank = 70, 140, 300, 6, 9
    A, B, scale, X, base = problem(rng, m, n, C, count, rank, type_)
    which = rng.integers(0, count - 1, C).astype(np.int32)
    mine = rng.random(C) < 0.4
    first = run(ctx, A, B, scale, which, X, base, type_)
    A2, B2, X2, base2, which2 = A.copy(), B.copy(), X.copy(), base.copy(), which.copy()
    which2[~mine] = rng.integers(-1, count + 1, int((~mine).sum()))
    A2[count - 1], B2[count - 1] = np.nan, np.inf
    X2[:, ~mine], base2[:, ~mine] = rng.choice([np.nan, np.inf, -np.inf, 1.0], (n, int((~mine).sum()))), np.nan
    second = run(ctx, A2, B2, scale, which2, X2, base2, type_)
    assert np.array_equal(first[:, mine], second[:, mine])
