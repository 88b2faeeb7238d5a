"""Layer norm, 4-bit products, adapters, rotary positions and the gated block as a block of a model calls them: one call's result as the next one's input, on one stream, without a wait between them.
Every step is held against its formula in float64 on the inputs that it was given, with the tolerances of its own tests; the formulas of the backward pass together against differences."""
import numpy as np
import pytest

import gated_reference
import hipabi
import mx_reference as mx
import test_gpu_adapters as adapters
import test_gpu_rotary as rotary
from elements import TYPES, fetch, stored
from test_gpu_gated import Arrays, draw
from test_gpu_gated import weights as dense
from test_gpu_layer_norm import EPS, check_forward, check_grad, check_statistics
from test_gpu_mxfp4 import product_tolerance, weights

pytestmark = pytest.mark.gpu


class Block:
    """Queries and keys of a layer and its feed-forward half, with adapters on the first projection and on both of the gated block's; attention itself is left out."""
    features, q, k, D, rot, ff, count, rank = 256, 4, 2, 64, 48, 520, 5, 12

    def __init__(self, ctx, rng, B, type_):
        self.ctx, self.B, self.type, n, m = ctx, B, type_, self.features, self.ff
        self.rows = rows = (self.q + self.k) * self.D
        self.a = Arrays(ctx, type_)
        put = lambda v: self.a.put(v)[0]
        self.host = {"gamma": (1 + 0.2 * rng.standard_normal(n)).astype(np.float32), "beta": (0.3 * rng.standard_normal(n)).astype(np.float32),
                     "pos": (rng.integers(0, 10 ** 5) + np.arange(B)).astype(np.int32), "freq": (10000.0 ** (-np.arange(self.rot // 2) / (self.rot // 2))).astype(np.float32),
                     "gq": (1 + 0.2 * rng.standard_normal(self.D)).astype(np.float32), "gk": (1 + 0.2 * rng.standard_normal(self.D)).astype(np.float32),
                     "which": adapters.requests(rng, B, self.count), "scale": (0.5 + rng.random(self.count)).astype(np.float32)}
        self.small = {name: ctx.array(v, v.dtype) for name, v in self.host.items()}
        low = lambda out: (draw(rng, type_, self.count, self.rank, n, size=n ** -0.5), draw(rng, type_, self.count, out, self.rank, size=self.rank ** -0.5))
        self.low = {"first": low(rows), "gate": low(m), "other": low(m)}
        self.dlow = {name: (put(A.reshape(-1, n)), put(V.reshape(-1, self.rank))) for name, (A, V) in self.low.items()}
        self.first, self.W1 = weights(ctx, rng, rows, n)
        self.out, self.W2 = weights(ctx, rng, n, rows)
        self.down, self.W3 = weights(ctx, rng, n, m)
        self.Wg, self.Wu = dense(rng, type_, m, n), dense(rng, type_, m, n)
        self.dWg, self.dWu = put(self.Wg), put(self.Wu)
        sizes = {"X": n, "N1": n, "P": rows, "Q": rows, "R": rows, "O": n, "N2": n, "G0": m, "U0": m, "H": m, "Y": n}
        self.d = {name: put(np.zeros((r, B))) for name, r in sizes.items()}
        self.sizes = sizes
        self.upload(rng)

    def upload(self, rng):
        self.d["X"].upload(stored(rng.standard_normal((self.features, self.B)), self.type).reshape(self.d["X"].shape))

    def reserve(self):
        c, t = self.ctx, self.type
        c.layer_norm_reserve(self.features, self.B, type=t)
        for W in (self.first, self.out, self.down):
            c.mxfp4_matmul_reserve(W, self.B)
        c.adapters_reserve(self.rows, self.features, self.B, self.rank, type=t)
        c.adapters_reserve(self.ff, self.features, self.B, self.rank, type=t)
        c.head_rotary_reserve(self.q, self.k, self.D, self.B, type=t)
        c.gated_reserve(self.ff, self.features, self.B, type=t)

    def run(self):
        c, d, s, B, t, n = self.ctx, self.d, self.small, self.B, self.type, self.features
        c.layer_norm(d["X"], n, B, s["gamma"], s["beta"], EPS, d["N1"], type=t)
        c.mxfp4_matmul(self.first, d["N1"], B, None, d["P"], type=t)
        c.adapters(*self.dlow["first"], s["scale"], self.count, self.rank, s["which"], self.rows, n, d["N1"], B, d["P"], d["Q"], type=t)
        c.head_rotary(d["Q"], self.q, self.k, self.D, B, s["pos"], s["freq"], self.rot, d["R"], "halves", 1.0, True, EPS, s["gq"], s["gk"], type=t)
        c.mxfp4_matmul(self.out, d["R"], B, None, d["O"], type=t)
        c.layer_norm(d["O"], n, B, s["gamma"], s["beta"], EPS, d["N2"], type=t)
        for name, to in (("gate", "G0"), ("other", "U0")):
            c.adapters(*self.dlow[name], s["scale"], self.count, self.rank, s["which"], self.ff, n, d["N2"], B, None, d[to], type=t)
        c.gated(self.dWg, self.dWu, self.ff, n, d["N2"], B, "silu", d["H"], None, None, d["G0"], d["U0"], type=t)
        c.mxfp4_matmul(self.down, d["H"], B, None, d["Y"], type=t)

    def fetch(self):
        return {name: fetch(self.d[name], r, self.B, self.type)[0] for name, r in self.sizes.items()}

    def check(self):
        v, h, t = self.fetch(), self.host, self.type

        def product(W, X, got):
            Xq = mx.dequantize(*mx.quantize(np.ascontiguousarray(X.T)), X.shape[0]).T
            assert np.all(np.abs(got - W @ Xq) <= product_tolerance(W, Xq, None, W @ Xq, "none", t))

        check_forward(v["N1"], v["X"], h["gamma"], h["beta"], t)
        product(self.W1, v["N1"], v["P"])
        adapters.check(v["Q"], *self.low["first"], h["scale"], h["which"], v["N1"], v["P"], t)
        want, tol, _ = rotary.forward(v["Q"], self.q, self.k, self.D, h["pos"], h["freq"], self.rot, "halves", 1.0, True, h["gq"], h["gk"], t, EPS)
        assert np.all(np.abs(v["R"] - want) <= tol)
        product(self.W2, v["R"], v["O"])
        check_forward(v["N2"], v["O"], h["gamma"], h["beta"], t)
        for name, to in (("gate", "G0"), ("other", "U0")):
            adapters.check(v[to], *self.low[name], h["scale"], h["which"], v["N2"], None, t)
        gated_reference.check(v["H"], gated_reference.forward(self.Wg, self.Wu, v["N2"], "silu", t, v["G0"], v["U0"])["H"])
        product(self.W3, v["H"], v["Y"])
        return v

    def free(self):
        for W in (self.first, self.out, self.down):
            W.free()
        self.a.free()
        for x in self.small.values():
            x.free()


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("B", [1, 3, 40, 300])
def test_a_block_of_a_served_model(ctx, B, type_):
    block = Block(ctx, np.random.default_rng(B), B, type_)
    block.run()
    assert block.check()["Y"].any()
    block.free()


@pytest.mark.parametrize("type_,B", [("f32", 5), ("bf16", 1), ("bf16", 270), ("f16", 33)])
def test_a_block_recorded_ahead_of_its_first_launch(type_, B):
    """Replayed with new columns, other adapters and positions, its own calls between the replays: the same bits as those."""
    rng = np.random.default_rng(B)
    ctx = hipabi.Context()
    try:
        block = Block(ctx, rng, B, type_)
        block.reserve()
        ctx.graph_begin()
        try:
            block.run()
        finally:
            graph = ctx.graph_end()
        for _ in range(3):
            block.upload(rng)
            block.host["which"], block.host["pos"] = adapters.requests(rng, B, block.count), rng.integers(0, 10 ** 6, B).astype(np.int32)
            for name in ("which", "pos"):
                block.small[name].upload(block.host[name])
            ctx.graph_launch(graph)
            first = block.check()
            block.run()
            second = block.fetch()
            for name in first:
                assert np.array_equal(first[name], second[name]), name
        ctx.graph_free(graph)
        block.free()
    finally:
        ctx.close()


def test_two_blocks_on_two_contexts_at_once():
    rng = np.random.default_rng(19)
    contexts = [hipabi.Context() for _ in range(2)]
    try:
        blocks = [Block(c, rng, 70, "bf16") for c in contexts]
        for _ in range(4):
            for b in blocks:
                b.run()
        for b in blocks:
            b.check()
            b.free()
    finally:
        for c in contexts:
            c.close()


def normed(X, gamma, beta):
    mean = X.mean(axis=0)
    return (X - mean) / np.sqrt(np.square(X - mean).mean(axis=0) + np.float64(np.float32(EPS))) * gamma[:, None] + beta[:, None]


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("B", [1, 33, 300])
def test_a_training_step(ctx, B, type_):
    """Layer norm, rotary positions and the gated block forward and back."""
    rng = np.random.default_rng(B + 100)
    q, k, D, rot, m, act = 3, 1, 32, 32, 150, "gelu"
    n = (q + k) * D
    X, dH = draw(rng, type_, n, B), draw(rng, type_, m, B, size=0.1)
    Wg, Wu = dense(rng, type_, m, n), dense(rng, type_, m, n)
    gamma, beta, gq, gk = ((c + 0.2 * rng.standard_normal(s)).astype(np.float32) for c, s in ((1, n), (0, n), (1, D), (1, D)))
    pos, freq = (100 + np.arange(B)).astype(np.int32), (10000.0 ** (-np.arange(rot // 2) / (rot // 2))).astype(np.float32)
    a = Arrays(ctx, type_)
    put = lambda v: a.put(v)[0]
    dX, dDh, dWg, dWu = put(X), put(dH), put(Wg), put(Wu)
    N, R, H, G, S, dR, dN, out, oWg, oWu = (put(np.zeros(s)) for s in ((n, B), (n, B), (m, B), (m, B), (m, B), (n, B), (n, B), (n, B), (m, n), (m, n)))
    small = [ctx.array(v, v.dtype) for v in (gamma, beta, gq, gk, pos, freq)]
    sums = [ctx.empty(s) for s in ((B,), (B,), (q + k, B), (D,), (D,), (n,), (n,))]
    (dGamma, dBeta, dGq, dGk, dPos, dFreq), (mean, rstd, rq, oGq, oGk, oGamma, oBeta) = small, sums
    ctx.layer_norm(dX, n, B, dGamma, dBeta, EPS, N, mean, rstd, type=type_)
    ctx.head_rotary(N, q, k, D, B, dPos, dFreq, rot, R, "pairs", 1.0, True, EPS, dGq, dGk, rq, type=type_)
    ctx.gated(dWg, dWu, m, n, R, B, act, H, G, S, type=type_)
    ctx.gated_grad(dWg, dWu, m, n, R, B, act, G, S, dDh, dR, oWg, oWu, type=type_)
    ctx.head_rotary_grad(N, dR, q, k, D, B, dPos, dFreq, rot, dN, "pairs", 1.0, True, dGq, dGk, rq, oGq, oGk, type=type_)
    ctx.layer_norm_grad(dX, dN, n, B, dGamma, mean, rstd, out, oGamma, oBeta, type=type_)
    get = lambda x, r, c: fetch(x, r, c, type_)[0]
    vN, vR, vG, vS, vdR, vdN = (get(x, r, B) for x, r in ((N, n), (R, n), (G, m), (S, m), (dR, n), (dN, n)))
    check_forward(vN, X, gamma, beta, type_)
    check_statistics(mean.download(), rstd.download(), X)
    want, tol, _ = rotary.forward(vN, q, k, D, pos, freq, rot, "pairs", 1.0, True, gq, gk, type_, EPS)
    assert np.all(np.abs(vR - want) <= tol)
    made = gated_reference.forward(Wg, Wu, vR, act, type_)
    for name, x in (("H", H), ("G", G), ("U", S)):
        gated_reference.check(get(x, m, B), made[name], name)
    back = gated_reference.backward(Wg, Wu, vR, act, vG, vS, dH, type_)
    for name, x, (r, c) in (("dX", dR, (n, B)), ("dWg", oWg, (m, n)), ("dWu", oWu, (m, n))):
        gated_reference.check(get(x, r, c), back[name], name)
    turned = rotary.backward(vN, vdR, q, k, D, pos, freq, rot, "pairs", 1.0, True, gq, gk, rq.download().reshape(q + k, B), type_)
    for name, got in (("dX", vdN), ("dq", oGq.download().astype(np.float64)), ("dk", oGk.download().astype(np.float64))):
        gated_reference.check(got, turned[name], name)
    check_grad(get(out, n, B), oGamma.download(), oBeta.download(), X, vdN, gamma, mean.download(), rstd.download(), type_)
    # the formulas together: along one direction of X, the loss's difference over 2 h, off by h^2 of its third derivative and 2^-52 / h of its size
    if type_ == "f32" and B == 33:
        e = lambda v: v.astype(np.float64)

        def loss(x):
            r, _, _ = rotary.forward(normed(x, e(gamma), e(beta)), q, k, D, pos, freq, rot, "pairs", 1.0, True, gq, gk, "f32", EPS)
            return np.sum(dH * gated_reference.gate(Wg @ r, act)[0] * (Wu @ r))

        direction, h = rng.standard_normal((n, B)), 1e-5
        difference = (loss(X + h * direction) - loss(X - h * direction)) / (2 * h)
        got = get(out, n, B)
        # three passes forward and three back, each with sums of fewer than 600 terms that are off by 2 u a term: 6 * 2 * 600 u = 2^-11.2 of the magnitudes that are added up
        assert abs(np.sum(got * direction) - difference) <= 2.0 ** -11 * np.sum(np.abs(got * direction))
    a.free()
    for x in small + sums:
        x.free()
