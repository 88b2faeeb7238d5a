"""LayerNormalization inside SparseOnnxModel, against float64.

Tolerances, u = 2^-24: of the normalisation alone those of so_layer_norm (no sum there runs through more than 40 additions one after the other, the formula adds 8 roundings).  In a
chain a product's rounding, at most 1e-6 of the largest output as everywhere for these layers, is a deviation of the norm's input: it moves a normalised entry by 1e-6 of max |x| rstd, twice that through the mean and once
more through rstd, and the next product adds its share over the row's absolute sum."""
import os

import numpy as np
import pytest

import datagen
import onnx_wire as ow
from test_gpu_model import _run_device

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def norm(X, g, b, eps):
    """X (B, features) in float64; the result and what so_layer_norm may be off by."""
    mean = X.mean(axis=1, keepdims=True)
    rstd = 1.0 / np.sqrt(np.square(X - mean).mean(axis=1, keepdims=True) + np.float64(np.float32(eps)))
    h = (X - mean) * rstd
    g, b = np.asarray(g, np.float64).reshape(-1), np.asarray(b, np.float64).reshape(-1)
    top = np.abs(X).max(axis=1, keepdims=True) * rstd
    return h * g + b, U * (48 * top * np.abs(g) + 48 * np.abs(h * g) + 2 * np.abs(b)), top


@pytest.mark.parametrize("shape,axis", [((70,), -1), ((70,), 1), ((1,), 1), ((9000,), 1), ((20000,), -1), ((3, 5, 7), 1), ((16, 8, 8), -3)])
@pytest.mark.parametrize("graph", ["0", "1"])          # SPARSEOPS_NO_GRAPH
def test_alone(backend, ctx, tmp_path, shape, axis, graph, monkeypatch):
    rng = np.random.default_rng(int(np.prod(shape)))
    g, b = (1 + 0.3 * rng.standard_normal(shape)).astype(np.float32), rng.standard_normal(shape).astype(np.float32)
    for with_bias in (True, False):
        nodes = [ow.node("LayerNormalization", ["x", "g"] + ["b"] * with_bias, ["y"], axis=axis, epsilon=1e-3)]
        path = ow.save(str(tmp_path / "n.onnx"), ow.model(nodes, [("x", (4,) + shape)], [("y", (4,) + shape)], [("g", g), ("b", b)], opset=17))
        monkeypatch.setenv("SPARSEOPS_NO_GRAPH", graph)
        model = backend.SparseOnnxModel(path)
        assert model.describe()[0].startswith("LayerNormalization")
        for B in (4, 1, 33, 300, 4):
            X = (rng.standard_normal((B,) + shape) + 2).astype(np.float32)
            want, tol, _ = norm(X.reshape(B, -1).astype(np.float64), g, b if with_bias else 0 * b, 1e-3)
            for Y in (model.run(X), model.run(X), _run_device(model, ctx, X)):
                assert Y.shape == (B,) + shape
                assert np.all(np.abs(Y.reshape(B, -1) - want) <= tol)


@pytest.mark.parametrize("B", [1, 24, 130])
def test_between_products(backend, ctx, tmp_path, B):
    """Gemm + Relu, LayerNormalization, Gemm, a residual Add, LayerNormalization with the default epsilon: recorded and launched, the same bits."""
    rng = np.random.default_rng(B)
    W1 = datagen.magnitude_prune(rng.standard_normal((96, 40)).astype(np.float32), .8)
    W2 = datagen.magnitude_prune(rng.standard_normal((96, 96)).astype(np.float32), .9)
    b1, b2, g1, c1, g2, c2 = (rng.standard_normal(96).astype(np.float32) for _ in range(6))
    nodes = [ow.node("Gemm", ["x", "W1", "b1"], ["a"], alpha=1.0, beta=1.0, transB=1), ow.node("Relu", ["a"], ["r"]),
             ow.node("LayerNormalization", ["r", "g1", "c1"], ["n"], epsilon=1e-6),
             ow.node("Gemm", ["n", "W2", "b2"], ["m"], alpha=1.0, beta=1.0, transB=1), ow.node("Add", ["m", "r"], ["s"]),
             ow.node("LayerNormalization", ["s", "g2", "c2"], ["y"])]
    inits = [("W1", W1), ("W2", W2), ("b1", b1), ("b2", b2), ("g1", g1), ("c1", c1), ("g2", g2), ("c2", c2)]
    path = ow.save(str(tmp_path / "c.onnx"), ow.model(nodes, [("x", (B, 40))], [("y", (B, 96))], inits, opset=17))
    X = rng.standard_normal((B, 40)).astype(np.float32)
    results = []
    for no_graph in ("0", "1"):
        os.environ["SPARSEOPS_NO_GRAPH"] = no_graph
        try:
            model = backend.SparseOnnxModel(path)
            assert [d.split()[0] for d in model.describe()][1] == "LayerNormalization" and "act=relu" in model.describe()[0]
            results += [model.run(X) for _ in range(3)] + [_run_device(model, ctx, X)]
        finally:
            del os.environ["SPARSEOPS_NO_GRAPH"]
    for Y in results[1:]:
        assert np.array_equal(Y, results[0])
    r = np.maximum(X.astype(np.float64) @ W1.T.astype(np.float64) + b1, 0)
    off_r = np.full((B, 1), 1e-6 * np.abs(r).max())
    n, tol, top = norm(r, g1, c1, 1e-6)
    off_n = tol + 3 * np.abs(g1) * (off_r / np.abs(r).max(axis=1, keepdims=True)) * top * (1 + np.abs(n - c1) / np.abs(g1))
    s = n @ W2.T.astype(np.float64) + b2 + r
    off_s = off_n @ np.abs(W2.T.astype(np.float64)) + 1e-6 * np.abs(s).max() + off_r + 2 * U * np.abs(s)
    y, tol, top = norm(s, g2, c2, 1e-5)
    rel = off_s.max(axis=1, keepdims=True) / np.abs(s).max(axis=1, keepdims=True)
    bound = tol + 3 * np.abs(g2) * rel * top * (1 + np.abs(y - c2) / np.abs(g2))
    assert np.all(np.abs(results[0] - y) <= bound), np.max(np.abs(results[0] - y) / bound)


@pytest.mark.parametrize("B", [1, 3, 5, 7, 20, 33])
def test_after_a_convolution(backend, ctx, tmp_path, B):
    """With convolutions the batch is carried in longer rows: what stands behind it (zeros, which without an epsilon become NaN) reaches no sample.  A sample's result is within the
    normalisation's tolerance of that of its own convolution, taken from a model that ends there."""
    rng = np.random.default_rng(40 + B)
    Wc = datagen.magnitude_prune(rng.standard_normal((8, 27)).astype(np.float32), .5).reshape(8, 3, 3, 3)
    bc, g, b = (rng.standard_normal(n).astype(np.float32) for n in (8, 8 * 36, 8 * 36))
    Wf = datagen.magnitude_prune(rng.standard_normal((10, 8 * 36)).astype(np.float32), .5)
    conv = ow.node("Conv", ["x", "Wc", "bc"], ["c"], kernel_shape=[3, 3], pads=[1, 1, 1, 1], strides=[1, 1], dilations=[1, 1], group=1)
    norm_node = ow.node("LayerNormalization", ["c", "g", "b"], ["n"], axis=1, epsilon=0.0)
    inits = [("Wc", Wc), ("bc", bc), ("g", g.reshape(8, 6, 6)), ("b", b.reshape(8, 6, 6)), ("Wf", Wf)]
    tail = [ow.node("Flatten", ["n"], ["f"], axis=1), ow.node("Gemm", ["f", "Wf"], ["y"], alpha=1.0, beta=1.0, transB=1)]
    image = [("x", (B, 3, 6, 6))]
    X = rng.standard_normal((B, 3, 6, 6)).astype(np.float32)
    make = lambda name, nodes, out: backend.SparseOnnxModel(ow.save(str(tmp_path / name), ow.model(nodes, image, [out], inits, opset=17)))
    c = make("c.onnx", [conv], ("c", (B, 8, 6, 6))).run(X).reshape(B, -1).astype(np.float64)
    want, tol, _ = norm(c, g, b, 0.0)
    model = make("n.onnx", [conv, norm_node], ("n", (B, 8, 6, 6)))
    for Y in (model.run(X), _run_device(model, ctx, X)):
        assert np.all(np.abs(Y.reshape(B, -1) - want) <= tol)
    whole = make("y.onnx", [conv, norm_node] + tail, ("y", (B, 10)))
    W = np.abs(Wf.T.astype(np.float64))
    # the product adds at most 288 entries of a row, each with two roundings
    bound = tol @ W + U * 2 * 288 * (np.abs(want) @ W)
    for Y in (whole.run(X), whole.run(X), _run_device(whole, ctx, X)):
        assert np.all(np.abs(Y - want @ Wf.T.astype(np.float64)) <= bound)
