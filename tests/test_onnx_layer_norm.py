"""LayerNormalization in the ONNX loader: what it refuses, without a GPU."""
import numpy as np
import pytest

import onnx_wire as ow


def norm_model(shape=(2, 6), scale=(6,), bias=(6,), inputs=None, outputs=("y",), **attrs):
    inits = [("g", np.ones(scale, np.float32)), ("b", np.zeros(bias, np.float32))]
    return ow.model([ow.node("LayerNormalization", list(inputs or ["x", "g", "b"]), list(outputs), **attrs)], [("x", shape)], [("y", shape)], inits, opset=17)


@pytest.mark.parametrize("payload,match", [
    (norm_model(axis=0), "over all axes but the batch"),
    (norm_model(axis=-2), "over all axes but the batch"),
    (norm_model(axis=2), "over all axes but the batch"),
    (norm_model(axis=2 ** 63 - 1), "over all axes but the batch"),
    (norm_model(axis=-3), "over all axes but the batch"),
    (norm_model((2, 3, 2, 1), axis=-1), "over all axes but the batch"),
    (norm_model((2, 3, 2, 1)), "over all axes but the batch"),                 # the default is the last axis
    (norm_model((2, 3, 2, 1), axis=2), "over all axes but the batch"),
    (norm_model(scale=(5,)), "Scale length"),
    (norm_model(scale=(1,)), "Scale length"),
    (norm_model((2, 3, 2, 1), scale=(3, 1, 1), axis=1), "Scale length"),
    (norm_model(bias=(7,)), "B length"),
    (norm_model(inputs=["x", "missing", "b"]), "Scale initializer"),
    (norm_model(inputs=["x", "x"]), "Scale initializer"),
    (norm_model(inputs=["x", "g", "missing"]), "B initializer"),
    (norm_model(inputs=["x"]), "input"),
    (norm_model(outputs=["y", "mean"]), "Mean and InvStdDev"),
    (norm_model(outputs=["y", "", "rstd"]), "Mean and InvStdDev"),
    (norm_model(stash_type=16), "stash_type"),
    (norm_model(epsilon=-1.0), "epsilon"),
    (norm_model(epsilon=float("nan")), "epsilon"),
    (norm_model(inputs=["z", "g", "b"]), "before it is produced"),
])
def test_refusals(backend, tmp_path, payload, match):
    path = ow.save(str(tmp_path / "bad.onnx"), payload)
    with pytest.raises(RuntimeError, match=match):
        backend.SparseOnnxModel(path)


@pytest.mark.parametrize("payload", [norm_model(), norm_model(axis=1), norm_model(axis=-1, epsilon=0.0), norm_model(inputs=["x", "g"]), norm_model(inputs=["x", "g", ""]), norm_model(outputs=["y", "", ""]),
                                     norm_model((2, 3, 2, 1), scale=(3, 2, 1), axis=1), norm_model((2, 3, 2, 1), scale=(6,), bias=(3, 2, 1), axis=-3)])
def test_accepted_as_far_as_the_gpu(backend, tmp_path, payload):
    if backend.device_available():
        pytest.skip("a GPU is present")
    path = ow.save(str(tmp_path / "ok.onnx"), payload)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        backend.SparseOnnxModel(path)
