"""Null contexts and handles are refused by the layer norm and 4-bit entry points, with a message; no GPU is needed for that."""
import ctypes as ct

import hipabi
from hipabi import SO_ERR_INVALID, SO_OK


def test_null_contexts_and_handles():
    lib = hipabi.load_library()
    refused = [
        ("so_layer_norm", (None, 0, 4, 4, None, 4, None, None, 1e-5, None, 4, None, None)),
        ("so_layer_norm_grad", (None, 0, 4, 4, None, 4, None, 4, None, None, None, None, 4, None, None)),
        ("so_layer_norm_reserve", (None, 0, 4, 4)),
        ("so_mxfp4_quantize", (None, 0, None, 4, 4, 4, None, None)),
        ("so_mxfp4_dequantize", (None, None, None, 4, 4, 0, None, 4)),
        ("so_mxfp4_matmul", (None, None, 0, None, 4, 4, None, None, 4, 0)),
        ("so_mxfp4_matmul_reserve", (None, None, 4)),
        ("so_mxfp4_matvec", (None, None, None, None, None)),
        ("so_mxfp4_dims", (None, None, None)),
    ]
    for name, args in refused:
        assert getattr(lib, name)(*args) == SO_ERR_INVALID, name
        assert lib.so_last_error().startswith(name.encode() + b":"), lib.so_last_error()
    h = ct.c_void_p()
    assert lib.so_mxfp4_create(None, None, None, 4, 4, ct.byref(h)) == SO_ERR_INVALID and not h.value
    assert lib.so_mxfp4_free(None, None) == SO_OK


def test_the_reference_of_the_tests():
    """What the GPU tests compare with, against the definition's own examples: ties to the even code, saturation, scales at their ends."""
    import numpy as np

    import mx_reference as mx
    X = np.zeros((4, 32))
    X[0, :14] = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0, -0.25, -0.75, -6.0, 4.0, 0.2, 0.26]
    X[1, 0] = 2.0 ** -149
    X[2, 0], X[2, 1] = 3.4028234663852886e38, -2.0 ** 126
    codes, scales = mx.quantize(X)
    assert scales[:, 0].tolist() == [127, 0, 252, 0]
    assert mx.dequantize(codes, scales, 32)[0, :14].tolist() == [0, 1, 1, 2, 2, 4, 4, 6, 0, -1, -6, 4, 0, 0.5]
    assert mx.dequantize(codes, scales, 32)[2, :2].tolist() == [6 * 2.0 ** 125, -2.0 ** 126]
    assert not mx.dequantize(codes, scales, 32)[1].any()
