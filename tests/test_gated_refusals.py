"""Null contexts are refused by the gated block's, the adapters' and the rotary positions' entry points, with a message, and the tests' own formulas hold; no GPU is needed for that."""
import numpy as np
import pytest

import hipabi
from gated_reference import ACTS, backward, gate
from hipabi import SO_ERR_INVALID


def test_null_contexts():
    lib = hipabi.load_library()
    refused = [
        ("so_gated", (None, 0, 4, 4, 4, None, None, 4, None, 4, 0, None, None, 4, None, 4, None, None, 4)),
        ("so_gated_grad", (None, 0, 4, 4, 4, None, None, 4, None, 4, 0, None, None, 4, None, 4, None, 4, None, None, 4, None, None, 4)),
        ("so_gated_reserve", (None, 0, 4, 4, 4)),
        ("so_adapters", (None, 0, 4, 4, 4, 1, 1, None, None, None, None, None, 4, None, 4, None, 4)),
        ("so_adapters_reserve", (None, 0, 4, 4, 4, 1)),
        ("so_head_rotary", (None, 0, 1, 1, 4, 4, None, 4, 0, None, None, 0.0, None, None, 0, 1.0, 0, None, 4, None)),
        ("so_head_rotary_grad", (None, 0, 1, 1, 4, 4, None, 4, None, 4, 0, None, None, None, None, None, 0, 1.0, 0, None, 4, None, None)),
        ("so_head_rotary_reserve", (None, 0, 1, 1, 4, 4)),
    ]
    for name, args in refused:
        assert getattr(lib, name)(*args) == SO_ERR_INVALID, name
        assert lib.so_last_error().startswith(name.encode() + b":"), lib.so_last_error()


@pytest.mark.parametrize("act", ACTS)
def test_slopes_against_differences(act):
    v = np.linspace(-9.0, 9.0, 1000)                       # none of them 0
    step = 1e-5
    difference = (gate(v + step, act)[0] - gate(v - step, act)[0]) / (2 * step)
    assert np.abs(gate(v, act)[1] - difference).max() < 1e-9       # third derivatives below 4, step^2 / 6 of them, and 2^-53 of 9 over 2 steps


@pytest.mark.parametrize("act", [a for a in ACTS if a != "relu"])
def test_gradients_against_differences(act):
    rng = np.random.default_rng(3)
    m, n, B = 7, 5, 4
    Wg, Wu, X, D = rng.standard_normal((m, n)), rng.standard_normal((m, n)), rng.standard_normal((n, B)), rng.standard_normal((m, B))
    loss = lambda Wg, Wu, X: float((D * gate(Wg @ X, act)[0] * (Wu @ X)).sum())
    got = backward(Wg, Wu, X, act, Wg @ X, Wu @ X, D, "f32")
    for name, at in (("dWg", 0), ("dWu", 1), ("dX", 2)):
        along = rng.standard_normal((Wg, Wu, X)[at].shape)
        moved = lambda s: [a + (s * along if i == at else 0.0) for i, a in enumerate((Wg, Wu, X))]
        difference = (loss(*moved(1e-5)) - loss(*moved(-1e-5))) / 2e-5
        assert abs(float((got[name][0] * along).sum()) - difference) < 1e-5
