"""An infinite entry of A x among finite ones that the element type does not hold: the result is the infinity that the formula has, since the finite ones stay finite between the products."""
import numpy as np
import pytest

from elements import TYPES
from test_gpu_adapters import run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("rank", [2, 18, 40, 200])
@pytest.mark.parametrize("C", [1, 20, 300])
def test_finite_entries_beside_an_infinite_one(ctx, C, rank, type_):
    n, m, count = 4, 6, 2
    A, B, X, base = np.zeros((count, rank, n)), np.zeros((count, m, rank)), np.full((n, C), 300.0), np.ones((m, C))
    A[0, 0, 0], A[0, rank - 1], A[1, 0, 0] = np.inf, 300.0, 1.0
    B[0, :, 0], B[0, :, rank - 1] = [1, 1, -1, -1, 0.5, -2], [-1, 1, 1, -1, -4, 3]
    B[0, :, 1:rank - 1], B[1] = 1.0, 0.25
    which = (np.arange(C) % 2).astype(np.int32)
    got = run(ctx, A, B, np.array([0.5, 2.0], np.float32), which, X, base, type_)
    want = np.where(which == 0, np.sign(B[0, :, :1]) * np.inf, 1 + 2 * 0.25 * 300.0)
    assert np.array_equal(got, want)
