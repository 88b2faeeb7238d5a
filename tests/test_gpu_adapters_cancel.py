"""Sums of A x that cancel in the second product: what is left of them is as exact as fp32's 24 bits of the sums let it be.

A x has two entries, x0 + 2^-8 x1 + 2^-16 x2 and x0 + 2^-8 x1, below 1 and in 24 bits at most, so that fp32 holds them as they are, in whatever order they are added; B takes their difference, 2^-16 x2, and the
result is that, rounded once.  Two numbers of 8 bits each would hold the first entry to 2^-17, as much as what is asked for.  u = 2^-24: in the second product at most 8 numbers that are not 0 are added up, each
addition off by 2 u of the entries' size at most."""
import numpy as np
import pytest

from elements import HALF_STEP, SMALLEST, TYPES, U
from test_gpu_adapters import run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("rank", [2, 17, 30, 100, 256])
@pytest.mark.parametrize("C", [1, 40, 70, 300])
def test_what_is_left_of_sums_that_cancel(ctx, C, rank, type_):
    rng = np.random.default_rng(C + rank)
    n, m, count = 3, 20, 3
    X = rng.integers(128, 256, (n, C)) / 256.0 * rng.choice([-1, 1], (1, C))      # 8 bits each, of one sign
    A, B = np.zeros((count, rank, n)), np.zeros((count, m, rank))
    first, second = 0, rank - 1                                                  # in the first and the last run of ranks
    size = 2.0 ** rng.integers(2, 5, count)                                     # 2^-16 of it is no subnormal number of fp16
    A[:, first], A[:, second, :2] = size[:, None] * [1, 2.0 ** -8, 2.0 ** -16], size[:, None] * [1, 2.0 ** -8]
    scale = rng.integers(-8, 9, (count, m)) / 8.0
    B[:, :, first], B[:, :, second] = scale, -scale
    which = rng.integers(0, count, C).astype(np.int32)
    got = run(ctx, A, B, None, which, X, None, type_)
    want = scale[which].T * size[which] * 2.0 ** -16 * X[2]
    off = 16 * U * np.abs(scale[which].T) * size[which] + SMALLEST[type_]
    assert np.all(np.abs(got - want) <= HALF_STEP[type_] * np.abs(want) + off), np.max(np.abs(got - want) / np.maximum(np.abs(want), 1e-30))
