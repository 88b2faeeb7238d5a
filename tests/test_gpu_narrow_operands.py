"""Dense operands of one to three columns without gaps, read through registers, whose last two steps of the contraction are not read whole: results against the formulas, with the tolerances of the
operators' own tests.  That no read passes an operand's end is tested on the host, in tests/test_operand_reads.py."""
import numpy as np
import pytest

import test_gpu_adapters as adapters
from elements import TYPES
from test_gpu_gated import run_backward, run_forward

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("rank", [5, 20, 40])
def test_adapters_of_one_to_three_columns(ctx, rank, type_):
    """Steps of 64, 128 or 256 bytes; lengths of 0 to 7 beyond a step's multiple."""
    rng = np.random.default_rng(rank)
    m, count = 9, 2
    for C in (1, 2, 3):
        for n in list(range(128, 136)) + [3 * 128 + 1, 5 * 128 + 5]:
            A, B, scale, X, base = adapters.problem(rng, m, n, C, count, rank, type_)
            which = (np.arange(C) % count).astype(np.int32)
            adapters.check(adapters.run(ctx, A, B, scale, which, X, base, type_, 0, 1), A, B, scale, which, X, base, type_)


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("B", [2, 3, 5])
def test_gated_blocks_of_two_to_five_columns(ctx, B, type_):
    rng = np.random.default_rng(B)
    for rest in (1, 2, 3, 5, 7):
        run_forward(ctx, rng, 20, 128 + rest, B, type_, "silu", 0, 1)
        run_backward(ctx, rng, 128 + rest, 20, B, type_, "silu", 0, 1)


@pytest.mark.parametrize("type_", TYPES)
@pytest.mark.parametrize("n", [1, 2, 3])
def test_gradients_of_one_to_three_features(ctx, n, type_):
    rng = np.random.default_rng(n)
    for m in (129, 131, 134, 65 * 64 + 3):
        run_backward(ctx, rng, m, n, 21, type_, "gelu", 0, 1)
