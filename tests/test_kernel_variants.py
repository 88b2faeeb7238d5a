"""The library holds no layer norm kernel that no call reaches, by the names in its code objects."""
import os
import re

import pytest

from conftest import PKG

pytest.importorskip("msgpack")
from test_kernel_scratch import code_objects, kernels          # noqa: E402

GROUP = {"f": 4, "DF16_": 8, "DF16b": 8}          # elements of 16 bytes, by the mangled type


def variants(kernel, numbers):
    """(elements of 16 bytes, the numbers) of every instantiation of a kernel template."""
    path = os.path.join(PKG, "libsparseops_hip.so")
    if not os.path.exists(path):
        pytest.skip("the library is not built")
    with open(path, "rb") as f:
        names = [k[".name"] for elf in code_objects(f.read()) for k in kernels(elf)]
    found = [re.search(kernel + r"I(f|DF16_|DF16b)" + r"Li(\d+)E" * numbers + "E", name) for name in names]
    return [(GROUP[m.group(1)],) + tuple(int(g) for g in m.groups()[1:]) for m in found if m]


def test_kernels_that_hold_all_features():
    """Lanes, rows a thread, threads: up to 16384 rows by lanes in 256 or 512 threads; with one lane a row 8192 in 256 or 1024, of 16-bit types 2048."""
    more = [(l, r, t) for l in (2, 4, 8) for t, rows in ((256, (1, 2, 4, 8, 16)), (512, (16, 32))) for r in rows]
    one = [(1, 1, 256), (1, 2, 256), (1, 1, 1024), (1, 2, 1024)]
    want = [(4,) + v for v in more + one + [(1, 4, 256), (1, 4, 1024), (1, 8, 1024)]] + 2 * [(8,) + v for v in more + one]
    assert sorted(variants("norm_whole_kernel", 3)) == sorted(want)


def test_gradients_of_one_workgroup():
    """Up to 8192 elements of whole groups: 2048 rows by lanes in fp32, 1024 in 16 bits."""
    want = [(v, l, r, t) for v, times in ((4, 1), (8, 2)) for l in (1, 2, 4, 8) for r, t in ((1, 256), (2, 256), (1, 1024), (2, 1024)) if v == 4 or (r, t) != (2, 1024) for _ in range(times)]
    assert sorted(variants("norm_grad_one_kernel", 3)) == sorted(want)
