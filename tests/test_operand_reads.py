"""Reads of the dense products' operands (csrc/dense.h) stay inside their matrices at every width, stride and length: the kernels' own index arithmetic, compiled for the host.  What such a read
brings from behind an end is of no use and dropped, so that no result shows it."""
import os
import shutil
import subprocess

import pytest

from conftest import PKG, ROOT


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    hipcc = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
    if not shutil.which(hipcc):
        pytest.skip("no hipcc")
    exe = str(tmp_path_factory.mktemp("cpp") / "operand_reads")
    subprocess.run([hipcc, "-x", "hip", "--offload-host-only", "-O2", "-std=c++17", "-Wno-unused-command-line-argument", "-I" + os.path.join(PKG, "csrc"), "-I" + os.path.join(ROOT, "include"),
                    os.path.join(ROOT, "tests", "cpp", "operand_reads.cpp"), "-o", exe], check=True)
    return exe


def test_no_group_passes_the_end_of_its_matrix(program):
    r = subprocess.run([program], timeout=120, stdout=subprocess.PIPE, text=True)
    assert r.returncode == 0, r.stdout
