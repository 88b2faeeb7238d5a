"""What the history holds: sources and results, nothing that a build leaves behind."""
import os
import subprocess

import pytest

from conftest import ROOT


def test_no_build_leftovers():
    """A compiler that is interrupted leaves its temporary output (NAME-HASH.o.tmp) beside the sources."""
    if not os.path.isdir(os.path.join(ROOT, ".git")):
        pytest.skip("not a git working tree")
    listed = subprocess.run(["git", "-C", ROOT, "ls-files"], capture_output=True, text=True)
    if listed.returncode:
        pytest.skip("git does not list the files")
    assert [f for f in listed.stdout.splitlines() if f.endswith((".tmp", ".o", ".so", ".a", ".s", ".hsaco", ".co", ".pyc"))] == []
