"""How rows of a paged cache are cut into parts, walked on the host."""
import os
import shutil
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.mark.parametrize("what", ["few", "many"])
def test_parts(tmp_path, what):
    compiler = shutil.which("g++")
    assert compiler, "needs a host C++ compiler"
    exe = str(tmp_path / "check")
    subprocess.run([compiler, "-O2", "-std=c++17", "-Wall", "-Werror", os.path.join(HERE, "paged_parts_check.cpp"), "-o", exe], check=True)
    for seed in range(4):
        got = subprocess.run([exe, what, str(seed)], stdout=subprocess.PIPE, text=True)
        assert got.returncode == 0, got.stdout
