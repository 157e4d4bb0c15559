"""How the chunks of an eviction wait for each other, walked on the host, and waits that are refused."""
import ctypes
import os
import shutil
import subprocess

import pytest

from intrasm_engine_amd import _lib
from test_long_generation_arguments import A, cache

HERE = os.path.dirname(os.path.abspath(__file__))


def test_whom_a_chunk_waits_for(tmp_path):
    compiler = shutil.which("g++")
    assert compiler, "needs a host C++ compiler"
    exe = str(tmp_path / "check")
    subprocess.run([compiler, "-O2", "-std=c++17", "-Wall", "-Werror", os.path.join(HERE, "evict_chunks_check.cpp"), "-o", exe], check=True)
    for seed in range(4):
        got = subprocess.run([exe, str(seed)], stdout=subprocess.PIPE, text=True)
        assert got.returncode == 0, got.stdout


@pytest.mark.parametrize("tries", [-1, (1 << 20) + 1])
def test_waits_that_are_refused(tries):
    c = cache()
    assert _lib.load().iex_evict_tokens_within(ctypes.byref(c), A, A, 100, 10, 2, A, tries, A, 1 << 40, None) == -1 and "looks" in _lib.last_error()
