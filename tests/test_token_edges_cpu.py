"""Token operators at their limits: the checks compiled and run on the CPU."""
import os
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, os.pardir, "cl-eden-kernel_b200", "csrc")


@pytest.fixture(scope="module")
def checks(tmp_path_factory):
    exe = str(tmp_path_factory.mktemp("token_edges") / "token_edges_test")
    subprocess.run(["/usr/bin/g++", "-std=c++17", "-O1", "-Wall", "-fsanitize=signed-integer-overflow", "-fno-sanitize-recover", "-I", CSRC,
                    os.path.join(HERE, "token_edges_test.cpp"), "-o", exe], check=True)
    return exe


@pytest.mark.parametrize("which", ["sizes", "overlaps", "calls", "scales"])
def test_checks(checks, which):
    r = subprocess.run([checks, which], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr
