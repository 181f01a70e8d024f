"""Refusals of the token operators: the checks compiled and run on the CPU, and the entry points without a context."""
import ctypes as C
import os
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, os.pardir, "cl-eden-kernel_b200", "csrc")


def test_descriptor_and_call_checks(tmp_path):
    exe = str(tmp_path / "token_check_test")
    subprocess.run(["/usr/bin/g++", "-std=c++17", "-O1", "-Wall", "-I", CSRC, os.path.join(HERE, "token_check_test.cpp"), "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout


def test_token_struct_sizes_match_header(enn):
    assert C.sizeof(enn.TokenFcDesc) == 24
    assert C.sizeof(enn.TokenNormDesc) == 11 * 4
    assert C.sizeof(enn.TokenGateDesc) == 6 * 4
    assert C.sizeof(enn.LogProbsDesc) == 32


def test_null_arguments(enn):
    h = C.c_void_p()
    byte, one = (C.c_int8 * 1)(), (C.c_float * 1)()
    assert enn.lib.enn_b200_token_fc_prepare(None, C.byref(enn.TokenFcDesc(m=1, k=1, n=1, out_dtype=enn.F32)), byte, one, None, C.byref(h)) == enn.INVALID_PARAMS
    assert enn.lib.enn_b200_token_norm_prepare(None, None, None, None, None, None, C.byref(h)) == enn.INVALID_PARAMS
    assert enn.lib.enn_b200_token_gate_prepare(None, None, C.byref(h)) == enn.INVALID_PARAMS
    assert enn.lib.enn_b200_log_probs_prepare(None, None, C.byref(h)) == enn.INVALID_PARAMS
    assert enn.lib.enn_b200_op_execute_rows(None, 0, None, 0, None, 0) == enn.INVALID_PARAMS
    assert enn.lib.enn_b200_oplist_add_op_n(None, None, None, 0, None, 0) == enn.INVALID_PARAMS
    assert enn.token_pitch(4097) == 4112 and enn.token_pitch(0) == 0


def test_constants_of_the_wrong_size(enn):
    with pytest.raises(ValueError):
        enn.token_fc(None, enn.TokenFcDesc(m=1, k=4, n=2, out_dtype=enn.F32), [1] * 7, [1.0] * 2)
