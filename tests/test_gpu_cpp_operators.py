"""Runs the self-checking C++ program for the quantiser, scaled GEMM and orthogonalisation classes."""
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "tests", "cpp"))

pytestmark = pytest.mark.gpu


def test_cpp_operators_program():
    import build_operators_test

    res = subprocess.run([build_operators_test.build()], capture_output=True, text=True, timeout=600)
    print(res.stdout)
    print(res.stderr, file=sys.stderr)
    assert res.returncode == 0, res.stdout + res.stderr
    assert "0 failure(s)" in res.stdout and res.stdout.count("PASS") == 4
