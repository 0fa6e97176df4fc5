"""Runs tests/csrc/test_rows.hip, a C++ caller of the templates behind the
operators between tokens and rows; it exits non-zero on any mismatch."""
import os
import subprocess

import pytest

pytestmark = pytest.mark.gpu
BIN = os.path.join(os.path.dirname(os.path.abspath(__file__)), "csrc", "test_rows")


def test_templates_from_cpp(dev):
    assert os.path.exists(BIN), "build tests/csrc first (make -C tests/csrc)"
    proc = subprocess.run([BIN], capture_output=True, text=True, timeout=110)
    assert proc.returncode == 0, proc.stdout[-2000:] + proc.stderr[-2000:]
    assert "passed" in proc.stdout
