"""Runs tests/csrc/test_rows_limits.hip: sizes that the templates between
tokens and rows refuse (no GPU needed: nothing is allocated or launched)."""
import os
import subprocess

CSRC = os.path.join(os.path.dirname(os.path.abspath(__file__)), "csrc")
BIN = os.path.join(CSRC, "test_rows_limits")


def test_templates_refuse_sizes_they_cannot_index():
    if not os.path.exists(BIN):
        subprocess.check_call(["make", "-C", CSRC, "test_rows_limits"])
    proc = subprocess.run([BIN], capture_output=True, text=True, timeout=110)
    assert proc.returncode == 0, proc.stdout[-2000:] + proc.stderr[-2000:]
    assert "passed" in proc.stdout
