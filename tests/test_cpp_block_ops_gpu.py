"""Runs the C++ program that puts the block operators of llmt's C++ interface in a row and checks each against loops."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BIN = os.path.join(ROOT, "tests", "cpp", "_build", "test_block_ops")


@pytest.mark.gpu
def test_block_operators_of_the_cpp_interface():
    assert os.path.exists(BIN), "run `python -m llmt_b200.build` (or __graft_entry__.build()) first"
    r = subprocess.run([BIN], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout[-2000:] + r.stderr[-2000:]
    assert "15 checks, 0 failures" in r.stdout
