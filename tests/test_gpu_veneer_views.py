"""Runs the C++ veneer's test program of the sequence-model operators on views (tests/cpp/sequence_views_test.cpp)."""
import os
import subprocess

import pytest

pytestmark = pytest.mark.gpu

BIN = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp", "sequence_views_test.bin")


def test_cpp_sequence_views_program():
    assert os.path.exists(BIN), "run __graft_entry__.build() first"
    r = subprocess.run([BIN], capture_output=True, text=True, timeout=110)
    assert r.returncode == 0, r.stdout + r.stderr
    assert " 0 failed" in r.stdout
