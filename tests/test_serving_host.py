"""The C++ host layer's attention and log probability calls (tests/cpp/test_host_serving.cpp, built by
__graft_entry__.build()): the checks of their arguments, and a run of them against sums in double."""
import os
import subprocess

import pytest

BIN = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp", "build", "test_host_serving")


def run(*args):
    assert os.path.exists(BIN), f"{BIN} is not built: run __graft_entry__.build()"
    p = subprocess.run([BIN, *args], capture_output=True, text=True, timeout=120)
    print(p.stdout, p.stderr)
    assert p.returncode == 0, p.stdout + p.stderr


def test_refusals():
    run("refusals")


@pytest.mark.gpu
def test_against_sums_in_double():
    run()
