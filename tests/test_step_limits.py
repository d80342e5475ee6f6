"""The tables of a serving step at their limits, without a GPU: the checks of tests/cpp/step_limits_test.cpp."""
import os
import subprocess

import pytest

BIN = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp", "_build", "step_limits_test")


@pytest.mark.parametrize("mode", ["places"])
def test_step_limits(mode):
    r = subprocess.run([BIN, mode], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and f"PASS {mode}" in r.stdout, r.stdout[-3000:] + r.stderr[-1000:]
