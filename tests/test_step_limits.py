"""The tables of a serving step at their limits, without a GPU: the checks of tests/cpp/step_limits_test.cpp."""
import os
import subprocess

import pytest

from tests import headref

BIN = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp", "_build", "step_limits_test")


@pytest.mark.parametrize("mode", ["places", "room"])
def test_step_limits(mode):
    r = subprocess.run([BIN, mode], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and f"PASS {mode}" in r.stdout, r.stdout[-3000:] + r.stderr[-1000:]


# change of each slot, max_new, max_len, free pages; the rows each gets of 8, with lengths of 10 and pages of 16
REFUSED = [
    ([10, 2], 16, 100, 9, [0, 2]),            # more than there are rows at all: in nobody's way
    ([9, 8], 9, 100, 9, [0, 8]),
    ([17, 8], 16, 100, 9, [0, 8]),            # above max_new
    ([5, 8], 16, 14, 9, [0, 0]),              # past max_len, both
    ([5, 4], 16, 14, 9, [0, 4]),
    ([6, 3, 2], 16, 100, 9, [6, 0, 0]),       # too late: two rows are left, but the sum has passed them
    ([6, 9, 2], 16, 100, 9, [6, 0, 2]),       # too large between them
    ([2, 8, 6], 16, 100, 0, [2, 0, 0]),
    ([7, 1, 0], 16, 100, 0, [0, 1, 0]),       # no page for the first; the second needs none
    ([2 ** 31 - 1, 3, 5], 2 ** 24, 2 ** 20, 9, [0, 3, 5]),
]


@pytest.mark.parametrize("change,max_new,max_len,spare,rows", REFUSED)
def test_who_is_refused(change, max_new, max_len, spare, rows):
    n = len(change)
    table = [[i] + [-1] * 6 for i in range(n)]
    length, _, _, starts, _, refused = headref.step(change, [10] * n, table, list(range(n, n + spare)), 16, n + spare, 8, max_new, max_len)
    assert [b - a for a, b in zip(starts, starts[1:])] == rows and length == [10 + r for r in rows]
    assert refused == sum(c > 0 and r == 0 for c, r in zip(change, rows))
