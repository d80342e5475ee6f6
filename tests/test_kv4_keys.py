"""Keys for the 4-bit cache that hold every unit with every code, and what attention makes of them, without a GPU
(tests/test_gpu_kv4_keys.py has it from the kernels)."""
import numpy as np
import pytest

from tests import headref


def keys(D):
    """Rows [510, D] of whole numbers, scale 1: in each group of 32 columns every unit, with all codes in changing columns.  One group of a row
    holds 1785 and has the unit 255; the second 255 rows have it elsewhere."""
    G = -(-D // 32)
    rows = np.zeros((510, D))
    for r, x in enumerate(rows):
        for g in range(G):
            w = min(32, D - 32 * g)
            code = (4 * np.arange(w) + r + g) % 15 - 7
            code[(r + g) % w] = 7 if r % 2 else -7  # makes the unit
            unit = 255 if g == (r % 255 + r // 255) % G else (r + 85 * g) % 255 + 1
            x[32 * g:32 * g + w] = code * unit
    assert (np.abs(rows).max(1) == 1785).all()
    return rows


def stored_from(x):
    """What is stored to become x: a group's largest a little smaller, as 7 u itself may take the unit u + 1 (its products round)."""
    y = x.copy()
    for g in range(0, x.shape[1], 32):
        part = y[:, g:g + 32]
        top = np.abs(part).max(1, keepdims=True)
        part[(np.abs(part) == top) & (top < 1785)] *= 1 - 2.0 ** -9
    return y


def outputs(x, m):
    """Columns 0 and 1 of a row that sees a key of which the query takes x, and m of zeros."""
    e = np.exp(x * 2 / 1785)
    return 1785 * e / (e + m), 1785 * m / (e + m)


@pytest.mark.parametrize("D", [64, 84, 128, 256])
def test_rows_cover_every_unit_and_code(D):
    x = keys(D)
    codes, scales = headref.quantize4(stored_from(x))
    assert np.array_equal(codes, x) and (scales == 1).all()
    for g in range(0, D, 32):
        w = min(32, D - g)
        seen = {(int(np.abs(row[g:g + w]).max()) // 7, int(c)) for row in x for c in row[g:g + w]}
        assert {u for u, _ in seen} == set(range(1, 256))
        if w == 32:
            assert {(u, c) for u in range(1, 256) for c in range(-7 * u, 7 * u + 1, u)} <= seen


def test_a_key_that_is_off_is_seen():
    """One step of the scale moves the output by more than three times what the kernels may be off by."""
    x, m = np.meshgrid(np.arange(-1785.0, 1786.0), np.arange(1, 128), indexing="ij")
    for d in (-1, 1):
        moved = np.abs(outputs(x + d, m)[0] / outputs(x, m)[0] - 1)
        assert moved.min() > 1.3e-4 > 3 * 3.6e-5
