"""Key/value cache without a GPU: the checks of tests/cpp/kv_calls_test.cpp (indexing, refusals) and the
plain restatement that the GPU tests compare with."""
import ctypes
import os
import subprocess

import numpy as np
import pytest

from open_rknpu2_lm_infer_amd import _lib
from tests import kvref

BIN = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp", "_build", "kv_calls_test")


@pytest.mark.parametrize("mode", ["index", "refusals"])
def test_kv_calls(mode):
    r = subprocess.run([BIN, mode], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and f"PASS {mode}" in r.stdout, r.stdout[-3000:] + r.stderr[-1000:]


def test_structs_match_header_sizes():
    assert ctypes.sizeof(_lib.KVConfig) == 16
    assert ctypes.sizeof(_lib.KVInfo) == 32
    assert ctypes.sizeof(_lib.KVBatch) == 48


def test_reference_quantize_matches_oracle(oracle):
    """The cache's rule is the activations' rule, but for a multiplication by 1/127 in the place of the division: scales
    differ by one step of f32 at most (the factor is off by half a step and the product rounded once more), and
    where they are equal so are the codes."""
    x = np.random.default_rng(1).standard_normal((40, 96)).astype(np.float32) * 10.0 ** np.arange(-10, 10).repeat(2)[:, None]
    x = x.astype(np.float32)
    for even in (False, True):
        c, s = kvref.quantize(x, even)
        q, so, bad = oracle.quantize(x, oracle.ROUND_EVEN if even else oracle.ROUND_AWAY)
        same = s.view(np.int32) == so.view(np.int32)
        assert bad == 0 and (np.abs(s.view(np.int32) - so.view(np.int32)) <= 1).all() and same.sum() >= 20
        assert np.array_equal(c[same], q[same]) and np.abs(c - q).max() <= 1
    c, s = kvref.quantize(np.array([[0.0, 0.0], [2.0 ** -70, 0.0], [np.nan, 1.0]], np.float32))
    assert s[0] == s[1] == 2.0 ** -64 and np.isnan(s[2]) and not c[0].any() and c[1, 0] == 0 and not c[2].any()


def test_reference_attention_by_hand():
    one = np.ones((1, 1), np.float32)
    # one token: its value; two equal keys: the mean; nothing seen: zeros
    kc, vc = np.array([[[1.0, 0.0]], [[1.0, 0.0]]]), np.array([[[3.0, 5.0]], [[7.0, 1.0]]])
    q = np.array([[[1.0, 2.0]]] * 3)
    o, tol = kvref.attend(q, kc, one.repeat(2, 0), vc, one.repeat(2, 0), [1, 2, 0], 0.5, 1, 2.0 ** -10)
    assert np.allclose(o[:, 0], [[3, 5], [5, 3], [0, 0]]) and (tol[:2] > 0).all() and not tol[2].any()
