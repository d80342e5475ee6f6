"""Rotary positions, head norms, 4-bit rows and the tables of a serving step without a GPU: the checks of
tests/cpp/step_calls_test.cpp, what the Python calls refuse, and the restatements that the GPU tests compare with."""
import ctypes
import math
import os
import subprocess
from types import SimpleNamespace

import numpy as np
import pytest
import torch

from open_rknpu2_lm_infer_amd import _lib
from open_rknpu2_lm_infer_amd import qlinear as ql
from tests import headref
from tests import test_kv_arguments
from tests.test_kv_arguments import reached  # noqa: F401

BIN = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp", "_build", "step_calls_test")


@pytest.mark.parametrize("mode", ["rules", "tables", "refusals"])
def test_step_calls(mode):
    r = subprocess.run([BIN, mode], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and f"PASS {mode}" in r.stdout, r.stdout[-3000:] + r.stderr[-1000:]


def test_structs_match_header_sizes():
    assert ctypes.sizeof(_lib.RopeConfig) == 72
    assert ctypes.sizeof(_lib.KVTables) == 112


class Tensor(test_kv_arguments.Tensor):
    def get_device(self):
        return self.device.index


ROPE = SimpleNamespace(handle=1, head_dim=64, device=0)
WS = SimpleNamespace(handle=1)
F16 = torch.float16


def test_rope_arguments(reached, monkeypatch):  # noqa: F811
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    x, pos = Tensor(5, 256, dtype=F16), Tensor(5)
    ql.rope(ROPE, x, pos, out=Tensor(5, 256, dtype=F16))
    ql.norm_rope(ROPE, x, pos, 3, None, Tensor(64, dtype=torch.float32), out=Tensor(5, 256, dtype=torch.float32))
    ql.norm_rope(None, x, None, 1, None, None, out=Tensor(5, 256, dtype=F16), head_dim=128)
    assert reached == ["qlin_rope_run", "qlin_rope_run_norm", "qlin_rope_run_norm"]
    bad = [
        lambda: ql.rope(ROPE, Tensor(5, 250, dtype=F16), pos, out=Tensor(5, 250, dtype=F16)),  # no whole heads
        lambda: ql.rope(ROPE, x, Tensor(4), out=x),
        lambda: ql.rope(ROPE, x, Tensor(5, dtype=torch.int64), out=x),
        lambda: ql.rope(ROPE, x, Tensor(5, device="cuda:1"), out=x),
        lambda: ql.rope(ROPE, x, pos, out=Tensor(5, 192, dtype=F16)),
        lambda: ql.rope(ROPE, x, pos, out=Tensor(5, 256, dtype=F16, device="cuda:1")),
        lambda: ql.rope(ROPE, x, None, out=x),
        lambda: ql.rope(SimpleNamespace(handle=1, head_dim=64, device=1), x, pos, out=x),
        lambda: ql.norm_rope(None, Tensor(5, 256, dtype=F16, device="cuda:1"), None, 1, None, None, head_dim=64,
                             out=Tensor(5, 256, dtype=F16, device="cuda:1")),
        lambda: ql.norm_rope(ROPE, x, pos, 5, None, None, out=x),  # more query heads than heads
        lambda: ql.norm_rope(ROPE, x, pos, 3, Tensor(128, dtype=torch.float32), None, out=x),
        lambda: ql.norm_rope(ROPE, x, pos, 3, Tensor(64, dtype=F16), None, out=x),
        lambda: ql.norm_rope(ROPE, x, None, 3, None, None, out=x),
        lambda: ql.norm_rope(None, x, pos, 3, None, None, out=x, head_dim=64),
        lambda: ql.norm_rope(ROPE, x, pos, 3, None, None, out=x, head_dim=128),
    ]
    for call in bad:
        with pytest.raises(AssertionError):
            call()
    assert len(reached) == 3
    with pytest.raises(KeyError):
        ql.Rope(64, layout="quarter")


def test_append_qkv_arguments(reached):  # noqa: F811
    cache = SimpleNamespace(handle=None, page_tokens=16, head_dim=64, columns=128, device=0)
    batch = ql.KVBatch(Tensor(3), Tensor(2), Tensor(2, 4), 5, 3, 64)
    x, g = Tensor(5, 512, dtype=F16), Tensor(64, dtype=torch.float32)
    ql.kv_append_qkv(WS, cache, batch, ROPE, x, 4, g, g, out=Tensor(5, 256, dtype=F16))
    ql.kv_append_qkv(WS, cache, batch, None, x, 4, out=Tensor(6, 256, dtype=F16))
    assert reached == ["qlin_kv_append_qkv"] * 2
    bad = [
        lambda: ql.kv_append_qkv(WS, cache, batch, ROPE, Tensor(5, 500, dtype=F16), 4, out=Tensor(5, 256, dtype=F16)),
        lambda: ql.kv_append_qkv(WS, cache, batch, ROPE, Tensor(4, 512, dtype=F16), 4, out=Tensor(5, 256, dtype=F16)),
        lambda: ql.kv_append_qkv(WS, cache, batch, ROPE, x, 4, out=Tensor(4, 256, dtype=F16)),
        lambda: ql.kv_append_qkv(WS, cache, batch, ROPE, x, 4, out=Tensor(5, 512, dtype=F16)),
        lambda: ql.kv_append_qkv(WS, cache, batch, SimpleNamespace(handle=1, head_dim=128, device=0), x, 4, out=Tensor(5, 256, dtype=F16)),
        lambda: ql.kv_append_qkv(WS, cache, batch, SimpleNamespace(handle=1, head_dim=64, device=1), x, 4, out=Tensor(5, 256, dtype=F16)),
        lambda: ql.kv_append_qkv(WS, cache, batch, ROPE, Tensor(5, 512, dtype=F16, device="cuda:1"), 4, out=Tensor(5, 256, dtype=F16)),
        lambda: ql.kv_append_qkv(WS, cache, batch, ROPE, x, 4, Tensor(32, dtype=torch.float32), out=Tensor(5, 256, dtype=F16)),
        lambda: ql.kv_append_qkv(WS, cache, batch, ROPE, x, 4, Tensor(64, dtype=torch.float32, device="cuda:1"), out=Tensor(5, 256, dtype=F16)),
    ]
    for call in bad:
        with pytest.raises(AssertionError):
            call()
    assert len(reached) == 2


def test_step_arguments(reached):  # noqa: F811
    cache = SimpleNamespace(handle=None, page_tokens=16, pages=20, device=0)

    def make(**kw):
        a = dict(length=Tensor(3), page_table=Tensor(3, 4), free_pages=Tensor(20), free_count=Tensor(1), rows=9, max_new=5,
                 max_len=64, row_start=Tensor(4), maps=False)
        return ql.KVStep(cache, **{**a, **kw})

    batch = ql.kv_step(WS, make(), Tensor(3))
    assert reached == ["qlin_kv_step"] and batch.rows == 9 and batch.c.max_new == 5 and batch.max_len == 64
    assert make(rows=3).batch.c.max_new == 3  # a batch's max_new is at most its rows
    for kw in (dict(length=Tensor(3, dtype=torch.int64)), dict(free_pages=Tensor(19)), dict(free_count=Tensor(2)),
               dict(row_start=Tensor(3)), dict(page_table=Tensor(2, 4)), dict(page_table=Tensor(3, 3)),
               dict(free_pages=Tensor(20, device="cuda:1")), dict(positions=Tensor(8)), dict(slots=Tensor(9)),
               dict(refused=Tensor(2)), dict(row_seq=Tensor(9, dtype=torch.int64)), dict(page_table=Tensor(3, 4, device="cuda:1"))):
        with pytest.raises(AssertionError):
            make(**kw)
    for change in (Tensor(2), Tensor(3, dtype=torch.int64), Tensor(3, device="cuda:1")):
        with pytest.raises(AssertionError):
            ql.kv_step(WS, make(), change)
    assert len(reached) == 1


# ------------------------------------------------------------------ the restatements, by hand


def test_reference_rotation_by_hand():
    w, a = headref.frequencies(4, 10000.0)
    assert np.allclose(w, [1, 0.01]) and a == 1
    x = np.arange(1.0, 7).reshape(1, 1, 6)
    left, right = headref.pairs(1, 4, "half")
    y, _ = headref.rotate(x, np.array([0]), w, 1.0, left, right)
    assert np.array_equal(x, y)
    y, off = headref.rotate(x, np.array([3]), w, 2.0, left, right)
    want = [1, 2 * (2 * math.cos(3) - 4 * math.sin(3)), 2 * (3 * math.cos(.03) - 5 * math.sin(.03)),
            2 * (4 * math.cos(3) + 2 * math.sin(3)), 2 * (5 * math.cos(.03) + 3 * math.sin(.03)), 6]
    assert np.allclose(y[0, 0], want, atol=1e-14) and 0 < off < 2e-6
    left, right = headref.pairs(2, 4, "interleaved")
    y, _ = headref.rotate(x, np.array([1]), w, 1.0, left, right)
    assert np.allclose(y[0, 0, 2:4], [3 * math.cos(1) - 4 * math.sin(1), 4 * math.cos(1) + 3 * math.sin(1)])
    # halving the frequencies, by each scaling's own way
    assert np.allclose(headref.frequencies(8, 1e4, "linear", 2.0)[0], headref.frequencies(8, 1e4)[0] / 2)
    far, near = headref.frequencies(8, 1e4, "base", 4.0)[0], headref.frequencies(8, 1e4)[0]
    assert far[0] == near[0] and math.isclose(far[3], near[3] / 4)  # the first as it is, the last divided
    for how in ("bands", "ramp"):
        w = headref.frequencies(64, 1e4, how, 8.0, 4096, 1.0, 4.0)[0] / headref.frequencies(64, 1e4)[0]
        assert w[0] == 1 and math.isclose(w[-1], 1 / 8) and (np.diff(w) <= 1e-15).all() and ((w < 0.99) & (w > 0.13)).any()


def test_reference_rows_in_4_bits_by_hand():
    x = np.zeros((1, 40), np.float32)
    x[0, 0], x[0, 1], x[0, 33] = 255 * 7, -255 * 3.5, 14.0  # scale 1, units 255 and 2 (or the next: products round)
    c, s = headref.quantize4(x)
    assert abs(s[0] - 1) < 1e-6 and c[0, 0] == 1785 and c[0, 1] in (-3 * 255, -4 * 255) and c[0, 33] in (14, 15) and not c[0, 2:33].any()
    r = np.random.default_rng(0).standard_normal((200, 100)).astype(np.float32) * 10.0 ** np.arange(-10, 10).repeat(10)[:, None].astype(np.float32)
    c, s = headref.quantize4(r)
    g = np.abs(np.pad(r, ((0, 0), (0, 28))).reshape(200, 4, 32)).max(-1).repeat(32, 1)[:, :100]
    # half a code of a unit that is a step of the row's scale too large at most
    assert (np.abs(c * s[:, None] - r) <= 0.5 * (g / 7 + s[:, None]) * 1.0001).all()
    c, s = headref.quantize4(np.array([[0.0, 0.0], [np.inf, 1.0]], np.float32))
    assert s[0] == 2.0 ** -64 and np.isnan(s[1]) and not c.any()


def test_reference_step_by_hand():
    # pages of 4; slot 0 grows by two pages, slot 1 gives a page back, slot 2 wants more than there is, slot 3 is idle
    length, table, free, starts, maps, refused = headref.step(
        [5, -3, 9, 0], [4, 6, 0, 3], [[7, -1, -1], [1, 2, -1], [-1] * 3, [5, -1, -1]], [9, 8], 4, 10, 20, 9, 12)
    assert length == [9, 3, 0, 3] and table == [[7, 2, 8], [1, -1, -1], [-1] * 3, [5, -1, -1]] and free == [9]
    assert starts == [0, 5, 5, 5, 5] and refused == 1
    assert maps == [(0, 4, 8), (0, 5, 9), (0, 6, 10), (0, 7, 11), (0, 8, 32)]
