"""Rotary positions and head norms on the GPU against the 64-bit restatement in tests/headref.py, within its bounds."""
import numpy as np
import pytest
import torch

from open_rknpu2_lm_infer_amd import qlinear as ql
from tests import headref

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
F16, F32 = torch.float16, torch.float32
EPS = {F16: 2.0 ** -10, F32: 2.0 ** -23}


def rand(shape, dtype, seed, size=1.0):
    return torch.from_numpy((np.random.default_rng(seed).standard_normal(shape) * size).astype(np.float32)).to(dtype)


def i32(x):
    return torch.as_tensor(np.asarray(x, np.int32), device=DEV)


def check(got, want, tol):
    got = got.double().cpu().numpy()
    assert np.array_equal(np.isnan(got), np.isnan(want))
    inf = np.isinf(want)
    assert np.array_equal(got[inf], want[inf])
    err = np.abs(np.where(inf | np.isnan(want), 0, got - np.where(inf, 0, np.nan_to_num(want))))
    assert (err <= tol).all(), (float(err.max()), float((err / np.maximum(tol, 1e-300)).max()), np.argwhere(err > tol)[:4])


def expected(x, dim, positions, q_heads, gammas, rope, first, layout, out_dtype, inverse=False):
    """Of rows x, a tensor on the host; the frequencies are the handle's own, which test_frequencies checks."""
    rows = x.shape[0]
    if rope is None:
        w, a, left, right = np.zeros(0), 1.0, np.zeros(0, int), np.zeros(0, int)
    else:
        w, a = np.array(rope.radians), rope.amplitude
        left, right = headref.pairs(first, rope.rotary_dim, layout)
    y, tol = headref.heads(x.double().numpy().reshape(rows, -1, dim), np.asarray(positions), q_heads, *gammas, 1e-6, w, a, left, right,
                           EPS[out_dtype], inverse)
    return y.reshape(rows, -1), tol.reshape(rows, -1)


# head dim, rotary columns, the first of them, layout, heads
SHAPES = [
    (128, 128, 0, "half", 40),
    (128, 64, 64, "interleaved", 5),
    (64, 64, 0, "interleaved", 3),
    (64, 16, 0, "half", 70),
    (256, 256, 0, "half", 2),
    (256, 128, 4, "half", 6),
    (96, 32, 8, "interleaved", 8),
    (84, 42, 20, "half", 15),      # pairs and the others no groups of eight
    (250, 250, 0, "half", 3),      # 32 lanes of pairs
    (250, 244, 3, "half", 3),      # more than 32 lanes
    (250, 246, 1, "interleaved", 3),
    (63, 62, 1, "half", 9),        # more than 8 lanes
    (127, 118, 9, "interleaved", 4),
    (2, 2, 0, "half", 1024),
    (3, 2, 1, "interleaved", 17),
    (5, 2, 0, "half", 1),
]


@pytest.mark.parametrize("D,n,first,layout,heads", SHAPES)
@pytest.mark.parametrize("form,dtype,out_dtype", [(f, a, b) for f in ("whole", "columns", "unaligned", "in place")
                                                  for a in (F16, F32) for b in (F16, F32) if f != "in place" or a == b])
def test_rope(dtype, out_dtype, D, n, first, layout, heads, form):
    rows = 7
    pos = [0, 1, 5, 4095, 32767, 1000003, 2]
    rope = ql.Rope(D, n, base=10000.0, first=first, layout=layout)
    x = rand((rows, heads * D), dtype, seed=D + n)
    print(f"[rope] {D} {n} {first} {layout} {heads} {dtype} {out_dtype} {form}", flush=True)
    want, tol = expected(x, D, pos, heads, (None, None), rope, first, layout, out_dtype)
    if form in ("whole", "in place"):
        xd = x.to(DEV)
        got = ql.rope(rope, xd, i32(pos), out=xd if form == "in place" else None, out_dtype=out_dtype)
        check(got, want, tol)
        if form == "whole":
            assert torch.equal(xd.cpu(), x)
    else:
        off = 8 if form == "columns" else 1
        wide = torch.full((rows, off + heads * D + (8 if form == "columns" else 3)), float("nan"), dtype=dtype, device=DEV)
        wide[:, off:off + heads * D] = x.to(DEV)
        out = torch.full((rows + 2, off + heads * D + off), 7.0, dtype=out_dtype, device=DEV)
        got = ql.rope(rope, wide[:, off:off + heads * D], i32(pos), out=out[:rows, off:off + heads * D])
        check(got, want, tol)
        assert (out[rows:] == 7).all() and (out[:, :off] == 7).all() and (out[:, off + heads * D:] == 7).all()


@pytest.mark.parametrize("scaling,kw", [
    ("plain", {}), ("linear", dict(factor=4.0)), ("base", dict(factor=8.0)),
    ("bands", dict(factor=8.0, original_len=8192, low=1.0, high=4.0)),
    ("ramp", dict(factor=16.0, original_len=4096, low=1.0, high=32.0)),
    ("ramp", dict(factor=32.0, original_len=10, low=1.0, high=32.0)),  # all pairs turn slowly: the ramp's ends meet
])
@pytest.mark.parametrize("D,n,base", [(128, 128, 1e6), (64, 2, 1e4), (96, 34, 5e5)])
def test_frequencies(scaling, kw, D, n, base):
    rope = ql.Rope(D, n, base=base, scaling=scaling, **kw)
    ref = {("original" if k == "original_len" else k): v for k, v in kw.items()}
    w, a = headref.frequencies(n, base, scaling, **ref)
    assert np.allclose(rope.radians, w, rtol=1e-13, atol=0) and abs(rope.amplitude - a) < 1e-13
    x, pos = rand((4, 3 * D), F32, seed=n), [0, 17, 70000, 131071]
    want, tol = expected(x, D, pos, 3, (None, None), rope, 0, "half", F32)
    check(ql.rope(rope, x.to(DEV), i32(pos)), want, tol)
    assert ql.Rope(D, n, scaling=scaling, amplitude=0.25, **kw).amplitude == 0.25


def test_far_positions():
    """Any int32: against angles reduced in whole numbers (turns a position as a fraction of 2^96)."""
    D = 128
    rope = ql.Rope(D, base=1e6)
    pos = [2 ** 31 - 1, -2 ** 31, -1, 2 ** 30 + 12345, 123456789, -7]
    x = rand((len(pos), D), F32, seed=3).double().numpy()
    turns = [int(w.as_integer_ratio()[0] * 2 ** 96 * 10 ** 30 // (w.as_integer_ratio()[1] * 6283185307179586476925286766559)) for w in rope.radians]
    t = np.array([[(p * f % 2 ** 96) / 2 ** 96 * 2 * np.pi for f in turns] for p in pos])
    y = np.concatenate([x[:, :64] * np.cos(t) - x[:, 64:] * np.sin(t), x[:, 64:] * np.cos(t) + x[:, :64] * np.sin(t)], 1)
    # as headref.rotate counts: 2^31 * w * 2^-51 quarter turns at most, two roundings of 2^-53 each of up to 2^31 * 0.64
    off = np.pi / 2 * (2.0 ** -26 + 2.0 ** 31 * 2.0 ** -51) + 8 * 2.0 ** -24
    size = np.abs(x[:, :64]) + np.abs(x[:, 64:])
    check(ql.rope(rope, torch.from_numpy(x).float().to(DEV), i32(pos)), y, off * np.concatenate([size, size], 1) + 2.0 ** -24 * np.abs(y))


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_turned_back(layout):
    """QLIN_ROPE_INVERSE is the transposed map: against its formula, and there and back again."""
    D, pos = 128, [3, 999, 70001]
    rope = ql.Rope(D, 96, first=16, layout=layout, amplitude=0.5)
    x = rand((3, 4 * D), F32, seed=9)
    want, tol = expected(x, D, pos, 4, (None, None), rope, 16, layout, F32, inverse=True)
    got = ql.rope(rope, x.to(DEV), i32(pos), flags=ql.QLIN_ROPE_INVERSE)
    check(got, want, tol)
    there = ql.rope(rope, x.to(DEV), i32(pos))
    # <R x, y> = <x, R' y>: f32 results, each off by its bound
    y = rand((3, 4 * D), F32, seed=10)
    back = ql.rope(rope, y.to(DEV), i32(pos), flags=ql.QLIN_ROPE_INVERSE).double().cpu()
    a, b = (there.double().cpu() * y.double()).sum(), (x.double() * back).sum()
    assert abs(a - b) < 2 * float((tol.max() * (x.abs().sum() + y.abs().sum())))
    once = ql.rope(ql.Rope(D, 96, first=16, layout=layout), x.to(DEV), i32(pos))
    again = ql.rope(ql.Rope(D, 96, first=16, layout=layout), once, i32(pos), flags=ql.QLIN_ROPE_INVERSE)
    check(again, x.double().numpy(), 4 * tol + 4 * 2.0 ** -20)


def test_nonfinite_values_stay_in_their_pair():
    D = 64
    x = rand((2, 3 * D), F16, seed=4)
    x[0, 70] = float("nan")   # head 1, column 6: pair 6
    x[1, 5] = float("inf")    # head 0
    rope = ql.Rope(D, 32, layout="half")
    got = ql.rope(rope, x.to(DEV), i32([3, 3])).cpu()
    bad = torch.zeros(2, 3 * D, dtype=torch.bool)
    bad[0, 70] = bad[0, 70 + 16] = bad[1, 5] = bad[1, 5 + 16] = True
    assert torch.equal(torch.isfinite(got), ~bad)
    assert torch.isnan(got[0, 70]) and torch.isnan(got[0, 86])


# ------------------------------------------------------------------ norms


@pytest.mark.parametrize("dtype,out_dtype", [(F16, F16), (F32, F32), (F16, F32)])
@pytest.mark.parametrize("D,n,first,layout,heads", SHAPES)
@pytest.mark.parametrize("which", ["both", "queries", "keys", "norms alone"])
def test_norm_rope(dtype, out_dtype, D, n, first, layout, heads, which):
    rows, q_heads = 5, (heads + 1) // 2
    pos = [0, 12, 4095, 100000, 7]
    rope = None if which == "norms alone" else ql.Rope(D, n, base=10000.0, first=first, layout=layout, amplitude=1.25)
    g = [(rand((D,), F32, seed=D + i, size=0.3) + 1.0) for i in range(2)]
    if which == "queries":
        g[1] = None
    if which == "keys":
        g[0] = None
    x = rand((rows, heads * D), dtype, seed=D + heads) * torch.tensor([1.0, 30.0, 0.01, 200.0, 3.0], dtype=dtype)[:, None]
    x[4, :D] = 0
    print(f"[norm] {D} {n} {first} {layout} {heads} {dtype} {out_dtype} {which}", flush=True)
    want, tol = expected(x, D, pos, q_heads, g, rope, first, layout, out_dtype)
    gd = [None if t is None else t.to(DEV) for t in g]
    got = ql.norm_rope(rope, x.to(DEV), i32(pos) if rope else None, q_heads, *gd, out_dtype=out_dtype, head_dim=D)
    check(got, want, tol)
    if dtype == out_dtype:
        xd = x.to(DEV)
        assert ql.norm_rope(rope, xd, i32(pos) if rope else None, q_heads, *gd, out=xd, head_dim=D) is xd
        assert torch.equal(xd, got)


def test_norms_of_extreme_rows():
    D = 64
    g = torch.ones(D, device=DEV)
    x = torch.zeros((6, D))
    x[0] = 2.0 ** 58 * (torch.arange(D) % 3 - 1.0)
    x[1] = 1e-30
    x[2, 3] = 2.0 ** 59
    x[4] = 1.0
    x[4, 7] = float("inf")
    x[5] = 1.0
    x[5, 9] = float("nan")
    y = ql.norm_rope(None, x.to(DEV), None, 1, g, None, head_dim=D).cpu()
    want, tol = expected(x[:4], D, [0] * 4, 1, (np.ones(D), None), None, 0, "half", F32)
    check(y[:4], want, tol)
    assert torch.isnan(y[4, 7]) and not y[4, :7].any() and torch.isnan(y[5]).all()
    # an eps that is no normal number leaves zeros zeros
    y = ql.norm_rope(None, torch.zeros((2, D), device=DEV), None, 1, g, None, eps=1e-42, head_dim=D)
    assert not y.any()
    # the largest fp16
    x = torch.full((1, D), 65504.0, dtype=F16, device=DEV)
    assert torch.equal(ql.norm_rope(None, x, None, 1, g, None, head_dim=D).cpu(), torch.ones((1, D), dtype=F16))


@pytest.mark.parametrize("rows", [0, 1, 2, 63, 700, 5000])
def test_any_number_of_rows(rows):
    """Each row's result is its own, however many workgroups a row has."""
    D, heads = 128, 20
    rope = ql.Rope(D, base=1e6)
    g = (rand((D,), F32, seed=1) + 2.0).to(DEV)
    x = rand((max(rows, 1), heads * D), F16, seed=rows).to(DEV)[:rows]
    pos = torch.arange(rows, dtype=torch.int32, device=DEV) * 7
    out = torch.full((rows + 1, heads * D), 5.0, dtype=F16, device=DEV)
    ql.norm_rope(rope, x, pos, 16, g, g, out=out[:rows])
    assert (out[rows:] == 5).all()
    for r in {0, rows // 2, rows - 1} if rows else ():
        one = ql.norm_rope(rope, x[r:r + 1], pos[r:r + 1], 16, g, g)
        assert torch.equal(one[0], out[r])
    if rows > 1:
        want, tol = expected(x[-2:].cpu(), D, pos[-2:].cpu().numpy(), 16, (g.cpu().numpy(),) * 2, rope, 0, "half", F16)
        check(out[rows - 2:rows], want, tol)


@pytest.mark.parametrize("D,n,first,layout,heads", [s for s in SHAPES if s[4] <= 8])
@pytest.mark.parametrize("rows", [1025, 2050, 2303])
@pytest.mark.parametrize("dtype", [F16, F32])
def test_many_rows_of_every_shape(D, n, first, layout, heads, rows, dtype):
    """Four rows a workgroup, the last one with fewer: a row's result is that of the row alone."""
    rope = ql.Rope(D, n, first=first, layout=layout)
    g = (rand((D,), F32, seed=1) + 2.0).to(DEV)
    x, pos = rand((rows, heads * D), dtype, seed=rows).to(DEV), torch.arange(rows, dtype=torch.int32, device=DEV) * 3
    out = torch.full((rows + 1, heads * D), 5.0, dtype=dtype, device=DEV)
    ql.norm_rope(rope, x, pos, heads // 2, g, None, out=out[:rows])
    assert (out[rows:] == 5).all()
    for r in (0, 1, 2, 3, 4, rows // 2, rows - 3, rows - 2, rows - 1):
        assert torch.equal(ql.norm_rope(rope, x[r:r + 1], pos[r:r + 1], heads // 2, g, None)[0], out[r]), r


def test_f32_rows_past_what_the_caches_hold():
    """40 million columns and a few: one row a workgroup again, results those of a few rows."""
    D, heads, rows = 128, 40, 7830
    rope, x = ql.Rope(D, layout="interleaved"), rand((rows, heads * D), F32, seed=3).to(DEV)
    pos = torch.arange(rows, dtype=torch.int32, device=DEV)
    out = torch.full((rows + 1, heads * D), 5.0, dtype=F32, device=DEV)
    ql.rope(rope, x, pos, out=out[:rows])
    assert (out[rows:] == 5).all()
    for a in range(0, rows, 700):
        assert torch.equal(ql.rope(rope, x[a:a + 700], pos[a:a + 700]), out[a:min(a + 700, rows)]), a


def test_streams_and_captured_rows():
    """On a stream of its own and in a graph, replayed with other rows and positions and eager calls in between."""
    D, heads, rows = 64, 6, 33
    rope = ql.Rope(D, layout="interleaved")
    x, pos = torch.zeros((rows, heads * D), dtype=F16, device=DEV), torch.zeros(rows, dtype=torch.int32, device=DEV)
    out = torch.empty_like(x)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ql.rope(rope, x, pos, out=out)
    st = torch.cuda.Stream()
    for rep in range(4):
        x.copy_(rand((rows, heads * D), F16, seed=rep).to(DEV))
        pos.copy_(torch.arange(rows, dtype=torch.int32, device=DEV) * (rep + 1) * 1000)
        out.fill_(3.0)
        g.replay()
        torch.cuda.synchronize()
        with torch.cuda.stream(st):
            eager = ql.rope(rope, x, pos)
        torch.cuda.synchronize()
        assert torch.equal(out, eager), rep
    del g
