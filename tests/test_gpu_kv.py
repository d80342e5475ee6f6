"""Key/value cache and its attention on the GPU against the 64-bit restatement in tests/kvref.py: stored rows
exactly, attention within the bound that kvref derives."""
import math

import numpy as np
import pytest
import torch

from open_rknpu2_lm_infer_amd import _lib
from open_rknpu2_lm_infer_amd import qlinear as ql
from open_rknpu2_lm_infer_amd import synth
from tests import kvref

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
F16, F32 = torch.float16, torch.float32
EPS = {F16: 2.0 ** -10, F32: 2.0 ** -23}


@pytest.fixture(scope="module")
def ws():
    w = ql.Workspace(1, 256, 256)
    yield w
    w.close()


def i32(x):
    return torch.as_tensor(np.asarray(x, np.int32), device=DEV)


class Setup:
    """Sequences of the given (length, new rows) whose tokens lie in scattered pages; rows on the host as f64."""

    def __init__(self, ws, seqs, kv_heads, dim, page, dtype, seed, q_heads=None, max_len=None, spare=3):
        self.ws, self.seqs, self.hk, self.D, self.P, self.dtype = ws, seqs, kv_heads, dim, page, dtype
        self.hq = q_heads or kv_heads
        self.rng = np.random.default_rng(seed)
        self.max_len = max(max(n for n, _ in seqs), 1) if max_len is None else max_len
        cols = max(1, -(-self.max_len // page))
        pages = len(seqs) * cols + spare
        self.table = self.rng.permutation(pages)[:len(seqs) * cols].reshape(len(seqs), cols).astype(np.int32)
        self.cache = ql.KVCache(kv_heads, dim, pages, page)
        self.starts = np.concatenate([[0], np.cumsum([n for _, n in seqs])])
        self.rows = int(self.starts[-1])

    def rand(self, *shape, size=1.0):
        x = (self.rng.standard_normal(shape) * size).astype(np.float32)
        return torch.from_numpy(x).to(self.dtype)

    def batch(self, lens=None, news=None, max_new=None, max_len=None, table=None):
        lens = [n for n, _ in self.seqs] if lens is None else lens
        news = [n for _, n in self.seqs] if news is None else news
        starts = np.concatenate([[0], np.cumsum(news)])
        return ql.KVBatch(i32(starts), i32(lens), i32(self.table if table is None else table), int(starts[-1]),
                          max(list(news) + [0]) if max_new is None else max_new, max_len or self.max_len)

    def fill(self, k, v):
        """Stores all tokens of every sequence: k, v [sum of lengths, kv_heads * D]."""
        b = self.batch(news=[n for n, _ in self.seqs])
        ql.kv_append(self.ws, self.cache, b, k.to(DEV), v.to(DEV))

    def history(self, size_k=1.0, size_v=1.0):
        n = sum(n for n, _ in self.seqs)
        k, v = self.rand(n, self.hk * self.D, size=size_k), self.rand(n, self.hk * self.D, size=size_v)
        return k, v

    def expected(self, q, k, v, out_dtype, scale=None, seqs=None):
        limbs = 1 if self.dtype == F16 and out_dtype == F16 else 2
        outs, tols, at = [], [], 0
        for i, (n, m) in enumerate(seqs or self.seqs):
            kc, ks = kvref.quantize(k[at:at + n].float().numpy().reshape(n, self.hk, self.D))
            vc, vs = kvref.quantize(v[at:at + n].float().numpy().reshape(n, self.hk, self.D))
            at += n
            r = int(self.starts[i])
            qi = q[r:r + m].double().numpy().reshape(m, self.hq, self.D)
            o, t = kvref.attend(qi, kc, ks, vc, vs, [n - m + j + 1 for j in range(m)], scale or self.D ** -0.5, limbs,
                                EPS[out_dtype])
            outs.append(o.reshape(m, self.hq * self.D))
            tols.append(t.reshape(m, self.hq * self.D))
        return np.concatenate(outs), np.concatenate(tols)


def check(got, want, tol):
    got = got.double().cpu().numpy()
    assert np.array_equal(np.isnan(got), np.isnan(want))
    err = np.abs(np.nan_to_num(got) - np.nan_to_num(want))
    assert (err <= tol).all(), (float(err.max()), float((err / np.maximum(tol, 1e-300)).max()), np.argwhere(err > tol)[:4])


# ------------------------------------------------------------------ append and read

STORE = [  # (length, new) of the sequences, kv heads, head dim, page
    ([(1, 1)], 1, 64, 16),
    ([(300, 1), (0, 0), (17, 17), (64, 2)], 8, 128, 64),
    ([(40, 33), (16, 16), (5, 1)], 3, 84, 16),
    ([(200, 200)], 2, 256, 32),
    ([(33, 20), (70, 3)], 5, 1, 16),
    ([(50, 50)], 2, 200, 128),
    ([(3, 5), (2, 4)], 2, 40, 16),  # more rows than tokens: the first have no token
]


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("seqs,hk,D,P", STORE)
@pytest.mark.parametrize("form", ["contiguous", "columns", "unaligned"])
def test_append_then_read(ws, dtype, seqs, hk, D, P, form):
    s = Setup(ws, seqs, hk, D, P, dtype, seed=D + P)
    k, v = s.rand(s.rows, hk * D, size=3.0), s.rand(s.rows, hk * D, size=0.01)
    k[0, 0] = 40.0
    v[s.rows // 2] = 0.0
    if form == "contiguous":
        kd, vd = k.to(DEV), v.to(DEV)
    else:  # columns of wider rows, as those of a qkv projection; or from an odd column on
        off = 4 * hk * D if form == "columns" else 3
        wide = torch.full((s.rows, off + 2 * hk * D + 5 * (form == "unaligned")), float("nan"), dtype=dtype, device=DEV)
        kd, vd = wide[:, off:off + hk * D], wide[:, off + hk * D:off + 2 * hk * D]
        kd.copy_(k)
        vd.copy_(v)
    half_even = form == "columns"
    b = s.batch()
    ql.kv_append(ws, s.cache, b, kd, vd, flags=ql.QLIN_ROUND_HALF_EVEN if half_even else 0)
    want = []
    for x in (k, v):
        c, sc = kvref.quantize(x.float().numpy().reshape(s.rows, hk, D), half_even)
        y = (c.astype(np.float32) * sc[..., None]).reshape(s.rows, hk * D)
        for i, (n, m) in enumerate(seqs):
            y[s.starts[i]:s.starts[i] + max(0, m - n)] = 0
        want.append(y)
    for out_dtype in (F16, F32):
        if form == "unaligned":
            buf = torch.full((s.rows + 2, 2 * hk * D + 7), 5.0, dtype=out_dtype, device=DEV)
            ko, vo = buf[:, 1:1 + hk * D], buf[:, 3 + hk * D:3 + 2 * hk * D]
            ql.kv_read(ws, s.cache, b, ko, vo)
            assert (buf[s.rows:] == 5).all() and (buf[:, 0] == 5).all() and (buf[:, 1 + hk * D:3 + hk * D] == 5).all()
            ko, vo = ko[:s.rows], vo[:s.rows]
        else:
            ko, vo = ql.kv_read(ws, s.cache, b, out_dtype=out_dtype)
        for o, w in zip((ko, vo), want):
            assert torch.equal(o.cpu(), torch.from_numpy(w).to(out_dtype))
    assert ws.status() == 0
    s.cache.close()


def test_rounding_ties(ws):
    """Rows whose x * (1/s) is exactly a half, and rows of the smallest values."""
    D = 64
    x = torch.zeros((4, D))
    x[0] = torch.arange(D) - 31.5
    x[0, 0] = 127.0
    x[1] = -x[0]
    x[2, 3], x[2, 4] = 2.0 ** -66, -(2.0 ** -64)  # under the smallest scale: a quarter rounds to 0, one to 1
    x[3, 0] = 3e38
    for even in (False, True):
        s = Setup(ws, [(4, 4)], 1, D, 16, F32, seed=1)
        b = s.batch()
        ql.kv_append(ws, s.cache, b, x.to(DEV), x.to(DEV), flags=ql.QLIN_ROUND_HALF_EVEN if even else 0)
        c, sc = kvref.quantize(x.numpy(), even)
        for o in ql.kv_read(ws, s.cache, b, out_dtype=F32):
            assert torch.equal(o.cpu(), torch.from_numpy(c.astype(np.float32) * sc[:, None]))
        assert float(c[2, 3]) == 0 and float(c[2, 4]) == -1


@pytest.mark.parametrize("dtype", [F16, F32])
def test_nonfinite_rows_are_poisoned_alone(ws, dtype):
    s = Setup(ws, [(20, 20)], 2, 72, 16, dtype, seed=3)
    k, v = s.history()
    k[4, 71], v[9, 100] = float("nan"), float("-inf")  # head 0 of token 4, head 1 of token 9
    ws.status()
    b = s.batch()
    ql.kv_append(ws, s.cache, b, k.to(DEV), v.to(DEV))
    assert ws.status() == _lib.QLIN_ERR_NONFINITE and ws.status() == 0
    ko, vo = ql.kv_read(ws, s.cache, b, out_dtype=F32)
    for o, x in ((ko, k), (vo, v)):
        c, sc = kvref.quantize(x.float().numpy().reshape(20, 2, 72))
        w = (c.astype(np.float32) * sc[..., None]).reshape(20, 144)
        assert np.array_equal(o.cpu().numpy(), w, equal_nan=True)
        assert np.isnan(w).sum() == 72
    q = s.rand(20, 144)
    out = ql.kv_attention(ws, s.cache, b, q.to(DEV))
    want, tol = s.expected(q, k, v, dtype)
    assert np.isnan(want[4:, :72]).all() and not np.isnan(want[:4]).any() and not np.isnan(want[:9, 72:]).any()
    check(out, want, tol)


# ------------------------------------------------------------------ attention

ATTEND = [  # (length, new), q heads, kv heads, head dim, page
    ([(1, 1)], 4, 1, 64, 16),
    ([(300, 1)], 32, 8, 128, 64),
    ([(127, 1), (128, 1), (129, 1), (0, 0), (15, 1), (16, 1), (17, 1), (31, 1), (33, 1), (1000, 1)], 8, 2, 128, 16),
    ([(50, 4), (4, 4), (3, 5), (0, 2), (700, 3)], 6, 2, 80, 32),  # rows without a token among them
    ([(90, 90), (260, 37)], 8, 2, 64, 64),
    ([(150, 20)], 16, 1, 128, 16),
    ([(333, 9), (20, 1)], 3, 3, 256, 128),
    ([(65, 65)], 5, 5, 1, 16),
    ([(2500, 2)], 8, 8, 33, 256),
]


@pytest.mark.parametrize("dtype,out_dtype", [(F16, F16), (F32, F32), (F16, F32), (F32, F16)])
@pytest.mark.parametrize("seqs,hq,hk,D,P", ATTEND)
def test_attention(ws, dtype, out_dtype, seqs, hq, hk, D, P):
    s = Setup(ws, seqs, hk, D, P, dtype, seed=len(seqs) + D, q_heads=hq)
    k, v = s.history(size_k=2.0)
    s.fill(k, v)
    q = s.rand(s.rows, hq * D, size=1.5)
    print(f"[kv] {seqs} {hq} {hk} {D} {P} {dtype}", flush=True)
    out = ql.kv_attention(ws, s.cache, s.batch(), q.to(DEV), out_dtype=out_dtype)
    check(out, *s.expected(q, k, v, out_dtype))
    assert ws.status() == 0
    s.cache.close()


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("seqs,hq,hk,D,P", [
    ([(2100, 1500)], 4, 2, 128, 64),            # a prompt with a past
    ([(600, 600), (33, 33), (257, 129), (0, 0)], 6, 2, 64, 32),
    ([(9000, 300)], 8, 1, 128, 64),             # few rows over a long past: cut along the tokens
    ([(700, 350)], 2, 1, 256, 16),
    ([(520, 513)], 3, 1, 100, 16),
])
def test_prompts(ws, dtype, seqs, hq, hk, D, P):
    s = Setup(ws, seqs, hk, D, P, dtype, seed=len(seqs) + D, q_heads=hq)
    k, v = s.history(size_k=2.0)
    s.fill(k, v)
    q = s.rand(s.rows, hq * D, size=1.5)
    print(f"[kv prompt] {seqs} {hq} {hk} {D} {P} {dtype}", flush=True)
    out = ql.kv_attention(ws, s.cache, s.batch(), q.to(DEV))
    check(out, *s.expected(q, k, v, dtype))
    s.cache.close()


def test_strides_and_rows_of_nobody(ws):
    """Queries as columns of qkv rows, outputs into wider rows at odd offsets; rows behind the last sequence and the
    columns beside the output stay as they were."""
    hq, hk, D = 4, 2, 72
    s = Setup(ws, [(100, 3), (0, 0), (41, 41)], hk, D, 32, F16, seed=5, q_heads=hq)
    k, v = s.history()
    s.fill(k, v)
    q = s.rand(s.rows, hq * D)
    want, tol = s.expected(q, k, v, F16)
    for off, wide in ((0, (hq + 2 * hk) * D), (1, hq * D + 3)):
        qkv = torch.full((s.rows + 4, wide), float("nan"), dtype=F16, device=DEV)
        qkv[:s.rows, off:off + hq * D] = q.to(DEV)
        out = torch.full((s.rows + 4, wide + 1), 7.0, dtype=F16, device=DEV)
        b = s.batch()
        b.c.rows += 4
        ql.kv_attention(ws, s.cache, b, qkv[:, off:off + hq * D], out=out[:, off:off + hq * D])
        check(out[:s.rows, off:off + hq * D], want, tol)
        assert (out[s.rows:] == 7).all() and (out[:, :off] == 7).all() and (out[:, off + hq * D:] == 7).all()


def test_unseen_tokens_do_not_matter(ws):
    """Pages hold NaN and huge rows behind the sequences' ends, and unused table columns hold ids of no page."""
    s = Setup(ws, [(70, 3), (16, 1), (33, 5)], 2, 64, 16, F16, seed=6, q_heads=8)
    b = s.batch(lens=[80] * 3, news=[80] * 3, max_len=80)
    junk = torch.full((240, 128), float("nan"), dtype=F16)
    junk[::2] = 60000.0
    ql.kv_append(ws, s.cache, b, junk.to(DEV), junk.to(DEV))
    assert ws.status() == _lib.QLIN_ERR_NONFINITE
    k, v = s.history()
    s.fill(k, v)
    q = s.rand(s.rows, 512)
    table = s.table.copy()
    table[1, 1:] = -5
    table[2, 3:] = 1 << 30
    out = ql.kv_attention(ws, s.cache, s.batch(table=table), q.to(DEV))
    check(out, *s.expected(q, k, v, F16))
    assert ws.status() == 0


@pytest.mark.parametrize("dtype", [F16, F32])
def test_scales_far_apart(ws, dtype):
    """Values of tokens spread over many powers of two, all-zero rows, and logits in the hundreds."""
    s = Setup(ws, [(400, 6)], 2, 64, 32, dtype, seed=8, q_heads=4)
    k, v = s.history(size_k=6.0)
    spread = 13 if dtype == F16 else 50
    f = 2.0 ** s.rng.integers(-spread, spread if dtype == F32 else 8, 400)
    v = (v.float() * torch.from_numpy(f.astype(np.float32))[:, None]).to(dtype)
    v[::7] = 0
    k[::11] = 0
    s.fill(k, v)
    q = s.rand(6, 256, size=4.0)
    q[1] = 0  # equal weights
    if dtype == F32:
        q[2] *= 1e-20
        q[3] *= 1e6
        k0 = q[3].clone()
    out = ql.kv_attention(ws, s.cache, s.batch(), q.to(DEV))
    check(out, *s.expected(q, k, v, dtype))


def test_nan_query_stays_in_its_row(ws):
    s = Setup(ws, [(90, 3), (50, 2)], 2, 128, 16, F16, seed=9, q_heads=4)
    k, v = s.history()
    s.fill(k, v)
    q = s.rand(5, 512)
    want, tol = s.expected(q, k, v, F16)
    q[1, 130] = float("nan")  # row 1, head 1
    want[1, 128:256] = np.nan
    check(ql.kv_attention(ws, s.cache, s.batch(), q.to(DEV)), want, tol)


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_nonfinite_f32_query_stays_in_its_row(ws, value):
    """The same for f32 queries, which are scaled by their largest value; few rows and many."""
    for seqs in ([(90, 3), (50, 2)], [(400, 300)]):
        s = Setup(ws, seqs, 2, 72, 16, F32, seed=9, q_heads=4)
        k, v = s.history()
        s.fill(k, v)
        q = s.rand(s.rows, 288)
        want, tol = s.expected(q, k, v, F32)
        q[1, 73] = value  # row 1, head 1
        want[1, 72:144] = np.nan
        check(ql.kv_attention(ws, s.cache, s.batch(), q.to(DEV)), want, tol)


def test_loose_bounds(ws):
    """Many sequences with one row each in a batch whose max_new and max_len promise far more: too many workgroups
    for results kept apart, so nothing is cut."""
    seqs = [(1 + 7 * i % 61, 1) for i in range(290)]
    s = Setup(ws, seqs, 1, 40, 16, F16, seed=14, q_heads=32, max_len=2560)
    k, v = s.history()
    s.fill(k, v)
    q = torch.zeros((2048, 32 * 40), dtype=F16)
    q[:290] = s.rand(290, 32 * 40)
    b = s.batch(max_new=2048)
    b.c.rows = 2048
    out = torch.full((2048, 32 * 40), 7.0, dtype=F16, device=DEV)
    ql.kv_attention(ws, s.cache, b, q.to(DEV), out=out)
    check(out[:290], *s.expected(q, k, v, F16))
    assert (out[290:] == 7).all() and ws.status() == 0


def test_prefix_without_room_for_its_results(ws):
    """More vectors than the scratch holds two results of: every sequence reads the prefix itself."""
    s = Setup(ws, [(2400, 2100), (2300, 2100)], 1, 64, 32, F16, seed=15, q_heads=32)
    k, v = s.history()
    k[2400:2400 + 192], v[2400:2400 + 192] = k[:192], v[:192]
    s.fill(k, v)
    q = s.rand(s.rows, 2048).to(DEV)
    plain = ql.kv_attention(ws, s.cache, s.batch(), q)
    pages, table = i32(s.table[0, :6]), s.table.copy()
    table[:, :6] = -1
    got = ql.kv_attention(ws, s.cache, s.batch(table=table), q, prefix_tokens=192, prefix_pages=pages)
    assert torch.equal(got, plain) and ws.status() == 0
    few = [0, 1, 2099, 2100, 4199]
    qs = q.cpu()
    for r in few:
        i, t = divmod(r, 2100)
        n = [2400, 2300][i]
        at = [0, 2400][i]
        kc, ks = kvref.quantize(k[at:at + n].float().numpy().reshape(n, 1, 64))
        vc, vs = kvref.quantize(v[at:at + n].float().numpy().reshape(n, 1, 64))
        o, tol = kvref.attend(qs[r:r + 1].double().numpy().reshape(1, 32, 64), kc, ks, vc, vs, [n - 2100 + t + 1], 0.125, 1, EPS[F16])
        check(got[r:r + 1], o.reshape(1, -1), tol.reshape(1, -1))


def test_bad_batches_are_flagged(ws):
    """Values in the device arrays outside the limits: flagged, nothing outside the buffers is touched, and
    sequences without fault get their results."""
    s = Setup(ws, [(40, 2), (40, 2), (40, 2)], 1, 64, 16, F16, seed=10, q_heads=2)
    k, v = s.history()
    s.fill(k, v)
    q = s.rand(6, 128)
    want, tol = s.expected(q, k, v, F16)
    assert ws.status() == 0
    table = s.table.copy()
    table[1, 0] = 1 << 20
    b = s.batch(table=table)
    out = ql.kv_attention(ws, s.cache, b, q.to(DEV))
    assert ws.status() == _lib.QLIN_ERR_PARAM
    check(out[[0, 1, 4, 5]], want[[0, 1, 4, 5]], tol[[0, 1, 4, 5]])
    assert torch.isnan(out[2:4]).all()
    for bad in (dict(lens=[40, 49, 40]), dict(lens=[40, -1, 40])):
        out = ql.kv_attention(ws, s.cache, s.batch(**bad), q.to(DEV))
        assert ws.status() == _lib.QLIN_ERR_PARAM
        check(out[[0, 1, 4, 5]], want[[0, 1, 4, 5]], tol[[0, 1, 4, 5]])
    before = ql.kv_read(ws, s.cache, s.batch(lens=[40] * 3, news=[40] * 3), out_dtype=F32)
    table[1] = [-1, -1, 10 ** 9]
    ql.kv_append(ws, s.cache, s.batch(table=table, lens=[0, 40, 0], news=[0, 2, 0]), torch.ones((2, 64), dtype=F16, device=DEV),
                 torch.ones((2, 64), dtype=F16, device=DEV))
    assert ws.status() == _lib.QLIN_ERR_PARAM
    after = ql.kv_read(ws, s.cache, s.batch(lens=[40] * 3, news=[40] * 3), out_dtype=F32)
    assert all(torch.equal(x, y) for x, y in zip(before, after))
    ko, _ = ql.kv_read(ws, s.cache, s.batch(table=table, lens=[0, 40, 0], news=[0, 2, 0]))
    assert torch.isnan(ko).all() and ws.status() == _lib.QLIN_ERR_PARAM
    # more rows than promised: those beyond are not touched
    out = torch.full((6, 128), 7.0, dtype=F16, device=DEV)
    ql.kv_attention(ws, s.cache, s.batch(max_new=1), q.to(DEV), out=out)
    assert ws.status() == _lib.QLIN_ERR_PARAM and (out[1::2] == 7).all()


# ------------------------------------------------------------------ a shared prefix


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("prefix,seqs,hq,hk,D,P", [
    (64, [(70, 1), (64, 1), (65, 1), (0, 0), (200, 1)], 8, 2, 128, 16),   # one with nothing of its own
    (256, [(300, 4), (257, 2), (100, 3), (2, 4)], 6, 2, 64, 32),          # shorter than the prefix; a row without a token
    (1024, [(1040 + i, 1 + i % 3) for i in range(40)], 4, 1, 128, 64),
    (2048, [(2050, 1)], 4, 2, 256, 128),
    (512, [(700, 150), (520, 8)], 3, 1, 96, 16),
])
def test_shared_prefix(ws, dtype, prefix, seqs, hq, hk, D, P):
    s = Setup(ws, seqs, hk, D, P, dtype, seed=prefix + D, q_heads=hq)
    k, v = s.history(size_k=2.0)
    # every sequence begins with the same rows, kept once
    shared = s.rand(prefix, hk * D, size=2.0), s.rand(prefix, hk * D)
    at = 0
    for n, _ in seqs:
        m = min(n, prefix)
        k[at:at + m], v[at:at + m] = shared[0][:m], shared[1][:m]
        at += n
    s.fill(k, v)
    pages = s.table[int(np.argmax([n for n, _ in seqs])), :prefix // P].copy()
    table = s.table.copy()
    table[:, :prefix // P] = -7  # these columns are not read
    q = s.rand(s.rows, hq * D, size=1.5)
    print(f"[kv prefix] {prefix} {seqs[:5]} {hq} {hk} {D} {P} {dtype}", flush=True)
    out = ql.kv_attention(ws, s.cache, s.batch(table=table), q.to(DEV), prefix_tokens=prefix, prefix_pages=i32(pages))
    want, tol = s.expected(q, k, v, dtype)
    check(out, want, tol)
    assert ws.status() == 0
    pages[0] = -1
    out = ql.kv_attention(ws, s.cache, s.batch(table=table), q.to(DEV), prefix_tokens=prefix, prefix_pages=i32(pages))
    assert ws.status() == _lib.QLIN_ERR_PARAM and torch.isnan(out).any()
    s.cache.close()


@pytest.mark.parametrize("new", [2, 150])
def test_rows_before_the_first_sequence(ws, new):
    """row_start[0] > 0: the rows before it are nobody's, with a prefix and without, few vectors and many."""
    hq, hk, D, P, skip = 8, 2, 64, 32, 5
    s = Setup(ws, [(200, new), (230, 1)], hk, D, P, F16, seed=new, q_heads=hq)
    k, v = s.history()
    k[200:328], v[200:328] = k[:128], v[:128]
    s.fill(k, v)
    q = s.rand(s.rows, hq * D)
    want, tol = s.expected(q, k, v, F16)
    b = ql.KVBatch(i32(s.starts + skip), i32([200, 230]), i32(s.table), s.rows + skip + 3, new, 230)
    qs = torch.full((b.rows, hq * D), float("nan"), dtype=F16)
    qs[skip:skip + s.rows] = q
    pages = i32(s.table[0, :4])
    for kw in ({}, dict(prefix_tokens=128, prefix_pages=pages)):
        out = torch.full((b.rows, hq * D), 7.0, dtype=F16, device=DEV)
        ql.kv_attention(ws, s.cache, b, qs.to(DEV), out=out, **kw)
        check(out[skip:skip + s.rows], want, tol)
        assert (out[:skip] == 7).all() and (out[skip + s.rows:] == 7).all()
    ko = torch.full((b.rows, hk * D), 7.0, dtype=F16, device=DEV)
    vo = ko.clone()
    ql.kv_read(ws, s.cache, b, ko, vo)
    for o in (ko, vo):
        assert (o[:skip] == 7).all() and (o[skip + s.rows:] == 7).all() and not (o[skip:skip + s.rows] == 7).all(1).any()
    assert ws.status() == 0
    s.cache.close()


# ------------------------------------------------------------------ as a program uses them


def test_long_offsets(ws):
    """Pages whose bytes lie past 2^32 of a cache."""
    cache = ql.KVCache(8, 256, 600, 4096)  # 5.03e9 bytes of keys
    s = Setup(ws, [(40, 2)], 8, 256, 16, F16, seed=11, q_heads=8)
    k, v = s.history()
    table = np.array([[599]], np.int32)
    b = ql.KVBatch(i32([0, 40]), i32([40]), i32(table), 40, 40, 4096)
    ql.kv_append(ws, cache, b, k.to(DEV), v.to(DEV))
    q = s.rand(2, 2048)
    b = ql.KVBatch(i32([0, 2]), i32([40]), i32(table), 2, 2, 4096)
    check(ql.kv_attention(ws, cache, b, q.to(DEV)), *s.expected(q, k, v, F16))
    # pages never written read as zeros
    ko, vo = ql.kv_read(ws, cache, ql.KVBatch(i32([0, 40]), i32([40]), i32([[598]]), 40, 40, 4096))
    assert not ko.any() and not vo.any()
    cache.close()


def test_streams_side_by_side():
    """Two workspaces on two streams, one cache, calls in flight together: the results of one stream alone."""
    wss = [ql.Workspace(1, 256, 256) for _ in range(2)]
    s = Setup(wss[0], [(3000, 2), (500, 1)], 4, 128, 64, F16, seed=12, q_heads=16)
    k, v = s.history()
    s.fill(k, v)
    qs = [s.rand(3, 2048).to(DEV) for _ in range(2)]
    b = s.batch()
    alone = [ql.kv_attention(wss[0], s.cache, b, q) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [torch.empty_like(a) for a in alone]
    for _ in range(10):
        for st, w, q, o in zip(streams, wss, qs, outs):
            with torch.cuda.stream(st):
                ql.kv_attention(w, s.cache, b, q, out=o)
    torch.cuda.synchronize()
    assert all(torch.equal(a, o) for a, o in zip(alone, outs))


@pytest.mark.parametrize("prefix", [0, 128])
def test_captured_decode_steps(prefix):
    """One decode step (append, attention) captured once and replayed while lengths, tables and rows change, with eager
    work of another workspace in between: every replay equals the eager calls bit for bit."""
    ws, other = ql.Workspace(1, 256, 256), ql.Workspace(1, 256, 256)
    hq, hk, D, P, B, top = 8, 2, 128, 16, 3, 600
    s = Setup(ws, [(top, 1)] * B, hk, D, P, F16, seed=13, q_heads=hq)
    k, v = s.rand(B * top, hk * D), s.rand(B * top, hk * D)
    s.fill(k.to(DEV), v.to(DEV))
    table = s.table.copy()
    pages = i32(table[0, :max(1, prefix // P)])
    table[:, :prefix // P] = table[0, :prefix // P]
    batch = s.batch(table=table)
    starts, length, tab = batch._keep
    x = torch.zeros((B, (hq + 2 * hk) * D), dtype=F16, device=DEV)
    out = torch.zeros((B, hq * D), dtype=F16, device=DEV)
    q, nk, nv = x[:, :hq * D], x[:, hq * D:(hq + hk) * D], x[:, (hq + hk) * D:]
    kw = dict(prefix_tokens=prefix, prefix_pages=pages) if prefix else {}

    def step(w, o):
        ql.kv_append(w, s.cache, batch, nk, nv)
        ql.kv_attention(w, s.cache, batch, q, out=o, **kw)

    step(ws, out)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step(ws, out)
    for rep, lens in enumerate([[prefix + 1, prefix + 40, 600], [200, 0, 333], [prefix + 17, 512, 129], [600, 600, 600]]):
        x.copy_(s.rand(*x.shape).to(DEV))
        length.copy_(i32(lens))
        starts.copy_(i32(np.concatenate([[0], np.cumsum([int(n > 0) for n in lens])])))
        out.fill_(5.0)
        g.replay()
        torch.cuda.synchronize()
        got = out.clone()
        ref = torch.full_like(out, 5.0)
        step(other, ref)
        torch.cuda.synchronize()
        assert torch.equal(got, ref), rep
        assert not torch.isnan(got).any()
    assert ws.status() == 0 and other.status() == 0
    del g


def test_decoder_layers_on_the_device():
    """Two layers' attention blocks as a decode loop runs them: RMSNorm and qkv projection, append, attention, o
    projection with the residual, against the same steps with attention computed in 64 bits from what the
    cache reads back."""
    hid, hq, hk, D, P, B = 512, 8, 2, 64, 16, 3
    ws = ql.Workspace(32, hid, (hq + 2 * hk) * D)
    layers = []
    for i in range(2):
        mk = lambda n, kk, j: ql.Weights.from_packed_device(  # noqa: E731
            8, kk, n, synth.codes(n, kk, 8, 50 + 2 * i + j, DEV), (torch.rand(n, device=DEV) + 0.5) / (73 * math.sqrt(kk)))
        layers.append((mk((hq + 2 * hk) * D, hid, 0), mk(hid, hq * D, 1), synth.gamma(hid, 60 + i, device=DEV),
                       ql.KVCache(hk, D, 12, P)))
    table = i32(np.random.default_rng(0).permutation(12).reshape(B, 4))
    for step, (lens, news) in enumerate([([20, 7, 0], [20, 7, 0]), ([21, 8, 0], [1, 1, 0]), ([23, 9, 12], [2, 1, 12])]):
        starts = np.concatenate([[0], np.cumsum(news)])
        rows = int(starts[-1])
        batch = ql.KVBatch(i32(starts), i32(lens), table, rows, max(news), 4 * P)
        full = ql.KVBatch(i32(np.concatenate([[0], np.cumsum(lens)])), i32(lens), table, sum(lens), max(lens), 4 * P)
        h = synth.activations(rows, hid, 70 + step, device=DEV)
        for wq, wo, gamma, cache in layers:
            qkv = ql.run(ws, wq, h, gamma=gamma)
            q, k, v = qkv[:, :hq * D], qkv[:, hq * D:(hq + hk) * D], qkv[:, (hq + hk) * D:]
            ql.kv_append(ws, cache, batch, k, v)
            att = ql.kv_attention(ws, cache, batch, q)
            ko, vo = (t.double().cpu().numpy().reshape(-1, hk, D) for t in ql.kv_read(ws, cache, full, out_dtype=F32))
            one, at = np.ones((ko.shape[0], hk), np.float32), 0
            for i, (n, m) in enumerate(zip(lens, news)):
                r = int(starts[i])
                want, tol = kvref.attend(q[r:r + m].double().cpu().numpy().reshape(m, hq, D), ko[at:at + n], one[at:at + n],
                                         vo[at:at + n], one[at:at + n], [n - m + j + 1 for j in range(m)], D ** -0.5, 1,
                                         EPS[F16])
                # codes * scale read back as f32 are off by half a step of the product: 2^-24 in a logit and a value
                check(att[r:r + m], want.reshape(m, hq * D), 1.01 * tol.reshape(m, hq * D) + 2.0 ** -22 * np.abs(vo).max())
                at += n
            h = ql.run(ws, wo, att, residual=h)
        assert torch.isfinite(h).all() and ws.status() == 0
