"""4-bit attention of very few vectors, whose columns are shared by classes of tokens: up to 4 vectors of a KV head (four classes,
pages of 64 and more) and up to 8 (two, pages of 32 and more), at lengths about the tiles, steps and parts, with prefixes, bad
pages, rows that see nothing and tokens nobody sees."""
import numpy as np
import pytest
import torch

from open_rknpu2_lm_infer_amd import _lib
from open_rknpu2_lm_infer_amd import qlinear as ql
from tests.test_gpu_kv import DEV, F16, F32, Setup, check, i32, ws  # noqa: F401
from tests.test_gpu_kv4 import four_bits  # noqa: F401

pytestmark = pytest.mark.gpu

EDGES = [1, 15, 16, 17, 31, 33, 48, 63, 64, 65, 127, 128, 129, 191, 193, 255, 256, 257, 300, 511, 513, 700]


@pytest.mark.parametrize("dtype,out_dtype", [(F16, F16), (F32, F32), (F16, F32), (F32, F16)])
@pytest.mark.parametrize("D", [1, 64, 84, 128, 200, 256])
@pytest.mark.parametrize("hq,new,P", [(1, 1, 64), (4, 1, 64), (3, 1, 128), (2, 2, 64), (1, 4, 64),  # four classes
                                      (4, 1, 32), (8, 1, 64), (5, 1, 64), (2, 4, 32), (1, 7, 128)])  # two
def test_lengths(ws, dtype, out_dtype, D, hq, new, P):  # noqa: F811
    seqs = [(n, min(new, 1 + i % new) if new > 1 else 1) for i, n in enumerate(EDGES)] + [(0, 0), (2, new), (0, new)]
    s = Setup(ws, seqs, 1, D, P, dtype, seed=D + hq, q_heads=hq)
    k, v = s.history(size_k=2.0)
    s.fill(k, v)
    q = s.rand(s.rows, hq * D, size=1.5)
    print(f"[classes] {D} {hq} {new} {P} {dtype} {out_dtype}", flush=True)
    out = ql.kv_attention(ws, s.cache, s.batch(max_new=new), q.to(DEV), out_dtype=out_dtype)
    check(out, *s.expected(q, k, v, out_dtype))
    assert ws.status() == 0
    s.cache.close()


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("hq,new,P,prefix", [(4, 1, 64, 512), (8, 1, 64, 192), (4, 2, 32, 320), (1, 4, 128, 1024)])
def test_prefixes_and_parts(ws, dtype, D, hq, new, P, prefix):  # noqa: F811
    """Own tokens behind a prefix that has parts of its own; one long sequence cut into many parts; and both as heads of several."""
    seqs = [(prefix + n, new) for n in (1, 63, 64, 65, 200, 257)] + [(prefix // 2, new), (prefix, new), (0, 0)]
    s = Setup(ws, seqs, 2, D, P, dtype, seed=D, q_heads=2 * hq)
    k, v = s.history(size_k=1.5)
    shared = s.rand(prefix, 2 * D, size=1.5), s.rand(prefix, 2 * D)
    at = 0
    for n, _ in seqs:
        m = min(n, prefix)
        k[at:at + m], v[at:at + m] = shared[0][:m], shared[1][:m]
        at += n
    s.fill(k, v)
    q = s.rand(s.rows, 2 * hq * D, size=1.5)
    want, tol = s.expected(q, k, v, dtype)
    table = s.table.copy()
    pages = i32(table[5, :prefix // P])
    table[:, :prefix // P] = -7
    out = ql.kv_attention(ws, s.cache, s.batch(table=table), q.to(DEV), prefix_tokens=prefix, prefix_pages=pages)
    check(out, want, tol)
    check(ql.kv_attention(ws, s.cache, s.batch(), q.to(DEV)), want, tol)
    assert ws.status() == 0
    s.cache.close()
    s = Setup(ws, [(5000, new)], 2, D, P, dtype, seed=D + 1, q_heads=2 * hq)
    k, v = s.history(size_k=1.5)
    s.fill(k, v)
    q = s.rand(s.rows, 2 * hq * D, size=1.5)
    check(ql.kv_attention(ws, s.cache, s.batch(), q.to(DEV)), *s.expected(q, k, v, dtype))
    s.cache.close()


@pytest.mark.parametrize("hq", [3, 8])
def test_bad_pages_and_junk(ws, hq):  # noqa: F811
    """A page outside the cache makes NaN of its sequence's rows that see it and of no others; NaN and infinities behind the ends,
    and ids of no page in columns nobody reads, change nothing."""
    D, P = 64, 64
    lens = [70, 64, 130, 1, 200]
    s = Setup(ws, [(n, 1) for n in lens], 2, D, P, F16, seed=7, q_heads=2 * hq)
    b = s.batch(lens=[256] * 5, news=[256] * 5, max_len=256)
    wide = np.full((5, 4), 0, np.int32)
    wide[:, :s.table.shape[1]] = s.table
    junk = torch.full((256, 2 * D), float("nan"), dtype=F16)
    junk[::3] = 60000.0
    for i, n in enumerate(lens):  # every page of the sequences holds junk first
        cols = -(-n // P)
        one = ql.KVBatch(i32([0, cols * P]), i32([cols * P]), i32(s.table[i:i + 1]), cols * P, cols * P, cols * P)
        ql.kv_append(ws, s.cache, one, junk[:cols * P].to(DEV), junk[:cols * P].to(DEV))
    ws.status()
    k, v = s.history()
    s.fill(k, v)
    q = s.rand(5, 2 * hq * D)
    want, tol = s.expected(q, k, v, F16)
    table = wide.copy()
    for i, n in enumerate(lens):
        table[i, -(-n // P):] = [-1, 1 << 30, -5, 99999][:4 - -(-n // P)]
    b = ql.KVBatch(i32(np.arange(6)), i32(lens), i32(table), 5, 1, 256)
    check(ql.kv_attention(ws, s.cache, b, q.to(DEV)), want, tol)
    assert ws.status() == 0
    table[2, 1] = s.cache.pages
    b = ql.KVBatch(i32(np.arange(6)), i32(lens), i32(table), 5, 1, 256)
    want[2] = np.nan
    check(ql.kv_attention(ws, s.cache, b, q.to(DEV)), want, tol)
    assert ws.status() == _lib.QLIN_ERR_PARAM
    s.cache.close()


def test_rows_before_and_behind_and_strides(ws):  # noqa: F811
    hq, hk, D, skip = 4, 2, 72, 3
    s = Setup(ws, [(100, 1), (0, 0), (41, 1), (300, 1)], hk, D, 64, F16, seed=5, q_heads=hq * hk)
    k, v = s.history()
    s.fill(k, v)
    q = s.rand(s.rows, hq * hk * D)
    want, tol = s.expected(q, k, v, F16)
    for off in (0, 1):
        wide = torch.full((s.rows + skip + 4, hq * hk * D + 9), float("nan"), dtype=F16, device=DEV)
        wide[skip:skip + s.rows, off:off + hq * hk * D] = q.to(DEV)
        out = torch.full_like(wide, 7.0)
        b = ql.KVBatch(i32(s.starts + skip), i32([100, 0, 41, 300]), i32(s.table), wide.shape[0], 1, 300)
        ql.kv_attention(ws, s.cache, b, wide[:, off:off + hq * hk * D], out=out[:, off:off + hq * hk * D])
        check(out[skip:skip + s.rows, off:off + hq * hk * D], want, tol)
        assert (out[:skip] == 7).all() and (out[skip + s.rows:] == 7).all() and (out[:, :off] == 7).all() and (out[:, off + hq * hk * D:] == 7).all()
    s.cache.close()


def test_logits_far_apart(ws):  # noqa: F811
    """Classes whose maxima are hundreds of bits apart, a class of which nothing is seen, and all weights on one token."""
    D = 64
    s = Setup(ws, [(80, 1), (256, 1), (18, 1)], 1, D, 64, F32, seed=9, q_heads=4)
    k, v = s.history()
    k[10] *= 60.0
    k[80 + 40] *= 100.0
    k[80 + 200] *= -100.0
    v[80:80 + 64] = 0
    s.fill(k, v)
    q = s.rand(3, 4 * D, size=4.0)
    q[1, :D] = 0
    check(ql.kv_attention(ws, s.cache, s.batch(), q.to(DEV)), *s.expected(q, k, v, F32))
    s.cache.close()
