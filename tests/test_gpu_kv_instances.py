"""Every instance of the attention kernels: padded heads of 64, 128 and 256, the three ways that fp16 and f32 meet, and
each pair of tiles (16, 32 and 128 vectors) for the sequences' own tokens and for a shared prefix."""
import numpy as np
import pytest
import torch

from open_rknpu2_lm_infer_amd import qlinear as ql
from tests.test_gpu_kv import DEV, F16, F32, Setup, check, i32

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ws():
    w = ql.Workspace(1, 256, 256)
    yield w
    w.close()


# (length, new) of the sequences, query heads, kv heads, tokens of the prefix, scale.  Vectors of a KV head: own
# max(new) * group, of the prefix rows * group; up to 16 the small tile, above 256 (fp16) or 512 the large one.
CASES = {
    "own few": ([(700, 2), (30, 1)], 8, 2, 0, -0.11),
    "own some": ([(700, 20), (90, 7)], 8, 2, 0, None),
    "own many": ([(700, 270), (300, 3)], 2, 1, 0, -0.17),
    "prefix few, own few": ([(700, 2), (650, 1)], 8, 2, 576, None),
    "prefix some, own few": ([(270 + 9 * i, 1) for i in range(20)], 8, 2, 256, 0.31),
    "prefix some, own some": ([(700, 20), (650, 3)], 8, 2, 576, None),
    "prefix many, own few": ([(130 + i % 50, 1) for i in range(180)], 3, 1, 128, 0.21),
    "prefix many, own many": ([(700, 270), (400, 2)], 2, 1, 384, None),
}


@pytest.mark.parametrize("dtype,out_dtype", [(F16, F16), (F16, F32), (F32, F16)])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("name", CASES)
def test_attention_instance(ws, name, D, dtype, out_dtype):
    seqs, hq, hk, prefix, scale = CASES[name]
    P = 32
    s = Setup(ws, seqs, hk, D, P, dtype, seed=len(name) + D, q_heads=hq)
    k, v = s.history(size_k=1.5)
    shared = s.rand(prefix, hk * D, size=1.5), s.rand(prefix, hk * D)
    at = 0
    for n, _ in seqs:
        m = min(n, prefix)
        k[at:at + m], v[at:at + m] = shared[0][:m], shared[1][:m]
        at += n
    s.fill(k, v)
    table, kw = s.table.copy(), {}
    if prefix:
        kw = dict(prefix_tokens=prefix, prefix_pages=i32(table[0, :prefix // P]))
        table[:, :prefix // P] = -1
    q = s.rand(s.rows, hq * D, size=1.5)
    out = ql.kv_attention(ws, s.cache, s.batch(table=table), q.to(DEV), out_dtype=out_dtype, scale=scale, **kw)
    check(out, *s.expected(q, k, v, out_dtype, scale=scale))
    assert ws.status() == 0
    s.cache.close()


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("new", [2, 300])
def test_equal_logits_at_the_largest_scale(ws, dtype, new):
    """Keys of zeros, or queries of zeros: every logit is 0 whatever the scale, and the result the mean."""
    s = Setup(ws, [(400, new)], 1, 64, 16, dtype, seed=31, q_heads=2)
    k, v = s.history()
    for zero in "kq":
        keys = k * 0 if zero == "k" else k
        s.fill(keys, v)
        q = s.rand(s.rows, 128) * (zero == "k")
        for scale in (2.0 ** 64, -2.0 ** 64):
            out = ql.kv_attention(ws, s.cache, s.batch(), q.to(DEV), scale=scale)
            check(out, *s.expected(q, keys, v, dtype, scale=scale))
    assert ws.status() == 0
    s.cache.close()


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("prefix", [0, 128])
def test_captured_chunks(prefix, dtype):
    """A step of many rows (append, attention) captured once and replayed while lengths, row starts and rows change:
    every replay equals the eager calls of another workspace bit for bit."""
    ws, other = ql.Workspace(1, 256, 256), ql.Workspace(1, 256, 256)
    hq, hk, D, P, top, new = 4, 2, 64, 16, 900, 300
    s = Setup(ws, [(top, new)] * 2, hk, D, P, dtype, seed=33, q_heads=hq)
    k, v = s.history()
    s.fill(k, v)
    table = s.table.copy()
    pages = i32(table[0, :max(1, prefix // P)])
    table[:, :prefix // P] = table[0, :prefix // P]
    batch = s.batch(table=table)
    starts, length, _ = batch._keep
    x = torch.zeros((2 * new, (hq + 2 * hk) * D), dtype=dtype, device=DEV)
    out = torch.zeros((2 * new, hq * D), dtype=dtype, device=DEV)
    q, nk, nv = x[:, :hq * D], x[:, hq * D:(hq + hk) * D], x[:, (hq + hk) * D:]
    kw = dict(prefix_tokens=prefix, prefix_pages=pages) if prefix else {}

    def step(w, o):
        ql.kv_append(w, s.cache, batch, nk, nv)
        ql.kv_attention(w, s.cache, batch, q, out=o, **kw)

    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step(ws, out)
    for lens, news in [([900, 700], [300, 300]), ([prefix + 40, 333], [40, 1]), ([0, 512], [0, 300]), ([prefix + 300, 450], [300, 170])]:
        x.copy_(s.rand(*x.shape).to(DEV))
        length.copy_(i32(lens))
        starts.copy_(i32(np.concatenate([[0], np.cumsum(news)])))
        out.fill_(5.0)
        g.replay()
        torch.cuda.synchronize()
        got = out.clone()
        ref = torch.full_like(out, 5.0)
        step(other, ref)
        torch.cuda.synchronize()
        assert torch.equal(got, ref), lens
        assert not torch.isnan(got).any() and (got[sum(news):] == 5).all()
    assert ws.status() == 0 and other.status() == 0
    del g


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("all_new", [False, True])  # tiles of 16 vectors, and of 32 (heads up to 128)
def test_few_vectors_in_fp16_are_rounded_once(ws, all_new, D):
    """fp16 rows in and out are held to the bound of probabilities of 22 bits and one rounding of the output.  Contexts are
    short and queries small, so that the bound's other parts, 2^-15 of the values together, leave a probability's rounding
    to 11 bits no room where values cancel."""
    lens = [2 + i % 5 for i in range(40)]
    s = Setup(ws, [(n, n if all_new else 1) for n in lens], 1, D, 16, F16, seed=D, q_heads=8)
    k, v = s.history()
    s.fill(k, v)
    q = s.rand(s.rows, 8 * D, size=0.2)
    out = ql.kv_attention(ws, s.cache, s.batch(), q.to(DEV))
    s.dtype = F32  # the bound of two fp16 values a probability
    check(out, *s.expected(q, k, v, F16))
    s.cache.close()
