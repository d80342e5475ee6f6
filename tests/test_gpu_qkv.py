"""From the rows of the qkv projection into the cache in one pass: the same bits as the norms and rotation into f32 rows
followed by append, for caches of both widths; those two are held to 64 bits by tests of their own."""
import numpy as np
import pytest
import torch

from open_rknpu2_lm_infer_amd import _lib
from open_rknpu2_lm_infer_amd import qlinear as ql
from tests.test_gpu_kv_errors import BAD

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
F16, F32 = torch.float16, torch.float32


@pytest.fixture(scope="module")
def ws():
    w = ql.Workspace(1, 256, 256)
    yield w
    w.close()


def i32(x):
    return torch.as_tensor(np.asarray(x, np.int32), device=DEV)


def rand(shape, dtype, seed, size=1.0):
    return torch.from_numpy((np.random.default_rng(seed).standard_normal(shape) * size).astype(np.float32)).to(dtype)


class Batch:
    """Sequences of (length, new rows) in scattered pages, two caches of one geometry."""

    def __init__(self, seqs, hk, D, P, bits, seed=0, spare=2):
        self.seqs, cols = seqs, max(1, -(-max(n for n, _ in seqs) // P))
        pages = len(seqs) * cols + spare
        self.table = np.random.default_rng(seed).permutation(pages)[:len(seqs) * cols].reshape(len(seqs), cols).astype(np.int32)
        self.caches = [ql.KVCache(hk, D, pages, P, bits=bits) for _ in range(2)]
        self.starts = np.concatenate([[0], np.cumsum([m for _, m in seqs])])
        self.rows, self.max_len = int(self.starts[-1]), max(n for n, _ in seqs)
        self.batch = ql.KVBatch(i32(self.starts), i32([n for n, _ in seqs]), i32(self.table), self.rows, max(m for _, m in seqs),
                                self.max_len)
        self.positions = [n - m + t for n, m in seqs for t in range(m)]

    def contents(self, ws):
        out = []
        for c in self.caches:
            n, P = c.pages, c.page_tokens
            b = ql.KVBatch(i32(np.arange(n + 1) * P), i32([P] * n), i32(np.arange(n).reshape(n, 1)), n * P, P, P)
            out.append(torch.cat(ql.kv_read(ws, c, b, out_dtype=F32), 1))
        return out

    def close(self):
        for c in self.caches:
            c.close()


def apart(ws, b, rope, qkv, hq, hk, D, gq, gk, out_dtype, flags=0):
    """The same by the calls that the pass joins, into the second cache."""
    heads = qkv[:, :(hq + hk) * D]
    pos = i32(b.positions) if rope else None
    q = ql.norm_rope(rope, heads, pos, hq, gq, gk, out_dtype=out_dtype, head_dim=D)[:, :hq * D]
    k = ql.norm_rope(rope, heads, pos, hq, gq, gk, out_dtype=F32, head_dim=D)[:, hq * D:]
    ql.kv_append(ws, b.caches[1], b.batch, k, qkv[:, (hq + hk) * D:].float(), flags=flags)
    return q


PASS = [  # sequences, query heads, kv heads, head dim, page, rotary columns, first, layout
    ([(1, 1)], 4, 1, 64, 16, 64, 0, "half"),
    ([(300, 1), (0, 0), (17, 17), (64, 2)], 32, 8, 128, 64, 128, 0, "half"),
    ([(40, 33), (16, 16), (5, 1)], 5, 3, 84, 16, 42, 20, "half"),
    ([(200, 200)], 2, 2, 256, 32, 128, 64, "interleaved"),
    ([(33, 20), (70, 3)], 7, 5, 3, 16, 2, 1, "interleaved"),
    ([(50, 50)], 3, 2, 250, 128, 244, 3, "half"),
    ([(90, 40), (31, 31)], 1, 1, 63, 16, 62, 0, "half"),
    ([(600, 600), (20, 1)], 16, 4, 128, 16, 64, 0, "interleaved"),
]


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("dtype,out_dtype", [(F16, F16), (F32, F32), (F16, F32), (F32, F16)])
@pytest.mark.parametrize("seqs,hq,hk,D,P,n,first,layout", PASS)
@pytest.mark.parametrize("norms", ["both", "none", "keys"])
def test_pass_equals_its_parts(ws, bits, dtype, out_dtype, seqs, hq, hk, D, P, n, first, layout, norms):
    b = Batch(seqs, hk, D, P, bits, seed=D)
    rope = ql.Rope(D, n, base=1e4, first=first, layout=layout)
    gq = (rand((D,), F32, 1, 0.3) + 1).to(DEV) if norms == "both" else None
    gk = (rand((D,), F32, 2, 0.3) + 1).to(DEV) if norms != "none" else None
    x = rand((b.rows, (hq + 2 * hk) * D), dtype, seed=D + hq, size=2.0).to(DEV)
    print(f"[qkv] {bits} {seqs} {hq} {hk} {D} {P} {n} {first} {layout} {dtype} {out_dtype} {norms}", flush=True)
    half_even = ql.QLIN_ROUND_HALF_EVEN if norms == "keys" else 0
    want = apart(ws, b, rope, x, hq, hk, D, gq, gk, out_dtype, half_even)
    got = ql.kv_append_qkv(ws, b.caches[0], b.batch, rope, x, hq, gq, gk, out_dtype=out_dtype, flags=half_even)
    assert torch.equal(got, want)
    one, two = b.contents(ws)
    assert torch.equal(one, two) and one.any()
    if dtype == out_dtype:  # queries in place, beside keys and values that stay
        y = x.clone()
        ql.kv_append_qkv(ws, b.caches[0], b.batch, rope, y, hq, gq, gk, out=y[:, :hq * D], flags=half_even)
        assert torch.equal(y[:, :hq * D], want) and torch.equal(y[:, hq * D:], x[:, hq * D:])
        assert torch.equal(b.contents(ws)[0], two)
    assert ws.status() == 0
    b.close()


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("D,n,first,hq,hk", [(128, 128, 0, 6, 2), (64, 32, 16, 3, 3), (84, 42, 20, 2, 1), (250, 244, 3, 1, 1)])
def test_many_rows(ws, bits, dtype, D, n, first, hq, hk):
    """Four rows a workgroup: ragged sequences whose rows are no multiples of four, idle ones, rows without a token."""
    b = Batch([(700, 700), (650, 301), (0, 0), (5, 3), (2, 6), (1, 1)], hk, D, 32, bits, seed=D)
    rope, g = ql.Rope(D, n, first=first), (rand((D,), F32, 1, 0.3) + 1).to(DEV)
    x = rand((b.rows, (hq + 2 * hk) * D), dtype, seed=D).to(DEV)
    want = apart(ws, b, rope, x, hq, hk, D, g, g, dtype)
    got = ql.kv_append_qkv(ws, b.caches[0], b.batch, rope, x, hq, g, g)
    assert torch.equal(got, want)
    one, two = b.contents(ws)
    assert torch.equal(one, two) and one.any() and ws.status() == 0
    b.close()


@pytest.mark.parametrize("new", [1, 2, 3, 5])
def test_many_sequences_of_few_rows(ws, new):
    """More than 2048 rows, of which a sequence has fewer than a workgroup's four, or one more."""
    b = Batch([(new + i % 3, new - (i % 5 == 4)) for i in range(2200)], 1, 64, 16, 8, seed=new)
    rope, x = ql.Rope(64), rand((b.rows, 6 * 64), F16, seed=new).to(DEV)
    want = apart(ws, b, rope, x, 4, 1, 64, None, None, F16)
    assert torch.equal(ql.kv_append_qkv(ws, b.caches[0], b.batch, rope, x, 4), want)
    one, two = b.contents(ws)
    assert torch.equal(one, two) and one.any() and ws.status() == 0
    b.close()


@pytest.mark.parametrize("bits", [8, 4])
def test_without_rotation_and_odd_rows(ws, bits):
    """No rope; rows from an odd column on, of an odd stride, outputs alike; rows of nobody before, behind and beside stay."""
    hq, hk, D = 3, 2, 72
    b = Batch([(40, 5), (9, 9), (0, 0), (3, 1)], hk, D, 16, bits)
    g = (rand((D,), F32, 1, 0.3) + 1).to(DEV)
    x = rand((b.rows, (hq + 2 * hk) * D), F16, seed=5).to(DEV)
    want = apart(ws, b, None, x, hq, hk, D, g, g, F16)
    skip = 3
    wide = torch.full((b.rows + skip + 4, (hq + 2 * hk) * D + 5), float("nan"), dtype=F16, device=DEV)
    rows = wide[:, 1:1 + (hq + 2 * hk) * D]
    rows[skip:skip + b.rows] = x
    out = torch.full((wide.shape[0], hq * D + 7), 7.0, dtype=F16, device=DEV)
    batch = ql.KVBatch(i32(b.starts + skip), i32([n for n, _ in b.seqs]), i32(b.table), wide.shape[0], 9, 40)
    ql.kv_append_qkv(ws, b.caches[0], batch, None, rows, hq, g, g, out=out[:, 3:3 + hq * D])
    assert torch.equal(out[skip:skip + b.rows, 3:3 + hq * D], want)
    assert (out[:skip] == 7).all() and (out[skip + b.rows:] == 7).all() and (out[:, :3] == 7).all() and (out[:, 3 + hq * D:] == 7).all()
    one, two = b.contents(ws)
    assert torch.equal(one, two) and ws.status() == 0
    b.close()


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("dtype", [F16, F32])
def test_nonfinite_rows_are_poisoned_alone(ws, bits, dtype):
    """A key or value head with Inf or NaN has the scale NaN and says so; a query's reaches its head alone and says nothing."""
    hq, hk, D = 2, 2, 64
    b = Batch([(20, 20)], hk, D, 16, bits)
    rope = ql.Rope(D)
    g = torch.ones(D, device=DEV)
    x = rand((20, 6 * D), dtype, seed=6)
    want = apart(ws, b, rope, x.to(DEV), hq, hk, D, g, g, dtype)
    x[2, 5] = float("nan")  # a query
    got = ql.kv_append_qkv(ws, b.caches[0], b.batch, rope, x.to(DEV), hq, g, g)
    assert ws.status() == 0
    keep = torch.ones(20, hq * D, dtype=torch.bool, device=DEV)
    keep[2, :D] = False
    assert torch.equal(got[keep], want[keep]) and torch.isnan(got[2, :D]).all()
    x[4, hq * D + D + 7] = float("inf")        # a key, head 1
    x[9, (hq + hk) * D + 3] = float("-inf")    # a value, head 0
    ql.kv_append_qkv(ws, b.caches[0], b.batch, rope, x.to(DEV), hq, g, g)
    assert ws.status() == _lib.QLIN_ERR_NONFINITE and ws.status() == 0
    clean = [t.clone() for t in ql.kv_read(ws, b.caches[1], b.batch, out_dtype=F32)]
    clean[0][4, D:] = float("nan")
    clean[1][9, :D] = float("nan")
    for got, want in zip(ql.kv_read(ws, b.caches[0], b.batch, out_dtype=F32), clean):
        assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got.nan_to_num(), want.nan_to_num())
    b.close()


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("starts,lens,rows,max_new,max_len,bad", BAD)
def test_nothing_is_stored_for_a_sequence_at_fault(ws, bits, starts, lens, rows, max_new, max_len, bad):
    hq, hk, D = 2, 2, 72
    b = Batch([(40, 2)] * 3, hk, D, 16, bits, seed=21)
    rope, g = ql.Rope(D, 64), torch.ones(D, device=DEV)
    x = rand((rows, 6 * D), F16, seed=7, size=9.0).to(DEV)
    batch = ql.KVBatch(i32(starts), i32(lens), i32(b.table), rows, max_new, max_len)
    out = torch.full((rows + 2, hq * D), 7.0, dtype=F16, device=DEV)
    assert ws.status() == 0
    ql.kv_append_qkv(ws, b.caches[0], batch, rope, x, hq, g, g, out=out)
    assert ws.status() == _lib.QLIN_ERR_PARAM and (out[rows:] == 7).all()
    good = sorted(set(range(3)) - set(bad))
    for i in good:
        n = starts[i + 1] - starts[i]
        one = ql.KVBatch(i32([0, n]), i32([lens[i]]), i32(b.table[i:i + 1]), n, n, max_len)
        q = ql.kv_append_qkv(ws, b.caches[1], one, rope, x[starts[i]:starts[i + 1]], hq, g, g)
        # where starts decrease, a row that two sequences claim has the queries of either
        only = [r for r in range(starts[i], starts[i + 1]) if not any(starts[j] <= r < starts[j + 1] for j in good if j != i)]
        assert len(only) >= n - 1 and torch.equal(q[[r - starts[i] for r in only]], out[only])
    one, two = b.contents(ws)
    assert torch.equal(one, two) and ws.status() == 0
    b.close()


@pytest.mark.parametrize("bits", [8, 4])
def test_bad_pages_and_rows_without_a_token(ws, bits):
    hq, hk, D = 2, 1, 64
    b = Batch([(40, 3), (2, 5), (20, 1)], hk, D, 16, bits)
    rope = ql.Rope(D)
    x = rand((b.rows, 4 * D), F16, seed=8).to(DEV)
    table = b.table.copy()
    table[0, 2] = 1 << 20  # tokens 37 .. 39
    batch = ql.KVBatch(i32(b.starts), i32([40, 2, 20]), i32(table), b.rows, 5, 40)
    q = ql.kv_append_qkv(ws, b.caches[0], batch, rope, x, hq)
    assert ws.status() == _lib.QLIN_ERR_PARAM and torch.isfinite(q).all()
    k, v = ql.kv_read(ws, b.caches[0], b.batch, out_dtype=F32)
    assert not k[:3].any() and not k[3:6].any() and k[6:].any(1).all() and v[6:].any(1).all()
    # the queries of rows whose page is at fault are good ones
    ql.kv_append_qkv(ws, b.caches[1], b.batch, rope, x, hq, out=(ref := torch.empty_like(q)))
    assert torch.equal(q, ref) and ws.status() == 0
    b.close()


def test_pages_past_4_gigabytes(ws):
    for bits, pages in ((8, 600), (4, 1100)):
        cache = ql.KVCache(8, 256, pages, 4096, bits=bits)
        assert (pages - 1) * cache.device_bytes // pages > 2 ** 32
        rope = ql.Rope(256)
        x = rand((40, 24 * 256), F16, seed=9).to(DEV)
        near = ql.KVBatch(i32([0, 40]), i32([40]), i32([[0]]), 40, 40, 4096)
        far = ql.KVBatch(i32([0, 40]), i32([40]), i32([[pages - 1]]), 40, 40, 4096)
        ql.kv_append_qkv(ws, cache, far, rope, x, 8)
        k, v = ql.kv_read(ws, cache, far, out_dtype=F32)
        assert not any(t.any() for t in ql.kv_read(ws, cache, near))
        ql.kv_append_qkv(ws, cache, near, rope, x, 8)
        assert all(torch.equal(a, c) for a, c in zip((k, v), ql.kv_read(ws, cache, near, out_dtype=F32))) and k.any()
        cache.close()


@pytest.mark.parametrize("bits", [8, 4])
def test_captured_passes(bits):
    """Captured once, replayed while rows, starts and lengths change, with eager work of another workspace in between."""
    ws, other = ql.Workspace(1, 256, 256), ql.Workspace(1, 256, 256)
    hq, hk, D, P, B = 4, 2, 128, 16, 3
    b = Batch([(300, 4)] * B, hk, D, P, bits)
    rope, g = ql.Rope(D, base=1e6), torch.ones(D, device=DEV)
    x, out = torch.zeros((4 * B, 8 * D), dtype=F16, device=DEV), torch.zeros((4 * B, hq * D), dtype=F16, device=DEV)
    starts, length, _ = b.batch._keep
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ql.kv_append_qkv(ws, b.caches[0], b.batch, rope, x, hq, g, g, out=out)
    for rep, (lens, news) in enumerate([([300, 20, 7], [4, 4, 4]), ([100, 0, 9], [1, 0, 2]), ([250, 33, 16], [0, 1, 3]), ([4, 4, 4], [4, 4, 4])]):
        x.copy_(rand(x.shape, F16, rep).to(DEV))
        length.copy_(i32(lens))
        starts.copy_(i32(np.concatenate([[0], np.cumsum(news)])))
        out.fill_(5.0)
        graph.replay()
        torch.cuda.synchronize()
        ref = torch.full_like(out, 5.0)
        ql.kv_append_qkv(other, b.caches[1], b.batch, rope, x, hq, g, g, out=ref)
        torch.cuda.synchronize()
        assert torch.equal(out, ref) and (out[sum(news):] == 5).all()
        one, two = b.contents(other)
        assert torch.equal(one, two), rep
    assert ws.status() == 0 and other.status() == 0
    del graph
    b.close()
