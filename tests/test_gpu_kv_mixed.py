"""Batches of a prompt among decoding and idle slots, most of whose workgroups have no row: what is stored, read and
reported, and that sequences of few rows beside one of many cost about as much as their launch."""
import time

import numpy as np
import pytest
import torch

from open_rknpu2_lm_infer_amd import _lib
from open_rknpu2_lm_infer_amd import qlinear as ql
from tests import headref, kvref
from tests.test_gpu_kv import DEV, F16, F32, i32

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ws():
    w = ql.Workspace(1, 256, 256)
    yield w
    w.close()


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("hk,D", [(8, 128), (3, 84), (1, 256), (5, 64), (17, 40)])
def test_prompts_among_decoding_slots(ws, bits, dtype, hk, D):
    """Rows and workgroups end at different places: each sequence holds its own rows and no other page is touched."""
    seqs = [(1, 1), (150, 131), (40, 1), (0, 0), (33, 2), (90, 17), (64, 0), (16, 16)]
    P, lens, news = 16, [n for n, _ in seqs], [m for _, m in seqs]
    cols = -(-max(lens) // P)
    pages = len(seqs) * cols + 5
    rng = np.random.default_rng(bits + D)
    table = rng.permutation(pages)[:len(seqs) * cols].reshape(len(seqs), cols).astype(np.int32)
    cache = ql.KVCache(hk, D, pages, P, bits=bits)
    starts = np.concatenate([[0], np.cumsum(news)])
    rows = int(starts[-1])
    batch = ql.KVBatch(i32(starts), i32(lens), i32(table), rows, max(news), max(lens))
    k, v = (torch.from_numpy(rng.standard_normal((rows, hk * D)).astype(np.float32)).to(dtype) for _ in range(2))
    ql.kv_append(ws, cache, batch, k.to(DEV), v.to(DEV))
    quantize = kvref.quantize if bits == 8 else headref.quantize4
    want = []
    for x in (k, v):
        c, s = quantize(x.float().numpy().reshape(rows, hk, D))
        want.append(torch.from_numpy((c.astype(np.float32) * s[..., None]).reshape(rows, hk * D)))
    for got, w in zip(ql.kv_read(ws, cache, batch, out_dtype=F32), want):
        assert torch.equal(got.cpu(), w)
    # the whole cache: what no row has been stored to is as it was made
    whole = ql.KVBatch(i32(np.arange(pages + 1) * P), i32([P] * pages), i32(np.arange(pages).reshape(pages, 1)), pages * P, P, P)
    slots = torch.tensor([table[i, (n - m + t) // P] * P + (n - m + t) % P for i, (n, m) in enumerate(seqs) for t in range(m)])
    for got, w in zip(ql.kv_read(ws, cache, whole, out_dtype=F32), want):
        full = torch.zeros((pages * P, hk * D))
        full[slots] = w
        assert torch.equal(got.cpu(), full)
    assert ws.status() == 0
    cache.close()


@pytest.mark.parametrize("bits", [8, 4])
def test_a_slot_at_fault_without_rows_is_reported(ws, bits):
    """One whose length cannot be, of no rows and of fewer than the batch's most: the word is set by append and by read."""
    cache = ql.KVCache(8, 128, 12, 16, bits=bits)
    x = torch.ones((41, 1024), dtype=F16, device=DEV)
    table = i32(np.arange(12).reshape(3, 4))
    for starts in ([0, 40, 40, 41], [0, 40, 41, 41]):
        for length in (-1, 65):
            b = ql.KVBatch(i32(starts), i32([40, length, 5]), table, 41, 40, 64)
            ql.kv_append(ws, cache, b, x, x)
            assert ws.status() == _lib.QLIN_ERR_PARAM
            ql.kv_read(ws, cache, b)
            assert ws.status() == _lib.QLIN_ERR_PARAM and ws.status() == 0
    cache.close()


@pytest.mark.parametrize("bits", [8, 4])
def test_missing_rows_cost_no_work(ws, bits):
    """One prompt of 512 tokens among 63 decoded tokens: 32768 workgroups, 575 of them with a row.  Storing takes 1.1 times as long as
    reading; where the others load a row and quantize it for nobody, 2.4 times and more."""
    lens, news = [512] + [1000] * 63, [512] + [1] * 63
    cache = ql.KVCache(8, 128, 64 * 16, 64, bits=bits)
    b = ql.KVBatch(i32(np.concatenate([[0], np.cumsum(news)])), i32(lens), i32(np.arange(1024).reshape(64, 16)), 575, 512, 1000)
    x = torch.randn((575, 1024), device=DEV).to(F16)
    out = torch.empty_like(x), torch.empty_like(x)

    def us(call):
        call()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            for _ in range(20):
                call()
        best = 1e9
        for _ in range(15):
            g.replay()
            torch.cuda.synchronize()
            a = time.perf_counter()
            for _ in range(5):
                g.replay()
            torch.cuda.synchronize()
            best = min(best, time.perf_counter() - a)
        return best / 100 * 1e6

    read, store = us(lambda: ql.kv_read(ws, cache, b, *out)), us(lambda: ql.kv_append(ws, cache, b, x, x))
    print(f"[mixed] {bits} bits: stored in {store:.1f} us, read in {read:.1f}", flush=True)
    assert store < 1.8 * read
    cache.close()
