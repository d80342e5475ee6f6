"""Key/value cache calls with faults in a batch's device arrays: what is stored, what is reported, and which results
stay right."""
import numpy as np
import pytest
import torch

from open_rknpu2_lm_infer_amd import _lib
from open_rknpu2_lm_infer_amd import qlinear as ql
from open_rknpu2_lm_infer_amd import synth
from tests.test_gpu_kv import DEV, F16, F32, Setup, check, i32

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ws():
    w = ql.Workspace(1, 256, 256)
    yield w
    w.close()


def whole_cache(s):
    """Every slot of the cache, [pages, page * columns] each of keys and values: every page as a full sequence."""
    n, P = s.cache.pages, s.P
    b = ql.KVBatch(i32(np.arange(n + 1) * P), i32([P] * n), i32(np.arange(n).reshape(n, 1)), n * P, P, P)
    return [x.view(n, -1) for x in ql.kv_read(s.ws, s.cache, b, out_dtype=F32)]


BAD = [  # row starts, lengths, rows of the tensors, max_new, max_len, the sequences at fault
    ([0, 2, 4, 6], [40, 49, 40], 6, 2, 40, [1]),     # past max_len: clamped, its rows would be tokens 38 and 39
    ([0, 2, 4, 6], [40, -1, 40], 6, 2, 40, [1]),
    ([0, 1, 3, 4], [40, 40, 40], 4, 1, 40, [1]),     # more rows than max_new: clamped, a row would take another's slot
    ([0, 3, 2, 4], [40, 40, 40], 4, 3, 40, [1]),     # decreasing
    ([0, 2, 5, 9], [40, 40, 40], 5, 3, 40, [2]),     # past the rows
    ([-1, 2, 4, 6], [40, 40, 40], 6, 3, 40, [0]),
]


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("starts,lens,rows,max_new,max_len,bad", BAD)
def test_append_stores_nothing_for_a_sequence_at_fault(ws, dtype, starts, lens, rows, max_new, max_len, bad):
    """The pages of a sequence whose row starts or length are out of the batch's limits keep what they held (they may
    be shared with others); the other sequences' rows are stored."""
    s = Setup(ws, [(40, 2)] * 3, 2, 72, 16, dtype, seed=21)
    k, v = s.history()
    s.fill(k, v)
    assert ws.status() == 0
    before = whole_cache(s)
    b = ql.KVBatch(i32(starts), i32(lens), i32(s.table), rows, max_new, max_len)
    new = s.rand(rows, 144, size=9.0).to(DEV), s.rand(rows, 144, size=9.0).to(DEV)
    ql.kv_append(ws, s.cache, b, *new)
    assert ws.status() == _lib.QLIN_ERR_PARAM
    after = whole_cache(s)
    good = [i for i in range(3) if i not in bad]
    owned = np.zeros(s.cache.pages, bool)
    owned[s.table[good].ravel()] = True
    for x, y in zip(before, after):
        assert torch.equal(x[~owned], y[~owned])
    # the good sequences hold what an append of theirs alone stores
    ref = Setup(ws, [(40, 2)] * 3, 2, 72, 16, dtype, seed=21)
    ref.fill(k, v)
    for i in good:
        n = starts[i + 1] - starts[i]
        one = ql.KVBatch(i32([0, n]), i32([lens[i]]), i32(s.table[i:i + 1]), n, n, max_len)
        ql.kv_append(ws, ref.cache, one, *(x[starts[i]:starts[i + 1]] for x in new))
    for x, y in zip(whole_cache(ref), after):
        assert torch.equal(x, y)
    assert ws.status() == 0
    s.cache.close()
    ref.cache.close()


def faulty_call(ws, nan=False):
    """A call that finds a length past max_len; with nan, the rows of another sequence hold one."""
    s = Setup(ws, [(40, 2)] * 2, 1, 64, 16, F16, seed=22)
    k = s.rand(4, 64)
    if nan:
        k[3, 5] = float("nan")
    ql.kv_append(ws, s.cache, s.batch(lens=[41, 40]), k.to(DEV), s.rand(4, 64).to(DEV))
    torch.cuda.synchronize()
    s.cache.close()


@pytest.mark.parametrize("K", [256, 250])  # through pinned blocks, through copies
def test_host_buffer_runs_leave_the_report_of_a_batch(K):
    w = ql.Workspace(4, 256, 256)
    packed, _, scales = synth.make_linear(128, K, 8, 5, device=DEV)
    lin = ql.Weights.from_packed_device(8, K, 128, packed, scales)
    A = synth.activations(4, K, 6).float().numpy()
    want = ql.run_host_f32(w, lin, A)
    faulty_call(w)
    assert np.array_equal(ql.run_host_f32(w, lin, A), want)
    assert w.status() == _lib.QLIN_ERR_PARAM and w.status() == 0
    # its own report of a row is the call's, whatever a batch left
    faulty_call(w)
    A[2, 3] = np.inf
    with pytest.raises(_lib.QlinError) as e:
        ql.run_host_f32(w, lin, A)
    assert e.value.rc == _lib.QLIN_ERR_NONFINITE
    assert w.status() == _lib.QLIN_ERR_PARAM
    w.close()


def test_status_reports_one_fault_after_the_other():
    w = ql.Workspace(1, 256, 256)
    faulty_call(w, nan=True)
    assert w.status(clear=False) == w.status(clear=False) == _lib.QLIN_ERR_PARAM
    assert w.status() == _lib.QLIN_ERR_PARAM
    assert w.status(clear=False) == _lib.QLIN_ERR_NONFINITE
    assert w.status() == _lib.QLIN_ERR_NONFINITE
    assert w.status() == 0
    w.close()


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("P", [16, 32])
@pytest.mark.parametrize("new,hq", [(2, 4), (150, 8)])  # few vectors and many
def test_bad_prefix_page_reaches_only_rows_that_see_it(ws, dtype, P, new, hq):
    """The prefix's second page is outside the cache: sequences that end before it keep their results."""
    seqs = [(P - 3, 2), (3 * P + new, new), (P, 1), (P + 1, 1), (5, 1)]
    s = Setup(ws, seqs, 2, 64, P, dtype, seed=23 + P, q_heads=hq)
    k, v = s.history()
    at = 0
    for n, _ in seqs:  # all begin with the longest sequence's tokens
        m = min(n, 3 * P)
        k[at:at + m], v[at:at + m] = k[P - 3:P - 3 + m].clone(), v[P - 3:P - 3 + m].clone()
        at += n
    s.fill(k, v)
    q = s.rand(s.rows, hq * 64)
    want, tol = s.expected(q, k, v, dtype)
    pages = s.table[1, :3].copy()
    kw = dict(prefix_tokens=3 * P, prefix_pages=i32(pages))
    check(ql.kv_attention(ws, s.cache, s.batch(), q.to(DEV), **kw), want, tol)
    assert ws.status() == 0
    pages[1] = s.cache.pages
    kw["prefix_pages"] = i32(pages)
    out = ql.kv_attention(ws, s.cache, s.batch(), q.to(DEV), **kw)
    assert ws.status() == _lib.QLIN_ERR_PARAM
    r = 0
    for n, m in seqs:
        for t in range(m):
            if n - m + t + 1 > P:
                want[r] = np.nan
            r += 1
    assert np.isnan(want).any() and not np.isnan(want).all()
    check(out, want, tol)
    s.cache.close()
