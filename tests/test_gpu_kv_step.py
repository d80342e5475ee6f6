"""Tables of a serving step on the GPU: equal to the plain account in tests/headref.py, number by number, and a whole
serving loop as a program runs it."""
import math

import numpy as np
import pytest
import torch

from open_rknpu2_lm_infer_amd import _lib
from open_rknpu2_lm_infer_amd import qlinear as ql
from tests import headref

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
F16 = torch.float16


@pytest.fixture(scope="module")
def ws():
    w = ql.Workspace(1, 256, 256)
    yield w
    w.close()


def i32(x):
    return torch.as_tensor(np.asarray(x, np.int32), device=DEV)


class Slots:
    """Slots with random lengths whose pages are scattered; some free pages; the plain account beside."""

    def __init__(self, seqs, page, max_len, rows, max_new, spare, seed, prefix=0, maps=True, lens=None, wide=0):
        rng = self.rng = np.random.default_rng(seed)
        self.page, self.prefix, self.rows, self.max_new, self.max_len = page, prefix, rows, max_new, max_len
        cols, shared = -(-max_len // page), prefix // page
        self.length = [int(x) for x in (rng.integers(0, max_len + 1, seqs) * (rng.random(seqs) > 0.2) if lens is None else lens)]
        own = [max(-(-n // page), shared) - shared for n in self.length]
        self.pages = sum(own) + spare + shared
        ids = [int(x) for x in rng.permutation(self.pages)]
        self.table = []
        for n in own:
            self.table.append([-9] * shared + [ids.pop() for _ in range(n)] + [-1] * (cols - shared - n))
        self.free = [ids.pop() for _ in range(spare)]
        self.cache = ql.KVCache(1, 64, max(self.pages, 1), page, bits=4)
        stack = np.full(max(self.pages, 1), -5, np.int32)
        stack[:spare] = self.free
        t = torch.full((seqs, cols + wide), -77, dtype=torch.int32, device=DEV)
        t[:, :cols] = i32(self.table).view(seqs, cols)
        self.whole = t
        out = lambda n, dtype=torch.int32: torch.full((n,), -3, dtype=dtype, device=DEV) if maps else None  # noqa: E731
        self.step = ql.KVStep(self.cache, i32(self.length), t[:, :cols], i32(stack), i32([spare]), rows, max_new, max_len, prefix,
                              row_seq=out(rows), positions=out(rows), slots=out(rows, torch.int64), refused=out(1), maps=maps)
        self.cols, self.seqs = cols, seqs

    def go(self, ws, change, call=None):
        s = self.step
        (call or (lambda: ql.kv_step(ws, s, i32(change))))()
        self.length, self.table, self.free, starts, maps, refused = headref.step(
            [int(c) for c in change], self.length, self.table, self.free, self.page, self.pages, self.rows, self.max_new, self.max_len,
            self.prefix)
        assert s.length.tolist() == self.length
        assert s.page_table.tolist() == self.table
        assert s.free_count.item() == len(self.free) and s.free_pages[:len(self.free)].tolist() == self.free
        assert s.row_start.tolist() == starts
        if s.row_seq is not None:
            assert s.refused.item() == refused
            got = list(zip(s.row_seq.tolist(), s.positions.tolist(), s.slots.tolist()))
            assert got[:len(maps)] == maps
        assert (self.whole[:, self.cols:] == -77).all()
        return starts, refused

    def close(self):
        self.cache.close()


STEPS = [  # slots, page, max_len, rows, max_new, spare pages, prefix
    (1, 16, 40, 8, 8, 3, 0),
    (64, 64, 4096, 256, 4, 40, 0),
    (7, 16, 100, 50, 100, 6, 32),
    (200, 32, 500, 300, 60, 20, 0),       # rows and pages run out
    (1024, 16, 64, 4096, 9, 300, 16),
    (1025, 16, 64, 4096, 9, 300, 16),     # more than one scan, three launches
    (3000, 16, 200, 9000, 40, 500, 0),
    (300, 16, 600, 20000, 600, 4000, 0),  # prompts
    (5, 4096, 9000, 10, 3, 1, 4096),
    (4096, 16, 64, 4096, 9, 900, 0),      # the most of one scan, one launch
    (4097, 16, 64, 4096, 9, 900, 0),      # two scans
    (9001, 16, 100, 5000, 20, 3000, 16),  # rows and pages run out in the second or third
    (9001, 16, 100, 200000, 20, 2000, 0),
]


@pytest.mark.parametrize("seqs,page,max_len,rows,max_new,spare,prefix", STEPS)
@pytest.mark.parametrize("seed", [1, 2])
def test_steps(ws, seqs, page, max_len, rows, max_new, spare, prefix, seed):
    s = Slots(seqs, page, max_len, rows, max_new, spare, seed, prefix, wide=seed - 1)
    print(f"[step] {seqs} {page} {max_len} {rows} {max_new} {spare} {prefix}", flush=True)
    some = 0
    for k in range(6):
        c = s.rng.integers(1, max_new + 2, seqs)
        what = s.rng.random(seqs)
        c = np.where(what < 0.3, 0, np.where(what < 0.6, -s.rng.integers(1, max_len + 2, seqs), np.where(what < 0.7, 1, c)))
        if k == 3:
            c = -np.minimum(s.rng.integers(0, 5, seqs), 4)
        if k == 4:
            c = np.full(seqs, max_new)
        starts, refused = s.go(ws, c)
        some += starts[-1]
    assert some > 0 and ws.status() == 0
    s.close()


def test_rows_behind_the_last_and_no_maps(ws):
    s = Slots(40, 16, 100, 200, 8, 30, 3)
    starts, _ = s.go(ws, [2] * 40)
    n = starts[-1]
    assert 0 < n < 200
    for t in (s.step.row_seq, s.step.positions, s.step.slots):
        assert (t[n:] == -3).all() and (t[:n] >= 0).all()
    s.close()
    for seqs in (40, 2000):
        s = Slots(seqs, 16, 100, 200, 8, 30, 3, maps=False)
        s.go(ws, [2] * seqs)
        s.go(ws, [-300] * seqs)
        assert s.length == [0] * seqs
        s.close()


@pytest.mark.parametrize("seqs", [30, 1500])
def test_nothing_to_do_and_ends(ws, seqs):
    """No change at all; everything given back at once (changes of -2^31 among them) and everything taken by one."""
    s = Slots(seqs, 16, 160, 4000, 160, 0, 4)
    s.go(ws, [0] * seqs)
    s.go(ws, [-2 ** 31 if i % 2 else -10 ** 6 for i in range(seqs)])
    assert len(s.free) == s.pages and s.length == [0] * seqs
    s.go(ws, [2 ** 31 - 1] * seqs)  # past every limit
    assert s.length == [0] * seqs
    s.go(ws, [160] + [0] * (seqs - 1))
    assert s.length[0] == 160
    s.go(ws, [1] + [0] * (seqs - 1))  # it is full
    assert s.length[0] == 160 and ws.status() == 0
    s.close()


def test_rows_of_none(ws):
    s = Slots(5, 16, 64, 0, 0, 4, 5)
    starts, refused = s.go(ws, [1, 0, -3, 2, 1])
    assert starts == [0] * 6 and refused == 3 and ws.status() == 0
    s.close()


@pytest.mark.parametrize("seqs", [3, 1400])
def test_numbers_outside_the_limits(ws, seqs):
    """Lengths, counts and ids that cannot be: said so, their slots left alone, the others served."""
    s = Slots(seqs, 16, 64, 50, 4, 9, 6, lens=[20] * seqs)
    s.step.length[1] = 65
    before = s.step.page_table[1].clone()
    ql.kv_step(ws, s.step, i32([1] * 3 + [0] * (seqs - 3)))
    assert ws.status() == _lib.QLIN_ERR_PARAM
    assert s.step.length[:3].tolist() == [21, 65, 21] and s.step.row_start[:4].tolist() == [0, 1, 1, 2] and s.step.refused.item() == 1
    assert torch.equal(s.step.page_table[1], before)
    s.step.length[1] = -1
    ql.kv_step(ws, s.step, i32([-1] * seqs))
    assert ws.status() == _lib.QLIN_ERR_PARAM and s.step.length[:3].tolist() == [20, -1, 20]
    s.step.length[1] = 20
    assert ws.status() == 0
    for count, taken in ((-4, 0), (s.pages + 3, s.pages)):
        s.step.free_count.fill_(count)
        s.step.free_pages.clamp_(min=0)
        ql.kv_step(ws, s.step, i32([0] * seqs))
        assert ws.status() == _lib.QLIN_ERR_PARAM and s.step.free_count.item() == taken
    # more pages given back than there are: the list is full and stays within its bounds
    ql.kv_step(ws, s.step, i32([-64] * seqs))
    assert ws.status() == _lib.QLIN_ERR_PARAM and s.step.free_count.item() == s.pages
    # an id of no page in the list is handed on, and said
    s.step.free_pages.fill_(10 ** 6)
    ql.kv_step(ws, s.step, i32([1] + [0] * (seqs - 1)))
    assert ws.status() == _lib.QLIN_ERR_PARAM and s.step.page_table[0, 0].item() == 10 ** 6
    # and on its way back
    s.step.free_count.fill_(0)
    ql.kv_step(ws, s.step, i32([-1] + [0] * (seqs - 1)))
    assert ws.status() == _lib.QLIN_ERR_PARAM and ws.status() == 0
    s.close()


def test_the_largest_number_of_slots(ws):
    n = 1 << 20
    cache = ql.KVCache(1, 64, 1024, 16, bits=4)
    length, table = torch.zeros(n, dtype=torch.int32, device=DEV), torch.full((n, 1), -1, dtype=torch.int32, device=DEV)
    step = ql.KVStep(cache, length, table, torch.arange(1024, dtype=torch.int32, device=DEV), i32([1024]), 5000, 9, 16)
    change = torch.zeros(n, dtype=torch.int32, device=DEV)
    change[::1000] = 3
    ql.kv_step(ws, step, change)
    assert step.refused.item() == 1049 - 1024 and step.row_start[-1].item() == 3 * 1024 and step.free_count.item() == 0
    at = torch.arange(1024, device=DEV)
    assert torch.equal(step.row_seq[:3 * 1024].view(-1, 3), (1000 * at)[:, None].expand(-1, 3).int())
    assert torch.equal(step.slots[:3 * 1024].view(-1, 3), (1023 - at)[:, None] * 16 + torch.arange(3, device=DEV))
    ql.kv_step(ws, step, -change)
    assert not step.length.any() and step.free_count.item() == 1024 and (table == -1).all() and ws.status() == 0
    cache.close()


@pytest.mark.parametrize("seqs", [20, 1100])
def test_captured_steps(seqs):
    """Captured once, replayed with other changes: every replay equals the plain account, with eager steps of another workspace between."""
    ws, other = ql.Workspace(1, 256, 256), ql.Workspace(1, 256, 256)
    s, t = (Slots(seqs, 16, 200, 500, 20, 60, 8) for _ in range(2))
    change = torch.zeros(seqs, dtype=torch.int32, device=DEV)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ql.kv_step(ws, s.step, change)
    for _ in range(5):
        c = s.rng.integers(-30, 22, seqs)
        change.copy_(i32(c))
        s.go(None, c, call=g.replay)
        t.go(other, c)
    assert ws.status() == 0 and other.status() == 0
    del g
    s.close()
    t.close()


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("dtype", [F16, torch.float32])
def test_a_serving_loop_on_the_device(bits, dtype):
    """Tables, the pass from the qkv rows and attention captured as one graph, replayed for prompts, decoded tokens, drafted
    tokens taken back and requests that end, slots reused by the next ones; against the same rows through calls of one
    request each, on caches of their own with tables made on the host: queries bit for bit."""
    hq, hk, D, P, B, rows, top = 4, 2, 64, 16, 5, 96, 200
    ws, other = ql.Workspace(1, 256, 256), ql.Workspace(1, 256, 256)
    cache = ql.KVCache(hk, D, 40, P, bits=bits)
    rope, g = ql.Rope(D, base=1e6), (torch.rand(D, device=DEV) + 0.5)
    step = ql.KVStep(cache, i32([0] * B), i32([[-1] * math.ceil(top / P)] * B), i32(np.random.default_rng(0).permutation(40)), i32([40]), rows,
                     40, top)
    change = torch.zeros(B, dtype=torch.int32, device=DEV)
    x = torch.zeros((rows, (hq + 2 * hk) * D), dtype=dtype, device=DEV)
    q, out = torch.zeros((rows, hq * D), dtype=dtype, device=DEV), torch.zeros((rows, hq * D), dtype=dtype, device=DEV)

    def run(w):
        batch = ql.kv_step(w, step, change)
        ql.kv_append_qkv(w, cache, batch, rope, x, hq, g, g, out=q)
        ql.kv_attention(w, cache, batch, q, out=out)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run(ws)
    # a cache of its own for every slot, its pages in order
    mine = [ql.KVCache(hk, D, math.ceil(top / P), P, bits=bits) for _ in range(B)]
    pages = i32([list(range(math.ceil(top / P)))])
    length = [0] * B
    rng = np.random.default_rng(1)
    for c in ([17, 40, 0, 1, 0], [1, 1, 33, 1, 0], [4, 4, 4, 4, 16], [-3, -1, 0, -4, 0], [1, 1, 1, 1, 1], [-500, 4, 4, -500, 4], [20, 1, 1, 40, 30],
              [0, 0, 0, 0, 0], [-500] * 5, [16, 16, 16, 16, 16]):
        x.copy_(torch.from_numpy(rng.standard_normal(tuple(x.shape)).astype(np.float32)))
        change.copy_(i32(c))
        out.fill_(5.0)
        graph.replay()
        torch.cuda.synchronize()
        r = 0
        for i, n in enumerate(c):
            length[i] = max(length[i] + n, 0)
            if n <= 0:
                continue
            b = ql.KVBatch(i32([0, n]), i32([length[i]]), pages, n, n, top)
            qi = ql.kv_append_qkv(other, mine[i], b, rope, x[r:r + n], hq, g, g)
            assert torch.equal(qi, q[r:r + n])
            want = ql.kv_attention(other, mine[i], b, qi)
            # the batch's max_new picks the tile and the parts: the same sums in another order.  A normalized head is at most
            # sqrt(64) * 1.5 long, so a logit's products sum up to 18 and an exponent is off by eta = ((64 + 8) 2^-23 +
            # 2^-21) 18 < 2^-12.5 at most, which moves either mean of values by 2 eta of the largest; fp16 adds 2^-11 for P
            # and 2^-11 for the output on either side
            tol = (4 * 2.0 ** -12.5 + (4 * 2.0 ** -11 if dtype == F16 else 2.0 ** -16)) * 1.01 * float(x[:, (hq + hk) * D:].abs().max())
            assert (out[r:r + n] - want).abs().max() <= tol
            r += n
        assert step.length.tolist() == length and (out[r:] == 5).all()
        assert step.positions[:r].tolist() == [length[i] - n + t for i, n in enumerate(c) for t in range(max(n, 0))]
    assert step.free_count.item() == 40 - 5 and ws.status() == 0 and other.status() == 0
    del graph
    for k in mine:
        k.close()
    cache.close()
