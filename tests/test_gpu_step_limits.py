"""The tables of a serving step at their limits on the GPU: ids of no page under rows, with few rows (one launch) and many (two), and
which slots are refused."""
import numpy as np
import pytest
import torch

from open_rknpu2_lm_infer_amd import _lib
from open_rknpu2_lm_infer_amd import qlinear as ql
from tests.test_step_limits import REFUSED

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


@pytest.fixture(scope="module")
def ws():
    w = ql.Workspace(1, 256, 256)
    yield w
    w.close()


def i32(x):
    return torch.as_tensor(np.asarray(x, np.int32), device=DEV)


class Step:
    """Slots that hold `held` tokens each, pages of 16 in the order of the slots; 100 free pages."""

    def __init__(self, seqs, held, rows, max_new, max_len=64, prefix=0, maps=True):
        cols, own, shared = -(-max_len // 16), -(-held // 16) - prefix // 16, prefix // 16
        self.pages = seqs * own + 100 + shared
        self.cache = ql.KVCache(1, 64, self.pages, 16)
        table = np.full((seqs, cols), -1, np.int32)
        table[:, :shared] = np.arange(shared)
        table[:, shared:shared + own] = shared + np.arange(seqs * own).reshape(seqs, own)
        free = np.arange(self.pages)
        free[:100] = shared + seqs * own + np.arange(100)
        self.table = i32(table)
        self.step = ql.KVStep(self.cache, i32([held] * seqs), self.table, i32(free), i32([100]), rows, max_new, max_len, prefix, maps=maps)

    def close(self):
        self.cache.close()


SIZES = [(5, 100), (1500, 8000), (5000, 6000), (40, 9000)]  # slots, rows: one workgroup, one of four slots a thread, two scans, two launches


@pytest.mark.parametrize("seqs,rows", SIZES)
@pytest.mark.parametrize("bad", [-1, -9, 10 ** 6, -2 ** 31, 2 ** 31 - 1, "pages"])
def test_an_id_of_no_page_under_a_row(ws, seqs, rows, bad):
    """The rest of a page that a slot holds already: the word says so, the rows on it have no slot, all others have theirs."""
    s = Step(seqs, 18, rows, 2)
    s.table[3, 1] = s.pages if bad == "pages" else bad
    change = torch.zeros(seqs, dtype=torch.int32, device=DEV)
    change[1:5] = 2
    ql.kv_step(ws, s.step, change)
    assert ws.status() == _lib.QLIN_ERR_PARAM and ws.status() == 0
    want = [-1 if i == 3 else (2 * i + 1) * 16 + 2 + t for i in range(1, 5) for t in range(2)]
    assert s.step.slots[:8].tolist() == want and s.step.positions[:8].tolist() == [18, 19] * 4
    assert s.step.row_seq[:8].tolist() == [1, 1, 2, 2, 3, 3, 4, 4]
    # an id that no row lies on is nobody's business
    s.step.slots.fill_(-3)
    change[3] = 0
    ql.kv_step(ws, s.step, change)
    assert ws.status() == 0 and (s.step.slots[:6] >= 0).all() and (s.step.slots[6:] == -3).all()
    s.close()


@pytest.mark.parametrize("seqs,rows", SIZES)
def test_an_id_of_no_page_from_the_list(ws, seqs, rows):
    """A page taken in the step: its table entry is what the list held, its rows have no slot."""
    s = Step(seqs, 16, rows, 3)
    s.step.free_pages[98] = -7
    change = torch.zeros(seqs, dtype=torch.int32, device=DEV)
    change[:3] = 3
    ql.kv_step(ws, s.step, change)
    assert ws.status() == _lib.QLIN_ERR_PARAM
    first = seqs
    assert s.table[:3, 1].tolist() == [first + 99, -7, first + 97]
    assert s.step.slots[:9].tolist() == [16 * (first + 99) + t for t in range(3)] + [-1] * 3 + [16 * (first + 97) + t for t in range(3)]
    s.close()


@pytest.mark.parametrize("seqs,rows", SIZES)
def test_ids_of_a_prefix_are_taken_as_they_are(ws, seqs, rows):
    """Rows among a prefix's tokens lie on what its columns say; the pages behind are looked at."""
    s = Step(seqs, 32, rows, 20, prefix=32)
    s.step.length[1] = 30
    s.table[1, 1] = -9
    change = torch.zeros(seqs, dtype=torch.int32, device=DEV)
    change[1] = 4
    ql.kv_step(ws, s.step, change)
    assert ws.status() == 0
    page = s.step.page_table[1, 2].item()
    assert s.step.slots[:4].tolist() == [-9 * 16 + 14, -9 * 16 + 15, page * 16, page * 16 + 1]
    s.table[1, 2] = -9
    ql.kv_step(ws, s.step, change)
    assert ws.status() == _lib.QLIN_ERR_PARAM and s.step.slots[:4].tolist() == [-1] * 4
    s.close()


@pytest.mark.parametrize("seqs,rows", SIZES)
def test_without_slots_held_pages_are_not_read(ws, seqs, rows):
    s = Step(seqs, 18, rows, 2, maps=False)
    s.table[3, 1] = -9
    ql.kv_step(ws, s.step, i32([2] * 5 + [0] * (seqs - 5)))
    assert ws.status() == 0 and s.step.length[:5].tolist() == [20] * 5
    s.close()


@pytest.mark.parametrize("slots", [3, 1500, 5000])
@pytest.mark.parametrize("change,max_new,max_len,spare,rows", REFUSED)
def test_who_is_refused(ws, slots, change, max_new, max_len, spare, rows):
    """The same slots alone, and among idle ones; those of the list are the last, so that sums come from all before."""
    n = len(change)
    cols = max(-(-min(max_len, 1024) // 16), 2)
    cache = ql.KVCache(1, 64, slots + 9, 16)
    table = torch.full((slots, cols), -1, dtype=torch.int32, device=DEV)
    table[:, 0] = torch.arange(slots, device=DEV)
    free = torch.arange(slots, 2 * slots + 9, dtype=torch.int32, device=DEV)[:slots + 9].clamp(max=slots + 8)
    step = ql.KVStep(cache, i32([10] * slots), table, free, i32([spare]), 8, max_new, min(max_len, 1024))
    ql.kv_step(ws, step, i32([0] * (slots - n) + change))
    assert step.length.tolist() == [10] * (slots - n) + [10 + r for r in rows]
    assert step.row_start[slots - n:].tolist() == [sum(rows[:i]) for i in range(n + 1)]
    assert step.refused.item() == sum(c > 0 and r == 0 for c, r in zip(change, rows)) and ws.status() == 0
    cache.close()
