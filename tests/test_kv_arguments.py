"""What the calls of the key/value cache do on the host: the Python ones (tensors and handles are stand-ins that say
what they are) and those of tests/cpp/kv_calls_test.cpp."""
import subprocess
from types import SimpleNamespace

import pytest
import torch

from open_rknpu2_lm_infer_amd import qlinear as ql
from tests.test_kv import BIN


class Tensor:
    """A device tensor as far as its description goes."""

    def __init__(self, *shape, dtype=torch.int32, device="cuda:0"):
        self.shape, self.dtype, self.device, self.is_cuda = shape, dtype, torch.device(device), True

    def numel(self):
        return int(torch.tensor(self.shape).prod())

    def dim(self):
        return len(self.shape)

    def stride(self, i=None):
        s = [1]
        for n in self.shape[:0:-1]:
            s.insert(0, s[0] * n)
        return tuple(s) if i is None else s[i]

    def is_contiguous(self):
        return True

    def data_ptr(self):
        return 0


def batch(**device):
    dev = lambda k: device.get(k, "cuda:0")  # noqa: E731
    return ql.KVBatch(Tensor(3, device=dev("row_start")), Tensor(2, device=dev("length")),
                      Tensor(2, 4, device=dev("page_table")), 5, 3, 64)


CACHE = SimpleNamespace(handle=None, page_tokens=16, head_dim=64, columns=128, device=0)
WS = SimpleNamespace(handle=None)


@pytest.fixture
def reached(monkeypatch):
    """Names of the entry points that were reached."""
    seen = []

    class Lib:
        def __getattr__(self, name):
            return lambda *a: seen.append(name) or 0

    monkeypatch.setattr(ql._lib, "load", lambda: Lib())
    monkeypatch.setattr(ql, "_raw_stream", lambda device: 0)
    return seen


def test_prefix_pages_and_tokens_come_together(reached):
    q, out = Tensor(5, 256, dtype=torch.float16), Tensor(5, 256, dtype=torch.float16)
    pages = Tensor(2)
    ql.kv_attention(WS, CACHE, batch(), q, out=out, prefix_pages=pages, prefix_tokens=32)
    ql.kv_attention(WS, CACHE, batch(), q, out=out)
    assert reached == ["qlin_kv_attention_prefix", "qlin_kv_attention"]
    with pytest.raises(AssertionError, match="prefix"):  # the table's columns of a prefix may hold anything
        ql.kv_attention(WS, CACHE, batch(), q, out=out, prefix_pages=pages)
    with pytest.raises(AssertionError):
        ql.kv_attention(WS, CACHE, batch(), q, out=out, prefix_tokens=32)
    with pytest.raises(AssertionError):
        ql.kv_attention(WS, CACHE, batch(), q, out=out, prefix_pages=pages, prefix_tokens=48)
    assert len(reached) == 2
    ql.kv_attention(WS, CACHE, batch(), q, out=out, prefix_pages=Tensor(0))  # a prefix of no pages
    assert reached[2] == "qlin_kv_attention"


def test_batch_lies_on_one_device():
    assert batch().device == torch.device("cuda:0")
    for name in ("row_start", "length", "page_table"):
        with pytest.raises(AssertionError, match="device"):
            batch(**{name: "cuda:1"})


def test_lds_of_many_vectors_is_asked_for_on_each_device():
    r = subprocess.run([BIN, "devices"], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and "PASS devices" in r.stdout, r.stdout[-3000:] + r.stderr[-1000:]


def test_limits_of_query_heads_and_scale():
    r = subprocess.run([BIN, "limits"], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and "PASS limits" in r.stdout, r.stdout[-3000:] + r.stderr[-1000:]
