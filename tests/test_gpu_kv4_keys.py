"""Keys and values of a 4-bit cache through the matrix core's operands, column by column: every unit with every code, for the kernels
of one, two and four classes of tokens, of one and two tiles of vectors and of many.

A query with a one in column d and zeros elsewhere makes token j's logit scale * k[j][d].  A sequence sees m tokens whose keys are zeros
and, last, the one that is looked at; values tell them apart: 1785 in column 0 of the last one's, 1785 in column 1 of the others' (code
7, unit 255, scale 1: exactly that).  With scale = 2 / 1785 the logit l lies within -2 .. 2, and the output is

  o[0] = 1785 e^l / (e^l + m),   o[1] = 1785 m / (e^l + m)

What an f32 evaluation may be off by: the logit is one exact product (the others are zeros) and a few roundings of 2^-23 of 2, the
exponents' maxima and differences 4 steps of 2^-23 of 2 log2 e + 8 < 11: eta = (8 * 2 + 4 * 11) 2^-23 < 2^-17, for numerator and
denominator 2 eta; P is kept to 22 bits, 2^-22; sums of up to 128 tokens 2 (128 / 8 + 64) 2^-23; quotient and output 2^-22.  In all 3.6e-5
of the result.  A key that is off by one step of the row's scale, the least there is, moves l by 2 / 1785 and o[0] by 1.12e-3 (1 - o[0] / 1785)
>= 1.12e-3 / (1 + e^2) = 1.3e-4 of itself.

Of values, with queries of zeros, the mean of the one that is looked at and m others is made: a value that is off by one step moves its
part by 1 / 1785 = 5.6e-4 of itself at least."""
import numpy as np
import pytest
import torch

from open_rknpu2_lm_infer_amd import qlinear as ql
from tests.test_gpu_kv import DEV, F16, F32, i32
from tests.test_kv4_keys import keys, outputs, stored_from

pytestmark = pytest.mark.gpu

TOL = (2 * 60 + 2 * (128 / 8 + 64) + 4) * 2.0 ** -23


@pytest.fixture(scope="module")
def ws():
    w = ql.Workspace(1, 256, 256)
    yield w
    w.close()


FORMS = [  # query heads of a KV head, new rows, page: what works on them
    (1, 1, 16),    # a tile without classes
    (5, 2, 16),
    (4, 1, 64),    # four classes
    (2, 2, 128),
    (8, 1, 32),    # two classes
    (4, 2, 64),
    (24, 1, 64),   # two tiles (heads of 256: one)
    (520, 1, 64),  # many vectors
]


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("D", [64, 84, 128, 256])
@pytest.mark.parametrize("hq,new,P", FORMS)
def test_every_key_column(ws, dtype, D, hq, new, P):
    """A sequence for each key and each hq columns; the key at changing places of its page.  With two rows the first does not see the
    key, whose mean of values is 1785 in column 1."""
    x = keys(D)
    n = len(x)
    cache = ql.KVCache(1, D, n, P, bits=4)
    place = 1 + np.arange(n) % (P - 1)
    k, v = np.zeros((2, n, P, D))
    v[..., 1] = 1785.0
    k[np.arange(n), place] = stored_from(x)
    v[np.arange(n), place] = 0.0
    v[np.arange(n), place, 0] = 1785.0
    whole = ql.KVBatch(i32(np.arange(n + 1) * P), i32([P] * n), i32(np.arange(n)[:, None]), n * P, P, P)
    ql.kv_append(ws, cache, whole, *(torch.from_numpy(t.reshape(n * P, D)).float().to(DEV) for t in (k, v)))
    got, _ = ql.kv_read(ws, cache, whole, out_dtype=F32)
    assert torch.equal(got.cpu().double().view(n, P, D)[np.arange(n), place], torch.from_numpy(x))
    row, first = (a.ravel() for a in np.meshgrid(np.arange(n), np.arange(0, D, hq), indexing="ij"))
    column = (first[:, None] + np.arange(hq)) % D
    seqs = len(row)
    q = torch.zeros((seqs, new, hq, D), dtype=dtype, device=DEV)
    q.scatter_(3, torch.from_numpy(column).to(DEV)[:, None, :, None].expand(seqs, new, hq, 1), 1.0)
    print(f"[keys] {D} {hq} {new} {P} {dtype} {seqs} sequences", flush=True)
    b = ql.KVBatch(i32(np.arange(seqs + 1) * new), i32(place[row] + 1), i32(row[:, None]), seqs * new, new, P)
    out = ql.kv_attention(ws, cache, b, q.view(-1, hq * D), out_dtype=F32, scale=2.0 / 1785).view(seqs, new, hq, D)
    for c, want in enumerate(outputs(x[row[:, None], column], place[row][:, None])):
        off = np.abs(out[:, -1, :, c].double().cpu().numpy() - want) / want
        assert (off <= TOL).all(), (c, float(off.max()), np.argwhere(off > TOL)[:4])
    assert not out[..., 2:].any() and not out[:, :-1, :, 0].any()
    assert (out[:, :-1, :, 1] / 1785 - 1).abs().max() <= TOL if new > 1 else True
    assert ws.status() == 0
    cache.close()


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("D", [64, 84, 128, 256])
@pytest.mark.parametrize("hq,new,P", FORMS)
def test_every_value_column(ws, dtype, D, hq, new, P):
    """The others hold 1785 in one column each, so that all scales are 1."""
    x = keys(D)
    n = len(x)
    cache = ql.KVCache(1, D, n, P, bits=4)
    place = 1 + np.arange(n) % (P - 1)
    v = np.zeros((n, P, D))
    v[np.arange(n), :, np.arange(n) % D] = 1785.0
    v[np.arange(n), place] = stored_from(x)
    whole = ql.KVBatch(i32(np.arange(n + 1) * P), i32([P] * n), i32(np.arange(n)[:, None]), n * P, P, P)
    v = torch.from_numpy(v.reshape(n * P, D)).float().to(DEV)
    ql.kv_append(ws, cache, whole, torch.zeros_like(v), v)
    q = torch.zeros((n * new, hq * D), dtype=dtype, device=DEV)
    print(f"[values] {D} {hq} {new} {P} {dtype}", flush=True)
    b = ql.KVBatch(i32(np.arange(n + 1) * new), i32(place + 1), i32(np.arange(n)[:, None]), n * new, new, P)
    out = ql.kv_attention(ws, cache, b, q, out_dtype=F32).view(n, new, hq, D)[:, -1].double().cpu().numpy()
    others = np.zeros((n, D))
    others[np.arange(n), np.arange(n) % D] = 1785.0
    m = place[:, None]
    want, size = (x + m * others) / (m + 1), (np.abs(x) + m * others) / (m + 1)
    off = np.abs(out - want[:, None])
    assert (off <= TOL * size[:, None]).all(), (float(off.max()), np.argwhere(off > TOL * size[:, None])[:4])
    assert ws.status() == 0
    cache.close()
