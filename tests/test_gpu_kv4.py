"""The key/value cache in 4 bits: every test of the 8-bit cache on the GPU again, with rows held to the rule for 4 bits, and
what is its own.  A code times its unit takes the place of a code in the restatement."""
import functools

import numpy as np
import pytest
import torch

from open_rknpu2_lm_infer_amd import _lib
from open_rknpu2_lm_infer_amd import qlinear as ql
from tests import headref, kvref
from tests.test_gpu_kv import (test_append_then_read, test_attention, test_bad_batches_are_flagged,  # noqa: F401
                               test_captured_decode_steps, test_decoder_layers_on_the_device, test_long_offsets,
                               test_loose_bounds, test_nan_query_stays_in_its_row, test_nonfinite_f32_query_stays_in_its_row,
                               test_nonfinite_rows_are_poisoned_alone, test_prefix_without_room_for_its_results,
                               test_prompts, test_rows_before_the_first_sequence, test_scales_far_apart,
                               test_shared_prefix, test_streams_side_by_side, test_strides_and_rows_of_nobody,
                               test_unseen_tokens_do_not_matter, ws)
from tests.test_gpu_kv import DEV, F16, F32, Setup, i32
from tests.test_gpu_kv_errors import (test_append_stores_nothing_for_a_sequence_at_fault,  # noqa: F401
                                      test_bad_prefix_page_reaches_only_rows_that_see_it)
from tests.test_gpu_kv_instances import (test_attention_instance, test_captured_chunks,  # noqa: F401
                                         test_equal_logits_at_the_largest_scale, test_few_vectors_in_fp16_are_rounded_once)

pytestmark = pytest.mark.gpu

_attend = kvref.attend
# Codes of 8 bits go to 127, a code times its unit to 1785.
UP = 1785.0 / 127.0


def attend4(q, kc, ks, vc, vs, seen, scale, limbs, out_eps):
    """kvref.attend, whose bound takes codes to be at most 127: values in units of 1785 / 127.  The kernel's exponents hold
    log2 of the scales as they are, log2(1785 / 127) = 3.82 more in size at most: 2 * 4 * 3.82 steps of 2^-23 of
    sum_j p_j |v_j|, which attend gives for values without their signs."""
    vs = np.asarray(vs, np.float64) * UP
    out, tol = _attend(q, kc, ks, vc / UP, vs, seen, scale, limbs, out_eps)
    size, _ = _attend(q, kc, ks, np.abs(vc) / UP, vs, seen, scale, limbs, out_eps)
    return out, tol + 2.0 ** -18 * np.nan_to_num(size)


@pytest.fixture(autouse=True)
def four_bits(monkeypatch):
    monkeypatch.setattr(ql, "KVCache", functools.partial(ql.KVCache, bits=4))
    monkeypatch.setattr(kvref, "quantize", headref.quantize4)
    monkeypatch.setattr(kvref, "attend", attend4)


def test_bytes():
    c = ql.KVCache(8, 128, 10, 64)
    assert c.bits == 4 and c.device_bytes == 10 * 8 * 64 * 144
    c.close()


@pytest.mark.parametrize("half_even", [False, True])
def test_rounding_and_units(ws, half_even):  # noqa: F811
    """Ties of codes, units at their ends, groups of zeros, rows below the smallest scale."""
    s = Setup(ws, [(9, 9)], 1, 72, 16, F32, seed=1)
    x = torch.zeros((9, 72))
    x[0, 0], x[0, 1:8], x[0, 40] = 1785.0, torch.tensor([127.5, -127.5, 382.5, -382.5, 637.5, 892.5, -1657.5]), 7.0  # scale 1, units 255 and 1
    x[1, 3], x[1, 40:44] = 1785.0, torch.tensor([0.5, 1.5, -2.5, 6.4])
    x[2] = 0.0
    x[3, 5] = 2.0 ** -80
    x[4] = torch.arange(72) * 3.0 ** -7
    x[5, 71] = -3e38
    x[6, 0], x[6, 33] = 1e30, 1e-30
    x[7] = 2.0 ** -64 * 1785 / 2 * torch.linspace(-1, 1, 72)
    x[8] = -1.0
    ql.kv_append(ws, s.cache, s.batch(), x.to(DEV), (-x).to(DEV), flags=ql.QLIN_ROUND_HALF_EVEN if half_even else 0)
    k, v = ql.kv_read(ws, s.cache, s.batch(), out_dtype=F32)
    for got, src in ((k, x), (v, -x)):
        c, sc = headref.quantize4(src.numpy(), half_even)
        assert torch.equal(got.cpu(), torch.from_numpy(c.astype(np.float32) * sc[:, None]))
    assert ws.status() == 0
    s.cache.close()


def test_every_code_and_unit(ws):  # noqa: F811
    """Every code of every unit through the operands of the matrix core: one token a sequence gives back its value row, and
    the logits of unit queries its keys."""
    D, n = 64, 255
    s = Setup(ws, [(n, 1)], 1, D, 16, F32, seed=2)
    x = torch.zeros((n, D))
    x[:, 0] = 1785.0  # scale 1
    for u in range(1, 256):  # the largest a little below seven units, which are rounded up to
        x[u - 1, 32:47] = torch.arange(-7, 8).float() * u
        x[u - 1, 32], x[u - 1, 46] = -7.0 * u + 0.3, 7.0 * u - 0.3
    s.fill(x, x)
    k, v = ql.kv_read(ws, s.cache, s.batch(news=[n]), out_dtype=F32)
    assert torch.equal(k[:, 32:47].cpu(), torch.arange(1.0, 256)[:, None] * torch.arange(-7.0, 8)) and torch.equal(k, v)
    # of each token alone: a softmax over one token is 1
    table = i32(np.repeat(s.table, n, 0))
    for new, hq in ((1, 1), (1, 40)):  # tiles of 16 and 32 vectors
        alone = ql.KVBatch(i32(np.arange(n + 1)), i32(np.arange(1, n + 1)), table, n, new, n)
        q = torch.zeros((n, hq * D), device=DEV)
        q.view(n, hq, D)[:, :, 0] = 30.0  # equal logits
        got = ql.kv_attention(ws, s.cache, alone, q, scale=1.0)
        want = torch.cumsum(k.double().cpu(), 0) / torch.arange(1, n + 1)[:, None]
        # sums of up to 255 values of up to 1785 in f32, P exact (equal): 2 * (n / 8 + 64) 2^-23 of the mean size, as kvref counts
        size = torch.cumsum(k.double().cpu().abs(), 0) / torch.arange(1, n + 1)[:, None]
        tol = 2.0 ** -15 * size + 1e-6
        err = (got.double().cpu().view(n, hq, D) - want[:, None]).abs()
        assert (err <= tol[:, None]).all()
    s.cache.close()


def test_many_vectors_of_every_unit(ws):  # noqa: F811
    """The same through the kernel for many vectors, keys told apart by their logits."""
    D, n = 128, 255
    s = Setup(ws, [(n, n)], 1, D, 32, F32, seed=3, q_heads=3)
    x = s.rand(n, D)
    for u in range(1, 256):
        x[u - 1, 0], x[u - 1, 32:47] = 1785.0 / 64, torch.arange(-7, 8).float() * (u - 0.04) / 64
    s.fill(x, x)
    q = s.rand(n, 3 * D, size=0.05)
    out = ql.kv_attention(ws, s.cache, s.batch(), q.to(DEV))
    want, tol = s.expected(q, x, x, F32)
    err = np.abs(out.double().cpu().numpy() - want)
    assert (err <= tol).all()
    s.cache.close()


def test_status_of_a_poisoned_row_is_of_its_own(ws):  # noqa: F811
    s = Setup(ws, [(20, 2)], 2, 64, 16, F16, seed=4)
    k = s.rand(2, 128)
    k[1, 70] = float("inf")
    ql.kv_append(ws, s.cache, s.batch(), k.to(DEV), s.rand(2, 128).to(DEV))
    assert ws.status() == _lib.QLIN_ERR_NONFINITE
    ko, vo = ql.kv_read(ws, s.cache, s.batch())
    assert torch.isnan(ko[1, 64:]).all() and torch.isfinite(ko[0]).all() and torch.isfinite(ko[1, :64]).all() and torch.isfinite(vo).all()
    s.cache.close()
