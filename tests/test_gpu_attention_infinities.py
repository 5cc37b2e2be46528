"""Infinite values that rows do see: their columns are infinite, whatever their weights are and wherever the other rows stop."""
import numpy as np
import pytest
import torch

from oracle import attention_oracle as ao
from tests.test_gpu_attention import Step

pytestmark = pytest.mark.gpu

COLUMNS = {3: float("inf"), 20: float("-inf")}     # and 9 holds both, at two keys


def infinite_step(lengths, heads, kv_heads, D, page, dtype, at, far, shared=0):
    """Request 0's values at the keys `at` and `at + 1` are infinite in some columns; with `far` its queries' scores there are some
    hundreds below the others'."""
    s = Step(lengths, heads, kv_heads, D, page, dtype, shared=shared, seed=41)
    clean = s.oracle()
    if far:     # all of request 0's rows have the same query, and the two keys are far below it
        s.query[:] = s.query[0, 0]
        for key in (at, at + 1):
            p = s.indices[s.indptr[0] + key // page]
            s.cache[p, 0, key % page] = (-40.0 * s.query[0, 0].float()).to(s.dtype)
        clean = s.oracle()
    for key in (at, at + 1):
        p = s.indices[s.indptr[0] + key // page]
        for c, x in COLUMNS.items():
            if key == at:
                s.cache[p, 1, key % page, :, c] = x
        s.cache[p, 1, key % page, :, 9] = float("inf") if key == at else float("-inf")
    return s, clean


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("far", [False, True])
@pytest.mark.parametrize("lengths,heads,kv_heads,D,page,at,shared", [
    ([(1, 300)], 8, 2, 64, 16, 100, 0), ([(1, 9000)], 4, 1, 128, 16, 4000, 0), ([(3, 700), (1, 50)], 4, 1, 128, 20, 17, 0),
    ([(1, 500)], 2, 1, 256, 16, 498, 0),                                                     # narrow tiles, whole and in parts
    ([(40, 300)], 4, 1, 64, 16, 100, 0), ([(40, 3000), (1, 20)], 4, 2, 128, 16, 1300, 0), ([(150, 700)], 4, 1, 96, 20, 610, 0),
    ([(40, 6000)], 128, 128, 32, 16, 2000, 0), ([(33, 400)], 2, 1, 256, 32, 5, 0),           # wide
    ([(1, 1200 + i) for i in range(1, 11)], 4, 1, 64, 16, 700, 70),                          # a shared prefix
    ([(1, 1200 + i) for i in range(1, 41)], 4, 1, 64, 16, 700, 70)])
def test_values_that_are_seen(gpu, lengths, heads, kv_heads, D, page, at, shared, far, dtype):
    s, clean = infinite_step(lengths, heads, kv_heads, D, page, dtype, at, far, shared)
    out, lse = s.plan(gpu).run(s.query.to(gpu), s.cache.to(gpu), return_lse=True)
    out, lse = out.cpu().double().numpy(), lse.cpu().double().numpy()
    want, want_lse, *bounds = clean
    tol, tol_lse = ao.attention_tolerances(want, want_lse, *bounds, D, s.scale, s.eps, s.denormal)
    odd = np.zeros(D, bool)
    odd[[3, 9, 20]] = True
    assert (np.abs(lse - want_lse) <= tol_lse).all()
    assert (np.abs(out - want)[..., ~odd] <= tol[..., ~odd]).all()
    for b, (n, k) in enumerate(lengths):
        for j in range(n):
            t, position = int(s.qo[b]) + j, k - n + j
            owns = b == 0 or at < shared * page      # (of the shared pages every request sees the keys)
            first, second = owns and position >= at, owns and position >= at + 1
            for c, x in COLUMNS.items():
                if first:
                    assert (out[t, :, c] == x).all(), (t, c, out[t, :, c])
                else:
                    assert (np.abs(out - want)[t, :, c] <= tol[t, :, c]).all()
            if second:
                assert np.isnan(out[t, :, 9]).all()
            elif first:
                assert (out[t, :, 9] == np.inf).all()


def test_a_row_whose_scores_are_all_minus_infinity_is_zero(gpu):
    """Also where the values beside them are infinite."""
    for lengths in ([(1, 200)], [(40, 200)]):
        s = Step(lengths, 4, 1, 64, 16, seed=42)
        s.query[:, :, :] = 0
        s.query[:, :, 0] = 1
        for p in s.indices:
            s.cache[p, 0, :, :, 0] = float("-inf")
        s.cache[s.indices[3], 1, 2] = float("inf")
        out, lse = s.plan(gpu).run(s.query.to(gpu), s.cache.to(gpu), return_lse=True)
        assert (out == 0).all() and torch.isneginf(lse).all()
