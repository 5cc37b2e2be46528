"""Softmax weights over the 8-bit cache: many small ones beside a large one count, and those of f16 queries of few rows go into the product in two
parts."""
import numpy as np
import pytest
import torch

from oracle import q8_oracle as qo
from tests.test_gpu_attention_q8 import Step
from tests.test_gpu_attention_q8_units import check

pytestmark = pytest.mark.gpu


def sink_step(lengths, heads, kv_heads, D, page, dtype, above, at, seed=30):
    """One key of every request stands about `above` over the others, whose scores are about 0, and its value is 0; theirs are about 1."""
    s = Step(lengths, heads, kv_heads, D, page, dtype, seed=seed, spread=0)
    c, rng = s.cache, np.random.default_rng(seed)
    q = np.where(rng.random(D) < 0.5, -1.0, 1.0)
    s.query = torch.from_numpy(np.broadcast_to(q, (s.T, heads, D)).astype(np.float32).copy()).to(s.dtype)
    owned = (c.codes & 127) != 127
    c.exponents[..., 0] = -9                                    # (the others' scores: a few tenths)
    c.exponents[..., 1] = -6
    c.codes[:, 1] = np.where(owned[:, 1], qo.encode(64 * (1 + 0.3 * rng.standard_normal(c.codes[:, 1].shape))), c.codes[:, 1])
    for b in range(len(lengths)):
        slot = int(s.indices[s.indptr[b] + at // page]) * page + at % page
        g = slot // 16
        top = above / (D * s.scale)                             # of every column of the key
        e = int(np.ceil(np.log2(top / 448)))
        had = qo.VALUES[c.codes[g * 16:g * 16 + 16, 0]] * 2.0 ** (-9 - max(e, -9))
        there = owned[g * 16:g * 16 + 16, 0]
        c.codes[g * 16:g * 16 + 16, 0] = np.where(there, qo.encode(np.where(there, had, 0)), c.codes[g * 16:g * 16 + 16, 0])
        c.exponents[g, :, 0] = max(e, -9)
        c.codes[slot, 0] = qo.encode(q * top * 2.0 ** -max(e, -9))
        c.codes[slot, 1] = 0
    return s


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("above", [9.0, 16.5, 18.0])
@pytest.mark.parametrize("lengths,heads,kv_heads,D,page", [
    ([(1, 7001)], 4, 2, 64, 16), ([(1, 900), (2, 700)], 4, 1, 128, 16), ([(1, 3000)], 4, 1, 80, 32),   # narrow tiles
    ([(40, 3000)], 4, 1, 64, 16), ([(40, 900), (35, 2001)], 4, 2, 128, 16), ([(40, 2000)], 2, 2, 256, 16)])   # wide
def test_one_key_far_above_many(gpu, lengths, heads, kv_heads, D, page, above, dtype):
    s = sink_step(lengths, heads, kv_heads, D, page, dtype, above, 100)
    out, lse = s.plan(gpu).run(s.query.to(gpu), s.pages(gpu), return_lse=True)
    check(s, out, lse)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("new", [1, 40])
def test_the_far_key_comes_late(gpu, new, dtype):
    """What was summed before it, and the weights that wait for their product, are scaled down by as much."""
    for at in (160, 1499, 2950):
        s = sink_step([(new, 3000)], 4, 1, 64, 16, dtype, 16.5, at)
        out, lse = s.plan(gpu).run(s.query.to(gpu), s.pages(gpu), return_lse=True)
        check(s, out, lse)


def cancelling_step(D, shared):
    """Requests of two to five keys (or as many behind a shared prefix) with nearly equal weights, and values of opposite signs that nearly cancel. (The rows of
    those that share are narrow tiles up to 128 of them; the wide ones have their weights in one part.)"""
    rng = np.random.default_rng(31)
    base = 16 * shared
    s = Step([(1, base + int(k)) for k in rng.integers(2, 6, 60 if shared else 96)], 4, 2, D, 16, "f16", seed=31, shared=shared, spread=0)
    c = s.cache
    owned = (c.codes[:, 1] & 127) != 127
    sign = np.where(np.arange(c.codes.shape[0]) % 2, -1.0, 1.0)[:, None, None]
    c.codes[:, 1] = np.where(owned, qo.encode(np.broadcast_to(sign * 240, c.codes[:, 1].shape)), c.codes[:, 1])
    s.query = s.query * 0.125
    return s


def bound(s, keys):
    """What two parts leave of a weight, 2^-22; the sums' (of weights and of their products) 2^-24 a term; the score's error; the output's rounding."""
    want, _, weighted, _, products = s.oracle()
    ds = s.scale * products * (s.D + 2) * 2.0 ** -24 + (1 + s.scale * products) * 2.0 ** -22
    return want, weighted * (2.0 ** -22 + 2 * (keys + 8) * 2.0 ** -24 + 2 * ds[..., None]) + np.abs(want) * 2.0 ** -11 * 1.01 + 2.0 ** -25


@pytest.mark.parametrize("D", [16, 64, 128, 256])
@pytest.mark.parametrize("shared", [0, 1])
def test_f16_weights_in_two_parts(gpu, D, shared):
    """f16 queries of few rows: two parts of 11 bits leave 2^-22 of a weight, where one would leave 2^-11 (and be off by several times the bound here)."""
    s = cancelling_step(D, shared)
    want, tol = bound(s, 16 * shared + 5)
    out = s.plan(gpu, max_q_len=1).run(s.query.to(gpu), s.pages(gpu)).cpu().double().numpy()
    err = np.abs(out - want)
    assert (err <= tol).all(), f"off by {(err / tol).max():.3g} of the bound"


@pytest.mark.parametrize("D", [64, 80, 128, 256])
def test_a_row_of_one_key_is_its_value(gpu, D):
    """f16, wide tiles, whose weights are rounded once: what O is divided by is rounded with them. Codes times 2^-6 are numbers of f16, so the first row of a prompt
    comes out as its key's value, and one whose keys have one value as that value."""
    s = Step([(40, 40)] * 24 + [(70, 70)] * 8, 4, 2, D, 16, "f16", seed=33, spread=0)
    c = s.cache
    for b in range(24, 32):
        table = s.indices[s.indptr[b]:s.indptr[b + 1]].astype(np.int64)
        slots = (table[:, None] * 16 + np.arange(16)).ravel()[:70]
        c.codes[slots, 1] = c.codes[slots[0], 1]
    out = s.plan(gpu).run(s.query.to(gpu), s.pages(gpu)).cpu().double().numpy()
    values = c.values()[:, 1]
    for b in range(32):
        v = np.repeat(values[int(s.indices[s.indptr[b]]) * 16], 2, axis=0)
        rows = out[s.qo[b]] if b < 24 else out[s.qo[b]:s.qo[b + 1]]
        # (sums in 32 bits: far less than half a step of f16, so the rounding takes it off)
        assert (np.abs(rows - v) <= 2.0 ** -20 * np.abs(v)).all(), b
