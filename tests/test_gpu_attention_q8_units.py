"""Attention over the 8-bit cache where groups, weights or both differ by more than a 16-bit type holds: a row's result is made of
the keys that it sees, and of each by its weight times its value."""
import numpy as np
import pytest
import torch

from oracle import attention_oracle as ao
from oracle import q8_oracle as qo
from tests.test_gpu_attention_q8 import Step

pytestmark = pytest.mark.gpu


def terms(s):
    """For every row: the largest weight times its group's 2^ev, and the greatest 2^ev, each over the sum of weights, and for every column the sum of |codes|, over
    the keys that the row sees."""
    G, c = s.Hq // s.H, s.cache
    values = c.values()
    sizes = 2.0 ** np.repeat(c.exponents[..., 1].astype(np.float64), qo.GROUP, axis=0)      # [slots, H]
    codes = np.abs(qo.VALUES[c.codes[:, 1]])
    largest, greatest, total = np.zeros((s.T, s.Hq)), np.zeros((s.T, s.Hq)), np.zeros((s.T, s.Hq, s.D))
    q = s.query.double().numpy()
    for b in range(len(s.qo) - 1):
        table = s.indices[s.indptr[b]:s.indptr[b + 1]].astype(np.int64)
        slots = (table[:, None] * s.page + np.arange(s.page)).ravel()
        length, n = (len(table) - 1) * s.page + int(s.last[b]), int(s.qo[b + 1] - s.qo[b])
        for i in range(n):
            seen = slots[:max(length - n + i + 1, 0)]
            if not len(seen):
                continue
            for x in range(s.Hq):
                score = s.scale * (values[seen, 0, x // G] @ q[s.qo[b] + i, x])
                p = np.exp(score - score.max())
                at = int(s.qo[b]) + i, x
                largest[at], greatest[at] = (p * sizes[seen, x // G]).max() / p.sum(), sizes[seen, x // G].max() / p.sum()
                total[at] = codes[seen, x // G].sum(0)
    return largest, greatest, total


def check(s, out, lse, weight_eps=2.0 ** -10):
    """The roundings, counted. A weight goes into the product as f16, off by half a step of itself (`weight_eps` / 2), or, below f16's normal numbers, by half their
    step, 2^-25, once when it is made and once when the units that it waits in grow: units in which the row's largest weight times size is at least 2^6, so 2^-30 of that
    largest, times the code. However small the weights, units are at most 2^100 below the greatest size: what is below f16's numbers there, 2^-115 of it,
    counts as nothing. The rest is the arithmetic's in 32 bits and the output's own rounding."""
    want, want_lse, weighted, values, products = s.oracle()
    largest, greatest, total = terms(s)
    tol, tol_lse = ao.attention_tolerances(want, want_lse, weighted, values, products, s.D, s.scale, weight_eps, 0.0)
    tol = tol + np.abs(want) * s.eps / 2 * 1.05 + ((largest * 2.0 ** -30 + greatest * 2.0 ** -115)[..., None] * total)
    smallest = 2.0 ** -25 if s.dtype == torch.float16 else 2.0 ** -134
    got = out.cpu().double().numpy().reshape(want.shape)
    err = np.abs(got - want)
    assert (err <= tol + smallest).all(), f"off by {np.nanmax(err / (tol + smallest)):.3g} of the bound at {np.unravel_index(np.nanargmax(err / (tol + smallest)), err.shape)}"
    assert (np.abs(lse.cpu().double().numpy() - want_lse) <= tol_lse).all()


LENGTHS = [(60, 200), (1, 130), (3, 90), (40, 40), (1, 500), (130, 333)]


def with_large_groups(low, gap, which, dtype, D, heads=4, kv_heads=2, light=0.0, seed=40):
    """V of 2^low in every group but the large ones, 2^gap above: those of a request's `last` keys, `first` ones or every `other` group. With `light`
    the scores of the large groups' keys are that much below the others' (about)."""
    s = Step(LENGTHS, heads, kv_heads, D, 16, dtype, seed=seed, spread=0)
    c = s.cache
    c.exponents[..., 1] = low
    sign = np.where(s.rng.random(D) < 0.5, -1.0, 1.0)
    if light:
        s.query = torch.from_numpy(np.broadcast_to(sign, (s.T, heads, D)).astype(np.float32).copy()).to(s.dtype)
    for b, (n, k) in enumerate(LENGTHS):
        table = s.indices[s.indptr[b]:s.indptr[b + 1]]
        large = {"last": table[-(-len(table) // 3):] if len(table) > 1 else table, "first": table[:max(1, len(table) // 3)], "other": table[1::2]}[which]
        c.exponents[large, :, 1] = low + gap
        if light:
            # q.k = -sum |k| where k goes against q
            slots = (large.astype(np.int64)[:, None] * 16 + np.arange(16)).ravel()
            there = (c.codes[slots, 0] & 127) != 127
            c.codes[slots, 0] = np.where(there, qo.encode(-sign * 64), c.codes[slots, 0])
            c.exponents[large, :, 0] = -6 + round(np.log2(light / (D * s.scale)))
    return s


@pytest.mark.parametrize("D", [64, 128, 80, 256])
@pytest.mark.parametrize("which", ["last", "first", "other"])
@pytest.mark.parametrize("low,gap,dtype", [(-6, 30, "bf16"), (-6, 45, "bf16"), (-6, 100, "bf16"), (-40, 140, "bf16"), (-100, 200, "bf16"), (-14, 22, "f16")])
def test_large_groups(gpu, low, gap, dtype, which, D):
    """Large groups that some rows see and others, of the same tile, do not."""
    s = with_large_groups(low, gap, which, dtype, D)
    out, lse = s.plan(gpu).run(s.query.to(gpu), s.pages(gpu), return_lse=True)
    check(s, out, lse)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("which", ["last", "first", "other"])
@pytest.mark.parametrize("gap,light", [(30, 16), (45, 32), (60, 32), (45, 64), (110, 64), (20, 32)])
def test_large_groups_of_little_weight(gpu, gap, light, which, D):
    """Values that are 2^gap larger under weights that are e^-light smaller, in turn more and less than what they lie among."""
    s = with_large_groups(-30, gap, which, "bf16", D, light=light)
    out, lse = s.plan(gpu).run(s.query.to(gpu), s.pages(gpu), return_lse=True)
    check(s, out, lse)


@pytest.mark.parametrize("which", ["last", "other"])
@pytest.mark.parametrize("rising", [False, True])
@pytest.mark.parametrize("size", [8, 14, 20])
def test_large_groups_and_scores_beyond_whole_numbers(gpu, size, rising, which):
    """Scores up to 2^size * 60, from 2^24 on none to which an exponent can be added in 32 bits. The keys' scores differ by 6 % and more, the sums are exact: where that is
    200 at least, a row is the value of its highest key, to the output's rounding (the others' weights are below e^-200, of values 2^40 larger at most)."""
    s = with_large_groups(-6, 40, which, "bf16", 64, seed=41)
    c = s.cache
    s.query = torch.ones_like(s.query)
    rank = s.rng.permuted(np.tile(np.arange(16), (c.codes.shape[0] // 16, 1)), axis=1).ravel()
    steps = np.array([2.0, 2.25, 2.5, 2.75, 3.0, 3.25, 3.5, 3.75, 4.0, 4.5, 5.0, 5.5, 6.0, 6.5, 7.0, 7.5])
    there = (c.codes[:, 0] & 127) != 127
    c.codes[:, 0] = np.where(there, qo.encode(np.broadcast_to(steps[rank][:, None, None], c.codes[:, 0].shape)), c.codes[:, 0])
    # a group's keys are above those of the next one along the request, or below
    order = np.zeros(c.exponents.shape[0], np.int64)
    for b in range(len(LENGTHS)):
        table = s.indices[s.indptr[b]:s.indptr[b + 1]]
        order[table] = np.arange(len(table)) - len(table) + 1 if rising else -np.arange(len(table))
    c.exponents[..., 0] = size + 2 * order[:, None]
    out, lse = s.plan(gpu).run(s.query.to(gpu), s.pages(gpu), return_lse=True)
    got, got_lse, values = out.cpu().double().numpy(), lse.cpu().double().numpy(), c.values()
    checked = 0
    for b, (n, k) in enumerate(LENGTHS):
        table = s.indices[s.indptr[b]:s.indptr[b + 1]].astype(np.int64)
        slots = (table[:, None] * 16 + np.arange(16)).ravel()
        for i in range(n):
            seen = slots[:k - n + i + 1]
            score = s.scale * values[seen, 0, 0].sum(1)
            top = np.argmax(score)
            if len(seen) > 1 and np.sort(score)[-2] > score[top] - 200:
                continue
            checked += 1
            want = values[seen[top], 1][:, None]
            at = int(s.qo[b]) + i
            # (two roundings in 32 bits and the output's)
            assert (np.abs(got[at].reshape(2, 2, 64) - want) <= (2.0 ** -8 + 2.0 ** -22) * np.abs(want)).all(), (b, i)
            assert (np.abs(got_lse[at] - score[top]) <= 2.0 ** -21 * score[top] + 2.0 ** -18).all()
    assert checked > 20
