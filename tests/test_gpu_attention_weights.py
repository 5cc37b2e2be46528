"""Softmax weights far below the largest: many of them together count, however small each is."""
import numpy as np
import pytest
import torch

from oracle import attention_oracle as ao
from tests.test_gpu_attention import Step

pytestmark = pytest.mark.gpu


def sink_step(lengths, heads, kv_heads, D, page, dtype, above, at, seed=30):
    """One key of every request stands `above` the others, whose scores are about 0, and its value is 0."""
    s = Step(lengths, heads, kv_heads, D, page, dtype, seed=seed)
    rng = np.random.default_rng(seed)
    q = rng.standard_normal(D).astype(np.float32)
    s.query = torch.from_numpy(np.broadcast_to(q, (s.T, heads, D)).copy()).to(s.dtype)
    s.cache[:, 0] *= 0.1
    s.cache[:, 1] = 1 + 0.3 * s.cache[:, 1]
    q = s.query[0, 0].float().numpy()
    for b in range(len(lengths)):
        p = s.indices[s.indptr[b] + at // page]
        s.cache[p, 0, at % page] = torch.from_numpy(q * (above / s.scale / (q * q).sum())).to(s.dtype)
        s.cache[p, 1, at % page] = 0
    return s


def check(s, out, lse):
    """As Step.check, but with a bound on a weight's rounding that has no floor at the type's smallest number. What is left of one:
    weights are at most 2^-7 of the type's range below it, half a step of the smallest numbers is 2^-25, and a base stands
    up to 1 above the largest score: 2^-31 of the largest weight."""
    want, want_lse, weighted, values, products = s.oracle()
    tol, tol_lse = ao.attention_tolerances(want, want_lse, weighted, values, products, s.D, s.scale, s.eps, 0.0)
    # (the output's own smallest numbers)
    tol = tol + values * 2.0 ** -31 * (s.denormal > 0) + s.denormal
    got = out.cpu().double().numpy().reshape(want.shape)
    err = np.abs(got - want)
    assert (err <= tol).all(), f"off by {np.nanmax(err / tol):.3g} of the bound, {np.nanmax(err / np.abs(want)):.3g} of the value"
    assert (np.abs(lse.cpu().double().numpy() - want_lse) <= tol_lse).all()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("above", [9.0, 16.5, 18.0])
@pytest.mark.parametrize("lengths,heads,kv_heads,D,page", [
    ([(1, 7001)], 4, 2, 64, 16), ([(1, 900), (2, 700)], 4, 1, 128, 16), ([(1, 3000)], 4, 1, 80, 20),   # narrow tiles
    ([(40, 3000)], 4, 1, 64, 16), ([(40, 900), (35, 2001)], 4, 2, 128, 20), ([(40, 6000)], 128, 128, 8, 16)])   # wide
def test_one_key_far_above_many(gpu, lengths, heads, kv_heads, D, page, above, dtype):
    s = sink_step(lengths, heads, kv_heads, D, page, dtype, above, 100)
    out, lse = s.plan(gpu).run(s.query.to(gpu), s.cache.to(gpu), return_lse=True)
    check(s, out, lse)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("new", [1, 40])
def test_the_far_key_comes_late(gpu, new, dtype):
    """What was summed before it, and the weights that wait for their product, are scaled down by as much."""
    for at in (160, 1499, 2950):
        s = sink_step([(new, 3000)], 4, 1, 64, 16, dtype, 16.5, at)
        out, lse = s.plan(gpu).run(s.query.to(gpu), s.cache.to(gpu), return_lse=True)
        check(s, out, lse)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("lengths,heads,kv_heads,D,page,shared", [
    ([(1, 40), (1, 700), (2, 65), (1, 2001)], 8, 2, 128, 16, 0), ([(4, 300), (1, 33)], 8, 2, 64, 16, 0), ([(1, 900)], 16, 1, 80, 20, 0),
    ([(3, 500), (1, 77)], 5, 1, 256, 32, 0), ([(1, 400 + 9 * i) for i in range(4)], 8, 2, 96, 8, 40)])
def test_few_rows_round_their_outputs_only(gpu, lengths, heads, kv_heads, D, page, shared, dtype):
    """Narrow tiles: the weights' two parts are off by 2^-16 (bf16) and 2^-22 of themselves, 32-bit sums by less, and the output's
    rounding is all that shows: the error's root mean square is that of the exact outputs rounded, to 1 %. (A weight in one
    part adds as much again as its own rounding, a quarter.)"""
    s = Step(lengths, heads, kv_heads, D, page, dtype, shared=shared, seed=31)
    out, lse = s.plan(gpu, max_q_len=max(n for n, _ in lengths)).run(s.query.to(gpu), s.cache.to(gpu), return_lse=True)
    s.check(out, lse)
    want = torch.from_numpy(s.oracle()[0])
    rms = lambda x: x.square().mean().sqrt().item()
    rounded = rms(want.to(s.dtype).double() - want)
    assert rms(out.cpu().double().reshape(want.shape) - want) <= 1.01 * rounded


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("lengths", [[(1, 900), (2, 40)], [(40, 700), (1, 33)]])
def test_scores_of_millions(gpu, lengths, dtype):
    """Scores up to 2^23 times log2(e), hundreds of thousands apart: a row is the value v of its highest key. In narrow tiles the
    weight w goes in as w1 + w2 with |w1 + w2 - w| <= (eps / 2)^2 w, so that o = v (w1 + w2) / w is nearer to v than the quarter step
    from which a value of the type would round to another: the same bits. In wide ones only w1 with |w1 - w| <= eps / 2 w does: o is
    off by eps / 2 |v|, and its rounding by eps / 2 |o|: eps (1 + eps / 4) |v| together."""
    s = Step(lengths, 8, 2, 128, 16, dtype, seed=32, scale_q=4096.0)
    s.cache[:, 0] *= 512
    out, lse = s.plan(gpu).run(s.query.to(gpu), s.cache.to(gpu), return_lse=True)
    out, lse = out.cpu(), lse.cpu().double()
    for b, (n, k) in enumerate(lengths):
        pages = torch.from_numpy(s.indices[s.indptr[b]:s.indptr[b + 1]].astype(np.int64))
        keys, values = (s.cache[pages, i].reshape(-1, 2, 128)[:k] for i in (0, 1))
        for j in range(n):
            t = int(s.qo[b]) + j
            for x in range(8):
                score = keys[:k - n + j + 1, x // 4].double() @ s.query[t, x].double() * s.scale
                top = score.topk(min(2, len(score)))
                if len(score) > 1 and top.values[0] - top.values[1] < 200 + 2.0 ** -16 * top.values.abs().max():
                    continue      # (too close to tell in 32 bits)
                v = values[top.indices[0], x // 4]
                if n * 4 > 32:
                    assert ((out[t, x].double() - v.double()).abs() <= s.eps * 1.01 * v.double().abs() + s.denormal).all()
                else:
                    assert torch.equal(out[t, x], v)
                assert abs(lse[t, x] - top.values[0]) <= 2.0 ** -16 * top.values[0].abs() + 1
