"""Head norms with the rotation and the K/V write against the formula in 64 bits; the cache holds the very bits that the
call returns for the key, the value's bits, and what it held everywhere else."""
import numpy as np
import pytest
import torch

import lmserve_amd as kvc
from oracle import attention_oracle as ao

pytestmark = pytest.mark.gpu

EPS = 1e-6
# half a step of the type, relative to the value, and half the smallest denormal
TYPES = {"bf16": (torch.bfloat16, 2.0 ** -8, 0.0), "f16": (torch.float16, 2.0 ** -11, 2.0 ** -25),
         "f32": (torch.float32, 2.0 ** -24, 0.0)}
# heads, kv heads, head_dim, rotary_dim, page
SHAPES = [(32, 8, 128, 128, 16), (28, 4, 128, 64, 16), (15, 5, 80, 32, 16), (4, 4, 64, 64, 8), (3, 1, 96, 96, 20), (2, 2, 256, 128, 16),
          (7, 1, 36, 36, 16), (5, 1, 33, 22, 5), (1, 1, 8, 8, 1), (6, 3, 16, 0, 16), (2, 1, 512, 512, 16), (2, 1, 1032, 256, 4),
          (9, 3, 40, 16, 64)]


def make(shape, dtype, T, seed=0, fused=True, off=0):
    hq, hk, D, rd, page = shape
    rng = np.random.default_rng(seed)
    t = lambda *s: torch.from_numpy(rng.standard_normal(s).astype(np.float32))
    td = TYPES[dtype][0]
    qkv = t(T, (hq + 2 * hk) * D + off).to(td)
    cut = qkv[:, off:]
    q, k, v = cut[:, :hq * D], cut[:, hq * D:(hq + hk) * D], cut[:, (hq + hk) * D:]
    if not fused:
        q, k, v = q.clone(), k.clone(), v.clone()
    qw, kw = (1 + 0.3 * t(D)).to(td), (1 + 0.3 * t(D)).to(td)
    longest = 600
    cs = kvc.make_cos_sin_cache(rd, longest, 10000.0, dtype=td)
    nb = -(-T // page) + 3
    slots = torch.from_numpy(rng.permutation(nb * page)[:T].astype(np.int64))
    pos = torch.from_numpy(rng.integers(0, longest, T).astype(np.int32))
    cache = t(nb, 2, page, hk, D).to(td)
    return q, k, v, qw, kw, cs, pos, slots, cache


def check(got, x, w, pos, cs, D, dtype):
    want, arith = ao.qk_norm_rotary_f64(x.double().numpy(), w.double().numpy(), pos.numpy(), cs.double().numpy(), D, EPS)
    half, denormal = TYPES[dtype][1:]
    err = np.abs(got.cpu().double().numpy().reshape(want.shape) - want)
    tol = (np.abs(want) + arith) * half * 1.01 + arith + denormal
    assert (err <= tol).all(), f"off by {(err / tol).max():.3g} of the bound"


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("T", [1, 7, 130])
def test_against_the_formula(gpu, shape, dtype, T):
    hq, hk, D, rd, page = shape
    q, k, v, qw, kw, cs, pos, slots, cache = make(shape, dtype, T)
    dev = [x.to(gpu) for x in (q, k, v, qw, kw)]
    # slices of one matrix stay slices
    row = torch.cat((q, k, v), 1).to(gpu)
    dq, dk, dv = row[:, :hq * D], row[:, hq * D:(hq + hk) * D], row[:, (hq + hk) * D:]
    dqw, dkw, dcs, dpos = dev[3], dev[4], cs.to(gpu), pos.to(gpu)
    qo, ko = kvc.qk_norm_rotary_pos_emb(dq, dk, dqw, dkw, dpos, dcs, D, EPS)
    check(qo, q, qw, pos, cs, D, dtype)
    check(ko, k, kw, pos, cs, D, dtype)
    # 64-bit positions, slots of either width, the page table: the same bits
    q8, k8 = kvc.qk_norm_rotary_pos_emb(dq, dk, dqw, dkw, dpos.long(), dcs, D, EPS)
    assert torch.equal(q8, qo) and torch.equal(k8, ko)
    want = cache.clone()
    want[slots // page, 0, slots % page] = ko.cpu().view(T, hk, D)
    want[slots // page, 1, slots % page] = v.reshape(T, hk, D)
    for st in (torch.int64, torch.int32):
        c = cache.to(gpu)
        q2, k2 = kvc.qk_norm_rotary_pos_emb_and_cache(dq, dk, dv, dqw, dkw, dpos, dcs, D, c, slots.to(gpu).to(st), EPS)
        assert torch.equal(q2, qo) and torch.equal(k2, ko) and torch.equal(c.cpu(), want)
    c = cache.to(gpu)
    _, none = kvc.qk_norm_rotary_pos_emb_and_cache(dq, dk, dv, dqw, dkw, dpos, dcs, D, c, slots.to(gpu), EPS, return_key=False)
    assert none is None and torch.equal(c.cpu(), want)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("shape", SHAPES)
def test_by_page_table_and_plan(gpu, shape, dtype):
    hq, hk, D, rd, page = shape
    lens = [1, 45, 17, 3]
    T = sum(lens)
    q, k, v, qw, kw, cs, _, _, _ = make(shape, dtype, T, seed=1)
    rng = np.random.default_rng(2)
    tables = [-(-n // page) for n in lens]
    nb = sum(tables) + 2
    ids = rng.permutation(nb)[:sum(tables)].astype(np.int32)
    indptr = np.cumsum([0] + tables).astype(np.int32)
    batch = np.repeat(np.arange(4), lens).astype(np.int32)
    pos = np.concatenate([np.arange(n) for n in lens]).astype(np.int32)
    slots = ids[indptr[batch] + pos // page].astype(np.int64) * page + pos % page
    last = np.array([(n - 1) % page + 1 for n in lens], np.int32)
    i = [torch.from_numpy(x).to(gpu) for x in (batch, pos, ids, indptr, last, slots)]
    cache = torch.zeros(nb, 2, page, hk, D, dtype=q.dtype, device=gpu)
    dq, dk, dv, dqw, dkw, dcs = (x.to(gpu) for x in (q, k, v, qw, kw, cs))
    by_slot = cache.clone()
    qo, ko = kvc.qk_norm_rotary_pos_emb_and_cache(dq, dk, dv, dqw, dkw, i[1], dcs, D, by_slot, i[5], EPS)
    check(qo, q, qw, torch.from_numpy(pos), cs, D, dtype)
    paged = cache.clone()
    q2, k2 = kvc.qk_norm_rotary_pos_emb_and_append_paged(dq, dk, dv, dqw, dkw, i[0], i[1], dcs, D, paged, i[2], i[3], i[4], EPS)
    assert torch.equal(q2, qo) and torch.equal(k2, ko) and torch.equal(paged, by_slot)
    for kw_plan in ({}, {"resolve_slots": True}, {"slots": i[5]}) if rd else ():    # (a plan takes a table)
        plan = kvc.PagedRotaryWritePlan(i[0], i[1], i[2], i[3], i[4], dcs, hq, hk, D, page, **kw_plan)
        c = cache.clone()
        q3, k3 = plan.run(dq, dk, dv, c, return_key=True, query_weight=dqw, key_weight=dkw, eps=EPS)
        assert torch.equal(q3, qo) and torch.equal(k3, ko) and torch.equal(c, by_slot)
        plain, _ = plan.run(dq, dk, dv, cache.clone())
        assert torch.equal(plain, kvc.rotary_pos_emb(dq, dk, i[1], dcs, D)[0])   # without weights: as before


@pytest.mark.parametrize("dtype", list(TYPES))
def test_unaligned_rows_tables_and_weights(gpu, dtype):
    shape = (8, 2, 128, 128, 16)
    q, k, v, qw, kw, cs, pos, slots, cache = make(shape, dtype, 33, off=1)
    D = 128
    wide = torch.zeros(33, 12 * D + 1, dtype=q.dtype, device=gpu)
    wide[:, 1:] = torch.cat((q, k, v), 1).to(gpu)
    odd = torch.empty(cs.numel() + 1, dtype=cs.dtype, device=gpu)
    odd[1:] = cs.flatten().to(gpu)
    weights = torch.empty(2 * D + 1, dtype=q.dtype, device=gpu)
    weights[1:] = torch.cat((qw, kw)).to(gpu)
    a, b = weights[1:1 + D], weights[1 + D:]
    for rows, table in ((wide[:, 1:], cs.to(gpu)), (torch.cat((q, k, v), 1).to(gpu), odd[1:].view(cs.shape))):
        c = cache.to(gpu)
        qo, ko = kvc.qk_norm_rotary_pos_emb_and_cache(rows[:, :8 * D], rows[:, 8 * D:10 * D], rows[:, 10 * D:], a, b, pos.to(gpu),
                                                      table, D, c, slots.to(gpu), EPS)
        check(qo, q, qw, pos, cs, D, dtype)
        check(ko, k, kw, pos, cs, D, dtype)
        assert torch.equal(c[slots.to(gpu) // 16, 1, slots.to(gpu) % 16].cpu().flatten(1), v)


def test_rows_of_zeros_large_rows_and_a_row_that_is_not_a_number(gpu):
    shape = (8, 2, 128, 128, 16)
    q, k, v, qw, kw, cs, pos, slots, cache = make(shape, "bf16", 5)
    q, k = q.clone(), k.clone()
    q[0] = 0
    q[1] = q[1] * 2.0 ** 60       # squares up to 2^125 or so: inside fp32's range
    q[2] = q[2] * 2.0 ** -60      # below eps: y = x w / sqrt(eps)
    q[3, :128] = float("nan")
    k[4, 128:] = float("inf")
    qo, ko = kvc.qk_norm_rotary_pos_emb(q.to(gpu), k.to(gpu), qw.to(gpu), kw.to(gpu), pos.to(gpu), cs.to(gpu), 128, EPS)
    assert (qo[0] == 0).all()
    check(qo[1:3], q[1:3], qw, pos[1:3], cs, 128, "bf16")
    assert torch.isnan(qo[3, :128]).all() and torch.isnan(ko[4, 128:]).all()
    check(qo[3:4, 128:], q[3:4, 128:], qw, pos[3:4], cs, 128, "bf16")
    check(ko[4:, :128], k[4:, :128], kw, pos[4:], cs, 128, "bf16")


@pytest.mark.parametrize("shape", [(8, 2, 128, 128, 16), (5, 1, 33, 22, 5)])
def test_in_place_and_skipped_tokens(gpu, shape):
    hq, hk, D, rd, page = shape
    q, k, v, qw, kw, cs, pos, slots, cache = make(shape, "bf16", 40, seed=3)
    dq, dk, dv, dqw, dkw, dcs = (x.to(gpu).contiguous() for x in (q, k, v, qw, kw, cs))
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=gpu)
    want_q, want_k = kvc.qk_norm_rotary_pos_emb(dq, dk, dqw, dkw, pos.to(gpu), dcs, D, EPS)
    plan = kvc.PagedRotaryWritePlan(i32([0] * 40), pos.to(gpu), i32([0]), i32([0, 1]), i32([1]), dcs, hq, hk, D, page,
                                    slots=slots.to(gpu))
    a, b, c = dq.clone(), dk.clone(), cache.to(gpu)
    plan.run(a, b, dv, c, query_out=a, key_out=b, query_weight=dqw, key_weight=dkw, eps=EPS)
    assert torch.equal(a, want_q) and torch.equal(b, want_k)
    # positions outside the table, slots outside the pool: nothing of the token is written
    bad = pos.clone()
    bad[3], bad[9] = -1, cs.shape[0]
    s = slots.clone()
    s[5], s[11] = -1, cache.shape[0] * page
    c = cache.to(gpu)
    kvc.qk_norm_rotary_pos_emb_and_cache(dq, dk, dv, dqw, dkw, bad.to(gpu), dcs, D, c, s.to(gpu), EPS)
    want = cache.clone()
    for t in range(40):
        if t not in (3, 5, 9, 11):
            want[slots[t] // page, 0, slots[t] % page] = want_k[t].cpu().view(hk, D)
            want[slots[t] // page, 1, slots[t] % page] = v[t].view(hk, D)
    assert torch.equal(c.cpu(), want)


def test_many_tokens_and_none(gpu):
    """More tokens than one dimension of a grid holds, and none at all."""
    shape = (2, 1, 64, 64, 16)
    q, k, v, qw, kw, cs, pos, slots, cache = make(shape, "bf16", 70001)
    qo, ko = kvc.qk_norm_rotary_pos_emb(q.to(gpu), k.to(gpu), qw.to(gpu), kw.to(gpu), pos.to(gpu), cs.to(gpu), 64, EPS)
    check(qo, q, qw, pos, cs, 64, "bf16")
    check(ko, k, kw, pos, cs, 64, "bf16")
    none, _ = kvc.qk_norm_rotary_pos_emb(q[:0].to(gpu), k[:0].to(gpu), qw.to(gpu), kw.to(gpu), pos[:0].to(gpu), cs.to(gpu), 64)
    assert none.shape == (0, 128)
    empty = torch.empty(0, 2, 16, 1, 64, dtype=q.dtype, device=gpu)
    q2, k2 = kvc.qk_norm_rotary_pos_emb_and_cache(q.to(gpu), k.to(gpu), v.to(gpu), qw.to(gpu), kw.to(gpu), pos.to(gpu),
                                                  cs.to(gpu), 64, empty, slots.to(gpu), EPS)
    assert torch.equal(q2, qo) and torch.equal(k2, ko)


def test_refusals(gpu):
    q, k, v, qw, kw, cs, pos, slots, cache = (x.to(gpu) for x in make((8, 2, 64, 64, 16), "bf16", 9))
    f = kvc.qk_norm_rotary_pos_emb
    with pytest.raises(TypeError, match="query_weight"):
        f(q, k, qw.float(), kw, pos, cs, 64)
    with pytest.raises(ValueError, match="key_weight"):
        f(q, k, qw, kw[:32], pos, cs, 64)
    for eps in (0.0, -1.0, float("nan"), float("inf")):
        with pytest.raises(ValueError, match="eps"):
            f(q, k, qw, kw, pos, cs, 64, eps)
    with pytest.raises(ValueError, match="GPU"):
        f(q, k, qw.cpu(), kw, pos, cs, 64)
    with pytest.raises(TypeError):
        f(q, k.half(), qw, kw, pos, cs, 64)
    with pytest.raises(ValueError, match="head_dim"):
        f(q, k, qw, kw, pos, cs, 60)
    g = kvc.qk_norm_rotary_pos_emb_and_cache
    with pytest.raises(ValueError, match="slot_mapping"):
        g(q, k, v, qw, kw, pos, cs, 64, cache, slots[:-1])
    with pytest.raises(TypeError):
        g(q, k, v.float(), qw, kw, pos, cs, 64, cache, slots)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=gpu)
    plan = kvc.PagedRotaryWritePlan(i32([0] * 9), pos, i32([0]), i32([0, 1]), i32([1]), cs, 8, 2, 64, 16, slots=slots)
    with pytest.raises(ValueError, match="together"):
        plan.run(q, k, v, cache, query_weight=qw)
    both = torch.zeros(9 * 8 * 64 + 64, dtype=q.dtype, device=gpu)
    with pytest.raises(ValueError, match="overlaps"):   # rows shifted against their own input
        plan.run(both[:9 * 512].view(9, 512), k, v, cache, query_out=both[64:].view(9, 512), query_weight=qw, key_weight=kw)
    with pytest.raises(ValueError, match="overlaps"):   # the key's rows are the cache's
        plan.run(q, cache.flatten()[:9 * 128].view(9, 128), v, cache, query_weight=qw, key_weight=kw)
