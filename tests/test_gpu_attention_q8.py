"""Attention over the 8-bit cache against the formula in 64 bits, on what the codes stand for. Every code that no request
owns is NaN: whatever reads beyond a request's keys shows."""
import numpy as np
import pytest
import torch

import lmserve_amd as kvc
from oracle import attention_oracle as ao
from oracle import q8_oracle as qo

pytestmark = pytest.mark.gpu

F8 = torch.float8_e4m3fn
# storage step of the outputs, of the weights in the product with V (f16, whatever the outputs are), half its smallest number
TYPES = {"bf16": (torch.bfloat16, 2.0 ** -7), "f16": (torch.float16, 2.0 ** -10)}
WEIGHT_EPS, DENORMAL = 2.0 ** -10, 2.0 ** -25


class Step:
    """A step's tensors: lengths = [(new tokens, keys)], the first `shared` pages of every table the same."""

    def __init__(self, lengths, heads, kv_heads, D, page, dtype="bf16", shared=0, seed=0, spare_rows=0, spread=2, k_size=0):
        self.rng = rng = np.random.default_rng(seed)
        self.dtype, self.eps = TYPES[dtype]
        self.page, self.H, self.Hq, self.D, self.shared = page, kv_heads, heads, D, shared
        tables = [-(-k // page) for _, k in lengths]
        own = [max(0, t - shared) for t in tables]
        P = shared + sum(own) + 2
        perm = rng.permutation(P)
        at, indices = shared, []
        for t, o in zip(tables, own):
            indices += [perm[:min(t, shared)], perm[at:at + o]]
            at += o
        self.indices = np.concatenate(indices).astype(np.int32) if indices else np.zeros(0, np.int32)
        self.indptr = np.cumsum([0] + tables).astype(np.int32)
        self.last = np.array([(k - 1) % page + 1 if k else 0 for _, k in lengths], np.int32)
        self.qo = np.cumsum([0] + [n for n, _ in lengths]).astype(np.int32)
        self.T = int(self.qo[-1]) + spare_rows
        raw = rng.integers(0, 256, (P * page // 16, qo.group_bytes(kv_heads, D)), dtype=np.uint8)
        c = self.cache = qo.Cache(raw.reshape(P, -1), kv_heads, D)
        c.codes[:] = 127
        # (of groups that no request owns: exponents of any size)
        c.exponents[:] = rng.integers(-100, 121, c.exponents.shape)
        done = np.zeros(P * page, bool)
        for b, (_, k) in enumerate(lengths):
            table = self.indices[self.indptr[b]:self.indptr[b + 1]].astype(np.int64)
            slots = (table[:, None] * page + np.arange(page)).ravel()[:k]
            slots = slots[~done[slots]]
            done[slots] = True
            x = rng.standard_normal((len(slots), 2, kv_heads, D))
            c.codes[slots] = qo.encode(x * 64)
            groups = np.unique(slots // 16)
            c.exponents[groups] = rng.integers(-spread, spread + 1, (len(groups), kv_heads, 2)) - 6
            c.exponents[groups, :, 0] += k_size
        self.query = torch.from_numpy(rng.standard_normal((self.T, heads, D)).astype(np.float32)).to(self.dtype)
        self.scale = D ** -0.5

    def pages(self, dev):
        return torch.from_numpy(self.cache.pages()).to(dev)

    def index(self, dev):
        return [torch.from_numpy(x).to(dev) for x in (self.qo, self.indices, self.indptr, self.last)]

    def plan(self, dev, **kw):
        kw.setdefault("shared_pages", self.shared)
        kw.setdefault("num_tokens", self.T)
        return kvc.PagedAttentionPlan(*self.index(dev), self.Hq, self.H, self.D, self.page, self.dtype, kv_dtype=F8, **kw)

    def oracle(self):
        P = self.cache.shape[0]
        values = self.cache.values().reshape(P, self.page, 2, self.H, self.D).transpose(0, 2, 1, 3, 4)
        return ao.paged_attention_f64(self.query.double().numpy(), values, self.qo, self.indices, self.indptr, self.last, self.scale)

    def check(self, out, lse=None, rows=None):
        """Outputs within the weights' rounding (half a step of f16, times the values' sizes), the arithmetic's and the outputs' own."""
        want, want_lse, *bounds = self.oracle()
        tol, tol_lse = ao.attention_tolerances(want, want_lse, *bounds, self.D, self.scale, WEIGHT_EPS, DENORMAL)
        tol = tol + np.abs(want) * (self.eps - WEIGHT_EPS) / 2 * 1.05
        got = out.detach().cpu().double().numpy().reshape(want.shape)
        rows = slice(0, int(self.qo[-1])) if rows is None else rows
        a, b = got[rows], want[rows]
        assert np.array_equal(np.isnan(a), np.isnan(b)), f"{np.isnan(a).sum()} NaN and not {np.isnan(b).sum()}"
        fine = ~np.isnan(b)
        err = np.abs(a - b)[fine] / tol[rows][fine]
        assert (err <= 1).all(), f"off by {err.max():.3g} of the bound"
        if lse is not None:
            a, b = lse.cpu().double().numpy()[rows], want_lse[rows]
            assert np.array_equal(np.isneginf(a), np.isneginf(b)) and np.array_equal(np.isnan(a), np.isnan(b))
            fine = np.isfinite(b)
            assert (np.abs(a - b)[fine] <= tol_lse[rows][fine]).all(), f"lse off by {np.abs(a - b)[fine].max():.3g}"


GEOMETRIES = [(8, 2, 128, 16), (32, 8, 64, 16), (7, 1, 128, 32), (4, 4, 80, 16), (6, 2, 96, 48), (2, 1, 256, 32), (3, 1, 16, 16),
              (16, 1, 48, 16), (40, 2, 64, 64), (5, 5, 144, 16)]


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("heads,kv_heads,D,page", GEOMETRIES)
def test_single_tokens(gpu, heads, kv_heads, D, page, dtype):
    s = Step([(1, 1), (1, 33), (1, 2), (1, 500), (1, page), (1, page + 1), (1, 129), (1, 64), (1, 1500)], heads, kv_heads, D, page, dtype)
    out, lse = s.plan(gpu).run(s.query.to(gpu), s.pages(gpu), return_lse=True)
    s.check(out, lse)
    again = kvc.paged_attention(s.query.to(gpu), s.pages(gpu), *s.index(gpu), max_q_len=1, num_kv_heads=kv_heads)
    assert again.shape == out.shape and torch.equal(again, out)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("heads,kv_heads,D,page", GEOMETRIES)
def test_chunks_and_single_tokens(gpu, heads, kv_heads, D, page, dtype):
    s = Step([(70, 70), (33, 161), (1, 40), (5, 5), (2, 300), (1, 1), (40, 600)], heads, kv_heads, D, page, dtype, seed=1)
    out, lse = s.plan(gpu).run(s.query.to(gpu), s.pages(gpu), return_lse=True)
    s.check(out, lse)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("heads,kv_heads,D,page", GEOMETRIES)
def test_shared_prefix(gpu, heads, kv_heads, D, page, dtype):
    shared = max(1, 200 // page)
    base = shared * page
    s = Step([(1, base + 1), (1, base + 90), (3, base + 40), (1, base), (1, base + 3), (40, base + 77), (2, base + 2)] +
             [(1, base + 5 * i + 1) for i in range(12)], heads, kv_heads, D, page, dtype, shared=shared, seed=2)
    out, lse = s.plan(gpu).run(s.query.to(gpu), s.pages(gpu), return_lse=True)
    s.check(out, lse)


@pytest.mark.parametrize("shared", [0, 2])
def test_no_keys_no_tokens_and_rows_behind_the_last_request(gpu, shared):
    s = Step([(1, 40), (0, 50), (2, 0), (0, 0), (5, 3), (1, 33)], 8, 2, 64, 16, seed=5, spare_rows=6)
    out = torch.full((s.T, 8, 64), 7.0, dtype=torch.bfloat16, device=gpu)
    lse = torch.full((s.T, 8), 7.0, device=gpu)
    s.plan(gpu, shared_pages=shared).run(s.query.to(gpu), s.pages(gpu), out=out, lse=lse)
    s.check(out, lse)
    n = int(s.qo[-1])
    assert (out[n:] == 7).all() and (lse[n:] == 7).all()
    assert (out[1:5] == 0).all() and torch.isneginf(lse[1:5]).all()


def test_pages_outside_the_cache_have_no_keys(gpu):
    s = Step([(1, 100), (40, 200), (1, 16)], 8, 2, 64, 16, seed=6)
    s.indices = s.indices.copy()
    s.indices[[0, 3, 8, 12]] = [-1, 1 << 30, s.cache.shape[0], -(1 << 31)]
    s.indices[-1] = -5           # all that the last request has
    out, lse = s.plan(gpu).run(s.query.to(gpu), s.pages(gpu), return_lse=True)
    s.check(out, lse)
    assert (out[-1] == 0).all()


@pytest.mark.parametrize("heads,kv_heads,D", [(8, 2, 128), (4, 1, 80), (2, 2, 256), (6, 3, 64)])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_groups_of_very_different_sizes(gpu, heads, kv_heads, D, dtype):
    """Exponents of K and V that differ by 2^20 within what one row sees, growing and falling along the keys; groups of zeros."""
    s = Step([(1, 700), (60, 700), (3, 90), (1, 40), (1, 16)], heads, kv_heads, D, 16, dtype, seed=7, spread=0)
    c = s.cache
    c.exponents[..., 1] = s.rng.integers(-20, 1, c.exponents.shape[:2])
    c.exponents[..., 0] = s.rng.integers(-16, -4, c.exponents.shape[:2])
    codes = c.codes.reshape(-1, 16, 2, kv_heads, D)
    first = s.indices[s.indptr[3]]
    codes[first] = 0             # a request whose first keys are zeros, with the exponents that the write gives them
    c.exponents[first] = qo.LEAST
    alone = s.indices[s.indptr[4]]
    codes[alone, :, 1] = 0
    c.exponents[alone, :, 1] = qo.LEAST
    out, lse = s.plan(gpu).run(s.query.to(gpu), s.pages(gpu), return_lse=True)
    s.check(out, lse)


@pytest.mark.parametrize("exponent", [-90, -40, 40, 100])
def test_values_near_the_ends_of_the_range(gpu, exponent):
    """V at 2^exponent (out of f16's range, so bf16 outputs), K small enough for scores below 2^24."""
    s = Step([(1, 300), (40, 200), (2, 17)], 4, 2, 64, 16, "bf16", seed=8, spread=0)
    s.cache.exponents[..., 1] = exponent
    out, lse = s.plan(gpu).run(s.query.to(gpu), s.pages(gpu), return_lse=True)
    s.check(out, lse)


@pytest.mark.parametrize("size", [3, 8])
def test_large_scores(gpu, size):
    s = Step([(1, 900), (50, 300), (1, 64), (4, 70)], 8, 2, 128, 16, "bf16", seed=9, k_size=size)
    out, lse = s.plan(gpu).run(s.query.to(gpu), s.pages(gpu), return_lse=True)
    s.check(out, lse)


@pytest.mark.parametrize("lengths", [[(1, 130), (3, 100), (1, 16)], [(50, 130), (200, 333)], [(1, 50), (40, 40), (17, 100)]])
@pytest.mark.parametrize("D", [64, 80, 256])
def test_nan_reaches_the_rows_that_see_it(gpu, lengths, D):
    """NaN codes among the keys: of V it makes its column NaN, of K the whole row, in the rows that see that key alone."""
    for plane in (1, 0):
        s = Step(lengths, 4, 2, D, 16, seed=10 + plane)
        for b, (n, k) in enumerate(lengths):
            # (one in a key makes whole rows NaN: only where the later rows see it)
            for at in {k - 1, max(0, k - n // 2 - 1)} if plane == 0 else {k - 1, max(0, k - n // 2 - 1), max(0, k - n), k // 3}:
                slot = int(s.indices[s.indptr[b] + at // 16]) * 16 + at % 16
                s.cache.codes[slot, plane, s.rng.integers(2), s.rng.integers(D, size=2)] = s.rng.choice([127, 255])
        nan = np.isnan(s.oracle()[0])
        assert nan.any() and not nan.all()
        out, lse = s.plan(gpu).run(s.query.to(gpu), s.pages(gpu), return_lse=True)
        s.check(out, lse)


def test_long_contexts_are_cut_and_joined(gpu):
    """Few rows over many keys, a workgroup a part, and wide tiles cut into ranges."""
    for lengths, heads, kv_heads, D in (([(1, 40001)], 8, 1, 128), ([(2, 5000), (1, 9000)], 4, 1, 64), ([(130, 6000)], 2, 1, 128), ([(64, 3000), (40, 9001)], 2, 2, 64)):
        s = Step(lengths, heads, kv_heads, D, 16, seed=11)
        out, lse = s.plan(gpu).run(s.query.to(gpu), s.pages(gpu), return_lse=True)
        s.check(out, lse)
        assert torch.equal(out, s.plan(gpu).run(s.query.to(gpu), s.pages(gpu)))


def test_many_requests(gpu):
    rng = np.random.default_rng(12)
    s = Step([(1, int(k)) for k in rng.integers(1, 200, 1500)], 4, 1, 64, 16, seed=12)
    out, lse = s.plan(gpu, max_q_len=1).run(s.query.to(gpu), s.pages(gpu), return_lse=True)
    s.check(out, lse)


def test_a_layer_of_a_large_pool(gpu):
    """Pages apart from one another, beyond 2^32 bytes; queries that are slices of a projection; the output in the query's place."""
    s = Step([(1, 100), (30, 90), (1, 33)], 8, 2, 128, 16, seed=13)
    n, page = s.cache.shape
    pool = torch.empty(40, 12000, page + 64 * 16, dtype=torch.uint8, device=gpu)
    ids = np.random.default_rng(0).permutation(12000)[:n]
    layer = pool[39][:, :page]
    layer[torch.from_numpy(ids).to(gpu)] = s.pages(gpu)
    index = s.index(gpu)
    index[1] = torch.from_numpy(ids[s.indices].astype(np.int32)).to(gpu)
    plan = kvc.PagedAttentionPlan(*index, 8, 2, 128, 16, s.dtype, s.T, kv_dtype=F8)
    wide = torch.empty(s.T, 12 * 128, dtype=s.dtype, device=gpu)
    wide[:, :1024] = s.query.flatten(1).to(gpu)
    out = plan.run(wide[:, :1024], layer)
    assert out.shape == (s.T, 1024)
    s.check(out)
    q = s.query.to(gpu)
    assert plan.run(q, layer, out=q) is q and torch.equal(q.flatten(1), out)


def test_recorded_steps_and_streams(gpu):
    """A plan of capacities, built and run in a graph that is replayed for other steps; the same plan on another stream."""
    big = Step([(1, 200), (40, 150), (1, 90), (3, 70)], 8, 2, 64, 16, seed=14, spare_rows=20)
    index, pages, q = big.index(gpu), big.pages(gpu), big.query.to(gpu)
    plan = kvc.PagedAttentionPlan(*index, 8, 2, 64, 16, big.dtype, big.T, kv_dtype=F8)
    out = torch.zeros_like(q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        plan.build()
        plan.run(q, pages, out=out)
    torch.cuda.synchronize()
    big.check(out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        plan.build()
        plan.run(q, pages, out=out)
    for i in range(4):
        # another step of the same capacities: other lengths over the same tables
        last = np.array([1 + (3 * i) % 16, 1 + (5 * i) % 16, 16 - i, 2 + i], np.int32)
        qo = np.cumsum([0, 1 + i, 40 - 9 * i, 1, 2]).astype(np.int32)
        big.last, big.qo = last, qo
        big.query = torch.from_numpy(np.random.default_rng(i).standard_normal((big.T, 8, 64)).astype(np.float32)).to(big.dtype)
        # every place of the tables is a key in one step or another
        table_slots = (big.indices.astype(np.int64)[:, None] * 16 + np.arange(16)).ravel()
        c = big.cache.codes[table_slots]
        big.cache.codes[table_slots] = np.where((c & 127) == 127, np.uint8(40 + i), c)
        index[0].copy_(torch.from_numpy(qo)), index[3].copy_(torch.from_numpy(last)), q.copy_(big.query)
        pages.copy_(big.pages(gpu))
        big.cache.exponents[:] = np.clip(big.cache.exponents, -8, -4)
        pages.copy_(big.pages(gpu))
        out.fill_(7)
        graph.replay()
        torch.cuda.synchronize()
        big.check(out)
        assert (out[int(qo[-1]):] == 7).all()


def test_refusals(gpu):
    s = Step([(1, 40)], 4, 2, 64, 16)
    q, pages, index = s.query.to(gpu), s.pages(gpu), s.index(gpu)
    plan = s.plan(gpu)
    with pytest.raises(TypeError):
        plan.run(q, torch.zeros(3, 2, 16, 2, 64, dtype=s.dtype, device=gpu))
    with pytest.raises(ValueError):
        plan.run(q, pages[:, :-16])
    with pytest.raises(ValueError):
        plan.run(q, torch.zeros(3, 2 * pages.shape[1], dtype=torch.uint8, device=gpu))
    with pytest.raises(TypeError):
        plan.run(q.half(), pages)
    with pytest.raises(ValueError, match="overlaps"):
        plan.run(q, pages, out=pages.view(s.dtype)[0, :256].view(1, 4, 64))
    for bad in (torch.float8_e5m2, torch.uint8, torch.float16):
        with pytest.raises(TypeError):
            kvc.PagedAttentionPlan(*index, 4, 2, 64, 16, s.dtype, 1, kv_dtype=bad)
    for D, page in ((72, 16), (64, 24), (272, 16)):
        with pytest.raises(TypeError):
            kvc.PagedAttentionPlan(*index, 4, 2, D, page, s.dtype, 1, kv_dtype=F8)
    with pytest.raises(ValueError):
        kvc.paged_attention(q, pages, *index)
    with pytest.raises(ValueError):
        kvc.paged_attention(q.flatten(1), pages, *index, num_kv_heads=2)
    wide = kvc.PagedAttentionPlan(*index, 4, 2, 64, 16, s.dtype, 1, kv_dtype=s.dtype)
    with pytest.raises(TypeError):
        wide.run(q, pages)


def test_one_plan_on_two_streams_at_once(gpu):
    """Every run has a workspace of its own."""
    s = Step([(1, 3000), (40, 900), (1, 700)], 8, 2, 128, 16, seed=21)
    plan, pages = s.plan(gpu), s.pages(gpu)
    q = [s.query.to(gpu), (s.query * 2).to(gpu)]
    want = [plan.run(x, pages) for x in q]
    s.check(want[0])
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(4):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(plan.run(q[i], pages))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])


def test_write_then_attend(gpu):
    """A prompt in chunks and single tokens, written and attended to through the eager calls, on what the write left."""
    H, HQ, D, page = 2, 8, 128, 32
    rng = np.random.default_rng(22)
    pool = kvc.allocate_q8_kv_caches(1, 20, page, H, D, gpu)[0].fill_(127)
    table = rng.permutation(20)[:10].astype(np.int32)
    i32 = dict(dtype=torch.int32, device=gpu)
    have = 0
    for new in (150, 1, 1, 33, 1, 14):
        k, v = (torch.from_numpy(rng.standard_normal((new, H, D)).astype(np.float32)).to(torch.bfloat16).to(gpu) for _ in range(2))
        q = torch.from_numpy(rng.standard_normal((new, HQ, D)).astype(np.float32)).to(torch.bfloat16).to(gpu)
        positions = torch.arange(have, have + new, **i32)
        have += new
        pages = -(-have // page)
        index = [torch.from_numpy(table[:pages]).to(gpu), torch.tensor([0, pages], **i32), torch.tensor([(have - 1) % page + 1], **i32)]
        kvc.append_paged_kv_cache_q8(k, v, torch.zeros(new, **i32), positions, pool, *index)
        out, lse = kvc.paged_attention(q, pool, torch.tensor([0, new], **i32), *index, return_lse=True, num_kv_heads=H)
        s = Step.__new__(Step)
        s.page, s.H, s.Hq, s.D, s.eps = page, H, HQ, D, 2.0 ** -7
        s.cache, s.query, s.scale = qo.Cache(pool.cpu().numpy(), H, D), q.cpu(), D ** -0.5
        s.qo, s.indices, s.indptr, s.last = np.array([0, new]), table[:pages], np.array([0, pages]), np.array([(have - 1) % page + 1])
        s.check(out, lse)
        # the rows that come back are those that were attended to
        bk, bv = kvc.read_paged_kv_cache_q8(torch.zeros(new, **i32), positions, pool, *index, H, D)
        assert (bk - k).abs().max() < 0.3 and (bv - v).abs().max() < 0.3


@pytest.mark.parametrize("lengths", [[(1, 100), (3, 40), (1, 16)], [(60, 200), (40, 40)]])
@pytest.mark.parametrize("scale,exponent", [(2.0 ** -60, -100), (1e-30, -100), (2.0 ** -120, 0), (2.0 ** -26, -100), (400.0, 120), (3e5, 118), (1e30, 100)])
def test_scales_of_any_size(gpu, lengths, scale, exponent):
    """A softmax scale whose product with a group's 2^e is no normal fp32. The small ones: groups of zeros among keys whose scores are then equal;
    the large ones: keys that lie in a column that the queries do not have, scores of 0."""
    s = Step(lengths, 4, 2, 64, 16, seed=23, spread=0)
    c = s.cache
    groups = np.unique(s.indices)[::2]
    by_group = c.codes.reshape(-1, 16, 2, 2, 64)
    if scale < 1:
        by_group[groups, :, 0] = 0
    else:
        s.query[..., 5] = 0
        there = (by_group[:, :, 0] & 127) != 127
        by_group[:, :, 0] = np.where(there, 0, by_group[:, :, 0])
        by_group[:, :, 0, :, 5] = np.where(there[..., 5], 120, by_group[:, :, 0, :, 5])
    c.exponents[groups, :, 0] = exponent
    s.scale = scale
    out, lse = s.plan(gpu, sm_scale=scale).run(s.query.to(gpu), s.pages(gpu), return_lse=True)
    s.check(out, lse)
