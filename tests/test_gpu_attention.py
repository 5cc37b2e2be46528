"""Attention over the paged cache against the formula in 64 bits. Everything the cache holds and no request owns is NaN:
whatever reads beyond a request's keys shows."""
import numpy as np
import pytest
import torch

import lmserve_amd as kvc
from lmserve_amd import _lib
from oracle import attention_oracle as ao

pytestmark = pytest.mark.gpu

TYPES = {"bf16": (torch.bfloat16, 2.0 ** -7, 0.0), "f16": (torch.float16, 2.0 ** -10, 2.0 ** -25)}


class Step:
    """A step's tensors: lengths = [(new tokens, keys)], the first `shared` pages of every table the same."""

    def __init__(self, lengths, heads, kv_heads, D, page, dtype="bf16", shared=0, seed=0, spare_rows=0, scale_q=1.0):
        rng = np.random.default_rng(seed)
        self.dtype, self.eps, self.denormal = TYPES[dtype]
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
        cache = np.full((P, 2, page, kv_heads, D), np.nan, np.float32)
        for b, (_, k) in enumerate(lengths):
            for i, p in enumerate(self.indices[self.indptr[b]:self.indptr[b + 1]]):
                used = min(page, k - i * page)
                if used > 0 and np.isnan(cache[p, :, :used]).any():
                    cache[p, :, :used] = rng.standard_normal((2, used, kv_heads, D))
        self.cache = torch.from_numpy(cache).to(self.dtype)
        self.query = (torch.from_numpy(rng.standard_normal((self.T, heads, D)).astype(np.float32)) * scale_q).to(self.dtype)
        self.scale = D ** -0.5

    def index(self, dev):
        return [torch.from_numpy(x).to(dev) for x in (self.qo, self.indices, self.indptr, self.last)]

    def plan(self, dev, **kw):
        kw.setdefault("shared_pages", self.shared)
        kw.setdefault("num_tokens", self.T)
        return kvc.PagedAttentionPlan(*self.index(dev), self.Hq, self.H, self.D, self.page, self.dtype, **kw)

    def oracle(self):
        return ao.paged_attention_f64(self.query.double().numpy(), self.cache.double().numpy(), self.qo, self.indices,
                                      self.indptr, self.last, self.scale)

    def check(self, out, lse=None, rows=None):
        want, want_lse, *bounds = self.oracle()
        tol, tol_lse = ao.attention_tolerances(want, want_lse, *bounds, self.D, self.scale, self.eps, self.denormal)
        got = out.detach().cpu().double().numpy().reshape(want.shape)
        rows = slice(0, int(self.qo[-1])) if rows is None else rows
        err = np.abs(got - want)[rows]
        assert (err <= tol[rows]).all(), f"off by {np.nanmax(err / tol[rows]):.3g} of the bound, NaN {np.isnan(err).sum()}"
        if lse is not None:
            a, b = lse.cpu().double().numpy()[rows], want_lse[rows]
            assert (np.isneginf(a) == np.isneginf(b)).all()
            fin = np.isfinite(b)
            assert (np.abs(a - b)[fin] <= tol_lse[rows][fin]).all(), f"lse off by {np.abs(a - b)[fin].max():.3g}"


GEOMETRIES = [(8, 2, 128, 16), (32, 8, 64, 16), (7, 1, 128, 16), (4, 4, 80, 20), (6, 2, 96, 8), (2, 1, 256, 32), (3, 1, 8, 1),
              (16, 1, 40, 5), (40, 2, 64, 64), (5, 5, 24, 16)]


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("heads,kv_heads,D,page", GEOMETRIES)
def test_single_tokens(gpu, heads, kv_heads, D, page, dtype):
    s = Step([(1, 1), (1, 33), (1, 2), (1, 500), (1, page), (1, page + 1), (1, 129)], heads, kv_heads, D, page, dtype)
    out, lse = s.plan(gpu).run(s.query.to(gpu), s.cache.to(gpu), return_lse=True)
    s.check(out, lse)
    again = kvc.paged_attention(s.query.to(gpu).flatten(1), s.cache.to(gpu), *s.index(gpu), max_q_len=1)
    assert again.shape == (s.T, heads * D) and torch.equal(again.view_as(out), out)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("heads,kv_heads,D,page", GEOMETRIES)
def test_chunks_and_single_tokens(gpu, heads, kv_heads, D, page, dtype):
    s = Step([(70, 70), (33, 161), (1, 40), (5, 5), (2, 300), (1, 1)], heads, kv_heads, D, page, dtype, seed=1)
    out, lse = s.plan(gpu).run(s.query.to(gpu), s.cache.to(gpu), return_lse=True)
    s.check(out, lse)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("heads,kv_heads,D,page", GEOMETRIES)
def test_shared_prefix(gpu, heads, kv_heads, D, page, dtype):
    shared = max(1, 200 // page)
    base = shared * page
    s = Step([(1, base + 1), (1, base + 90), (3, base + 40), (1, base), (1, base + 3), (40, base + 77), (2, base + 2)] +
             [(1, base + 5 * i + 1) for i in range(12)], heads, kv_heads, D, page, dtype, shared=shared, seed=2)
    out, lse = s.plan(gpu).run(s.query.to(gpu), s.cache.to(gpu), return_lse=True)
    s.check(out, lse)


def test_rows_of_the_prefix_stop_inside_it(gpu):
    """Requests whose own tokens lie in the shared pages see them up to their position only."""
    s = Step([(30, 64), (1, 50), (20, 70), (5, 64)], 8, 2, 64, 16, shared=4, seed=3)
    out, lse = s.plan(gpu).run(s.query.to(gpu), s.cache.to(gpu), return_lse=True)
    s.check(out, lse)


def test_requests_that_begin_with_other_pages_are_computed_by_themselves(gpu):
    s = Step([(1, 80), (1, 90), (1, 100), (4, 85)], 8, 2, 64, 16, shared=4, seed=4)
    other = Step([(1, 80), (1, 90), (1, 100), (4, 85)], 8, 2, 64, 16, shared=0, seed=4)
    out = other.plan(gpu, shared_pages=4).run(other.query.to(gpu), other.cache.to(gpu))
    other.check(out)
    # one request of four begins with a page of its own
    cache = torch.cat((s.cache, s.cache[s.indices[:1]]))
    s.cache = cache
    s.indices = s.indices.copy()
    s.indices[s.indptr[2]] = cache.shape[0] - 1
    s.check(s.plan(gpu).run(s.query.to(gpu), s.cache.to(gpu)))
    # fewer pages than are said to be shared, and more than there are
    for pages in (1, 5, 6, 7, 10 ** 6):
        s.check(s.plan(gpu, shared_pages=pages).run(s.query.to(gpu), s.cache.to(gpu)))


@pytest.mark.parametrize("shared", [0, 2])
def test_no_keys_no_tokens_and_rows_behind_the_last_request(gpu, shared):
    """Requests without pages, without tokens, with more tokens than keys; buffers longer than the step."""
    s = Step([(1, 40), (0, 50), (2, 0), (0, 0), (5, 3), (1, 33)], 8, 2, 64, 16, shared=0, seed=5, spare_rows=6)
    out = torch.full((s.T, 8, 64), 7.0, dtype=torch.bfloat16, device=gpu)
    lse = torch.full((s.T, 8), 7.0, device=gpu)
    s.plan(gpu, shared_pages=shared).run(s.query.to(gpu), s.cache.to(gpu), out=out, lse=lse)
    s.check(out, lse)
    n = int(s.qo[-1])
    assert (out[n:] == 7).all() and (lse[n:] == 7).all()
    rows = [1, 2]        # of the request without pages
    assert (out[rows] == 0).all() and torch.isneginf(lse[rows]).all()
    assert (out[3:5] == 0).all()      # tokens before the first key


def test_pages_outside_the_cache_have_no_keys(gpu):
    s = Step([(1, 70), (3, 100), (1, 16)], 8, 2, 128, 16, seed=6)
    s.indices = s.indices.copy()
    s.indices[1], s.indices[6], s.indices[-1] = -1, s.cache.shape[0], 1 << 30
    out, lse = s.plan(gpu).run(s.query.to(gpu), s.cache.to(gpu), return_lse=True)
    s.check(out, lse)
    assert (out[4] == 0).all() and torch.isneginf(lse[4]).all()


@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("new", [3, 24, 150])
def test_masked_keys_and_values_do_not_reach_the_result(gpu, bad, new):
    """The last keys of a chunk are infinite or NaN: the tokens before them do not see them."""
    s = Step([(new, 2 * new + 60), (1, 33)], 8, 2, 128, 16, seed=7)
    clean = s.oracle()
    length = 2 * new + 60
    page, at = s.indices[(length - 2) // 16], (length - 2) % 16
    s.cache[page, 1, at] = bad
    s.cache[page, 0, at, :, 3] = float("nan")
    out, lse = s.plan(gpu).run(s.query.to(gpu), s.cache.to(gpu), return_lse=True)
    got = out.cpu().double().numpy()
    want, want_lse, *bounds = clean
    tol, _ = ao.attention_tolerances(want, want_lse, *bounds, s.D, s.scale, s.eps, s.denormal)
    keep = [t for t in range(s.T) if t not in (new - 2, new - 1)]
    assert (np.abs(got - want)[keep] <= tol[keep]).all()
    assert np.isnan(got[[new - 2, new - 1]]).all() and torch.isnan(lse[new - 2:new]).all()   # the key's NaN is theirs
    # a value alone, in a few columns: the tokens that see it have it in those columns
    s.cache[page, 0, at] = torch.randn(2, 128).to(torch.bfloat16)
    s.cache[page, 1, at] = 1.0
    s.cache[page, 1, at, :, 5::17] = bad
    out = s.plan(gpu).run(s.query.to(gpu), s.cache.to(gpu)).cpu().double().numpy()
    assert (np.abs(out - want)[keep] <= tol[keep]).all()
    cols = np.zeros(128, bool)
    cols[5::17] = True
    assert np.isfinite(out[new - 2:new][:, :, ~cols]).all()
    assert (np.isnan(out[new - 2:new][:, :, cols]) if np.isnan(bad) else out[new - 2:new][:, :, cols] == bad).all()


def test_large_scores(gpu):
    """Scores of some thousands: one key takes all the weight, in whichever block it lies."""
    s = Step([(1, 700), (40, 333)], 8, 2, 128, 16, seed=8, scale_q=64.0)
    out, lse = s.plan(gpu).run(s.query.to(gpu), s.cache.to(gpu), return_lse=True)
    s.check(out, lse)


def test_strided_queries_and_caches(gpu):
    """Slices of a fused projection, rows that start off 16 bytes, one layer of a pool kept block by block."""
    s = Step([(1, 90), (17, 40)], 8, 2, 64, 16, seed=9)
    q, cache = s.query.to(gpu), s.cache.to(gpu)
    want = s.plan(gpu).run(q, cache)
    s.check(want)
    wide = torch.zeros(s.T, 12 * 64, dtype=q.dtype, device=gpu)
    wide[:, :8 * 64] = q.flatten(1)
    assert torch.equal(s.plan(gpu).run(wide[:, :8 * 64], cache), want.flatten(1))
    odd = torch.zeros(s.T, 8 * 64 + 3, dtype=q.dtype, device=gpu)
    odd[:, 3:] = q.flatten(1)
    assert torch.equal(s.plan(gpu).run(odd[:, 3:], cache), want.flatten(1))
    pool = torch.full((cache.shape[0], 3) + cache.shape[1:], float("nan"), dtype=q.dtype, device=gpu)
    pool[:, 1] = cache
    assert torch.equal(s.plan(gpu).run(q, pool[:, 1]), want)


def test_a_long_context_is_split_and_joined(gpu):
    """One request over many workgroups; its keys also beyond 2^31 bytes into the cache."""
    s = Step([(1, 20011), (2, 1700)], 4, 1, 128, 16, seed=10)
    out, lse = s.plan(gpu).run(s.query.to(gpu), s.cache.to(gpu), return_lse=True)
    s.check(out, lse)
    P = s.cache.shape[0]
    far = (1 << 32) // (2 * 16 * 128 * 2) + 5
    big = torch.empty((far + P, 2, 16, 1, 128), dtype=s.dtype, device=gpu)
    big[far:] = s.cache.to(gpu)
    s.indices = s.indices + far
    moved, moved_lse = s.plan(gpu).run(s.query.to(gpu), big, return_lse=True)
    assert torch.equal(moved, out) and torch.equal(moved_lse, lse)


def test_many_requests(gpu):
    """More requests than the layout takes in one pass of its scan."""
    rng = np.random.default_rng(11)
    lengths = [(int(rng.integers(0, 3)), int(rng.integers(0, 20))) for _ in range(2500)]
    s = Step(lengths, 2, 1, 16, 4, seed=11)
    out, lse = s.plan(gpu).run(s.query.to(gpu), s.cache.to(gpu), return_lse=True)
    s.check(out, lse)


def test_the_same_call_twice_gives_the_same_bits(gpu):
    s = Step([(1, 5000), (1, 1200), (60, 400)] + [(1, 300)] * 20, 8, 2, 128, 16, shared=10, seed=12)
    plan = s.plan(gpu)
    q, cache = s.query.to(gpu), s.cache.to(gpu)
    first = plan.run(q, cache)
    for _ in range(5):
        plan.build()
        assert torch.equal(plan.run(q, cache), first)


def test_on_another_stream_and_two_at_once(gpu):
    s = Step([(1, 900), (1, 1200), (60, 400)], 8, 2, 128, 16, seed=13)
    q, cache = s.query.to(gpu), s.cache.to(gpu)
    plan = s.plan(gpu)
    want = plan.run(q, cache)
    s.check(want)
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(10):
        for st in streams:
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                got.append(plan.run(q, cache))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)


def test_refusals(gpu):
    s = Step([(1, 40), (2, 20)], 8, 2, 64, 16)
    q, cache = s.query.to(gpu), s.cache.to(gpu)
    idx = s.index(gpu)
    plan = s.plan(gpu)
    with pytest.raises(ValueError, match="multiple"):
        kvc.PagedAttentionPlan(*idx, 7, 2, 64, 16, torch.bfloat16, num_tokens=3)
    with pytest.raises(TypeError, match="head_dim"):
        kvc.PagedAttentionPlan(*idx, 8, 2, 60, 16, torch.bfloat16, num_tokens=3)
    with pytest.raises(TypeError, match="head_dim"):
        kvc.PagedAttentionPlan(*idx, 8, 2, 264, 16, torch.bfloat16, num_tokens=3)
    with pytest.raises(TypeError):
        kvc.PagedAttentionPlan(*idx, 8, 2, 64, 16, torch.float32, num_tokens=3)
    with pytest.raises(TypeError):
        kvc.PagedAttentionPlan(*idx, 8, 2, 64, 16, torch.int8, num_tokens=3)
    with pytest.raises(TypeError, match="int32"):
        kvc.PagedAttentionPlan(idx[0].long(), *idx[1:], 8, 2, 64, 16, torch.bfloat16, num_tokens=3)
    with pytest.raises(ValueError, match="batch_size"):
        kvc.PagedAttentionPlan(idx[0][:-1], *idx[1:], 8, 2, 64, 16, torch.bfloat16, num_tokens=3)
    with pytest.raises(ValueError, match="scale"):
        kvc.PagedAttentionPlan(*idx, 8, 2, 64, 16, torch.bfloat16, num_tokens=3, sm_scale=0.0)
    with pytest.raises(ValueError, match="scale"):
        kvc.PagedAttentionPlan(*idx, 8, 2, 64, 16, torch.bfloat16, num_tokens=3, sm_scale=float("inf"))
    with pytest.raises(ValueError, match="kv_layout"):
        kvc.PagedAttentionPlan(*idx, 8, 2, 64, 16, torch.bfloat16, num_tokens=3, kv_layout="HND")
    with pytest.raises(ValueError):
        plan.run(q[:2], cache)
    with pytest.raises(TypeError):
        plan.run(q.half(), cache)
    with pytest.raises(ValueError):
        plan.run(q, cache[..., :32])
    with pytest.raises(ValueError):
        plan.run(q, cache.transpose(2, 3))
    with pytest.raises(ValueError):
        plan.run(q, cache, out=torch.empty(3, 8 * 64, dtype=torch.bfloat16, device=gpu)[:2])
    with pytest.raises(ValueError, match="lse"):
        plan.run(q, cache, lse=torch.empty(3, 7, device=gpu))
    with pytest.raises(ValueError, match="GPU"):
        plan.run(q.cpu(), cache)
    with pytest.raises(ValueError, match="aligned"):
        flat = torch.empty(cache.numel() + 1, dtype=cache.dtype, device=gpu)
        plan.run(q, flat[1:].view(cache.shape))
