"""Head norms, rotation, K/V write and attention as a model's layers use them: one after another over one step's index
tensors, eager and recorded into a hipGraph that later steps replay."""
import numpy as np
import pytest
import torch

import lmserve_amd as kvc
from oracle import attention_oracle as ao

pytestmark = pytest.mark.gpu

EPS = 1e-5
PAGE, HQ, HK, D, RD, LAYERS = 16, 8, 2, 64, 64, 2
B, T, PAGES = 12, 200, 160
SHARED = 4
SENTINEL = 1.5


class Requests:
    """Requests that begin with the same pages, and their tables as they grow."""

    def __init__(self, seed):
        self.rng = np.random.default_rng(seed)
        self.free = [int(x) for x in self.rng.permutation(np.arange(SHARED, PAGES))]
        self.tables, self.lens = [], []

    def begin(self, shares=True):
        self.tables.append(list(range(SHARED)) if shares else [])
        self.lens.append(SHARED * PAGE if shares else 0)

    def step(self, new):
        """`new[i]` more tokens for request i (those with none sit the step out)."""
        inputs = []
        for i, n in enumerate(new):
            if n == 0:
                continue
            while len(self.tables[i]) * PAGE < self.lens[i] + n:
                self.tables[i].append(self.free.pop())
            self.lens[i] += n
            inputs.append(kvc.InferInput(i, [0] * n, n, self.lens[i] - n, self.lens[i], list(self.tables[i])))
        return inputs


def new_step(gpu, cos_sin, **kw):
    return kvc.KVWriteStep(HK, D, PAGE, torch.bfloat16, gpu, max_requests=B, max_tokens=T, max_block_ids=PAGES * 4,
                           cos_sin_cache=cos_sin, num_heads=HQ, with_attention=True, shared_pages=SHARED, **kw)


class Buffers:
    def __init__(self, gpu, caches):
        z = lambda *s: torch.zeros(*s, dtype=torch.bfloat16, device=gpu)
        self.qkv = [z(T, (HQ + 2 * HK) * D) for _ in range(LAYERS)]
        cut = lambda a, b: [x[:, a * D:b * D] for x in self.qkv]
        self.q, self.k, self.v = cut(0, HQ), cut(HQ, HQ + HK), cut(HQ + HK, HQ + 2 * HK)
        self.q_out = [z(T, HQ * D) for _ in range(LAYERS)]
        self.out = [z(T, HQ, D) for _ in range(LAYERS)]
        self.caches = caches

    def fill(self, rng, gpu):
        for l in range(LAYERS):
            self.qkv[l].copy_(torch.from_numpy(rng.standard_normal(self.qkv[l].shape).astype(np.float32)))
            self.out[l].fill_(SENTINEL)


def caches_of(gpu, seed=1):
    """Pages of a prompt that every request begins with, and NaN behind them."""
    rng = np.random.default_rng(seed)
    c = np.full((LAYERS, PAGES, 2, PAGE, HK, D), np.nan, np.float32)
    c[:, :SHARED] = rng.standard_normal(c[:, :SHARED].shape)
    return list(torch.from_numpy(c).to(torch.bfloat16).to(gpu))


def weights_of(gpu, seed=2):
    rng = np.random.default_rng(seed)
    w = lambda: (1 + 0.3 * torch.from_numpy(rng.standard_normal(D).astype(np.float32))).to(torch.bfloat16).to(gpu)
    return [(w(), w()) for _ in range(LAYERS)]


def check_layer(host, order, inputs, x, weights, q_out, out, cache, cos_sin):
    """The layer's outputs against the formulas: the rotation's within its roundings, and the attention's on the queries
    and the cache as they were written."""
    n = sum(r.input_len for r in inputs)
    pos = host.position_ids
    for got, t, w in ((q_out[:n], x[:n, :HQ * D], weights[0]), (None, x[:n, HQ * D:(HQ + HK) * D], weights[1])):
        want, arith = ao.qk_norm_rotary_f64(t.double().cpu().numpy(), w.double().cpu().numpy(), pos,
                                            cos_sin.double().cpu().numpy(), D, EPS)
        if got is None:
            s = torch.from_numpy(host.slot_mapping)
            got = cache[:, 0].reshape(-1, HK * D)[s.to(cache.device)]
        err = np.abs(got.double().cpu().numpy().reshape(want.shape) - want)
        assert (err <= (np.abs(want) + arith) * 2.0 ** -8 * 1.01 + arith).all()
    want, lse, *bounds = ao.paged_attention_f64(q_out.double().cpu().numpy().reshape(T, HQ, D), cache.double().cpu().numpy(),
                                                host.cu_seqlens_q, host.kv_block_indices, host.kv_block_indptrs,
                                                host.kv_last_block_lens, D ** -0.5)
    tol, _ = ao.attention_tolerances(want, lse, *bounds, D, D ** -0.5, 2.0 ** -7, 0.0)
    err = np.abs(out.double().cpu().numpy() - want)[:n]
    assert (err <= tol[:n]).all()
    assert (out[n:].float() == SENTINEL).all()


def plan_of_steps():
    """What the requests of six steps do: chunks and single tokens, requests that end and begin, one that shares nothing."""
    r = Requests(3)
    for shares in (True, True, True, False, True, True):
        r.begin(shares)
    return r, [[70, 40, 5, 30, 1, 1], [1, 1, 33, 1, 1, 0], [1] * 6, [0, 0, 1, 0, 0, 0], [1, 90, 1, 1, 0, 64], [1, 1, 0, 1, 1, 1]]


def test_a_recorded_layer_sequence_serves_later_steps(gpu):
    cos_sin = kvc.make_cos_sin_cache(RD, 4096, 10000.0, dtype=torch.bfloat16).to(gpu)
    weights = weights_of(gpu)
    buf, eager = Buffers(gpu, caches_of(gpu)), Buffers(gpu, caches_of(gpu))
    step, other = new_step(gpu, cos_sin), new_step(gpu, cos_sin)
    reqs, steps = plan_of_steps()
    graph = None
    for i, new in enumerate(steps):
        inputs = reqs.step(new)
        for b in (buf, eager):
            b.fill(np.random.default_rng(100 + i), gpu)
        step.set_requests(inputs)
        if graph is None:
            graph = step.capture(buf.k, buf.v, buf.caches, queries=buf.q, query_outs=buf.q_out, norm_weights=weights, eps=EPS,
                                 attention_outs=buf.out)
            torch.cuda.synchronize()
            for o in buf.out:
                o.fill_(SENTINEL)
        graph.replay()
        other.set_requests(inputs)
        other.build_index()
        for l in range(LAYERS):
            q, _ = other.rotate_and_append(eager.q[l], eager.k[l], eager.v[l], eager.caches[l], query_out=eager.q_out[l],
                                           query_weight=weights[l][0], key_weight=weights[l][1], eps=EPS)
            other.attend(q, eager.caches[l], out=eager.out[l])
        torch.cuda.synchronize()
        host = kvc.make_kv_index_inputs(inputs, PAGE)
        n = len(host.position_ids)
        for l in range(LAYERS):
            assert torch.equal(buf.q_out[l][:n], eager.q_out[l][:n]) and torch.equal(buf.out[l], eager.out[l]), (i, l)
            assert torch.equal(buf.caches[l].view(torch.int16), eager.caches[l].view(torch.int16)), (i, l)
            check_layer(host, host.order, inputs, buf.qkv[l], weights[l], buf.q_out[l], buf.out[l], buf.caches[l], cos_sin)
        torch.randn(64, 64, device=gpu) @ torch.randn(64, 64, device=gpu)    # the program's own work between replays


def test_plain_writes_with_attention_and_without_rotation(gpu):
    """A step without a cos/sin table: `append`, then `attend`, recorded; and the standalone functions give the formula's too."""
    step = kvc.KVWriteStep(HK, D, PAGE, torch.bfloat16, gpu, max_requests=B, max_tokens=T, max_block_ids=PAGES * 4,
                           num_heads=HQ, with_attention=True)
    buf = Buffers(gpu, caches_of(gpu))
    reqs, steps = plan_of_steps()
    graph = None
    for i, new in enumerate(steps[:4]):
        inputs = reqs.step(new)
        buf.fill(np.random.default_rng(200 + i), gpu)
        step.set_requests(inputs)
        if graph is None:
            graph = step.capture(buf.k, buf.v, buf.caches, queries=buf.q, attention_outs=buf.out)
            for o in buf.out:
                o.fill_(SENTINEL)
        graph.replay()
        torch.cuda.synchronize()
        host = kvc.make_kv_index_inputs(inputs, PAGE)
        dev = kvc.to_device(host, PAGE, gpu)
        n = len(host.position_ids)
        shared = kvc.common_prefix_pages([r.block_ids for r in inputs])
        for l in range(LAYERS):
            want, lse, *bounds = ao.paged_attention_f64(
                buf.q[l].double().cpu().numpy().reshape(T, HQ, D), buf.caches[l].double().cpu().numpy(), host.cu_seqlens_q,
                host.kv_block_indices, host.kv_block_indptrs, host.kv_last_block_lens, D ** -0.5)
            tol, _ = ao.attention_tolerances(want, lse, *bounds, D, D ** -0.5, 2.0 ** -7, 0.0)
            alone = kvc.paged_attention(buf.q[l][:n], buf.caches[l], dev.cu_seqlens_q, dev.kv_block_indices,
                                        dev.kv_block_indptrs, dev.kv_last_block_lens, shared_pages=shared)
            for got in (buf.out[l][:n], alone.view(n, HQ, D)):
                assert (np.abs(got.double().cpu().numpy() - want[:n]) <= tol[:n]).all(), (i, l)
            assert (buf.out[l][n:].float() == SENTINEL).all()


def test_two_recorded_sequences_at_once(gpu):
    """Two steps' graphs replayed on two streams, and eager runs on a third meanwhile: none meets another's workspace."""
    cos_sin = kvc.make_cos_sin_cache(RD, 4096, 10000.0, dtype=torch.bfloat16).to(gpu)
    weights = weights_of(gpu)
    bufs = [Buffers(gpu, caches_of(gpu, 5 + i)) for i in range(2)]
    steps = [new_step(gpu, cos_sin) for _ in range(2)]
    want, graphs = [], []
    for i in range(2):
        r = Requests(20 + i)
        for _ in range(6):
            r.begin()
        inputs = r.step([60, 30 + i, 1, 1, 20, 1])
        bufs[i].fill(np.random.default_rng(30 + i), gpu)
        steps[i].set_requests(inputs)
        graphs.append(steps[i].capture(bufs[i].k, bufs[i].v, bufs[i].caches, queries=bufs[i].q, query_outs=bufs[i].q_out,
                                       norm_weights=weights, eps=EPS, attention_outs=bufs[i].out))
        torch.cuda.synchronize()
        want.append([o.clone() for o in bufs[i].out])
    eager_want = steps[0].attend(bufs[0].q_out[0], bufs[0].caches[0], out=torch.full_like(want[0][0], SENTINEL))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for _ in range(8):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                for o in bufs[i].out:
                    o.fill_(SENTINEL)
                graphs[i].replay()
        with torch.cuda.stream(streams[2]):
            got.append(steps[0].attend(bufs[0].q_out[0], bufs[0].caches[0], out=torch.full_like(want[0][0], SENTINEL)))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(a, b) for a, b in zip(bufs[i].out, want[i]))
    assert all(torch.equal(g, eager_want) for g in got)


def test_the_output_may_be_the_query_and_nothing_else_that_is_read(gpu):
    r = Requests(9)
    for _ in range(4):
        r.begin()
    inputs = r.step([50, 1, 12, 1])
    host = kvc.make_kv_index_inputs(inputs, PAGE)
    dev = kvc.to_device(host, PAGE, gpu)
    n = len(host.position_ids)
    cache = torch.randn(PAGES, 2, PAGE, HK, D, device=gpu).to(torch.bfloat16)
    idx = (dev.cu_seqlens_q, dev.kv_block_indices, dev.kv_block_indptrs, dev.kv_last_block_lens)
    rows = torch.randn(n + 1, HQ * D, device=gpu).to(torch.bfloat16)
    for kw in ({}, {"shared_pages": SHARED}):
        q = rows[:n].clone()
        want = kvc.paged_attention(q, cache, *idx, **kw)
        assert torch.equal(kvc.paged_attention(q, cache, *idx, out=q, **kw), want) and torch.equal(q, want)
    with pytest.raises(ValueError, match="overlap"):
        kvc.paged_attention(rows[:n], cache, *idx, out=rows[1:])
    wide = torch.randn(n, 2 * HQ * D, device=gpu).to(torch.bfloat16)
    with pytest.raises(ValueError, match="overlap"):
        kvc.paged_attention(wide[:, :HQ * D], cache, *idx, out=wide.flatten()[:n * HQ * D].view(n, HQ * D))
    with pytest.raises(ValueError, match="overlap"):
        kvc.paged_attention(rows[:n], cache, *idx, out=cache.flatten()[:n * HQ * D].view(n, HQ * D))
    plan = kvc.PagedAttentionPlan(*idx, HQ, HK, D, PAGE, torch.bfloat16, n)
    out = torch.empty(n, HQ, D, dtype=torch.bfloat16, device=gpu)
    with pytest.raises(ValueError, match="overlap"):
        plan.run(rows[:n], cache, out=out, lse=out.view(torch.float32).flatten()[:n * HQ].view(n, HQ))


def test_refusals(gpu):
    cos_sin = kvc.make_cos_sin_cache(RD, 4096, 10000.0, dtype=torch.bfloat16).to(gpu)
    args = dict(max_requests=2, max_tokens=8, max_block_ids=8)
    with pytest.raises(ValueError, match="num_heads"):
        kvc.KVWriteStep(HK, D, PAGE, torch.bfloat16, gpu, with_attention=True, **args)
    plain = kvc.KVWriteStep(HK, D, PAGE, torch.bfloat16, gpu, **args)
    x = torch.zeros(8, HK * D, dtype=torch.bfloat16, device=gpu)
    cache = torch.zeros(8, 2, PAGE, HK, D, dtype=torch.bfloat16, device=gpu)
    with pytest.raises(ValueError, match="without attention"):
        plain.attend(x, cache)
    with pytest.raises(ValueError, match="without attention"):
        plain.capture([x], [x], [cache], queries=[x], attention_outs=[x])
    with pytest.raises(ValueError, match="queries"):
        plain.capture([x], [x], [cache], norm_weights=[(x[0, :D], x[0, :D])])
    step = kvc.KVWriteStep(HK, D, PAGE, torch.bfloat16, gpu, cos_sin_cache=cos_sin, num_heads=HK, with_attention=True, **args)
    with pytest.raises(ValueError, match="query_outs"):
        step.capture([x], [x], [cache], queries=[x], attention_outs=[x])
    with pytest.raises(ValueError, match="together"):
        step.rotate_and_append(x, x, x, cache, query_weight=x[0, :D].clone())
