"""Steps over an 8-bit pool as a model runs them: rotation, write, attention, eager and recorded, against the formulas in 64
bits on what the cache then holds."""
import numpy as np
import pytest
import torch

import lmserve_amd as kvc
from oracle import attention_oracle as ao
from oracle import q8_oracle as qo
from oracle import rope_oracle as ro

pytestmark = pytest.mark.gpu
F8 = torch.float8_e4m3fn
H, HQ, D, PAGE, LAYERS, BLOCKS = 2, 8, 64, 16, 2, 40
TOKENS = 64


def step_of(gpu, **kw):
    return kvc.KVWriteStep(H, D, PAGE, torch.bfloat16, gpu, max_requests=6, max_tokens=TOKENS, max_block_ids=60, num_heads=HQ,
                           with_attention=True, kv_dtype=F8, **kw)


class Requests:
    """Requests that grow from step to step over blocks of their own."""

    def __init__(self, seed):
        self.rng = np.random.default_rng(seed)
        self.free = list(self.rng.permutation(BLOCKS))
        self.have, self.blocks = [0] * 4, [[] for _ in range(4)]

    def next(self, new):
        out = []
        for b, n in enumerate(new):
            if n == 0:
                continue
            self.have[b] += n
            while len(self.blocks[b]) * PAGE < self.have[b]:
                self.blocks[b].append(int(self.free.pop()))
            out.append(kvc.InferInput(seq_id=b, input_ids=[0] * n, filled_token_len=self.have[b] - n, input_len=n,
                                      context_len=self.have[b], block_ids=list(self.blocks[b])))
        return out


def projections(rng, gpu, layers=LAYERS):
    qkv = [torch.from_numpy(rng.standard_normal((TOKENS, (HQ + 2 * H) * D)).astype(np.float32)).to(torch.bfloat16).to(gpu) for _ in range(layers)]
    return [(x[:, :HQ * D], x[:, HQ * D:(HQ + H) * D], x[:, (HQ + H) * D:]) for x in qkv]


def check(step, query, attended, cache, rows):
    pages = qo.Cache(cache.cpu().numpy(), H, D).values().reshape(-1, PAGE, 2, H, D).transpose(0, 2, 1, 3, 4)
    b = step.num_requests
    index = [t.cpu().numpy() for t in (step.cu_seqlens_q[:b + 1], step.kv_indices, step.kv_indptr[:b + 1], step.kv_last_page_len[:b])]
    want, lse, *bounds = ao.paged_attention_f64(query[:rows].double().cpu().numpy().reshape(rows, HQ, D), pages, *index, D ** -0.5)
    tol, _ = ao.attention_tolerances(want, lse, *bounds, D, D ** -0.5, 2.0 ** -10, 2.0 ** -25)
    tol = tol + np.abs(want) * (2.0 ** -7 - 2.0 ** -10) / 2 * 1.05
    assert (np.abs(attended[:rows].double().cpu().numpy().reshape(want.shape) - want) <= tol).all()


STEPS = [(30, 5, 17, 1), (1, 1, 1, 1), (1, 20, 1, 12), (1, 1, 1, 1), (0, 1, 2, 3)]


@pytest.mark.parametrize("rotate,norms", [(False, False), (True, False), (True, True)])
@pytest.mark.parametrize("recorded", [False, True])
def test_a_model_s_steps(gpu, rotate, norms, recorded):
    g = torch.Generator().manual_seed(0)
    cs = kvc.make_cos_sin_cache(D, 256, 10000.0, dtype=torch.bfloat16)
    step = step_of(gpu, **({"cos_sin_cache": cs.to(gpu)} if rotate else {}))
    weights = [tuple((1 + 0.2 * torch.randn(D, generator=g)).to(torch.bfloat16).to(gpu) for _ in range(2)) for _ in range(LAYERS)] if norms else None
    pool = kvc.allocate_q8_kv_caches(LAYERS, BLOCKS, PAGE, H, D, gpu)
    pool.random_(0, 256, generator=torch.Generator(device=gpu).manual_seed(1))
    oracles = [qo.Cache(pool[l].cpu().numpy(), H, D) for l in range(LAYERS)]
    reqs = Requests(3)
    buffers = projections(reqs.rng, gpu)
    q_outs = [torch.zeros(TOKENS, HQ * D, dtype=torch.bfloat16, device=gpu) for _ in range(LAYERS)]
    outs = [torch.zeros_like(q) for q in q_outs]
    graph = None
    for n, new in enumerate(STEPS):
        inputs = reqs.next(new)
        tokens = sum(new)
        for (q, k, v), (q1, k1, v1) in zip(buffers, projections(reqs.rng, gpu)):
            q.copy_(q1), k.copy_(k1), v.copy_(v1)
        step.set_requests(inputs)
        queries = [q for q, _, _ in buffers]
        if recorded and graph is None:
            # its eager pass writes this step; recording runs nothing
            graph = step.capture([k for _, k, _ in buffers], [v for _, _, v in buffers], list(pool), queries=queries,
                                 query_outs=q_outs if rotate else None, norm_weights=weights, attention_outs=outs)
        elif recorded:
            graph.replay()
        else:
            step.build_index()
            for l, (q, k, v) in enumerate(buffers):
                if rotate:
                    q, _ = step.rotate_and_append(q, k, v, pool[l], query_out=q_outs[l], **(dict(query_weight=weights[l][0], key_weight=weights[l][1]) if norms else {}))
                else:
                    step.append(k, v, pool[l])
                step.attend(q, pool[l], out=outs[l])
        torch.cuda.synchronize()
        slots = step.slot_mapping[:tokens].cpu().numpy()
        positions = step.positions[:tokens].cpu().numpy()
        for l, (q, k, v) in enumerate(buffers):
            q, k, v = q[:tokens], k[:tokens], v[:tokens]
            if rotate:
                # the rotated keys are the operator's own: its rounding is its tests' matter, the write has to be of them to the bit
                call = (lambda *a: kvc.qk_norm_rotary_pos_emb(a[0], a[1], *weights[l], *a[2:])) if norms else kvc.rotary_pos_emb
                rq, k = call(q.contiguous(), k.contiguous(), step.positions[:tokens], cs.to(gpu), D)
                assert torch.equal(q_outs[l][:tokens], rq)
                q = rq
                if not norms:
                    want, _ = ro.rotary_pos_emb_f64(buffers[l][0][:tokens].double().cpu().numpy(), buffers[l][1][:tokens].double().cpu().numpy(),
                                                    positions, cs.double().numpy(), D)
                    assert (np.abs(rq.double().cpu().numpy() - want) <= 2.0 ** -8 * np.abs(want) * 1.01 + 2.0 ** -18).all()
            oracles[l].write(k.double().cpu().numpy().reshape(tokens, H, D), v.double().cpu().numpy().reshape(tokens, H, D), slots)
            assert np.array_equal(pool[l].cpu().numpy(), oracles[l].pages()), (n, l)
            check(step, q, outs[l], pool[l], tokens)


def test_what_a_step_refuses(gpu):
    for bad in (dict(kv_dtype=torch.uint8), dict(kv_dtype=torch.float8_e5m2)):
        with pytest.raises(TypeError):
            kvc.KVWriteStep(H, D, PAGE, torch.bfloat16, gpu, 1, 1, 1, **bad)
    for heads, dim, page, dtype in ((H, 72, 16, torch.bfloat16), (H, 64, 20, torch.bfloat16), (H, 64, 16, torch.float32)):
        with pytest.raises(TypeError):
            kvc.KVWriteStep(heads, dim, page, dtype, gpu, 1, 1, 1, kv_dtype=F8)
    step = step_of(gpu)
    pool = kvc.allocate_q8_kv_caches(1, 4, PAGE, H, D, gpu)
    rows = torch.zeros(TOKENS, H, D, dtype=torch.bfloat16, device=gpu)
    with pytest.raises(ValueError, match="cos/sin"):
        step.rotate_and_append(torch.zeros(TOKENS, HQ * D, dtype=torch.bfloat16, device=gpu), rows.flatten(1), rows.flatten(1), pool[0])
    with pytest.raises(ValueError):
        step.append(rows[:5], rows[:5], pool[0])
    with pytest.raises(TypeError):
        step.append(rows, rows, torch.zeros(4, 2, PAGE, H, D, dtype=torch.bfloat16, device=gpu))


def test_operators_of_the_dispatcher(gpu):
    import lmserve_amd.torch_ops  # noqa: F401
    rng = np.random.default_rng(0)
    k, v = (torch.from_numpy(rng.standard_normal((20, H, D)).astype(np.float32)).to(torch.bfloat16).to(gpu) for _ in range(2))
    a, b = (kvc.allocate_q8_kv_caches(1, 4, PAGE, H, D, gpu)[0].zero_() for _ in range(2))
    slots = torch.arange(20, device=gpu)
    torch.ops.kvcache.reshape_and_cache_q8(k, v, a, slots)
    i32 = dict(dtype=torch.int32, device=gpu)
    torch.ops.kvcache.append_paged_kv_cache_q8(k, v, torch.zeros(20, **i32), slots.int(), b, torch.arange(2, **i32),
                                               torch.tensor([0, 2], **i32), torch.tensor([4], **i32))
    assert torch.equal(a, b) and a.any()


@pytest.mark.parametrize("norms", [False, True])
@pytest.mark.parametrize("key_out", [False, True])
@pytest.mark.parametrize("recorded", [False, True])
def test_tokens_beyond_the_cos_sin_table_are_left_alone(gpu, recorded, key_out, norms):
    """A table that ends inside a request's context, inside a group: the tokens that have no row are not written either, and the
    codes and exponents that their groups hold stay, whatever the rotated keys' memory held before."""
    rows = 37
    cs = kvc.make_cos_sin_cache(D, rows, 10000.0, dtype=torch.bfloat16).to(gpu)
    step = step_of(gpu, cos_sin_cache=cs)
    g = torch.Generator().manual_seed(0)
    weights = [(1 + 0.2 * torch.randn(D, generator=g)).to(torch.bfloat16).to(gpu) for _ in range(2)] if norms else [None, None]
    pool = kvc.allocate_q8_kv_caches(1, BLOCKS, PAGE, H, D, gpu)
    pool.random_(0, 256, generator=torch.Generator(device=gpu).manual_seed(1))
    oracle = qo.Cache(pool[0].cpu().numpy(), H, D)
    reqs = Requests(5)
    (q, k, v), = projections(reqs.rng, gpu, 1)
    q_out = torch.zeros(TOKENS, HQ * D, dtype=torch.bfloat16, device=gpu)
    k_out = torch.zeros(TOKENS, H * D, dtype=torch.bfloat16, device=gpu) if key_out else None
    graph = None
    for new in ((26, 33, 5), (5, 1, 20), (1, 1, 1), (0, 4, 30)):
        inputs = reqs.next(new)
        tokens = sum(new)
        for t, x in zip((q, k, v), projections(reqs.rng, gpu, 1)[0]):
            t.copy_(x)
        step.set_requests(inputs)
        # what earlier steps may have left where the rotation writes nothing
        junk = torch.full((TOKENS, H * D), 3e38, dtype=torch.bfloat16, device=gpu)
        if key_out:
            k_out.copy_(junk)
        del junk
        q_out.fill_(7)
        if recorded and graph is None:
            def body():
                step.build_index()
                step.rotate_and_append(q, k, v, pool[0], query_out=q_out, key_out=k_out, query_weight=weights[0], key_weight=weights[1])
            body()      # (writing a step twice is writing it once)
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                body()
        if recorded:
            graph.replay()
        else:
            step.build_index()
            step.rotate_and_append(q, k, v, pool[0], query_out=q_out, key_out=k_out, query_weight=weights[0], key_weight=weights[1])
        torch.cuda.synchronize()
        positions = step.positions[:tokens].cpu().numpy()
        slots = step.slot_mapping[:tokens].cpu().numpy()
        there = positions < rows
        assert (q_out[:tokens].cpu()[torch.from_numpy(~there)] == 7).all()
        call = (lambda *a: kvc.qk_norm_rotary_pos_emb(a[0], a[1], *weights, *a[2:])) if norms else kvc.rotary_pos_emb
        _, rk = call(q[:tokens].contiguous(), k[:tokens].contiguous(), step.positions[:tokens].clamp(max=rows - 1), cs, D)
        oracle.write(rk.double().cpu().numpy().reshape(tokens, H, D), v[:tokens].double().cpu().numpy().reshape(tokens, H, D),
                     np.where(there, slots, -1))
        assert np.array_equal(pool[0].cpu().numpy(), oracle.pages()), new
    assert max(reqs.have) > rows + PAGE
    # without the rotation every token of the step is written
    before = pool.clone()
    step.append(k, v, pool[0])
    oracle.write(k[:tokens].double().cpu().numpy().reshape(tokens, H, D), v[:tokens].double().cpu().numpy().reshape(tokens, H, D), slots)
    assert np.array_equal(pool[0].cpu().numpy(), oracle.pages()) and not torch.equal(before, pool)


def test_what_a_rotating_step_refuses(gpu):
    """As over 16 bits: a table that is not one at construction, rows of another number or width at every call."""
    cs = kvc.make_cos_sin_cache(D, 64, 10000.0, dtype=torch.bfloat16).to(gpu)
    args = (H, D, PAGE, torch.bfloat16, gpu, 4, TOKENS, 20)
    for error, kw in ((TypeError, dict(cos_sin_cache=cs.half(), num_heads=HQ)), (ValueError, dict(cos_sin_cache=cs.t(), num_heads=HQ)),
                      (ValueError, dict(cos_sin_cache=cs[0], num_heads=HQ))):
        with pytest.raises(error):
            kvc.KVWriteStep(*args, kv_dtype=F8, **kw)
    with pytest.raises((TypeError, ValueError, RuntimeError)):
        kvc.KVWriteStep(*args, kv_dtype=F8, cos_sin_cache=cs.cpu(), num_heads=HQ)
    pool = kvc.allocate_q8_kv_caches(1, BLOCKS, PAGE, H, D, gpu).zero_()
    step = kvc.KVWriteStep(*args, kv_dtype=F8, cos_sin_cache=cs, num_heads=HQ)
    reqs = Requests(6)
    step.set_requests(reqs.next((20, 5)))
    step.build_index()
    (q, k, v), = projections(reqs.rng, gpu, 1)
    half = TOKENS // 2
    with pytest.raises(ValueError):      # (of a step without query heads)
        kvc.KVWriteStep(*args, kv_dtype=F8, cos_sin_cache=cs).rotate_and_append(q, k, v, pool[0])
    for bad in ((q[:half], k, v), (q, k[:half], v), (q, k, v[:half]), (q[:, D:], k, v), (q.reshape(2 * TOKENS, -1), k, v),
                (q.reshape(-1), k, v), (q, torch.cat((k, k), 1), v), (q, k, torch.cat((v, v), 1)), (q, k, v[:, D:])):
        with pytest.raises(ValueError):
            step.rotate_and_append(*bad, pool[0])
    for bad in ((q.half(), k, v), (q, k.half(), v), (q, k, v.half())):
        with pytest.raises(TypeError):
            step.rotate_and_append(*bad, pool[0])
    with pytest.raises(ValueError):
        step.rotate_and_append(q, k, v, pool[0], query_out=torch.empty(half, HQ * D, dtype=torch.bfloat16, device=gpu))
    with pytest.raises(ValueError):
        step.rotate_and_append(q, k, v, pool[0], query_weight=torch.ones(D, dtype=torch.bfloat16, device=gpu))
    torch.cuda.synchronize()
    assert not pool.any()
    rotated, _ = step.rotate_and_append(q, k, v, pool[0])
    assert rotated.shape == (TOKENS, HQ * D) and pool.any()
    # rows of any layout are rows
    apart = q.reshape(TOKENS, HQ, D).transpose(1, 2).contiguous().transpose(1, 2)
    again, _ = step.rotate_and_append(apart, k, v, pool[0])
    n = step.num_tokens
    assert torch.equal(again.reshape(TOKENS, -1)[:n], rotated[:n])
