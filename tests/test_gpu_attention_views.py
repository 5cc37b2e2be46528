"""Attention plans over index tensors that are views."""
import pytest
import torch

import lmserve_amd as kvc
from tests.test_gpu_attention import Step

pytestmark = pytest.mark.gpu


def test_index_tensors_that_are_views_serve_later_steps(gpu):
    """Columns of a matrix of indices: what is written into them is what the next build lays out, eager and recorded."""
    first, then = (Step(lengths, 8, 2, 64, 16, seed=5) for lengths in ([(1, 90), (3, 40), (1, 33)], [(2, 40), (1, 70), (2, 64)]))
    assert first.T == then.T and first.indices.size >= then.indices.size
    n = first.indices.size
    table = torch.zeros(n + 1, 4, dtype=torch.int32, device=gpu)
    columns = [table[:4, 0], table[:n, 1], table[:4, 2], table[:3, 3]]

    def write(s):
        for column, x in zip(columns, (s.qo, s.indices, s.indptr, s.last)):
            column[:x.size].copy_(torch.from_numpy(x))

    write(first)
    plan = kvc.PagedAttentionPlan(*columns, 8, 2, 64, 16, torch.bfloat16, num_tokens=first.T)
    first.check(plan.run(first.query.to(gpu), first.cache.to(gpu)))
    write(then)
    plan.build()
    q, cache = then.query.to(gpu), then.cache.to(gpu)
    want = plan.run(q, cache)
    then.check(want)
    out = torch.empty_like(want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan.build()
        plan.run(q, cache, out=out)
    for s in (first, then, first, then):
        write(s)
        q.copy_(s.query)
        graph.replay()
        torch.cuda.synchronize()
        if s is then:
            assert torch.equal(out, want)
