"""Attention calls whose outputs lie where the launch reads: refused before anything runs."""
import pytest
import torch

import lmserve_amd as kvc
from tests.test_gpu_attention import Step

pytestmark = pytest.mark.gpu


def test_outputs_on_the_page_table_or_the_layout_are_refused(gpu):
    s = Step([(1, 90), (3, 40)], 8, 2, 64, 16)
    q, cache = s.query.to(gpu), s.cache.to(gpu)
    idx = s.index(gpu)
    room = torch.zeros(4096, dtype=torch.int32, device=gpu)
    n = idx[1].numel()
    room[:n] = idx[1]
    idx[1] = room[:n]
    plan = kvc.PagedAttentionPlan(*idx, 8, 2, 64, 16, torch.bfloat16, num_tokens=s.T)
    want = plan.run(q, cache)
    s.check(want)
    values = s.T * 8 * 64
    halves = room.view(torch.bfloat16)
    layout = plan._buffer.view(torch.bfloat16)
    assert layout.numel() >= values and halves.numel() >= values
    for out in (halves[:values], layout[:values]):
        with pytest.raises(ValueError, match="overlaps"):
            plan.run(q, cache, out=out.view(s.T, 8, 64))
        with pytest.raises(ValueError, match="overlaps"):
            plan.run(q, cache, lse=out.view(torch.float32)[:s.T * 8].view(s.T, 8))
    with pytest.raises(ValueError, match="overlaps"):
        kvc.paged_attention(q, cache, *idx, out=halves[:values].view(s.T, 8, 64))
    # right behind the table is apart from it
    at = -(-n * 2 // 8) * 8
    assert torch.equal(plan.run(q, cache, out=halves[at:at + values].view(s.T, 8, 64)), want)
    assert torch.equal(room[:n].cpu(), torch.from_numpy(s.indices))


def test_norm_outputs_on_what_is_read_are_refused(gpu):
    g = torch.Generator().manual_seed(0)
    r = lambda *shape: torch.randn(*shape, generator=g).to(torch.bfloat16).to(gpu)
    q, k, v, qw, kw = r(9, 512), r(9, 128), r(9, 128), r(64), r(64)
    table = torch.zeros(16384, dtype=torch.bfloat16, device=gpu)
    cs = table[:100 * 128].view(100, 128)
    cs.copy_(kvc.make_cos_sin_cache(64, 100, 10000.0, dtype=torch.bfloat16))
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=gpu)
    slots = torch.arange(9, dtype=torch.int64, device=gpu)
    plan = kvc.PagedRotaryWritePlan(i32([0] * 9), i32(list(range(9))), i32([0]), i32([0, 1]), i32([9]), cs, 8, 2, 64, 16, slots=slots)
    cache = torch.zeros(2, 2, 16, 2, 64, dtype=torch.bfloat16, device=gpu)
    before = table.clone()
    with pytest.raises(ValueError, match="overlaps"):
        plan.run(q, k, v, cache, query_out=table[-4608 - 64 * 50:-64 * 50].view(9, 512), query_weight=qw, key_weight=kw)
    with pytest.raises(ValueError, match="overlaps"):
        plan.run(q, k, v, cache, key_out=table[:9 * 128].view(9, 128), query_weight=qw, key_weight=kw)
    with pytest.raises(ValueError, match="overlaps"):
        plan.run(q, k, v, table[:2 * 4096].view(2, 2, 16, 2, 64), query_weight=qw, key_weight=kw)
    assert torch.equal(table, before) and (cache == 0).all()
