"""A workspace of more than 2^32 rows of partials: as many single tokens behind a shared prefix as a plan takes of this many heads."""
import pytest
import torch

import lmserve_amd as kvc

pytestmark = pytest.mark.gpu


def test_partials_beyond_2_to_the_32_rows(gpu):
    """Every row's softmax is over two keys, one of the prefix and one of its own: both parts are joined, from slots on both sides of 2^32 rows."""
    R, H, D, OWN = 8448, 32768, 8, 16
    torch.cuda.empty_cache()
    free = torch.cuda.mem_get_info()[0]
    if free < 200 << 30:
        pytest.skip(f"{free >> 30} GiB of the card are free, 200 are needed")
    i32 = dict(dtype=torch.int32, device=gpu)
    g = torch.Generator(device=gpu).manual_seed(0)
    cache = torch.randn(1 + OWN, 2, 1, H, D, device=gpu, generator=g, dtype=torch.bfloat16)
    query = torch.empty(R, H, D, device=gpu, dtype=torch.bfloat16).normal_(generator=g)
    table = torch.zeros(R, 2, **i32)
    table[:, 1] = 1 + torch.arange(R, **i32) % OWN
    index = [torch.arange(R + 1, **i32), table.view(-1), 2 * torch.arange(R + 1, **i32), torch.ones(R, **i32)]
    plan = kvc.PagedAttentionPlan(*index, H, H, D, 1, torch.bfloat16, R, max_q_len=1, shared_pages=1)
    assert plan._workspace_bytes > (1 << 32) * 36
    print(f"workspace of {plan._workspace_bytes >> 30} GiB", flush=True)
    out = plan.run(query, cache)
    torch.cuda.synchronize()
    worst = 0.0
    shared = cache[0].float()
    for b0 in range(0, R, 256):
        own = cache[1 + torch.arange(b0, b0 + 256, device=gpu) % OWN].float()      # [256, 2, 1, H, D]
        q = query[b0:b0 + 256].float()
        s = torch.stack(((q * shared[0, 0]).sum(-1), (q * own[:, 0, 0]).sum(-1)), -1) * D ** -0.5
        p = s.softmax(-1)
        a, b = p[..., :1] * shared[1, 0], p[..., 1:] * own[:, 1, 0]
        want = a + b
        # the output's rounding; that of the prefix's weight, whose rows are wide tiles; what two parts of 8 bits leave of the other, 32 bits' in
        # products and sums, and in scores of up to some 2^5
        tol = want.abs() * 2.0 ** -8 * 1.01 + a.abs() * 2.0 ** -8 * 1.01 + (a.abs() + b.abs()) * 2.0 ** -15
        worst = max(worst, ((out[b0:b0 + 256].float() - want).abs() / tol).max().item())
    del out, query, cache, plan, own, q, s, p, a, b, want, tol, shared
    torch.cuda.empty_cache()
    assert worst <= 1, f"off by {worst:.3g} of the bound"
