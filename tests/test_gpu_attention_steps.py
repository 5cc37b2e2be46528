"""Steps at the edges of the layout: offsets that decrease, more wide requests than are looked at one by one, keys beyond 32-bit
offsets, ranges of keys that end inside the windows that the wide tiles read."""
import numpy as np
import pytest
import torch

import lmserve_amd as kvc
from tests.test_gpu_attention import Step

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shared", [0, 1])
@pytest.mark.parametrize("which", ["qo", "indptr"])
def test_offsets_that_decrease_are_not_computed(gpu, which, shared):
    s = Step([(5, 40), (5, 40), (5, 40)], 8, 2, 64, 16, seed=1)
    bad = getattr(s, which).copy()
    bad[2] = bad[0]                      # request 0's rows or pages again for request 2
    setattr(s, which, bad)
    out = torch.full((s.T, 8, 64), 7.0, dtype=torch.bfloat16, device=gpu)
    lse = torch.full((s.T, 8), 7.0, device=gpu)
    s.plan(gpu, shared_pages=shared).run(s.query.to(gpu), s.cache.to(gpu), out=out, lse=lse)
    torch.cuda.synchronize()
    assert (out == 7).all() and (lse == 7).all()


@pytest.mark.parametrize("new", [40, 41, 64, 65])
def test_wide_tiles_at_every_end_of_a_window(gpu, new):
    """Chunks whose keys end 31 to 97 behind a window's begin, with contexts of odd lengths."""
    for D, page in ((64, 16), (128, 16), (128, 20), (96, 32)):
        s = Step([(new, new), (new, new + 31), (new, new + 32), (new, new + 33), (new, 64 * 3 - 1), (new, 64 * 3), (new, 64 * 3 + 1)],
                 4, 1, D, page, seed=new)
        out, lse = s.plan(gpu).run(s.query.to(gpu), s.cache.to(gpu), return_lse=True)
        s.check(out, lse)


def test_more_wide_requests_than_are_looked_at_one_by_one(gpu):
    """1100 requests of 12 tokens and 4 heads to a key head: the same bits whatever order the layout's counters took."""
    rng = np.random.default_rng(4)
    s = Step([(12, 12 + int(k)) for k in rng.integers(0, 40, 1100)], 4, 1, 64, 16, seed=2)
    q, cache = s.query.to(gpu), s.cache.to(gpu)
    plan = s.plan(gpu)
    out, lse = plan.run(q, cache, return_lse=True)
    s.check(out, lse)
    for _ in range(3):
        plan.build()
        assert torch.equal(plan.run(q, cache), out)


def test_pages_beyond_32_bit_offsets(gpu):
    """A cache of 6 GiB whose requests' pages lie at its end: byte offsets beyond 2^32."""
    H, D, page = 2, 128, 16
    pages = (6 << 30) // (2 * page * H * D * 2)
    s = Step([(1, 70), (40, 300), (1, 500)], 8, H, D, page, seed=3)
    small = s.cache.to(gpu)
    big = torch.zeros(pages, 2, page, H, D, dtype=torch.bfloat16, device=gpu)
    n = small.shape[0]
    big[pages - n:] = small
    idx = s.index(gpu)
    idx[1] = idx[1] + (pages - n)
    out, lse = kvc.paged_attention(s.query.to(gpu), big, *idx, return_lse=True)
    s.check(out, lse)
