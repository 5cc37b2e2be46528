"""Steps whose tiles are cut at the keys and joined, as the layout's lists show it: narrow tiles in spite of a wrong hint."""
import pytest
import torch

from tests.test_gpu_attention import Step

pytestmark = pytest.mark.gpu


def layout(plan):
    """Wide items, entries of narrow and of wide tiles that are joined, and whether the shared prefix is in wide tiles."""
    torch.cuda.synchronize()
    return plan._buffer[:16].view(torch.int32).tolist()


@pytest.mark.parametrize("lengths,heads,kv_heads,D,max_q_len", [
    ([(900, 900)], 32, 8, 128, 1), ([(600, 900)], 32, 8, 128, 1), ([(700, 700)], 32, 32, 256, 1), ([(900, 900)], 16, 2, 256, 2),
    ([(20, 704), (20, 224)], 128, 128, 256, 20), ([(1500, 100)], 8, 8, 128, 1)])
def test_a_hint_of_fewer_tokens_than_requests_have_is_no_limit(gpu, lengths, heads, kv_heads, D, max_q_len):
    """Few keys in all, whose narrow tiles are cut all the same: every row is written."""
    s = Step(lengths, heads, kv_heads, D, 16, seed=20)
    out = torch.full((s.T, heads, D), float("nan"), dtype=torch.bfloat16, device=gpu)
    lse = torch.full((s.T, heads), float("nan"), device=gpu)
    plan = s.plan(gpu, max_q_len=max_q_len)
    plan.run(s.query.to(gpu), s.cache.to(gpu), out=out, lse=lse)
    wide, narrow_entries, _, _ = layout(plan)
    assert wide == 0 and narrow_entries > 0
    s.check(out, lse)
