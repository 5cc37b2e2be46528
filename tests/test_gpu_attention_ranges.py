"""Steps whose tiles are cut at the keys and joined, as the layout's lists show it: narrow tiles in spite of a wrong hint, wide ones and
prefixes in ranges of the least length and in long ones."""
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


@pytest.mark.parametrize("dtype,page", [("bf16", 16), ("f16", 16), ("bf16", 20), ("f16", 64)])
@pytest.mark.parametrize("lengths,heads,kv_heads,D,items,entries", [
    ([(42, 700)], 4, 1, 64, 2 * 2, 8 + 3),                       # two tiles of two ranges, 16 rows an entry
    ([(33, 1100), (1, 5), (50, 513)], 8, 2, 128, 3 * 2 + 2 * 2, 9 + 13),
    ([(11, 9000)], 4, 1, 64, 18, 44),                            # more parts than an entry of several rows has: one a row
    ([(40, 1600)], 512, 512, 8, 1, 0),                           # a range of 26 windows, whole: its pages are looked up twice
    ([(40, 6000)], 128, 128, 8, 4, 3)])                          # and four of 1500 keys
def test_wide_tiles_are_cut(gpu, lengths, heads, kv_heads, D, items, entries, dtype, page):
    s = Step(lengths, heads, kv_heads, D, page, dtype, seed=21)
    plan = s.plan(gpu)
    out, lse = plan.run(s.query.to(gpu), s.cache.to(gpu), return_lse=True)
    print(lengths, heads, kv_heads, "layout", layout(plan))
    s.check(out, lse)
    wide, _, wide_entries, _ = layout(plan)
    assert (wide, wide_entries) == (items, entries)


@pytest.mark.parametrize("dtype,page", [("bf16", 16), ("f16", 20)])
@pytest.mark.parametrize("keys,rows,wide", [(1100, 20, False), (1100, 100, False), (1100, 150, True), (4096, 20, False),
                                            (4096, 100, True), (4096, 150, True)])
def test_a_prefix_is_cut(gpu, keys, rows, wide, dtype, page):
    """The rows of requests that share 1100 or 4096 keys, in narrow tiles and in wide ones, over several ranges."""
    shared = keys // page
    s = Step([(1, shared * page + 1 + 7 * i % 60) for i in range(rows // 4)], 4, 1, 64, page, dtype, shared=shared, seed=22)
    plan = s.plan(gpu)
    out, lse = plan.run(s.query.to(gpu), s.cache.to(gpu), return_lse=True)
    print(keys, rows, "layout", layout(plan))
    s.check(out, lse)
    items, _, _, shared_wide = layout(plan)
    assert bool(shared_wide) == wide
    if wide:
        assert items >= 2 * -(-s.T * 4 // 128)


def test_a_prefix_and_chunks_in_ranges_side_by_side(gpu):
    """Wide tiles of a prefix and of requests of their own in one list, cut at the same length."""
    s = Step([(1, 1600 + i) for i in range(1, 41)] + [(36, 2000), (40, 1700)], 4, 1, 64, 16, shared=100, seed=23)
    plan = s.plan(gpu)
    out, lse = plan.run(s.query.to(gpu), s.cache.to(gpu), return_lse=True)
    print("layout", layout(plan))
    s.check(out, lse)
    items, narrow_entries, wide_entries, shared_wide = layout(plan)
    assert shared_wide and narrow_entries >= 40 and wide_entries > 0 and items > 6
