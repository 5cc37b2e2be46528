"""Tensors that have no strides (sparse ones) where rows, caches or index arrays belong: a Python exception, not the end of the process."""
import pytest
import torch

import lmserve_amd as kvc

pytestmark = pytest.mark.gpu
H, HQ, D, PAGE, T = 2, 4, 64, 16, 8
F8 = torch.float8_e4m3fn


class Step:
    def __init__(self, gpu):
        bf, i32 = dict(dtype=torch.bfloat16, device=gpu), dict(dtype=torch.int32, device=gpu)
        self.q, self.k, self.v = (torch.ones(T, h * D, **bf) for h in (HQ, H, H))
        self.k3, self.v3 = self.k.view(T, H, D), self.v.view(T, H, D)
        self.cache = torch.zeros(4, 2, PAGE, H, D, **bf)
        self.q8 = kvc.allocate_q8_kv_caches(1, 4, PAGE, H, D, gpu)[0].zero_()
        self.slots = torch.arange(T, device=gpu)
        self.index = [torch.zeros(T, **i32), torch.arange(T, **i32)]
        self.pages = [torch.arange(1, **i32), torch.tensor([0, 1], **i32), torch.tensor([T], **i32)]
        self.cs = kvc.make_cos_sin_cache(D, 64, dtype=torch.bfloat16).to(gpu)
        self.qo = torch.tensor([0, T], **i32)
        self.plan = kvc.PagedKVWritePlan(*self.index, *self.pages, H, D, PAGE, torch.bfloat16)
        self.rotary = kvc.PagedRotaryWritePlan(*self.index, *self.pages, self.cs, HQ, H, D, PAGE)


CALLS = {
    "reshape_and_cache": lambda s: (kvc.reshape_and_cache, [s.k3, s.v3, s.cache, s.slots]),
    "append": lambda s: (kvc.append_paged_kv_cache, [s.k3, s.v3, *s.index, s.cache, *s.pages]),
    "write_plan": lambda s: (s.plan.append, [s.k3, s.v3, s.cache]),
    "rotary_plan": lambda s: (s.rotary.run, [s.q, s.k, s.v, s.cache]),
    "rotary": lambda s: (lambda *a: kvc.rotary_pos_emb(*a, D), [s.q, s.k, s.index[1], s.cs]),
    "rotary_append": lambda s: (lambda q, k, v, b, p, cs, c, *pages: kvc.rotary_pos_emb_and_append_paged(q, k, v, b, p, cs, D, c, *pages),
                                [s.q, s.k, s.v, *s.index, s.cs, s.cache, *s.pages]),
    "write_q8": lambda s: (kvc.reshape_and_cache_q8, [s.k3, s.v3, s.q8, s.slots]),
    "append_q8": lambda s: (kvc.append_paged_kv_cache_q8, [s.k3, s.v3, *s.index, s.q8, *s.pages]),
    "read_q8": lambda s: (lambda c, x: kvc.read_cache_q8(c, x, H, D), [s.q8, s.slots]),
    "attention": lambda s: (kvc.paged_attention, [s.q.view(T, HQ, D), s.cache, s.qo, *s.pages]),
    "attention_q8": lambda s: (lambda *a: kvc.paged_attention(*a, num_kv_heads=H), [s.q.view(T, HQ, D), s.q8, s.qo, *s.pages]),
}


@pytest.mark.parametrize("name", CALLS)
def test_a_sparse_tensor_is_refused(gpu, name):
    s = Step(gpu)
    call, args = CALLS[name](s)
    call(*args)
    torch.cuda.synchronize()
    # (kv_last_page_len, the last one, is not read where tokens have positions)
    for i, t in enumerate(args[:-1] if name in ("rotary_append", "append_q8") else args):
        print(name, i, flush=True)
        bad = list(args)
        bad[i] = t.to_sparse()
        with pytest.raises((RuntimeError, TypeError, ValueError, NotImplementedError)):
            call(*bad)
    torch.cuda.synchronize()
    call(*args)
    torch.cuda.synchronize()
