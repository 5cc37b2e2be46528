"""What the attention's and the normed rotation's C entries refuse before they launch anything, and the host arithmetic
beside them. Every call here returns before its first launch."""
import ctypes

import numpy as np
import pytest

import lmserve_amd as kvc
from lmserve_amd import _lib

OK, INVALID, UNSUPPORTED, STAGING = _lib.KVC_OK, _lib.KVC_ERR_INVALID_ARG, _lib.KVC_ERR_UNSUPPORTED, _lib.KVC_ERR_STAGING
BF16, F16, F32 = 0, 1, 2


def create(out, **kw):
    a = dict(qo=4096, idx=8192, ptr=12288, last=16384, batch=3, tokens=7, nidx=9, hq=8, hk=2, d=64, page=16, max_q=0, shared=0,
             scale=0.125, dtype=BF16)
    a.update(kw)
    return _lib.lib().kvc_attention_plan_create(*a.values(), ctypes.byref(out) if out is not None else None)


def test_dtype_codes_are_those_of_the_header():
    from lmserve_amd.rotary import _DTYPES
    import torch
    assert (_DTYPES[torch.bfloat16], _DTYPES[torch.float16], _DTYPES[torch.float32]) == (BF16, F16, F32)


@pytest.mark.parametrize("change,code,word", [
    (dict(dtype=F32), UNSUPPORTED, "dtype"), (dict(dtype=9), UNSUPPORTED, "dtype"), (dict(batch=-1), INVALID, "negative"),
    (dict(tokens=-1), INVALID, "negative"), (dict(nidx=-1), INVALID, "negative"), (dict(shared=-1), INVALID, "negative"),
    (dict(max_q=-1), INVALID, "negative"), (dict(hq=0), INVALID, "heads"), (dict(hk=0), INVALID, "heads"),
    (dict(hq=7), INVALID, "multiple"), (dict(hq=-8, hk=-2), INVALID, "heads"), (dict(d=0), UNSUPPORTED, "head_dim"),
    (dict(d=60), UNSUPPORTED, "head_dim"), (dict(d=264), UNSUPPORTED, "head_dim"), (dict(page=0), INVALID, "page_size"),
    (dict(page=(1 << 20) + 1), INVALID, "page_size"), (dict(scale=0.0), INVALID, "scale"), (dict(scale=-1.0), INVALID, "scale"),
    (dict(scale=float("inf")), INVALID, "scale"), (dict(scale=float("nan")), INVALID, "scale"),
    (dict(batch=1 << 24), UNSUPPORTED, "too many"), (dict(nidx=1 << 31), UNSUPPORTED, "too many"),
    (dict(tokens=1 << 28), UNSUPPORTED, "too many"), (dict(hq=1 << 16, hk=1 << 16), UNSUPPORTED, "too many"),
    (dict(qo=None), INVALID, "null"), (dict(idx=None), INVALID, "null"), (dict(ptr=None), INVALID, "null"),
    (dict(last=None), INVALID, "null")])
def test_plans_that_are_refused(change, code, word):
    h = ctypes.c_void_p(5)
    assert create(h, **change) == code and h.value is None
    assert word in _lib.last_error()


def test_runs_that_are_refused():
    L = _lib.lib()
    assert create(None) == INVALID
    h = ctypes.c_void_p()
    assert create(h) == OK and h.value
    need, work = L.kvc_attention_plan_bytes(h), L.kvc_attention_workspace_bytes(h)
    assert need > 0 and work > 0 and L.kvc_attention_plan_bytes(None) < 0 and L.kvc_attention_workspace_bytes(None) < 0
    assert L.kvc_attention_plan_build(None, 1 << 20, need, None) == INVALID
    assert L.kvc_attention_plan_build(h, None, need, None) == STAGING
    assert L.kvc_attention_plan_build(h, (1 << 20) + 16, need, None) == STAGING
    assert L.kvc_attention_plan_build(h, 1 << 20, need - 1, None) == STAGING
    page = 2 * 16 * 2 * 64
    good = dict(q=1 << 20, qs=512, cache=1 << 24, ps=page, pages=4, out=2 << 20, lse=None, ws=1 << 30, wb=work)

    def run(plan=h, **kw):
        a = dict(good)
        a.update(kw)
        return L.kvc_attention_plan_run(plan, *a.values(), None)

    assert run(plan=None) == INVALID
    assert run() == INVALID and "not built" in _lib.last_error()     # every other argument is in order
    for change, word in ((dict(q=None), "null"), (dict(out=None), "null"), (dict(ws=None), "null"), (dict(cache=None), "null"),
                         (dict(pages=-1), "geometry"), (dict(pages=1 << 31), "geometry"), (dict(ps=page - 8), "geometry"),
                         (dict(ps=1 << 31), "geometry"), (dict(qs=504), "stride"), (dict(q=(1 << 20) + 8), "aligned"),
                         (dict(qs=516), "aligned"), (dict(ps=page + 4), "aligned"), (dict(cache=(1 << 24) + 8), "aligned"),
                         (dict(out=(2 << 20) + 4), "aligned"), (dict(lse=(3 << 20) + 2), "aligned"), (dict(ws=(1 << 30) + 128), "aligned")):
        assert run(**change) == INVALID and word in _lib.last_error(), change
    assert run(wb=work - 1) == STAGING
    assert L.kvc_attention_plan_destroy(h) == OK and L.kvc_attention_plan_destroy(None) == OK


def test_empty_steps_need_no_launch():
    L = _lib.lib()
    for change in (dict(batch=0), dict(tokens=0), dict(batch=0, qo=None, idx=None, ptr=None, last=None, nidx=0)):
        h = ctypes.c_void_p()
        assert create(h, **change) == OK
        need = L.kvc_attention_plan_bytes(h)
        assert L.kvc_attention_plan_build(h, 1 << 20, need, None) == OK
        assert L.kvc_attention_plan_run(h, None, 0, None, 0, 0, None, None, None, 0, None) == OK
        L.kvc_attention_plan_destroy(h)


@pytest.mark.parametrize("tokens,batch,hq,hk,shared", [(1, 1, 1, 1, 0), (256, 256, 32, 8, 0), (2048, 4, 28, 4, 0), (256, 256, 32, 8, 256),
                                                       (8192, 512, 64, 64, 8), (100000, 100000, 8, 1, 0), (1, 1, 65535, 65535, 1)])
def test_sizes_of_plans_stay_in_bounds(tokens, batch, hq, hk, shared):
    """Workspaces grow with the rows of a launch's tiles, not with the contexts: below 2 GiB where the queries are below 0.5."""
    h = ctypes.c_void_p()
    assert create(h, tokens=tokens, batch=batch, hq=hq, hk=hk, d=128, nidx=1 << 20, shared=shared, max_q=0) == OK
    L = _lib.lib()
    assert 0 < L.kvc_attention_plan_bytes(h) < 1 << 30
    work = L.kvc_attention_workspace_bytes(h)
    assert 0 < work < (8 << 30)
    h2 = ctypes.c_void_p()
    assert create(h2, tokens=tokens, batch=batch, hq=hq, hk=hk, d=128, nidx=1 << 30, shared=shared, max_q=0) == OK
    assert L.kvc_attention_workspace_bytes(h2) == work
    L.kvc_attention_plan_destroy(h)
    L.kvc_attention_plan_destroy(h2)


def test_normed_rotations_that_are_refused():
    L = _lib.lib()
    good = dict(q=1 << 20, k=2 << 20, qw=3 << 20, kw=4 << 20, eps=1e-6, pos=7 << 20, pb=4, cs=8 << 20, maxp=100, tokens=4,
                hq=8, hk=2, d=64, rd=64, qs=512, ks=128, qo=5 << 20, ko=6 << 20, qos=512, kos=128, dtype=BF16)

    def run(**kw):
        a = dict(good)
        a.update(kw)
        return L.kvc_qk_norm_rotary_pos_emb(*a.values(), None)

    for change, code in ((dict(dtype=9), UNSUPPORTED), (dict(d=0), INVALID), (dict(q=None), INVALID), (dict(k=None), INVALID),
                         (dict(qw=None), INVALID), (dict(kw=None), INVALID), (dict(qo=None), INVALID), (dict(pos=None), INVALID),
                         (dict(pb=2), UNSUPPORTED), (dict(qs=504), INVALID), (dict(ks=64), INVALID), (dict(eps=-1.0), INVALID),
                         (dict(eps=float("nan")), INVALID), (dict(rd=66), INVALID), (dict(rd=63), INVALID), (dict(tokens=-1), INVALID),
                         (dict(qo=(1 << 20) + 2), INVALID), (dict(qo=2 << 20), INVALID), (dict(ko=1 << 20), INVALID)):
        assert run(**change) == code, change
    assert run(tokens=0) == OK


def test_common_prefix_pages():
    f = kvc.common_prefix_pages
    assert f([]) == 0 and f([[1, 2, 3]]) == 3 and f([[1, 2, 3], []]) == 0
    assert f([[1, 2, 3], [1, 2, 4], [1, 2]]) == 2
    assert f([[1, 2, 3], [1, 9, 3], [1, 2, 3]]) == 1
    assert f([[5, 2], [4, 2]]) == 0
    assert f(t for t in ([7] * 4, [7] * 6)) == 4
    assert f([np.arange(1000, dtype=np.int32), list(range(999)) + [5, 6]]) == 999


def test_what_is_written_may_not_be_what_is_read():
    """The arrays beside the rows, against everything that is written: index arrays and the attention plan's buffer; the norm's
    weights, tables and indices and its outputs and cache planes. (A run of the attention needs a plan that was built.)"""
    L = _lib.lib()
    h = ctypes.c_void_p()
    assert create(h) == OK
    need = L.kvc_attention_plan_bytes(h)
    for at in (4096, 8192, 12288, 16384):        # the index arrays that `create` gives
        at = at // 256 * 256
        assert L.kvc_attention_plan_build(h, at, need, None) == INVALID and "overlaps" in _lib.last_error()
    L.kvc_attention_plan_destroy(h)
    page = 2 * 16 * 2 * 64 * 2
    good = dict(q=1 << 20, k=2 << 20, v=3 << 20, qw=4 << 20, kw=5 << 20, eps=1e-6, pos=6 << 20, pb=4, cs=7 << 20, maxp=100, tokens=4,
                hq=8, hk=2, d=64, rd=64, qs=512, ks=128, vs=128, qo=8 << 20, ko=9 << 20, qos=512, kos=128, kc=16 << 20,
                vc=(16 << 20) + page // 2, slots=10 << 20, sb=8, bs=16, bstride=page // 2, sstride=128, nb=8, dtype=BF16)

    def run(**kw):
        a = dict(good)
        a.update(kw)
        return L.kvc_qk_norm_rotary_pos_emb_and_cache(*a.values(), None)

    ends = dict(qw=128, kw=128, pos=16, cs=100 * 2 * 64 * 2, slots=32)      # bytes of the arrays
    outs = dict(qo=4 * 512 * 2, ko=4 * 128 * 2, kc=8 * page, vc=8 * page - page // 2)
    for array, n in ends.items():
        for out in outs:
            at = good[out] if out != "vc" else good["kc"] + page // 2
            for where in (at, at + 16, at - n + 16):
                if out == "vc" and where < good["vc"]:
                    continue
                assert run(**{array: where}) == INVALID and "overlaps" in _lib.last_error(), (array, out, where - at)
    paged = dict(q=1 << 20, k=2 << 20, v=3 << 20, qw=4 << 20, kw=5 << 20, eps=1e-6, batch=6 << 20, pos=7 << 20, cs=8 << 20, maxp=100,
                 nnz=4, hq=8, hk=2, d=64, rd=64, qs=512, ks=128, vs=128, qo=9 << 20, ko=10 << 20, qos=512, kos=128, cache=16 << 20,
                 idx=11 << 20, ptr=12 << 20, b=3, n=9, page=16, stride=page // 2, pages=8, dtype=BF16)
    for array in ("qw", "kw", "batch", "pos", "cs", "idx", "ptr"):
        for out in ("qo", "ko", "cache"):
            a = dict(paged)
            a[array] = paged[out] + 16
            assert L.kvc_qk_norm_rotary_pos_emb_and_append_paged(*a.values(), None) == INVALID and "overlaps" in _lib.last_error(), (array, out)
