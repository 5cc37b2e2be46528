"""The 8-bit cache's sizes, its oracle's pinning, and what its C entries refuse before they launch anything."""
import numpy as np
import pytest
import torch

import lmserve_amd as kvc
from lmserve_amd import _lib
from oracle import q8_oracle as qo

OK, INVALID, UNSUPPORTED = _lib.KVC_OK, _lib.KVC_ERR_INVALID_ARG, _lib.KVC_ERR_UNSUPPORTED


def test_sizes():
    assert kvc.q8_page_bytes(8, 128, 16) == 2 * 16 * 8 * 128 + 128
    assert kvc.q8_page_bytes(8, 128, 64) == 4 * kvc.q8_page_bytes(8, 128, 16)
    assert kvc.q8_page_bytes(1, 16, 16) == 640 and kvc.q8_page_bytes(65, 16, 16) == 33280 + 256
    for bad in ((0, 128, 16), (8, 120, 16), (8, 0, 16), (8, 272, 16), (8, 128, 24), (8, 128, 0), (70000, 16, 16)):
        with pytest.raises((TypeError, ValueError)):
            kvc.q8_page_bytes(*bad)
    plan = kvc.plan_q8_cache(1 << 30, 1 << 31, 0, 32, 8, 128, 16)
    assert plan.num_gpu_blocks == (1 << 30) // (32 * 32896) and plan.num_host_blocks == (1 << 31) // (32 * 32896)
    assert plan.num_disk_blocks == 0 and plan.kv_block_size * 2 == 32896
    assert kvc.allocate_q8_kv_caches(2, 3, 32, 4, 64, device="cpu").shape == (2, 3, kvc.q8_page_bytes(4, 64, 32))


def test_the_oracle_rounds_as_the_type_does():
    """Against torch's own conversion: every code, halves between them and what lies next to these."""
    values = qo.VALUES
    assert np.array_equal(values, torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy(), equal_nan=True)
    codes = values[:127]
    half = (codes[1:] + codes[:-1]) / 2
    x = np.concatenate([codes, half, np.nextafter(half, 0), np.nextafter(half, 448), half * (1 + 2.0 ** -20), half * (1 - 2.0 ** -20)])
    x = np.concatenate([x, -x])
    want = torch.from_numpy(x).to(torch.float32)
    assert np.array_equal(qo.encode(want.double().numpy()), want.to(torch.float8_e4m3fn).view(torch.uint8).numpy())
    assert qo.exponent(448.0) == 0 and qo.exponent(np.nextafter(448.0, 500)) == 1 and qo.exponent(0.0) == -100
    assert qo.exponent(3.4e38) == 120 and qo.exponent(224.0) == -1


def test_the_oracle_keeps_places_apart():
    rng = np.random.default_rng(0)
    raw = rng.integers(0, 256, (3, qo.group_bytes(3, 32) * 2), dtype=np.uint8)
    c = qo.Cache(raw, 3, 32)
    assert np.array_equal(c.pages(), raw)
    # the header's formula, byte by byte
    for _ in range(200):
        g, t, h, d = rng.integers(6), rng.integers(16), rng.integers(3), rng.integers(32)
        group = raw.reshape(6, -1)[g]
        assert c.codes[g * 16 + t, 0, h, d] == group[(((h * 4 + t // 4) * 2 + d // 16) * 4 + t % 4) * 16 + d % 16]
        assert c.codes[g * 16 + t, 1, h, d] == group[16 * 3 * 32 + (h * 32 + d) * 16 + t]
        assert c.exponents[g, h, 1] == int(group[2 * 16 * 3 * 32 + 2 * h + 1]) - 127


def test_calls_that_are_refused():
    L = _lib.lib()
    page = kvc.q8_page_bytes(2, 64, 32)
    write = dict(k=1 << 20, v=2 << 20, cache=16 << 20, slots=3 << 20, sb=8, n=5, h=2, d=64, page=32, ks=128, vs=128, ps=page, pages=4, dtype=0)
    read = dict(cache=16 << 20, slots=3 << 20, sb=8, k=1 << 20, v=2 << 20, n=5, h=2, d=64, page=32, ks=128, vs=128, ps=page, pages=4, dtype=0)
    append = dict(k=1 << 20, v=2 << 20, batch=3 << 20, pos=4 << 20, cache=16 << 20, idx=5 << 20, ptr=6 << 20, last=None, n=5, b=2, ni=9,
                  h=2, d=64, page=32, ks=128, vs=128, ps=page, pages=4, dtype=0)
    back = dict(batch=3 << 20, pos=4 << 20, cache=16 << 20, idx=5 << 20, ptr=6 << 20, last=None, k=1 << 20, v=2 << 20, n=5, b=2, ni=9,
                h=2, d=64, page=32, ks=128, vs=128, ps=page, pages=4, dtype=0)
    common = [(dict(h=0), INVALID), (dict(h=-2), INVALID), (dict(h=70000), INVALID), (dict(d=8), UNSUPPORTED), (dict(d=0), UNSUPPORTED),
              (dict(d=72), UNSUPPORTED), (dict(d=272), UNSUPPORTED), (dict(page=24), UNSUPPORTED), (dict(page=0), UNSUPPORTED),
              (dict(page=-16), UNSUPPORTED), (dict(page=1 << 21), UNSUPPORTED), (dict(n=-1), INVALID), (dict(pages=-1), INVALID),
              (dict(pages=1 << 31), INVALID), (dict(ps=page - 16), INVALID), (dict(ps=1 << 32), INVALID), (dict(ps=page + 8), INVALID),
              (dict(ks=120), INVALID), (dict(vs=127), INVALID), (dict(ks=129), INVALID), (dict(dtype=2), UNSUPPORTED), (dict(dtype=-1), UNSUPPORTED),
              (dict(k=None), INVALID), (dict(v=None), INVALID), (dict(cache=None), INVALID), (dict(k=(1 << 20) + 8), INVALID),
              (dict(cache=(16 << 20) + 8), INVALID), (dict(k=(16 << 20) + 64), INVALID), (dict(v=(16 << 20) - 16), INVALID)]
    for fn, good, more in (
            (L.kvc_reshape_and_cache_q8, write, [(dict(slots=None), INVALID), (dict(sb=2), UNSUPPORTED), (dict(slots=16 << 20), INVALID)]),
            (L.kvc_read_cache_q8, read, [(dict(slots=None), INVALID), (dict(sb=1), UNSUPPORTED), (dict(slots=1 << 20), INVALID),
                                         (dict(v=1 << 20), INVALID), (dict(v=(1 << 20) + 1024), INVALID)]),
            (L.kvc_append_paged_kv_cache_q8, append, [(dict(batch=None), INVALID), (dict(pos=None), INVALID), (dict(idx=None), INVALID),
                                                      (dict(ptr=None), INVALID), (dict(b=-1), INVALID), (dict(ni=1 << 31), INVALID),
                                                      (dict(idx=(16 << 20) + 4), INVALID)]),
            (L.kvc_read_paged_kv_cache_q8, back, [(dict(batch=None), INVALID), (dict(idx=(2 << 20) + 4), INVALID), (dict(ptr=1 << 20), INVALID)])):
        for change, code in common + more:
            a = dict(good)
            a.update(change)
            assert fn(*a.values(), None) == code, (fn.__name__, change, _lib.last_error())
            assert fn.__name__ in _lib.last_error()
        for change in (dict(n=0), dict(pages=0)):
            a = dict(good)
            a.update(change)
            assert fn(*a.values(), None) == OK, change


def test_no_cpu_path():
    k = torch.zeros(3, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="GPU"):
        kvc.reshape_and_cache_q8(k, k, torch.zeros(2, kvc.q8_page_bytes(2, 64, 16), dtype=torch.uint8), torch.arange(3))


def test_attention_plans_over_8_bits_that_are_refused():
    import ctypes
    L = _lib.lib()
    good = dict(qo=4096, idx=8192, ptr=12288, last=16384, batch=3, tokens=7, nidx=9, hq=8, hk=2, d=64, page=32, max_q=0, shared=0,
                scale=0.125, dtype=0)

    def create(fn, **kw):
        a = dict(good)
        a.update(kw)
        h = ctypes.c_void_p()
        return fn(*a.values(), ctypes.byref(h)), h

    for change, code in ((dict(d=72), UNSUPPORTED), (dict(d=8), UNSUPPORTED), (dict(d=272), UNSUPPORTED), (dict(page=20), UNSUPPORTED),
                         (dict(page=8), UNSUPPORTED), (dict(page=0), INVALID), (dict(dtype=2), UNSUPPORTED), (dict(hq=7), INVALID),
                         (dict(scale=0.0), INVALID), (dict(batch=-1), INVALID), (dict(qo=None), INVALID),
                         (dict(page=1 << 20, hk=64, hq=64, d=256), UNSUPPORTED)):
        rc, h = create(L.kvc_attention_plan_create_q8, **change)
        assert rc == code and h.value is None, change
        assert "kvc_attention_plan_create_q8" in _lib.last_error()
    rc, h = create(L.kvc_attention_plan_create_q8)
    rc16, h16 = create(L.kvc_attention_plan_create)
    assert rc == rc16 == OK
    work, page = L.kvc_attention_workspace_bytes(h), kvc.q8_page_bytes(2, 64, 32)
    run = dict(q=1 << 20, qs=512, cache=1 << 24, ps=page, pages=4, out=2 << 20, lse=None, ws=1 << 30, wb=work)

    def go(fn, plan, **kw):
        a = dict(run)
        a.update(kw)
        return fn(plan, *a.values(), None)

    assert go(L.kvc_attention_plan_run_q8, None) == INVALID
    for fn, plan, bits in ((L.kvc_attention_plan_run_q8, h16, 16), (L.kvc_attention_plan_run, h, 8)):
        assert go(fn, plan) == INVALID and f"{bits} bits" in _lib.last_error()
    assert go(L.kvc_attention_plan_run_q8, h) == INVALID and "not built" in _lib.last_error()     # every other argument is in order
    for change, word in ((dict(q=None), "null"), (dict(out=None), "null"), (dict(cache=None), "null"), (dict(ps=page - 16), "geometry"),
                         (dict(ps=1 << 32), "geometry"), (dict(pages=-1), "geometry"), (dict(qs=504), "stride"), (dict(ps=page + 8), "aligned"),
                         (dict(cache=(1 << 24) + 8), "aligned"), (dict(q=(1 << 20) + 8), "aligned"), (dict(ws=(1 << 30) + 64), "aligned")):
        assert go(L.kvc_attention_plan_run_q8, h, **change) == INVALID and word in _lib.last_error(), change
    assert go(L.kvc_attention_plan_run_q8, h, wb=work - 1) == _lib.KVC_ERR_STAGING
    for x in (h, h16):
        L.kvc_attention_plan_destroy(x)


def test_blocks_of_bytes_on_disk(tmp_path):
    """The disk tier holds 8-bit blocks as bytes."""
    rng = np.random.default_rng(0)
    shape = (6, 2, kvc.q8_page_bytes(2, 64, 16))
    host = rng.integers(0, 256, shape, dtype=np.uint8)
    tier = kvc.DiskTier(str(tmp_path / "blocks.npy"), shape, np.uint8)
    try:
        tier.save_blocks(host, np.array([0, 3, 5]), np.array([4, 1, 0]))
        back = np.zeros_like(host)
        tier.load_blocks(back, np.array([4, 1, 0]), np.array([2, 1, 4]))
    finally:
        tier.close()
    assert np.array_equal(back[[2, 1, 4]], host[[0, 3, 5]]) and not back[[0, 3, 5]].any()
