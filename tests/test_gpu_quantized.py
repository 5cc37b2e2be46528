"""The write into the 8-bit cache and the way back against their definition in 64 bits: every byte of the cache is compared."""
import numpy as np
import pytest
import torch

import lmserve_amd as kvc
from oracle.q8_oracle import VALUES, Cache, group_bytes

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
GEOMETRIES = [(1, 16, 16), (8, 64, 16), (4, 128, 16), (5, 80, 32), (2, 256, 16), (3, 48, 64), (7, 112, 48), (2, 144, 16), (8, 128, 160)]


def pool(rng, pages, H, D, page):
    """Pages of any bytes, NaN codes among them; what a group's first place does not begin anew keeps exponents of the format."""
    raw = rng.integers(0, 256, (pages * page // 16, group_bytes(H, D)), dtype=np.uint8)
    raw[:, 32 * H * D:32 * H * D + 2 * H] = rng.integers(27, 248, (raw.shape[0], 2 * H))
    return raw.reshape(pages, -1)


def rows(rng, T, H, D, dtype, kind="normal"):
    x = rng.standard_normal((T, H, D)) * 2.0 ** rng.integers(-6, 7, (T, H, 1))
    if kind == "odd":
        # borders of the exponent, halves of steps, the type's smallest and largest numbers, zeros, infinities, NaN
        tiny, huge = (2.0 ** -133, 3e38) if dtype == "bf16" else (2.0 ** -24, 65504.0)
        special = np.array([448, -448, 449, 450, 464, 1.0625, 1.1875, -1.0625, 2.0 ** -9, 2.0 ** -10, 2.0 ** -11, 0.0, -0.0, tiny, -tiny,
                            huge, -huge, np.inf, -np.inf, np.nan])
        pick = rng.integers(0, len(special), x.shape)
        x = np.where(rng.random(x.shape) < 0.02, special[pick], x * 2.0 ** rng.integers(-12, 9, (T, 1, 1)))
        x[rng.random((T, H)) < 0.1] = 0
        x[rng.random((T, H)) < 0.05] = np.nan
        x[rng.random((T, H)) < 0.05] *= 2.0 ** -120
    return torch.from_numpy(x).to(TYPES[dtype])


class Step:
    """Requests of `page`-sized tables over a shuffled pool, and calls that write their tokens."""

    def __init__(self, lengths, H, D, page, dtype, seed, kind="normal"):
        self.rng = rng = np.random.default_rng(seed)
        self.H, self.D, self.page, self.dtype, self.kind = H, D, page, dtype, kind
        tables = [-(-n // page) for n in lengths]
        self.indptr = np.cumsum([0] + tables).astype(np.int32)
        self.pages = sum(tables) + 2
        self.indices = rng.permutation(self.pages)[:sum(tables)].astype(np.int32)
        self.have = [0] * len(lengths)
        self.raw = pool(rng, self.pages, H, D, page)
        self.oracle = Cache(self.raw, H, D)

    def call(self, new):
        """New tokens of every request -> (key, value, batch, positions, slots)."""
        batch = np.repeat(np.arange(len(new)), new).astype(np.int32)
        positions = np.concatenate([np.arange(h, h + n) for h, n in zip(self.have, new)]).astype(np.int32)
        self.have = [h + n for h, n in zip(self.have, new)]
        slots = self.indices[self.indptr[batch] + positions // self.page].astype(np.int64) * self.page + positions % self.page
        k, v = (rows(self.rng, len(batch), self.H, self.D, self.dtype, self.kind) for _ in range(2))
        self.oracle.write(k.double().numpy(), v.double().numpy(), slots)
        return k, v, batch, positions, slots

    def last(self):
        return np.array([(h - 1) % self.page + 1 if h else 0 for h in self.have], np.int32)

    def tables(self, dev):
        return [torch.from_numpy(x).to(dev) for x in (self.indices, self.indptr, self.last())]


def same(cache, oracle, what=""):
    got, want = cache.cpu().numpy(), oracle.pages()
    got, want = (x.reshape(-1, oracle.raw.shape[1]) for x in (got, want))
    bad = np.argwhere(got != want)
    assert not len(bad), f"{what}: {len(bad)} bytes differ, the first at {bad[0]} (of groups of {want.shape[1]}): " \
                         f"{got[tuple(bad[0])]} and not {want[tuple(bad[0])]}"


@pytest.mark.parametrize("kind", ["normal", "odd"])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("H,D,page", GEOMETRIES)
def test_calls_that_go_on_with_groups(gpu, H, D, page, dtype, kind):
    """Prompts, chunks and single tokens one call after another, by slots of both widths and by the page table."""
    s = Step([90, 17, 40, 16, 70], H, D, page, dtype, seed=H * D + page, kind=kind)
    cache = torch.from_numpy(s.raw).to(gpu)
    calls = [(33, 1, 5, 16, 1), (1, 1, 1, 0, 1), (20, 14, 1, 0, 30)] + [(1, 0, 1, 0, 1)] * 14
    for i, new in enumerate(calls):
        k, v, batch, positions, slots = s.call(new)
        k, v = k.to(gpu), v.to(gpu)
        if i % 3 == 0:
            kvc.append_paged_kv_cache_q8(k, v, torch.from_numpy(batch).to(gpu), torch.from_numpy(positions).to(gpu), cache, *s.tables(gpu))
        else:
            kvc.reshape_and_cache_q8(k, v, cache, torch.from_numpy(slots.astype(np.int64 if i % 3 == 1 else np.int32)).to(gpu))
        same(cache, s.oracle, f"call {i}")


@pytest.mark.parametrize("T,H,D,page", [(1, 1, 16, 16), (15, 2, 64, 32), (257, 8, 128, 16), (1000, 2, 80, 16), (5000, 1, 64, 64), (300, 40, 32, 16)])
def test_many_requests_and_long_ones(gpu, T, H, D, page):
    rng = np.random.default_rng(T)
    lengths = []
    while sum(lengths) < T:
        lengths.append(int(min(T - sum(lengths), rng.choice([1, 1, 2, 15, 16, 17, 400]))))
    s = Step([n + 20 for n in lengths], H, D, page, "bf16", seed=T)
    cache = torch.from_numpy(s.raw).to(gpu)
    for new in ([int(x) for x in rng.integers(0, 20, len(lengths))], lengths):
        k, v, _, _, slots = s.call(new)
        if len(slots):
            kvc.reshape_and_cache_q8(k.to(gpu), v.to(gpu), cache, torch.from_numpy(slots).to(gpu))
    same(cache, s.oracle)


def test_tokens_without_a_place(gpu):
    """Slots outside the cache, tokens outside a request's table: skipped, and they part the runs beside them."""
    H, D, page = 2, 64, 16
    s = Step([64], H, D, page, "bf16", seed=9)
    cache = torch.from_numpy(s.raw).to(gpu)
    p = s.indices.astype(np.int64) * page
    slots = np.array([p[0], p[0] + 1, -1, p[1] + 3, p[1] + 4, s.pages * page, -5, p[2], 1 << 40, p[3] + 15, -1 << 40], np.int64)
    k, v = (rows(s.rng, len(slots), H, D, "bf16") for _ in range(2))
    s.oracle.write(k.double().numpy(), v.double().numpy(), slots)
    kvc.reshape_and_cache_q8(k.to(gpu), v.to(gpu), cache, torch.from_numpy(slots).to(gpu))
    same(cache, s.oracle, "slots")
    # the same by a page table with ids that the cache does not have, positions beyond the table, requests that are not there
    batch = np.array([0, 0, -1, 1, 0, 0, 2, 0, 0], np.int32)
    positions = np.array([0, 1, 2, 3, 16, 32, 5, -1, 64], np.int32)
    indices, indptr = np.array([s.indices[3], -1, s.pages, 0, 7], np.int32), np.array([0, 3, 3], np.int32)
    k, v = (rows(s.rng, len(batch), H, D, "bf16") for _ in range(2))
    s.oracle.write(k.double().numpy(), v.double().numpy(), np.where(np.isin(np.arange(9), [0, 1]), p[3] + positions, -1))
    kvc.append_paged_kv_cache_q8(k.to(gpu), v.to(gpu), *[torch.from_numpy(x).to(gpu) for x in (batch, positions)], cache,
                                 *[torch.from_numpy(x).to(gpu) for x in (indices, indptr, np.zeros(2, np.int32))])
    same(cache, s.oracle, "page table")


def test_rows_of_a_projection_and_rows_that_have_to_be_copied(gpu):
    H, D, page = 4, 64, 16
    s = Step([40, 40, 40], H, D, page, "f16", seed=3)
    cache = torch.from_numpy(s.raw).to(gpu)
    for i in range(3):
        k, v, _, _, slots = s.call((10, 1, 12))
        slots = torch.from_numpy(slots).to(gpu)
        if i == 0:      # slices of one matrix
            both = torch.cat((k.flatten(1), v.flatten(1)), 1).to(gpu)
            k, v = both[:, :H * D].unflatten(1, (H, D)), both[:, H * D:].unflatten(1, (H, D))
        elif i == 1:    # heads apart, and rows at an odd address
            k = k.to(gpu).transpose(0, 1).contiguous().transpose(0, 1)
            v = torch.cat((v.flatten()[:1], v.flatten()))[1:].to(gpu)
            v = torch.empty(v.numel() + 1, dtype=v.dtype, device=gpu)[1:].copy_(v).view(-1, H, D)
        else:
            k, v = k.to(gpu), v.to(gpu)
        kvc.reshape_and_cache_q8(k, v, cache, slots)
        same(cache, s.oracle, str(i))


def test_pages_of_a_pool(gpu):
    """A layer of a pool whose pages lie apart; places beyond 2^31 bytes."""
    H, D, page = 8, 128, 16
    s = Step([30, 30], H, D, page, "bf16", seed=5)
    big = torch.empty(90000, 2, kvc.q8_page_bytes(H, D, page) // 2 + 64, dtype=torch.uint8, device=gpu)
    wide = big.view(90000, -1)[:, :kvc.q8_page_bytes(H, D, page)]
    assert wide.stride(0) > wide.shape[1]
    ids = np.array([3, 89999, 70001, 40000, 12345, 80000], np.int64)[:s.pages]
    wide[torch.from_numpy(ids).to(gpu)] = torch.from_numpy(s.raw).to(gpu)
    for new in ((17, 5), (3, 20)):
        k, v, _, _, slots = s.call(new)
        far = torch.from_numpy(ids[slots // page] * page + slots % page).to(gpu)
        kvc.reshape_and_cache_q8(k.to(gpu), v.to(gpu), wide, far)
        same(wide[torch.from_numpy(ids).to(gpu)], s.oracle)
    got = kvc.read_cache_q8(wide, far, H, D)
    want = s.oracle.values()[slots]
    for g, w in zip(got, (want[:, 0], want[:, 1])):
        assert torch.equal(g.cpu(), torch.from_numpy(w).to(torch.bfloat16))


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("H,D,page", GEOMETRIES)
def test_read_back(gpu, H, D, page, dtype):
    """Any bytes, in any order, more than once: the value that the code stands for, rounded once."""
    rng = np.random.default_rng(H + D)
    pages = 12
    raw = pool(rng, pages, H, D, page)
    oracle = Cache(raw, H, D)
    cache = torch.from_numpy(raw).to(gpu)
    order = np.concatenate([np.arange(pages * page), rng.integers(0, pages * page, 200), [-1, pages * page, 5, 5, 6, 7]])
    want = torch.from_numpy(oracle.values()[np.clip(order, 0, pages * page - 1)]).to(TYPES[dtype])
    skipped = torch.from_numpy((order < 0) | (order >= pages * page))
    want[skipped] = 7
    for slots in (order.astype(np.int64), order.astype(np.int32)):
        k, v = (torch.full((len(order), H, D), 7.0, dtype=TYPES[dtype], device=gpu) for _ in range(2))
        got = kvc.read_cache_q8(cache, torch.from_numpy(slots).to(gpu), H, D, TYPES[dtype], key=k, value=v)
        assert got[0] is k and got[1] is v
        for g, w in ((k, want[:, 0]), (v, want[:, 1])):
            assert torch.equal(torch.isnan(g.cpu()), torch.isnan(w)) and torch.equal(g.cpu().nan_to_num(1), w.nan_to_num(1))
    # by a page table: one request whose pages are shuffled
    table = rng.permutation(pages).astype(np.int32)
    positions = rng.permutation(pages * page)[:333].astype(np.int32)
    k, v = kvc.read_paged_kv_cache_q8(torch.zeros(333, dtype=torch.int32, device=gpu)[:len(positions)], torch.from_numpy(positions).to(gpu),
                                      cache, torch.from_numpy(table).to(gpu), torch.tensor([0, pages], dtype=torch.int32, device=gpu),
                                      torch.tensor([page], dtype=torch.int32, device=gpu), H, D, TYPES[dtype])
    want = torch.from_numpy(oracle.values()[table[positions // page] * page + positions % page]).to(TYPES[dtype])
    for g, w in ((k, want[:, 0]), (v, want[:, 1])):
        assert torch.equal(torch.isnan(g.cpu()), torch.isnan(w)) and torch.equal(g.cpu().nan_to_num(1), w.nan_to_num(1))


def test_what_was_written_comes_back_within_half_a_step(gpu):
    """A value is off by at most half a step of its code, 2^-4 of itself or 2^-10 of the scale; a group that was rounded again by a step."""
    H, D, page = 4, 64, 16
    s = Step([200], H, D, page, "bf16", seed=8)
    cache = torch.from_numpy(s.raw).to(gpu)
    k, v, _, _, slots = s.call((200,))
    at = torch.from_numpy(slots).to(gpu)
    kvc.reshape_and_cache_q8(k.to(gpu), v.to(gpu), cache, at)
    for got, x in zip(kvc.read_cache_q8(cache, at, H, D), (k, v)):
        x, got = x.double().numpy(), got.double().cpu().numpy()
        top = np.stack([np.abs(x[g:g + 16]).max((0, 2)) for g in range(0, 200, 16)]).repeat(16, 0)[:200, :, None]
        assert (np.abs(got - x) <= np.maximum(np.abs(x) * 2.0 ** -4, top / 224 * 2.0 ** -10)).all()


def test_slices_of_one_buffer_and_streams(gpu):
    """Reads into the two halves of one matrix; a write and a read on another stream; a recorded write and read, replayed."""
    H, D, page = 2, 64, 32
    s = Step([300, 300], H, D, page, "bf16", seed=4)
    cache = torch.from_numpy(s.raw).to(gpu)
    side = torch.cuda.Stream()
    k, v, _, _, slots = s.call((33, 50))
    at = torch.from_numpy(slots).to(gpu)
    k, v = k.to(gpu), v.to(gpu)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        kvc.reshape_and_cache_q8(k, v, cache, at)
        both = torch.empty(83, 2 * H * D, dtype=torch.bfloat16, device=gpu)
        kvc.read_cache_q8(cache, at, H, D, key=both[:, H * D:], value=both[:, :H * D])
    torch.cuda.current_stream().wait_stream(side)
    same(cache, s.oracle)
    want = torch.from_numpy(s.oracle.values()[slots]).to(torch.bfloat16).flatten(2)
    assert torch.equal(both.cpu(), torch.cat((want[:, 1], want[:, 0]), 1))
    # recorded, with buffers that are written anew before every replay; rows behind the step's have no slot
    key, value = torch.zeros(64, H, D, dtype=torch.bfloat16, device=gpu), torch.zeros(64, H, D, dtype=torch.bfloat16, device=gpu)
    where = torch.full((64,), -1, dtype=torch.int64, device=gpu)
    back_k, back_v = torch.zeros_like(key), torch.zeros_like(key)

    def body():
        kvc.reshape_and_cache_q8(key, value, cache, where)
        kvc.read_cache_q8(cache, where, H, D, key=back_k, value=back_v)
    with torch.cuda.stream(side):
        body()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        body()
    for new in ((1, 1), (40, 7), (1, 1), (2, 60), (1, 0)):
        k, v, _, _, slots = s.call(new)
        n = len(slots)
        where.fill_(-1)
        key[:n], value[:n], where[:n] = k.to(gpu), v.to(gpu), torch.from_numpy(slots).to(gpu)
        graph.replay()
        torch.cuda.synchronize()
        same(cache, s.oracle, str(new))
        want = torch.from_numpy(s.oracle.values()[slots]).to(torch.bfloat16)
        assert torch.equal(back_k[:n].cpu(), want[:, 0]) and torch.equal(back_v[:n].cpu(), want[:, 1])


def test_blocks_move_with_their_exponents(gpu):
    """Copy on write, gather and scatter, the swap to the host and back, on a pool of two layers."""
    H, D, page, L = 2, 64, 16, 2
    layers = [Step([100], H, D, page, "bf16", seed=20 + l) for l in range(L)]
    pool8 = kvc.allocate_q8_kv_caches(L, 16, page, H, D, gpu)
    assert pool8.shape == (L, 16, kvc.q8_page_bytes(H, D, page)) and pool8.dtype == torch.uint8
    pool8.zero_()
    slots = torch.arange(100, device=gpu)
    for l, s in enumerate(layers):
        k, v, *_ = s.call((100,))
        kvc.reshape_and_cache_q8(k.to(gpu), v.to(gpu), pool8[l], slots)
    before = [kvc.read_cache_q8(pool8[l], slots, H, D) for l in range(L)]
    kvc.copy_blocks(pool8, {i: [8 + i] for i in range(7)})
    worker = kvc.KVWorker(pool8, 16)
    try:
        worker.copy_kv_sync([kvc.BlockMapping.from_pairs((8 + i, i) for i in range(7))], kvc.Device.GPU, kvc.Device.Host)
        pool8.zero_()
        worker.copy_kv_sync([kvc.BlockMapping.from_pairs((i, 15 - i) for i in range(7))], kvc.Device.Host, kvc.Device.GPU)
    finally:
        worker.close()
    moved = (15 - slots // page) * page + slots % page
    for l in range(L):
        for a, b in zip(before[l], kvc.read_cache_q8(pool8[l], moved, H, D)):
            assert torch.equal(a, b)
    buffer = kvc.gather_blocks(pool8, torch.tensor([15, 14, 9], device=gpu))
    pool8.zero_()
    kvc.scatter_blocks(pool8, torch.tensor([1, 2, 3], device=gpu), buffer)
    for a, b in zip(before[1], kvc.read_cache_q8(pool8[1], slots[:32] + page, H, D)):
        assert torch.equal(a[:32], b)


def test_refusals(gpu):
    H, D, page = 2, 64, 16
    cache = kvc.allocate_q8_kv_caches(1, 4, page, H, D, gpu)[0]
    k = torch.zeros(3, H, D, dtype=torch.bfloat16, device=gpu)
    at = torch.arange(3, device=gpu)
    write = kvc.reshape_and_cache_q8
    for bad, error in (((k, k, cache[:, :-1], at), ValueError), ((k, k, cache.view(torch.int8), at), TypeError),
                       ((k, k, cache[None], at), ValueError), ((k, k[:2], cache, at), ValueError), ((k, k, cache, at[:2]), ValueError),
                       ((k.float(), k.float(), cache, at), TypeError), ((k, k.half(), cache, at), TypeError),
                       ((k.flatten(1), k, cache, at), ValueError), ((k, k[:, :1], cache, at), ValueError),
                       ((k[..., :8], k[..., :8], cache, at), TypeError), ((k.cpu(), k, cache, at), ValueError),
                       ((k, k, cache.cpu(), at), ValueError), ((k, k, cache, at.cpu()), ValueError)):
        with pytest.raises(error):
            write(*bad)
    inside = cache.view(torch.bfloat16)[0, :3 * H * D].view(3, H, D)
    with pytest.raises(ValueError, match="overlaps"):
        write(inside, k, cache, at)
    with pytest.raises(ValueError, match="overlaps"):
        kvc.read_cache_q8(cache, at, H, D, key=inside, value=k)
    with pytest.raises(ValueError, match="overlaps"):
        kvc.read_cache_q8(cache, at, H, D, key=k, value=k)
    with pytest.raises(TypeError):
        kvc.read_cache_q8(cache, at, H, D, torch.float32)
    with pytest.raises(ValueError):
        kvc.read_cache_q8(cache, at, H, D, torch.float16, key=k)
    with pytest.raises(ValueError):
        kvc.read_cache_q8(cache, at, H, D, key=k[:2])
    none = torch.zeros(0, H, D, dtype=torch.bfloat16, device=gpu)
    write(none, none, cache, at[:0])
    write(k, k, cache[:0], at)
    assert kvc.read_cache_q8(cache, at[:0], H, D)[0].shape == (0, H, D)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_large_calls_are_what_smaller_ones_are(gpu, dtype):
    """Sizes from which rows go past the caches, against the same tokens in calls below them."""
    H, D, page, T = 8, 128, 16, 33000
    g = torch.Generator(device=gpu).manual_seed(1)
    k, v = (torch.randn(T, H, D, generator=g, device=gpu).to(TYPES[dtype]) for _ in range(2))
    slots = torch.randperm(T // 16 + 9, generator=g, device=gpu)[torch.arange(T, device=gpu) // 16] * 16 + torch.arange(T, device=gpu) % 16
    one = kvc.allocate_q8_kv_caches(1, T // 16 + 9, page, H, D, gpu)[0]
    one.fill_(40)
    many = one.clone()
    kvc.reshape_and_cache_q8(k, v, one, slots)
    for t in range(0, T, 4000):
        kvc.reshape_and_cache_q8(k[t:t + 4000], v[t:t + 4000], many, slots[t:t + 4000])
    assert torch.equal(one, many)
    got = kvc.read_cache_q8(one, slots, H, D, TYPES[dtype])
    for t in range(0, T, 4000):
        for a, b in zip(got, kvc.read_cache_q8(one, slots[t:t + 4000], H, D, TYPES[dtype])):
            assert torch.equal(a[t:t + 4000], b)
    assert (got[0] - k).abs().max() < 0.3 and (got[1] - v).abs().max() < 0.3


def test_a_group_in_another_order_or_twice_harms_no_other(gpu):
    """Places of one group in falling order, twice, and in two parts of a call: its own contents are undefined, every other group's are right."""
    H, D, page = 4, 128, 32
    s = Step([64, 64], H, D, page, "bf16", seed=31)
    cache = torch.from_numpy(s.raw).to(gpu)
    base = s.indices.astype(np.int64) * page
    bad = [base[0] + 7, base[0] + 6, base[0] + 5, base[0] + 6, base[0] + 1, base[0] + 2, base[0] + 15, base[0] + 15]
    good = [base[1] + i for i in range(20)] + [base[2] + 16 + i for i in range(3)]
    slots = np.array(bad[:3] + good[:9] + bad[3:6] + good[9:] + bad[6:], np.int64)
    k, v = (rows(s.rng, len(slots), H, D, "bf16") for _ in range(2))
    keep = [i for i, t in enumerate(slots) if t not in bad]
    # (the good tokens are one run of the call with a break inside a group: what follows it goes on with the group)
    first, second = [i for i in keep if i < 12], [i for i in keep if i > 12]
    for part in (first, second):
        s.oracle.write(k[part].double().numpy(), v[part].double().numpy(), slots[part])
    for part in (slice(0, 12), slice(12, None)):
        kvc.reshape_and_cache_q8(k[part].to(gpu), v[part].to(gpu), cache, torch.from_numpy(slots[part]).to(gpu))
    group = group_bytes(H, D)
    got, want = cache.cpu().numpy().reshape(-1, group), s.oracle.pages().reshape(-1, group)
    others = np.delete(np.arange(len(got)), base[0] // 16)
    assert np.array_equal(got[others], want[others])
    back = kvc.read_cache_q8(cache, torch.from_numpy(slots[::-1].copy()).to(gpu), H, D)      # any order, twice the same
    where = torch.from_numpy(Cache(cache.cpu().numpy(), H, D).values()[slots[::-1]]).to(torch.bfloat16)
    for g, w in zip(back, (where[:, 0], where[:, 1])):
        assert torch.equal(torch.isnan(g.cpu()), torch.isnan(w)) and torch.equal(g.cpu().nan_to_num(1), w.nan_to_num(1))


def test_writes_on_two_streams_at_once(gpu):
    """Calls that write different groups of the same pages side by side."""
    H, D, page = 8, 64, 64
    s = Step([64 * 8], H, D, page, "f16", seed=32)
    cache = torch.from_numpy(s.raw).to(gpu)
    k, v = (rows(s.rng, 512, H, D, "f16") for _ in range(2))
    slots = (s.indices.astype(np.int64)[:, None] * page + np.arange(page)).ravel()
    s.oracle.write(k.double().numpy(), v.double().numpy(), slots)
    halves = [np.flatnonzero(np.arange(512) // 16 % 2 == h) for h in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    given = [(k[h].to(gpu), v[h].to(gpu), torch.from_numpy(slots[h]).to(gpu)) for h in halves]
    torch.cuda.synchronize()
    for _ in range(3):
        for stream, (a, b, at) in zip(streams, given):
            with torch.cuda.stream(stream):
                kvc.reshape_and_cache_q8(a, b, cache, at)
    torch.cuda.synchronize()
    same(cache, s.oracle)
