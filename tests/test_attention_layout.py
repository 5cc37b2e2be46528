"""The attention plan's capacities against the work that its layout can make of a step, without a GPU: what is cut must have
somewhere to be joined. The rules of the line of work are restated here."""
import ctypes
import random

import pytest

from lmserve_amd import _lib

TILE, TILE_WORK, MIN_SHARE, MIN_PART, MAX_GROUPS = 16, 64, 1024, 256, 1024


def ceil(a, b):
    return -(-a // b)


def plan_bytes(lens, hq, hk, d, page, max_q, pages=None, tokens=None):
    tokens = sum(n for n, _ in lens) if tokens is None else tokens
    pages = sum(ceil(k, page) for _, k in lens) if pages is None else pages
    h = ctypes.c_void_p()
    L = _lib.lib()
    assert L.kvc_attention_plan_create(4096, 8192, 12288, 16384, len(lens), tokens, pages, hq, hk, d, page, max_q, 0, d ** -0.5, 0,
                                       ctypes.byref(h)) == _lib.KVC_OK
    got = L.kvc_attention_plan_bytes(h)
    L.kvc_attention_plan_destroy(h)
    return got


def narrow_rows(lens, hq, hk, page, max_q, pages=None):
    rows = sum(n for n, _ in lens) * (hq // hk)
    pages = sum(ceil(k, page) for _, k in lens) if pages is None else pages
    most = 16 if rows * (pages * page // len(lens)) > 1 << 18 else 32
    return 1 << 31 if 0 < max_q * (hq // hk) <= most else most


def parts_of_narrow_tiles(lens, hq, hk, d, most, places=False):
    """How many parts every narrow tile of a step is cut into, its tiles end to end on the line of work; with `places` the last
    workgroup that has one as well."""
    group = hq // hk
    wide = sum(n for n, _ in lens) * group > most
    groups = max(1, min(MAX_GROUPS, (1024 if wide else 256 * (4 if d <= 64 else 2 if d <= 128 else 1)) // hk))
    tiles = []
    for n, k in lens:
        if n == 0 or n * group > most:
            continue

        def before(i):
            first = max(0, min(k, k - n + ceil(TILE, group)))
            return i * (first + TILE_WORK) + (i * (i - 1) // 2 * TILE // group if i >= 2 else 0)
        tiles += [before(i + 1) - before(i) for i in range(ceil(n * group, TILE))]
    share = max(ceil(sum(tiles), groups), MIN_SHARE)
    sliver = share // 2 if share <= MIN_SHARE else min(share // 2, MIN_PART)
    at, parts = 0, []
    for work in tiles:
        first = min((at + sliver - 1) // share, groups - 1)
        last = 0 if at + work < sliver else (at + work - sliver) // share
        count = max(last - first, 0) + 1
        parts.append((first + count - 1, count) if places else count)
        at += work
    return parts


def check(lens, hq, hk, d, page, max_q):
    """Where a tile is cut, the plan has room for its rows' entries: it is as large as one whose requests could have keys enough."""
    most = narrow_rows(lens, hq, hk, page, max_q)
    cut = max(parts_of_narrow_tiles(lens, hq, hk, d, most), default=1) > 1
    if cut:
        long = ceil(942, page)
        if narrow_rows(lens, hq, hk, page, max_q, long) != most:
            return False      # (other tiles with more keys: nothing to compare with)
        assert plan_bytes(lens, hq, hk, d, page, max_q) == plan_bytes(lens, hq, hk, d, page, max_q, pages=long), lens
    return cut


@pytest.mark.parametrize("lens,hq,hk,d,max_q", [
    ([(900, 900)], 32, 8, 128, 1), ([(600, 900)], 32, 8, 128, 1), ([(700, 700)], 32, 32, 256, 1), ([(900, 900)], 16, 2, 256, 2),
    ([(20, 704), (20, 224)], 128, 128, 256, 20), ([(1500, 100)], 8, 8, 128, 1), ([(3000, 0)], 2, 1, 64, 1)])
def test_tiles_that_are_cut_are_joined(lens, hq, hk, d, max_q):
    assert check(lens, hq, hk, d, 16, max_q)


def test_tiles_that_are_cut_are_joined_in_steps_as_they_come():
    rng, cuts = random.Random(5), 0
    for _ in range(4000):
        hk = rng.choice([1, 2, 8, 32, 128, 512])
        hq, d, page = hk * rng.choice([1, 2, 4, 7]), rng.choice([64, 128, 256]), rng.choice([1, 16, 20])
        left, lens = rng.randint(0, 941), []
        for _ in range(rng.randint(1, 8)):
            k = rng.randint(0, left)
            left -= k
            lens.append((rng.choice([0, 1, 3, 20, 200, 1500]) if rng.random() < .5 else min(k, rng.choice([1, 5, 20, 900])), k))
        cuts += check(lens, hq, hk, d, page, rng.choice([0, 1, 4, 20]))
    assert cuts > 200


def test_small_steps_need_no_join():
    """What cannot be cut has no entries: a decode step of short requests and a chunk of few tokens are one launch."""
    for lens, hq, hk, max_q in (([(1, 200)] * 4, 32, 8, 1), ([(1, 900)], 32, 8, 1), ([(1, 16)] * 50, 32, 8, 1), ([(4, 100)] * 4, 32, 8, 4)):
        rows = sum(n for n, _ in lens) * (hq // hk)
        long = ceil(1100, 16)
        assert narrow_rows(lens, hq, hk, 16, max_q, long) == narrow_rows(lens, hq, hk, 16, max_q)
        assert plan_bytes(lens, hq, hk, 128, 16, max_q, pages=long) - plan_bytes(lens, hq, hk, 128, 16, max_q) == ceil(rows * 32, 256) * 256


# ---- workspaces
def workspace(lens, hq, hk, d, page, max_q=0, shared=0, pages=None, tokens=None, batch=None):
    tokens = sum(n for n, _ in lens) if tokens is None else tokens
    pages = sum(ceil(k, page) for _, k in lens) if pages is None else pages
    h = ctypes.c_void_p()
    L = _lib.lib()
    assert L.kvc_attention_plan_create(4096, 8192, 12288, 16384, len(lens) if batch is None else batch, tokens, pages, hq, hk, d, page, max_q,
                                       shared, d ** -0.5, 0, ctypes.byref(h)) == _lib.KVC_OK
    got = L.kvc_attention_workspace_bytes(h)
    L.kvc_attention_plan_destroy(h)
    return got


MB = 1 << 20


@pytest.mark.parametrize("limit,tokens,batch,keys,hq,hk,d,max_q,shared", [
    (5 * MB, 20, 1, 900, 32, 8, 128, 0, 0), (1 * MB, 33, 1, 40, 32, 8, 128, 0, 0), (9 * MB, 20, 1, 900, 32, 8, 256, 0, 0),
    (9 * MB, 256, 256, 256 * 4096, 32, 8, 128, 1, 0), (190 * MB, 256, 256, 256 * 4096, 32, 8, 128, 0, 0),
    (180 * MB, 2048, 4, 4 * 32768, 28, 4, 128, 0, 0), (400 * MB, 16384, 256, 256 * 1024, 32, 8, 128, 0, 256),
    (300 * MB, 16384, 2, 32768, 32, 8, 128, 0, 64), (1 * MB, 1, 1, 4096, 1, 1, 64, 1, 0)])
def test_workspaces_are_what_a_step_can_need(limit, tokens, batch, keys, hq, hk, d, max_q, shared):
    assert 0 < workspace([(0, 0)], hq, hk, d, 16, max_q, shared, pages=keys // 16, tokens=tokens, batch=batch) <= limit


def slots_of_wide_tiles(lens, group, residents, most, chunk):
    """Slots that wide tiles take when no range is to be longer than `chunk`, one of the layout's candidates."""
    return sum(ceil(n * group, 128) * ceil(k, chunk) for n, k in lens if n * group > most and k > chunk)


def test_slots_of_wide_tiles_are_there_whatever_the_ranges_are():
    rng = random.Random(6)
    fullest = 0
    for _ in range(1500):
        hk, group, page = rng.choice([1, 4, 8, 64, 512]), rng.choice([1, 4, 7]), rng.choice([1, 16])
        d = 64
        lens = []
        for _ in range(rng.randint(1, 12)):
            n = rng.choice([0, 1, 5, 9, 33, 128, 700])
            lens.append((n, n + rng.choice([0, 10, 500, 1000, 5000, 40000])))
        most = narrow_rows(lens, hk * group, hk, page, 0)
        rows = sum(n for n, _ in lens) * group
        if rows <= most:
            continue
        residents, groups = max(1, 512 // hk), max(1, min(MAX_GROUPS, 1024 // hk))
        # (a line that may be longer than its least shares reaches every workgroup)
        parts = sum(ceil(k, page) * page for _, k in lens) > MIN_SHARE * groups
        work = sum(ceil(n * group, 128) * k for n, k in lens if n * group > most)
        have = workspace(lens, hk * group, hk, d, page)
        for x in range(64):
            chunk = ceil(max(512, ceil(work * 16, residents * (x + 1))), 64) * 64
            slots = slots_of_wide_tiles(lens, group, residents, most, chunk)
            need = (2 * groups * 16 * parts + slots * 128) * hk * (d + 1) * 4
            assert need <= have, (lens, hk, group, x)
            fullest = max(fullest, need / have)
    assert fullest > 0.9


def test_slots_of_shared_prefixes_are_there():
    """Every request's tokens are few and all share: a first part of every tile, of the prefix's tiles, and the prefix's ranges."""
    rng = random.Random(7)
    for _ in range(1500):
        hk, group, page, d = rng.choice([1, 4, 8, 64]), rng.choice([1, 4, 7]), rng.choice([1, 16]), 64
        shared = rng.choice([16, 512, 1024, 4096]) // page
        lens = [(rng.choice([0, 1, 2, 4]), shared * page + rng.randint(1, 300)) for _ in range(rng.randint(1, 300))]
        T = sum(n for n, _ in lens)
        if not T:
            continue
        most = narrow_rows(lens, hk * group, hk, page, 0)
        shares = [n for n, _ in lens if 0 < n * group <= most]
        rows = sum(shares) * group
        wide = rows > 128 or (rows > 16 and rows * shared * page > 1 << 18)
        groups = max(1, min(MAX_GROUPS, (1024 if T * group > most or wide else 1024) // hk))
        narrow = sum(ceil(n * group, 16) for n in shares) + (0 if wide else ceil(rows, 16))
        work = (ceil(rows, 128) * shared * page if wide else 0) + sum(ceil(n * group, 128) * k for n, k in lens if n * group > most)
        residents = max(1, 512 // hk)
        have = workspace(lens, hk * group, hk, d, page, 0, shared)
        for x in range(64):
            chunk = ceil(max(512, ceil(work * 16, residents * (x + 1))), 64) * 64
            slots = slots_of_wide_tiles(lens, group, residents, most, chunk) + (ceil(rows, 128) * ceil(shared * page, chunk) if wide else 0)
            assert ((2 * groups + narrow) * 16 + slots * 128) * hk * (d + 1) * 4 <= have, (lens, hk, group, x)


def test_slots_of_narrow_tiles_are_there():
    """The last part that leaves a partial is in one of the workgroups that have slots."""
    rng = random.Random(8)
    for _ in range(3000):
        hk, group, page, d = rng.choice([1, 2, 8, 64]), rng.choice([1, 4, 7]), rng.choice([1, 16]), 64
        lens = [(n, max(0, n + rng.choice([-5, 0, 50, 900, 3000, 20000]))) for n in
                (rng.choice([1, 1, 2, 8, 40, 900]) for _ in range(rng.randint(1, 20)))]
        max_q = rng.choice([0, 1, 2])
        most = narrow_rows(lens, hk * group, hk, page, max_q)
        if any(n * group > most for n, _ in lens):
            continue
        parts = parts_of_narrow_tiles(lens, hk * group, hk, d, most, True)
        last = max((group for group, count in parts if count > 1), default=-1)
        have = workspace(lens, hk * group, hk, d, page, max_q) // (16 * hk * (d + 1) * 4)
        assert 2 * (last + 1) <= have, (lens, hk, group)


def test_slots_of_the_longest_requests_are_there():
    """Requests of nearly 2^31 keys under so many rows that an even share of the work is a longer range than any request has: none is cut."""
    longest = (1 << 31) - 1 - 8192
    for hk, group, n, requests in ((1, 1, 1 << 20, 1), (8, 1, 1 << 20, 2), (1, 8, 1 << 22, 3)):
        lens = [(n, longest)] * requests
        residents = max(1, 512 // hk)
        work = sum(ceil(n * group, 128) * k for n, k in lens)
        assert ceil(work * 16, residents * 64) > longest
        have = workspace(lens, hk * group, hk, 64, 1024)
        for x in range(64):
            chunk = ceil(min(max(512, ceil(work * 16, residents * (x + 1))), longest), 64) * 64
            assert slots_of_wide_tiles(lens, group, residents, 32, chunk) * 128 * hk * 65 * 4 <= have, (lens, x)
