"""Calls of the operators of a paged cache that is held in 8 bits, as a forward pass makes them.

`write`: keys and values of a step are quantised as they are written. `read`: cached keys and values come back in 16 bits, as
a hand-over to a worker with a 16-bit cache wants them. `attention`: the queries of a step over the 8-bit cache, causal, with
fewer key/value heads than query heads; where `shared` is given, the first `shared` tokens of every request lie in the same pages.

The cache: a page is `page / 16` groups of 16 tokens. A group holds, one after another, the codes (8-bit floating point with 4
bits of exponent and 3 of mantissa) of K and of V and their exponents, padded to whole 128 bytes:
    K [head][token / 4][dim / 16][token % 4][dim % 16],  V [head][dim][token],  exponents [head][K, V], plus 127.
A value is its code times 2 to the power of its exponent, one for the 16 tokens, a head, and K or V: the least from -100 on with which the
largest magnitude of the group's tokens is at most 448. A group's first token begins it anew; where a later call adds
tokens, the exponent may grow, and what the group holds is then rounded to the coarser codes.

`run` is either the plain form in elementary torch operations, or the calls of this package."""
import random

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
GROUP, LEAST, MOST, LARGEST = 16, -100, 120, 448.0
_F8 = torch.float8_e4m3fn


def _rows(name, op, form, tokens, requests, kv_heads, head_dim, dtype, page=16, behind=0):
    c = {"op": op, "form": form, "tokens": tokens, "requests": requests, "kv_heads": kv_heads, "head_dim": head_dim,
         "dtype": dtype, "page": page, "behind": behind}
    return dict(c, name=name) if name else c


def _attn(name, requests, chunk_requests, chunk, low, high, shared, heads, kv_heads, head_dim, dtype, page=16,
          plan=True, lse=False, lengths=0):
    c = {"op": "attention", "requests": requests, "chunk_requests": chunk_requests, "chunk": chunk, "low": low,
         "high": high, "shared": shared, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, "dtype": dtype,
         "page": page, "plan": plan, "lse": lse, "lengths": lengths}
    return dict(c, name=name) if name else c


def listed():
    return [
        # one token of one request, into a group that holds some already: what a layer pays when nobody else is served
        _rows("write-one-token", "write", "paged", 1, 1, 4, 128, "bf16", behind=901),
        # a decode step of a full batch, by the slots that a step keeps for all its layers
        _rows("write-decode-256", "write", "slots", 256, 256, 8, 128, "bf16", behind=1000),
        # a prefill chunk of three requests behind what they have, heads of 80, larger pages
        _rows("write-odd-heads", "write", "paged", 717, 3, 5, 80, "f16", page=32, behind=77),
        # a long prompt at once
        _rows("write-prompt-16384", "write", "slots", 16384, 2, 8, 128, "bf16"),
        # a short context
        _rows("read-one-request", "read", "paged", 900, 1, 8, 64, "f16"),
        # the contexts of a prefill's requests, for a decode worker with a 16-bit cache
        _rows("read-contexts-131001", "read", "slots", 131001, 7, 8, 128, "bf16"),
        # one request with a short context: latency; the index tensors are new with every call
        _attn("attend-one-request", 1, 0, 0, 900, 900, 0, 32, 8, 64, "bf16", plan=False),
        # a decode step of a full batch, contexts as they come
        _attn("attend-decode-256", 256, 0, 0, 1, 4095, 0, 32, 8, 128, "bf16"),
        # one request far into a long document
        _attn("attend-long-document", 1, 0, 0, 131001, 131001, 0, 64, 8, 128, "bf16", lse=True),
        # a decode step behind one long system prompt
        _attn("attend-shared-prompt", 256, 0, 0, 1, 512, 4096, 32, 8, 128, "bf16"),
        # a prefill chunk of four requests with long contexts behind them
        _attn("attend-chunks-2048", 4, 4, 512, 1024, 32768, 0, 28, 4, 128, "bf16"),
        # chunks and single tokens in one step, behind a shared prompt, larger pages
        _attn("attend-mixed-step", 63, 3, 259, 300, 2500, 1024, 32, 8, 64, "f16", page=32, lse=True),
    ]


def _spread(rng, low, high):
    """Spread over the logarithm, both ends included."""
    return max(low, min(high, round(low * (high / low) ** rng.random())))


def draw(rng):
    heads, kv_heads, head_dim = rng.choice([(32, 8, 64), (32, 8, 128), (28, 4, 128), (64, 8, 128), (8, 1, 128),
                                            (32, 32, 128), (40, 8, 80), (15, 5, 80), (16, 2, 256), (7, 7, 64)])
    page = rng.choice([16, 16, 16, 32, 64, 48])
    dtype = rng.choice(["bf16", "f16"])
    kind = rng.choice(["write", "write", "read", "decode", "shared", "chunks", "mixed"])
    if kind in ("write", "read"):
        tokens = _spread(rng, 1, min(16384 if kind == "write" else 131072, (1 << 27) // (kv_heads * head_dim)))
        return _rows(None, kind, rng.choice(["slots", "paged"]), tokens, rng.randint(1, min(tokens, 256)), kv_heads,
                     head_dim, dtype, page, rng.choice([0, rng.randint(1, 999)]))
    lengths, plan, lse = rng.randint(0, 999), rng.random() < 0.8, rng.random() < 0.5
    if kind == "chunks":
        requests, chunk = rng.randint(1, 4), _spread(rng, 2, 512)
        high = _spread(rng, chunk, 16384)
        return _attn(None, requests, requests, chunk, chunk, high, 0, heads, kv_heads, head_dim, dtype, page, plan, lse,
                     lengths)
    if kind == "mixed":
        chunk = _spread(rng, 2, 400)
        return _attn(None, rng.randint(4, 60), rng.randint(1, 3), chunk, chunk, chunk + _spread(rng, 1, 2000),
                     page * rng.choice([0, 5, 20]), heads, kv_heads, head_dim, dtype, page, plan, lse, lengths)
    requests = _spread(rng, 1, 256)
    high = _spread(rng, 1, min(131072, 400000 // requests))
    if kind == "decode":
        return _attn(None, requests, 0, 0, max(1, high // 3), high, 0, heads, kv_heads, head_dim, dtype, page, plan, lse,
                     lengths)
    high = min(high, 1000)
    return _attn(None, requests, 0, 0, 1, high, page * _spread(rng, 1, 4096 // page), heads, kv_heads, head_dim, dtype,
                 page, plan, lse, lengths)


# ---------------------------------------------------------------- the cache
def _group_bytes(heads, dim):
    return -(-(2 * GROUP * heads * dim + 2 * heads) // 128) * 128


def _values(cache, heads, dim):
    """The cache's contents as the numbers they are: codes `[groups, codes of a group]`, exponents plus 127 `[groups, heads, 2]`."""
    groups = cache.view(-1, _group_bytes(heads, dim))
    codes = 2 * GROUP * heads * dim
    return {"codes": groups[:, :codes].view(_F8), "exponents": groups[:, codes:codes + 2 * heads].reshape(-1, heads, 2)}


def _exponent(top):
    """The least exponent with which magnitudes up to `top` are at most 448 = 0.875 * 2**9."""
    mantissa, power = torch.frexp(top)
    return torch.where(top > 0, power - 9 + (mantissa > 0.875), LEAST).clamp(LEAST, MOST)


def _power(exponent):
    """2**exponent, exactly."""
    return torch.ldexp(torch.ones((), device="cuda"), exponent)


def _put(groups, at, k, v, exponents):
    """Codes `[n, 16, H, D]` and exponents `[n, H, 2]` into groups `[N, bytes]`."""
    n, _, H, D = k.shape
    half = GROUP * H * D
    groups[at, :half] = k.view(torch.uint8).reshape(n, 4, 4, H, D // 16, 16).permute(0, 3, 1, 4, 2, 5).reshape(n, half)
    groups[at, half:2 * half] = v.view(torch.uint8).permute(0, 2, 3, 1).reshape(n, half)
    groups[at, 2 * half:2 * half + 2 * H] = (exponents + 127).to(torch.uint8).reshape(n, 2 * H)


def _get(groups, at, H, D):
    """Codes of K and V as bytes `[n, 16, H, D]` and exponents `[n, H, 2]` of groups `[N, bytes]`."""
    half = GROUP * H * D
    rows = groups[at]
    n = rows.shape[0]
    k = rows[:, :half].reshape(n, H, 4, D // 16, 4, 16).permute(0, 2, 4, 1, 3, 5).reshape(n, GROUP, H, D)
    v = rows[:, half:2 * half].reshape(n, H, D, GROUP).permute(0, 3, 1, 2)
    return k, v, rows[:, 2 * half:2 * half + 2 * H].reshape(n, H, 2).int() - 127


# ---------------------------------------------------------------- inputs
def _lengths(case):
    """(new tokens, context length) of every request: by the case alone."""
    if case["op"] != "attention":
        rng, B, T = random.Random(case["behind"]), case["requests"], case["tokens"]
        new = [T // B + (1 if b < T % B else 0) for b in range(B)]
        return [(n, n + rng.randint(0, case["behind"])) for n in new]
    rng = random.Random(case["lengths"])
    out = []
    for b in range(case["requests"]):
        new = case["chunk"] if b < case["chunk_requests"] else 1
        out.append((new, case["shared"] + max(new, rng.randint(case["low"], case["high"]))))
    return out


def _normal(gen, shape, dtype):
    return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32).to(dtype)


def _filled(gen, pages, page, H, D):
    """A cache whose every token was written: heads of other sizes, some columns of K larger than the rest."""
    groups = torch.zeros(pages * page // GROUP, _group_bytes(H, D), dtype=torch.uint8, device="cuda")
    size = torch.exp2(torch.randint(-2, 3, (2, H, 1), generator=gen, device="cuda").float())
    size = size * (1 + 3 * (torch.rand(2, H, D, generator=gen, device="cuda") < 0.03).float())
    size[0] /= size[0].square().mean(dim=1, keepdim=True).sqrt()
    step = max(1, (1 << 26) // (GROUP * H * D))
    for g in range(0, groups.shape[0], step):
        n = min(step, groups.shape[0] - g)
        codes, exponents = [], []
        for which in range(2):
            x = torch.randn(n, GROUP, H, D, generator=gen, device="cuda") * size[which]
            e = _exponent(x.abs().amax(dim=(1, 3)))
            codes.append((x * _power(-e)[:, None, :, None]).to(_F8))
            exponents.append(e)
        _put(groups, slice(g, g + n), codes[0], codes[1], torch.stack(exponents, dim=2))
    return groups.view(pages, -1)


def _tables(case, gen):
    page, lengths = case["page"], _lengths(case)
    common = case.get("shared", 0) // page
    tables = [-(-n // page) for _, n in lengths]
    pages = common + sum(t - common for t in tables) + 3
    order = torch.randperm(pages, generator=gen, device="cuda")
    parts, at = [], common
    for t in tables:
        parts += [order[:common], order[at:at + t - common]]
        at += t - common
    i32 = dict(dtype=torch.int32, device="cuda")
    new = [n for n, _ in lengths]
    return {"lengths": lengths, "tables": tables, "pages": pages, "indices": torch.cat(parts).to(torch.int32),
            "indptr": torch.tensor([sum(tables[:b]) for b in range(len(tables) + 1)], **i32),
            "last": torch.tensor([(n - 1) % page + 1 for _, n in lengths], **i32),
            "qo_indptr": torch.tensor([sum(new[:b]) for b in range(len(new) + 1)], **i32)}


def _rows_tensors(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    T, H, D, page = case["tokens"], case["kv_heads"], case["head_dim"], case["page"]
    s = _tables(case, gen)
    new = torch.tensor([n for n, _ in s["lengths"]], device="cuda")
    start = torch.tensor([n - k for k, n in s["lengths"]], device="cuda")
    batch = torch.repeat_interleave(torch.arange(len(s["lengths"]), device="cuda"), new)
    positions = torch.arange(T, device="cuda") - s["qo_indptr"][batch] + start[batch]
    slots = s["indices"][s["indptr"][batch] + positions // page].long() * page + positions % page
    s.update(batch=batch.to(torch.int32), positions=positions.to(torch.int32), slots=slots,
             cache=_filled(gen, s["pages"], page, H, D))
    if case["op"] == "write":
        # rows as a fused projection leaves them: slices of one matrix
        qkv = _normal(gen, (T, 6 * H * D), _TYPES[case["dtype"]])
        s.update(key=qkv[:, 4 * H * D:5 * H * D].unflatten(1, (H, D)), value=qkv[:, 5 * H * D:].unflatten(1, (H, D)))
        # for the plain form: the groups that are written, each one's first new token, and the group of every token
        group, member = torch.unique_consecutive(slots // GROUP, return_inverse=True)
        first = torch.full_like(group, GROUP).scatter_reduce_(0, member, slots % GROUP, "amin")
        s.update(group=group, member=member, first=first)
    return s


def _attention_tensors(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    D, hq, hk = case["head_dim"], case["heads"], case["kv_heads"]
    s = _tables(case, gen)
    tokens = sum(n for n, _ in s["lengths"])
    s["query"] = _normal(gen, (tokens, (hq + 2 * hk) * D), _TYPES[case["dtype"]])[:, :hq * D].unflatten(1, (hq, D))
    s["cache"] = _filled(gen, s["pages"], case["page"], hk, D)
    return s


def prepare(case, seed):
    if case["op"] != "attention":
        return dict(_rows_tensors(case, seed), case=case)
    state = _attention_tensors(case, seed)
    state["max_q_len"] = max(n for n, _ in state["lengths"])
    if own and case["plan"]:
        import lmserve_amd as kvc
        state["plan"] = kvc.PagedAttentionPlan(
            state["qo_indptr"], state["indices"], state["indptr"], state["last"], case["heads"], case["kv_heads"],
            case["head_dim"], case["page"], _TYPES[case["dtype"]], num_tokens=state["query"].shape[0],
            max_q_len=state["max_q_len"], shared_pages=case["shared"] // case["page"], kv_dtype=_F8)
    return dict(state, case=case)


# ---------------------------------------------------------------- one pass
def run(state):
    case = state["case"]
    if case["op"] == "write":
        return _run_write(state, case) if own else _plain_write(state, case)
    if case["op"] == "read":
        return _run_read(state, case) if own else _plain_read(state, case)
    return _run_attention(state, case) if own else _plain_attention(state, case)


def _run_write(s, case):
    import lmserve_amd as kvc
    if case["form"] == "slots":
        kvc.reshape_and_cache_q8(s["key"], s["value"], s["cache"], s["slots"])
    else:
        kvc.append_paged_kv_cache_q8(s["key"], s["value"], s["batch"], s["positions"], s["cache"], s["indices"],
                                     s["indptr"], s["last"])
    return _values(s["cache"], case["kv_heads"], case["head_dim"])


def _run_read(s, case):
    import lmserve_amd as kvc
    H, D, dtype = case["kv_heads"], case["head_dim"], _TYPES[case["dtype"]]
    if case["form"] == "slots":
        k, v = kvc.read_cache_q8(s["cache"], s["slots"], H, D, dtype)
    else:
        k, v = kvc.read_paged_kv_cache_q8(s["batch"], s["positions"], s["cache"], s["indices"], s["indptr"], s["last"],
                                          H, D, dtype)
    return {"key": k, "value": v}


def _run_attention(s, case):
    import lmserve_amd as kvc
    if case["plan"]:
        got = s["plan"].run(s["query"], s["cache"], return_lse=case["lse"])
    else:
        got = kvc.paged_attention(s["query"], s["cache"], s["qo_indptr"], s["indices"], s["indptr"], s["last"],
                                  max_q_len=s["max_q_len"], shared_pages=case["shared"] // case["page"],
                                  return_lse=case["lse"], num_kv_heads=case["kv_heads"])
    return {"out": got[0], "lse": got[1]} if case["lse"] else {"out": got}


def _plain_write(s, case):
    H, D = case["kv_heads"], case["head_dim"]
    groups = s["cache"].view(-1, _group_bytes(H, D))
    old_k, old_v, old_exponents = _get(groups, s["group"], H, D)
    lane = torch.arange(GROUP, device="cuda")[None, :, None, None]
    live = lane < s["first"][:, None, None, None]
    began = (s["first"] > 0)[:, None]
    codes, exponents = [], []
    for which, new, old in ((0, s["key"], old_k), (1, s["value"], old_v)):
        x = torch.zeros(old.shape, device="cuda")
        x[s["member"], s["slots"] % GROUP] = new.float()
        fresh = torch.zeros(old.shape[:2], dtype=torch.bool, device="cuda")
        fresh[s["member"], s["slots"] % GROUP] = True
        had = old_exponents[:, :, which]
        e = _exponent(x.abs().amax(dim=(1, 3)))
        e = torch.where(began, torch.maximum(e, had), e)
        kept = old.contiguous().view(_F8).float() * _power(had - e)[:, None, :, None]
        x = torch.where(live, kept, x * _power(-e)[:, None, :, None]).to(_F8).view(torch.uint8)
        codes.append(torch.where(live | fresh[:, :, None, None], x, old))
        exponents.append(e)
    _put(groups, s["group"], codes[0], codes[1], torch.stack(exponents, dim=2))
    return _values(s["cache"], H, D)


def _plain_read(s, case):
    H, D, dtype = case["kv_heads"], case["head_dim"], _TYPES[case["dtype"]]
    groups, half = s["cache"].view(-1, _group_bytes(H, D)), GROUP * H * D
    at, t = s["slots"] // GROUP, s["slots"] % GROUP
    power = _power(groups[:, 2 * half:2 * half + 2 * H].reshape(-1, H, 2).int() - 127)[at]
    k = groups[:, :half].view(_F8).view(-1, H, 4, D // 16, 4, 16)[at, :, t // 4, :, t % 4].reshape(-1, H, D)
    v = groups[:, half:2 * half].view(_F8).view(-1, H, D, GROUP)[at, :, :, t]
    return {"key": (k.float() * power[..., :1]).to(dtype), "value": (v.float() * power[..., 1:]).to(dtype)}


def _plain_attention(s, case):
    hq, hk, D, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    group, scale = hq // hk, D ** -0.5
    tokens = s["query"].shape[0]
    out = torch.empty(tokens, hq, D, dtype=s["query"].dtype, device="cuda")
    lse = torch.empty(tokens, hq, dtype=torch.float32, device="cuda")
    indices, pages = s["indices"].long(), s["cache"].view(s["pages"], page // GROUP, -1)
    half = GROUP * hk * D
    lengths, tables = s["lengths"], s["tables"]
    first_token, first_page = [0], [0]
    for (n, _), t in zip(lengths, tables):
        first_token.append(first_token[-1] + n)
        first_page.append(first_page[-1] + t)
    b = 0
    while b < len(lengths):
        # requests next to each other with as many new tokens go together, padded to the longest of them
        n, e, longest = lengths[b][0], b, 0
        while e < len(lengths) and lengths[e][0] == n:
            wide = max(longest, tables[e])
            if e > b and (e - b + 1) * wide * page * max(hk * D, hq * n) > 1 << 29:
                break
            longest, e = wide, e + 1
        R, L = e - b, longest * page
        table = torch.zeros(R, longest, dtype=torch.long, device="cuda")
        if R == 1:
            table[0] = indices[first_page[b]:first_page[e]]
        else:
            inside = torch.arange(longest, device="cuda")[None] < (s["indptr"][b + 1:e + 1] - s["indptr"][b:e])[:, None]
            table[inside] = indices[first_page[b]:first_page[e]]
        ends = (s["indptr"][b + 1:e + 1] - s["indptr"][b:e] - 1) * page + s["last"][b:e]
        limit = ends[:, None] - n + 1 + torch.arange(n, device="cuda")[None]          # keys that a token sees
        q = s["query"][first_token[b]:first_token[e]].reshape(R, n, hk, group, D)
        rows = pages[table.reshape(-1)].view(R, L // GROUP, -1)
        power = _power(rows[..., 2 * half:2 * half + 2 * hk].reshape(R, L // GROUP, hk, 2).int() - 127)
        codes_k = rows[..., :half].view(_F8).view(R, L // GROUP, hk, 4, D // 16, 4, 16)
        codes_v = rows[..., half:2 * half].view(_F8).view(R, L // GROUP, hk, D, GROUP)
        heads = max(1, min(hk, (1 << 30) // max(1, R * n * group * L)))               # key heads at a time
        for h in range(0, hk, heads):
            H = min(heads, hk - h)
            k = codes_k[:, :, h:h + H].float() * power[:, :, h:h + H, 0, None, None, None, None]
            k = k.permute(0, 2, 4, 6, 1, 3, 5).reshape(R, H, D, L)
            v = codes_v[:, :, h:h + H].float() * power[:, :, h:h + H, 1, None, None]
            v = v.permute(0, 2, 1, 4, 3).reshape(R, H, L, D)
            qh = q[:, :, h:h + H].float().permute(0, 2, 1, 3, 4).reshape(R, H, n * group, D)
            scores = torch.matmul(qh * scale, k).reshape(R, H, n, group, L)
            seen = torch.arange(L, device="cuda")[None, None] < limit[:, :, None]
            scores.masked_fill_(~seen[:, None, :, None, :], float("-inf"))
            top = scores.amax(dim=4, keepdim=True)
            weights = scores.sub_(top).exp_()
            total = weights.sum(dim=4, keepdim=True)
            o = torch.matmul(weights.reshape(R, H, n * group, L), v).reshape(R, H, n, group, D) / total
            to = slice(first_token[b], first_token[e])
            out[to].reshape(R, n, hk, group, D)[:, :, h:h + H] = o.permute(0, 2, 1, 3, 4).to(out.dtype)
            lse[to].reshape(R, n, hk, group)[:, :, h:h + H] = (top + total.log())[..., 0].permute(0, 2, 1, 3)
        b = e
    return {"out": out, "lse": lse} if case["lse"] else {"out": out}


# ---------------------------------------------------------------- work and exact values
def work(case):
    D, hk = case["head_dim"], case["kv_heads"]
    if case["op"] != "attention":
        T, row = case["tokens"], 2 * hk * D
        groups = sum(-(-n // GROUP) - (n - k) // GROUP for k, n in _lengths(case))
        index = T * 8 + 2 * hk * groups
        return {"bytes": T * row * 2 + T * row + index, "flops": T * row * (3 if case["op"] == "write" else 1)}
    hq, tokens, keys, pairs = case["heads"], 0, 0, 0
    for n, length in _lengths(case):
        tokens += n
        keys += length - case["shared"]
        pairs += n * length - n * (n - 1) // 2
    keys += case["shared"]
    return {"bytes": keys * 2 * hk * D + keys // GROUP * 2 * hk + 4 * tokens * hq * D + (4 * tokens * hq if case["lse"] else 0)
            + 4 * keys // case["page"], "flops": 4 * pairs * hq * D}


def exact(case, seed):
    return {"write": _exact_write, "read": _exact_read, "attention": _exact_attention}[case["op"]](case, seed)


def _code_value(byte):
    """What 8 bits stand for, in 64: sign, 4 bits of exponent over 2**-7, 3 of mantissa."""
    byte = byte.long()
    power, mantissa = (byte >> 3) & 15, (byte & 7).double()
    size = torch.where(power > 0, (8 + mantissa) * torch.exp2(power.double() - 10), mantissa * 2.0 ** -9)
    return torch.where(byte >= 128, -size, size)


def _nearest(x):
    """The value of 4 bits of mantissa, steps of 2**-9 at least, next to x; half way to the even one."""
    size = x.abs().clamp(min=2.0 ** -6)
    step = torch.exp2(torch.floor(torch.log2(size)) - 3)
    step = torch.where(size / step >= 16, step * 2, torch.where(size / step < 8, step / 2, step))
    return torch.round(x / step) * step


def _cells(s, case):
    """Every token's K and V of the cache in 64 bits, `[group, token, head, dim]`, their codes' values and exponents."""
    H, D = case["kv_heads"], case["head_dim"]
    raw = s["cache"].view(-1, _group_bytes(H, D))
    n = raw.shape[0]
    value = _code_value(raw[:, :32 * H * D])
    k = value[:, :16 * H * D].view(n, H, 4, D // 16, 4, 16).transpose(3, 4).reshape(n, H, 16, D).transpose(1, 2)
    v = value[:, 16 * H * D:].view(n, H, D, 16).permute(0, 3, 1, 2)
    return k, v, raw[:, 32 * H * D:32 * H * D + 2 * H].view(n, H, 2).double() - 127


def _exact_write(case, seed):
    s = _rows_tensors(case, seed)
    H, D = case["kv_heads"], case["head_dim"]
    k, v, exponents = _cells(s, case)
    slots = s["slots"]
    where, what = slots // 16, slots % 16
    parts = []
    for which, codes, rows in ((0, k.clone(), s["key"].double()), (1, v.clone(), s["value"].double())):
        n = codes.shape[0]
        first = torch.full((n,), 16, device="cuda", dtype=torch.long).index_reduce_(0, where, what, "amin")
        top = torch.zeros(n, H, device="cuda", dtype=torch.float64).index_reduce_(0, where, rows.abs().amax(dim=2), "amax")
        need = torch.ceil(torch.log2(top / 448))
        need = torch.where(top > 448 * torch.exp2(need), need + 1, torch.where(top <= 448 * torch.exp2(need - 1), need - 1, need))
        need = need.nan_to_num(neginf=-100.0).clamp(-100, 120)
        before = exponents[:, :, which]
        touched = (first < 16)[:, None]
        grown = torch.where(touched & (first > 0)[:, None], torch.maximum(need, before), torch.where(touched, need, before))
        older = torch.arange(16, device="cuda")[None, :] < first[:, None]
        moved = _nearest(codes * torch.exp2(before - grown)[:, None, :, None])
        codes = torch.where((older & touched)[:, :, None, None], moved, codes)
        codes[where, what] = _nearest(rows * torch.exp2(-grown[where])[:, :, None])
        exponents[:, :, which] = grown
        parts.append(codes)
    n = k.shape[0]
    k = parts[0].transpose(1, 2).reshape(n, H, 4, 4, D // 16, 16).transpose(3, 4).reshape(n, -1)
    v = parts[1].permute(0, 2, 3, 1).reshape(n, -1)
    return {"codes": torch.cat((k, v), dim=1), "exponents": (exponents + 127).to(torch.uint8)}


def _exact_read(case, seed):
    s = _rows_tensors(case, seed)
    k, v, exponents = _cells(s, case)
    power = torch.exp2(exponents)
    at, t = s["slots"] // 16, s["slots"] % 16
    return {"key": k[at, t] * power[at, :, 0, None], "value": v[at, t] * power[at, :, 1, None]}


def _exact_attention(case, seed):
    s = _attention_tensors(case, seed)
    hq, hk, D, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    group = hq // hk
    tokens = s["query"].shape[0]
    out = torch.zeros(tokens, hq, D, dtype=torch.float64, device="cuda")
    lse = torch.zeros(tokens, hq, dtype=torch.float64, device="cuda")
    t = p = 0
    for (n, length), used in zip(s["lengths"], s["tables"]):
        table = s["indices"][p:p + used].long()
        k, v, exponents = _cells({"cache": s["cache"].view(s["pages"], -1)[table].contiguous()}, case)
        k = (k * torch.exp2(exponents[:, None, :, :1])).reshape(used * page, hk, D)[:length]
        v = (v * torch.exp2(exponents[:, None, :, 1:])).reshape(used * page, hk, D)[:length]
        for h in range(hk):
            z = torch.matmul(s["query"][t:t + n, h * group:(h + 1) * group].double().reshape(n * group, D),
                             k[:, h].T.contiguous()) / D ** 0.5
            if n > 1:
                future = torch.ones(n, length, dtype=torch.bool, device="cuda").triu(length - n + 1)
                z = torch.where(future.repeat_interleave(group, dim=0), -torch.inf, z)
            norm = torch.logsumexp(z, dim=1)
            out[t:t + n, h * group:(h + 1) * group] = (torch.exp(z - norm[:, None]) @ v[:, h].contiguous()).view(n, group, D)
            lse[t:t + n, h * group:(h + 1) * group] = norm.view(n, group)
        t, p = t + n, p + used
    return {"out": out, "lse": lse} if case["lse"] else {"out": out}
