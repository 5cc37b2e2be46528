"""Calls of the attention layer's operators around the paged cache, as a forward pass makes them.

`norm_rotate`: queries and keys normed head by head (root mean square, a weight per lane), rotated by their positions, and
the rotated key and the value written into the token's cache slot, in one call. `attention`: the queries of a step over
the paged cache, causal, with fewer key/value heads than query heads; where `shared` is given, the first `shared` tokens
of every request lie in the same pages, as a common system prompt does.

`run` is either the plain form in elementary torch operations, or the calls of this package."""
import random

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
EPS = 1e-6


def _norm(name, form, tokens, requests, heads, kv_heads, head_dim, rotary_dim, dtype, page=16):
    c = {"op": "norm_rotate", "form": form, "tokens": tokens, "requests": requests, "heads": heads,
         "kv_heads": kv_heads, "head_dim": head_dim, "rotary_dim": rotary_dim, "dtype": dtype, "page": page}
    return dict(c, name=name) if name else c


def _attn(name, requests, chunk_requests, chunk, low, high, shared, heads, kv_heads, head_dim, dtype, page=16,
          plan=True, lse=False, lengths=0):
    c = {"op": "attention", "requests": requests, "chunk_requests": chunk_requests, "chunk": chunk, "low": low,
         "high": high, "shared": shared, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, "dtype": dtype,
         "page": page, "plan": plan, "lse": lse, "lengths": lengths}
    return dict(c, name=name) if name else c


def listed():
    return [
        # one token of one request: what a layer pays when nobody else is served
        _norm("norm-one-token", "paged", 1, 1, 28, 4, 128, 128, "bf16"),
        # a decode step of a full batch, through the plan that a step keeps for all its layers
        _norm("norm-decode-256", "plan", 256, 256, 32, 8, 128, 128, "bf16"),
        # a prefill chunk of four requests, by slot mapping
        _norm("norm-chunk-2048", "slots", 2048, 4, 28, 4, 128, 128, "f16"),
        # heads of 80 rotated in part, in 32 bits, an odd number of tokens, without a cache
        _norm("norm-odd-heads", "rotate", 717, 3, 15, 5, 80, 32, "f32"),
        # a long prompt at once
        _norm("norm-prompt-16384", "paged", 16384, 2, 64, 8, 128, 128, "bf16"),
        # one request with a short context: latency; the index tensors are new with every call
        _attn("attend-one-request", 1, 0, 0, 900, 900, 0, 32, 8, 64, "bf16", plan=False),
        # a decode step of a full batch, contexts as they come
        _attn("attend-decode-256", 256, 0, 0, 1, 4095, 0, 32, 8, 128, "bf16"),
        # one request far into a long document
        _attn("attend-long-document", 1, 0, 0, 131001, 131001, 0, 64, 8, 128, "bf16", lse=True),
        # a decode step behind one long system prompt
        _attn("attend-shared-prompt", 256, 0, 0, 1, 512, 4096, 32, 8, 128, "bf16"),
        # few requests behind a prompt that the batch shares, seven query heads to a key head
        _attn("attend-shared-few", 13, 0, 0, 5, 900, 2000, 28, 4, 128, "f16", lse=True),
        # a prefill chunk of four requests with long contexts behind them
        _attn("attend-chunks-2048", 4, 4, 512, 1024, 32768, 0, 28, 4, 128, "bf16"),
        # chunks and single tokens in one step, behind a shared prompt
        _attn("attend-mixed-step", 63, 3, 259, 300, 2500, 1024, 32, 8, 64, "f16"),
    ]


def _spread(rng, low, high):
    """Spread over the logarithm, both ends included."""
    return max(low, min(high, round(low * (high / low) ** rng.random())))


def draw(rng):
    heads, kv_heads, head_dim = rng.choice([(32, 8, 64), (32, 8, 128), (28, 4, 128), (64, 8, 128), (8, 1, 128),
                                            (32, 32, 128), (40, 8, 80), (15, 5, 80), (16, 2, 256), (7, 7, 64)])
    page = rng.choice([16, 16, 16, 8, 32, 64, 20])
    if rng.random() < 0.4:
        tokens = _spread(rng, 1, 16384)
        rotary = rng.choice([head_dim, head_dim, head_dim // 2 // 16 * 16])
        return _norm(None, rng.choice(["rotate", "slots", "paged", "plan"]), tokens, rng.randint(1, min(tokens, 256)),
                     heads, kv_heads, head_dim, rotary, rng.choice(["bf16", "f16", "f32"]), page)
    dtype = rng.choice(["bf16", "f16"])
    lengths, plan, lse = rng.randint(0, 999), rng.random() < 0.8, rng.random() < 0.5
    kind = rng.choice(["decode", "shared", "chunks", "mixed"])
    if kind == "chunks":
        requests, chunk = rng.randint(1, 4), _spread(rng, 2, 512)
        high = _spread(rng, chunk, 16384)
        return _attn(None, requests, requests, chunk, chunk, high, 0, heads, kv_heads, head_dim, dtype, page, plan, lse,
                     lengths)
    if kind == "mixed":
        chunk = _spread(rng, 2, 400)
        return _attn(None, rng.randint(4, 60), rng.randint(1, 3), chunk, chunk, chunk + _spread(rng, 1, 2000),
                     page * rng.choice([0, 5, 64]), heads, kv_heads, head_dim, dtype, page, plan, lse, lengths)
    requests = _spread(rng, 1, 256)
    high = _spread(rng, 1, min(131072, 400000 // requests))
    if kind == "decode":
        return _attn(None, requests, 0, 0, max(1, high // 3), high, 0, heads, kv_heads, head_dim, dtype, page, plan, lse,
                     lengths)
    high = min(high, 1000)
    return _attn(None, requests, 0, 0, 1, high, page * _spread(rng, 1, 4096 // page), heads, kv_heads, head_dim, dtype,
                 page, plan, lse, lengths)


# ---------------------------------------------------------------- inputs
def _lengths(case):
    """(new tokens, context length) of every request: by the case alone."""
    rng = random.Random(case["lengths"])
    out = []
    for b in range(case["requests"]):
        new = case["chunk"] if b < case["chunk_requests"] else 1
        out.append((new, case["shared"] + max(new, rng.randint(case["low"], case["high"]))))
    return out


def _normal(gen, shape, dtype):
    return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32).to(dtype)


def _cos_sin(rotary_dim, positions, dtype):
    half = torch.arange(0, rotary_dim, 2, device="cuda", dtype=torch.float64) / rotary_dim
    angles = torch.arange(positions, device="cuda", dtype=torch.float64)[:, None] / 500000.0 ** half[None, :]
    angles = torch.cat((angles, angles), dim=1)
    return torch.cat((angles.cos(), angles.sin()), dim=1).to(dtype)


def _norm_tensors(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype, T, D, page = _TYPES[case["dtype"]], case["tokens"], case["head_dim"], case["page"]
    hq, hk, B = case["heads"], case["kv_heads"], case["requests"]
    # rows as a fused projection leaves them: slices of one matrix
    qkv = _normal(gen, (T, (hq + 2 * hk) * D), dtype)
    new = [T // B + (1 if b < T % B else 0) for b in range(B)]
    tables = [-(-n // page) for n in new]
    pages = sum(tables) + 3
    order = torch.randperm(pages, generator=gen, device="cuda")
    batch = torch.repeat_interleave(torch.arange(B, device="cuda"), torch.tensor(new, device="cuda"))
    first = torch.tensor([sum(new[:b]) for b in range(B)], device="cuda")
    positions = torch.arange(T, device="cuda") - first[batch]
    indptr = torch.tensor([sum(tables[:b]) for b in range(B + 1)], device="cuda")
    indices = order[:sum(tables)]
    slots = indices[indptr[batch] + positions // page] * page + positions % page
    i32 = torch.int32
    return {
        "query": qkv[:, :hq * D], "key": qkv[:, hq * D:(hq + hk) * D], "value": qkv[:, (hq + hk) * D:],
        "query_weight": (1 + 0.2 * torch.randn(D, generator=gen, device="cuda")).to(dtype),
        "key_weight": (1 + 0.2 * torch.randn(D, generator=gen, device="cuda")).to(dtype),
        "cos_sin": _cos_sin(case["rotary_dim"], max(new), dtype),
        "cache": torch.zeros(pages, 2, page, hk, D, dtype=dtype, device="cuda"),
        "batch": batch.to(i32), "positions": positions.to(i32), "slots": slots, "indices": indices.to(i32),
        "indptr": indptr.to(i32), "last": torch.tensor([(n - 1) % page + 1 for n in new], dtype=i32, device="cuda"),
    }


def _attention_tensors(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype, D, page = _TYPES[case["dtype"]], case["head_dim"], case["page"]
    hq, hk = case["heads"], case["kv_heads"]
    lengths = _lengths(case)
    common = case["shared"] // page
    tables = [-(-n // page) for _, n in lengths]
    pages = common + sum(t - common for t in tables) + 3
    order = torch.randperm(pages, generator=gen, device="cuda")
    parts, at = [], common
    for t in tables:
        parts += [order[:common], order[at:at + t - common]]
        at += t - common
    new = [n for n, _ in lengths]
    tokens = sum(new)
    cache = torch.empty(pages, 2, page, hk, D, dtype=dtype, device="cuda")
    step = max(1, (1 << 27) // (2 * page * hk * D))
    for p in range(0, pages, step):
        cache[p:p + step] = _normal(gen, (min(step, pages - p), 2, page, hk, D), dtype)
    i32 = torch.int32
    return {
        "query": _normal(gen, (tokens, (hq + 2 * hk) * D), dtype)[:, :hq * D], "cache": cache,
        "qo_indptr": torch.tensor([sum(new[:b]) for b in range(len(new) + 1)], dtype=i32, device="cuda"),
        "indices": torch.cat(parts).to(i32),
        "indptr": torch.tensor([sum(tables[:b]) for b in range(len(tables) + 1)], dtype=i32, device="cuda"),
        "last": torch.tensor([(n - 1) % page + 1 for _, n in lengths], dtype=i32, device="cuda"),
        "lengths": lengths, "tables": tables,
    }


def prepare(case, seed):
    if case["op"] == "norm_rotate":
        state = _norm_tensors(case, seed)
        if own and case["form"] == "plan":
            import lmserve_amd as kvc
            state["plan"] = kvc.PagedRotaryWritePlan(
                state["batch"], state["positions"], state["indices"], state["indptr"], state["last"], state["cos_sin"],
                case["heads"], case["kv_heads"], case["head_dim"], case["page"], slots=state["slots"])
    else:
        state = _attention_tensors(case, seed)
        state["max_q_len"] = max(n for n, _ in state["lengths"])
        if own and case["plan"]:
            import lmserve_amd as kvc
            state["plan"] = kvc.PagedAttentionPlan(
                state["qo_indptr"], state["indices"], state["indptr"], state["last"], case["heads"], case["kv_heads"],
                case["head_dim"], case["page"], _TYPES[case["dtype"]], num_tokens=state["query"].shape[0],
                max_q_len=state["max_q_len"], shared_pages=case["shared"] // case["page"])
    return dict(state, case=case)


# ---------------------------------------------------------------- one pass
def run(state):
    case = state["case"]
    if case["op"] == "norm_rotate":
        return _run_norm(state, case) if own else _plain_norm(state, case)
    return _run_attention(state, case) if own else _plain_attention(state, case)


def _run_norm(s, case):
    import lmserve_amd as kvc
    norm = (s["query_weight"], s["key_weight"])
    if case["form"] == "rotate":
        q, k = kvc.qk_norm_rotary_pos_emb(s["query"], s["key"], *norm, s["positions"], s["cos_sin"], case["head_dim"], EPS)
        return {"query": q, "key": k}
    if case["form"] == "slots":
        q, k = kvc.qk_norm_rotary_pos_emb_and_cache(s["query"], s["key"], s["value"], *norm, s["positions"], s["cos_sin"],
                                                    case["head_dim"], s["cache"], s["slots"], EPS)
        return {"query": q, "key": k, "cache": s["cache"]}
    if case["form"] == "paged":
        q, k = kvc.qk_norm_rotary_pos_emb_and_append_paged(
            s["query"], s["key"], s["value"], *norm, s["batch"], s["positions"], s["cos_sin"], case["head_dim"], s["cache"],
            s["indices"], s["indptr"], s["last"], EPS)
        return {"query": q, "key": k, "cache": s["cache"]}
    q, _ = s["plan"].run(s["query"], s["key"], s["value"], s["cache"], query_weight=norm[0], key_weight=norm[1], eps=EPS)
    return {"query": q, "cache": s["cache"]}


def _run_attention(s, case):
    import lmserve_amd as kvc
    if case["plan"]:
        got = s["plan"].run(s["query"], s["cache"], return_lse=case["lse"])
    else:
        got = kvc.paged_attention(s["query"], s["cache"], s["qo_indptr"], s["indices"], s["indptr"], s["last"],
                                  max_q_len=s["max_q_len"], shared_pages=case["shared"] // case["page"],
                                  return_lse=case["lse"])
    return {"out": got[0], "lse": got[1]} if case["lse"] else {"out": got}


def _plain_norm(s, case):
    T, D, rd, dtype = case["tokens"], case["head_dim"], case["rotary_dim"], _TYPES[case["dtype"]]
    row = s["cos_sin"].float()[s["positions"].long()][:, None, :]
    cos, sin = row[..., :rd], row[..., rd:]

    def rotated(x, weight):
        x = x.reshape(T, -1, D).float()
        x = x / (x.square().mean(dim=2, keepdim=True) + EPS).sqrt() * weight.float()
        turn, rest = x[..., :rd], x[..., rd:]
        crossed = torch.cat((-turn[..., rd // 2:], turn[..., :rd // 2]), dim=2)
        return torch.cat((turn * cos + crossed * sin, rest), dim=2).to(dtype)

    q, k = rotated(s["query"], s["query_weight"]), rotated(s["key"], s["key_weight"])
    out = {"query": q.reshape(T, -1), "key": k.reshape(T, -1)}
    if case["form"] == "rotate":
        return out
    page, cache = case["page"], s["cache"]
    cache[s["slots"] // page, 0, s["slots"] % page] = k
    cache[s["slots"] // page, 1, s["slots"] % page] = s["value"].reshape(T, -1, D)
    out["cache"] = cache
    if case["form"] == "plan":
        del out["key"]
    return out


def _plain_attention(s, case):
    hq, hk, D, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    group, scale = hq // hk, D ** -0.5
    tokens = s["query"].shape[0]
    out = torch.empty(tokens, hq, D, dtype=s["query"].dtype, device="cuda")
    lse = torch.empty(tokens, hq, dtype=torch.float32, device="cuda")
    indices = s["indices"].long()
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
        heads = max(1, min(hk, (1 << 30) // max(1, R * n * group * L)))               # key heads at a time
        for h in range(0, hk, heads):
            H = min(heads, hk - h)
            pages = s["cache"][table.reshape(-1), :, :, h:h + H].float().reshape(R, longest, 2, page, H, D)
            k = pages[:, :, 0].reshape(R, L, H, D).permute(0, 2, 3, 1).contiguous()
            v = pages[:, :, 1].reshape(R, L, H, D).permute(0, 2, 1, 3).contiguous()
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
    out = out.reshape(tokens, hq * D)
    return {"out": out, "lse": lse} if case["lse"] else {"out": out}


# ---------------------------------------------------------------- work and exact values
def work(case):
    D, hq, hk = case["head_dim"], case["heads"], case["kv_heads"]
    E = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "norm_rotate":
        T = case["tokens"]
        longest = -(-T // case["requests"])
        read = T * (hq + hk) * D * E + min(T, longest) * 2 * case["rotary_dim"] * E + 2 * D * E + 4 * T
        wrote = T * hq * D * E + (T * hk * D * E if case["form"] != "plan" else 0)
        if case["form"] != "rotate":
            read += T * hk * D * E + 8 * T
            wrote += 2 * T * hk * D * E
        return {"bytes": read + wrote, "flops": T * (hq + hk) * (4 * D + 3 * case["rotary_dim"])}
    tokens = keys = 0
    pairs = 0
    for n, length in _lengths(case):
        tokens += n
        keys += length - case["shared"]
        pairs += n * length - n * (n - 1) // 2
    keys += case["shared"]
    return {"bytes": keys * 2 * hk * D * E + 2 * tokens * hq * D * E + (4 * tokens * hq if case["lse"] else 0)
            + 4 * keys // case["page"], "flops": 4 * pairs * hq * D}


def exact(case, seed):
    return _exact_norm(case, seed) if case["op"] == "norm_rotate" else _exact_attention(case, seed)


def _exact_norm(case, seed):
    s = _norm_tensors(case, seed)
    T, D, rd = case["tokens"], case["head_dim"], case["rotary_dim"]
    table = s["cos_sin"].double().index_select(0, s["positions"].long()).unsqueeze(1)

    def one(rows, weight):
        x = rows.double().view(T, rows.shape[1] // D, D)
        power = torch.einsum("thd,thd->th", x, x) / D
        y = x * torch.rsqrt(power + EPS).unsqueeze(2) * weight.double()
        z = y.clone()
        half = rd // 2
        a, b = y[..., :half], y[..., half:rd]
        z[..., :half] = a * table[..., :half] - b * table[..., rd:rd + half]
        z[..., half:rd] = b * table[..., half:rd] + a * table[..., rd + half:]
        return z

    q, k = one(s["query"], s["query_weight"]), one(s["key"], s["key_weight"])
    out = {"query": q.flatten(1), "key": k.flatten(1)}
    if case["form"] != "rotate":
        pages, _, page, hk, _ = s["cache"].shape
        planes = torch.zeros(2, pages * page, hk, D, dtype=torch.float64, device="cuda")
        planes[0].index_copy_(0, s["slots"], k)
        planes[1].index_copy_(0, s["slots"], s["value"].double().view(T, hk, D))
        out["cache"] = planes.view(2, pages, page, hk, D).transpose(0, 1).contiguous()
    if case["form"] == "plan":
        del out["key"]
    return out


def _exact_attention(case, seed):
    s = _attention_tensors(case, seed)
    hq, hk, D, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    group = hq // hk
    tokens = s["query"].shape[0]
    out = torch.zeros(tokens, hq, D, dtype=torch.float64, device="cuda")
    lse = torch.zeros(tokens, hq, dtype=torch.float64, device="cuda")
    query = s["query"].view(tokens, hq, D)
    t = p = 0
    for (n, length), used in zip(s["lengths"], s["tables"]):
        table = s["indices"][p:p + used].long()
        for h in range(hk):
            k = s["cache"][table, 0, :, h].reshape(used * page, D)[:length].double()
            v = s["cache"][table, 1, :, h].reshape(used * page, D)[:length].double()
            for g in range(h * group, (h + 1) * group):
                z = query[t:t + n, g].double() @ k.T / D ** 0.5
                if n > 1:
                    future = torch.ones(n, length, dtype=torch.bool, device="cuda").triu(length - n + 1)
                    z = torch.where(future, -torch.inf, z)
                norm = torch.logsumexp(z, dim=1)
                out[t:t + n, g] = torch.exp(z - norm[:, None]) @ v
                lse[t:t + n, g] = norm
        t, p = t + n, p + used
    out = out.view(tokens, hq * D)
    return {"out": out, "lse": lse} if case["lse"] else {"out": out}
