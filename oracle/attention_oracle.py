"""Attention over a paged cache and the normed rotation by their formulas, in 64 bits, request by request (NumPy).

Restates the interface the reference's wrappers have (runtime/worker/llm_worker/models/layers/attention.py:87-99): causal,
query head x reads key head x // (Hq / H), request b's tokens stand at the end of its keys. Test infrastructure only.
"""
from __future__ import annotations

import numpy as np


def paged_attention_f64(query, cache, qo_indptr, kv_indices, kv_indptr, kv_last_page_len, scale):
    """query [T, Hq, D], cache [P, 2, page, H, D] (float64). Returns out [T, Hq, D], lse [T, Hq], and what bounds the error of
    arithmetic: weighted [T, Hq, D] = sum p |v|, values [T, Hq, D] = sum |v|, products [T, Hq] = max sum |q| |k|.
    Rows of no request are NaN; rows without keys are 0, their lse -inf."""
    query, cache = np.asarray(query, np.float64), np.asarray(cache, np.float64)
    T, Hq, D = query.shape
    P, _, page, H, _ = cache.shape
    G = Hq // H
    out, lse = np.full((T, Hq, D), np.nan), np.full((T, Hq), np.nan)
    weighted, values, products = np.zeros((T, Hq, D)), np.zeros((T, Hq, D)), np.zeros((T, Hq))
    for b in range(len(qo_indptr) - 1):
        table = np.asarray(kv_indices[kv_indptr[b]:kv_indptr[b + 1]], np.int64)
        length = max(len(table) - 1, 0) * page + int(kv_last_page_len[b]) if len(table) else 0
        n = int(qo_indptr[b + 1] - qo_indptr[b])
        there = np.repeat((table >= 0) & (table < P), page)[:length]
        rows = cache[np.clip(table, 0, P - 1)] if len(table) else cache[:0]
        keys = rows[:, 0].reshape(-1, H, D)[:length]
        vals = rows[:, 1].reshape(-1, H, D)[:length]
        for j in range(n):
            t = int(qo_indptr[b]) + j
            seen = there & (np.arange(length) <= length - n + j)
            k, v = keys[seen], vals[seen]
            for x in range(Hq):
                if not len(k):
                    out[t, x], lse[t, x] = 0, -np.inf
                    continue
                s = scale * (k[:, x // G] @ query[t, x])
                m = s.max()
                p = np.exp(s - m)
                out[t, x] = p @ v[:, x // G] / p.sum()
                lse[t, x] = m + np.log(p.sum())
                weighted[t, x] = p @ np.abs(v[:, x // G]) / p.sum()
                values[t, x] = np.abs(v[:, x // G]).sum(0)
                products[t, x] = (np.abs(k[:, x // G]) @ np.abs(query[t, x])).max()
    return out, lse, weighted, values, products


def attention_tolerances(out, lse, weighted, values, products, D, scale, dtype_eps, denormal):
    """Bounds of |out - exact| and |lse - exact| by counting roundings.

    A score is D products summed in 32 bits: off by at most (D + 2) 2^-24 sum|q||k|, times the scale, and by 2^-22 of the
    exponent's own size for scale, maximum and difference; a weight by that (relative) and by half a step of the storage type
    (dtype_eps / 2; or half the smallest denormal of f16, of weights that are scaled up by 2^7 and more against a base that stands up to
    1 above the largest score: 2^-6 of that, as a part of the largest weight); sums of weights and of weighted values by 2^-24 a
    term in the chains of up to 600 terms the sizes here make; the output is rounded once more."""
    ds = scale * products * (D + 2) * 2.0 ** -24 + (1 + scale * products) * 2.0 ** -22
    chain = 600 * 2.0 ** -24
    rel = 2 * ds + 2 * chain
    tol = weighted * (dtype_eps / 2 + rel[..., None]) * 1.05 + np.abs(out) * dtype_eps / 2 * 1.05 + values * denormal * 2.0 ** -6 + denormal
    return tol, ds + chain + np.abs(np.where(np.isfinite(lse), lse, 0)) * 2.0 ** -22 + 2.0 ** -22


def qk_norm_rotary_f64(x, weight, positions, cos_sin, D, eps):
    """x [T, heads * D] normed head by head (root mean square, times weight), then its first rotary_dim lanes rotated
    (runtime/worker/llm_worker/ops/triton/rotary_embedding.py:5-66). Returns ([T, heads, D], bound on the error of 32-bit
    arithmetic before the last rounding)."""
    x, weight, cos_sin = np.asarray(x, np.float64), np.asarray(weight, np.float64), np.asarray(cos_sin, np.float64)
    T = x.shape[0]
    x = x.reshape(T, -1, D)
    y = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * weight
    rd = cos_sin.shape[1] // 2
    half = rd // 2
    row = cos_sin[np.asarray(positions, np.int64)][:, None, :]
    a, b = y[..., :half], y[..., half:rd]
    out, size = y.copy(), np.abs(y)
    out[..., :half] = a * row[..., :half] - b * row[..., rd:rd + half]
    out[..., half:rd] = b * row[..., half:rd] + a * row[..., rd + half:]
    size[..., :half] = np.abs(a * row[..., :half]) + np.abs(b * row[..., rd:rd + half])
    size[..., half:rd] = np.abs(b * row[..., half:rd]) + np.abs(a * row[..., rd + half:])
    # the mean: D/2 squares summed in a chain at most, half of which shows in the root; root, reciprocal, three products, a sum
    return out, size * (D / 4 + 8) * 2.0 ** -24
