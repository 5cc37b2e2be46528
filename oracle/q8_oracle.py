"""The 8-bit cache by its definition, in 64 bits, token by token (NumPy). Test infrastructure only.

Beside the 16-bit write of runtime/worker/llm_worker/models/layers/attention.py:76-85: groups of 16 tokens, e4m3 codes, one
exponent a group, head, and K or V."""
from __future__ import annotations

import numpy as np

GROUP, LEAST, MOST = 16, -100, 120


def _code_values():
    byte = np.arange(256)
    power, mantissa = byte >> 3 & 15, byte & 7
    size = np.where(power > 0, (1 + mantissa / 8) * 2.0 ** (power - 7), mantissa * 2.0 ** -9)
    size[byte & 127 == 127] = np.nan
    return np.where(byte > 127, -size, size)


VALUES = _code_values()


def encode(x):
    """The code next to x, ties to the even one; NaN for what is not finite (and, of finite numbers, |x| <= 448 only)."""
    x = np.asarray(x, np.float64)
    size, table = np.abs(np.where(np.isfinite(x), x, 0)), VALUES[:127]
    assert (size <= 448).all()
    up = np.clip(np.searchsorted(table, size), 1, 126)
    low = up - 1
    to_up, to_low = table[up] - size, size - table[low]
    code = np.where((to_up < to_low) | ((to_up == to_low) & (up % 2 == 0)), up, low)
    code = np.where(np.signbit(x), code + 128, code)
    return np.where(np.isfinite(x), code, 127).astype(np.uint8)


def exponent(top):
    for e in range(LEAST, MOST):
        if top <= 448 * 2.0 ** e:
            return e
    return MOST


def group_bytes(H, D):
    return (2 * GROUP * H * D + 2 * H + 127) // 128 * 128


class Cache:
    """codes [slots, 2, H, D] and exponents [groups, H, 2] of pages of uint8."""

    def __init__(self, pages, H, D):
        self.shape, self.H, self.D = pages.shape, H, D
        self.raw = pages.reshape(-1, group_bytes(H, D)).copy()
        n, half = self.raw.shape[0], GROUP * H * D
        k = self.raw[:, :half].reshape(n, H, 4, D // 16, 4, 16).transpose(0, 2, 4, 1, 3, 5).reshape(n, GROUP, H, D)
        v = self.raw[:, half:2 * half].reshape(n, H, D, GROUP).transpose(0, 3, 1, 2)
        self.codes = np.stack((k, v), 2).reshape(n * GROUP, 2, H, D)
        self.exponents = self.raw[:, 2 * half:2 * half + 2 * H].reshape(n, H, 2).astype(np.int64) - 127

    def pages(self):
        n, half, H, D = self.raw.shape[0], GROUP * self.H * self.D, self.H, self.D
        codes = self.codes.reshape(n, GROUP, 2, H, D)
        raw = self.raw.copy()
        raw[:, :half] = codes[:, :, 0].reshape(n, 4, 4, H, D // 16, 16).transpose(0, 3, 1, 4, 2, 5).reshape(n, half)
        raw[:, half:2 * half] = codes[:, :, 1].transpose(0, 2, 3, 1).reshape(n, half)
        raw[:, 2 * half:2 * half + 2 * H] = (self.exponents + 127).reshape(n, 2 * H)
        return raw.reshape(self.shape)

    def values(self):
        """[slots, 2, H, D]"""
        e = np.repeat(self.exponents, GROUP, axis=0).transpose(0, 2, 1)[..., None]
        return VALUES[self.codes] * 2.0 ** e

    def write(self, key, value, slots):
        """Rows [T, H, D] at slots (below 0, or beyond the cache: none), whose groups are written from one run of the call each."""
        rows = np.stack((np.asarray(key, np.float64), np.asarray(value, np.float64)), 1)
        slots = np.asarray(slots, np.int64)
        runs, t = [], 0
        while t < len(slots):
            end = t + 1
            while end < len(slots) and slots[end] == slots[end - 1] + 1 and slots[end] % GROUP:
                end += 1
            if 0 <= slots[t] < len(self.codes):
                runs.append((t, end))
            t = end
        for t, end in runs:
            g, first = divmod(int(slots[t]), GROUP)
            at = g * GROUP
            for h in range(self.H):
                for w in range(2):
                    x = rows[t:end, w, h]
                    e = exponent(np.abs(np.where(np.isfinite(x), x, 0)).max())
                    if first:
                        had = int(np.clip(self.exponents[g, h, w], LEAST, MOST))
                        if e > had:
                            old = self.codes[at:at + first, w, h]
                            self.codes[at:at + first, w, h] = encode(VALUES[old] * 2.0 ** (had - e))
                        e = max(e, had)
                    self.codes[at + first:at + first + end - t, w, h] = encode(x * 2.0 ** -e)
                    self.exponents[g, h, w] = e
