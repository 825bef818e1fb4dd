"""Plain float64 forms of the operators on ragged rows (include/rtxllm/kv8.h and the windowed attention of
include/rtxllm/paged_kv.h), on numpy arrays, one block, row and head at a time."""

from __future__ import annotations

import numpy as np

NONE = 0xFFFFFFFF


def to_e4m3(y):
    """The nearest OCP e4m3 number (four significant bits, steps of 2^-9 at least), ties to the even one."""
    y = np.asarray(y, np.float64)
    _, e = np.frexp(np.maximum(np.abs(y), 2.0 ** -6))
    step = 2.0 ** (e - 4)
    return np.round(y / step) * step


def quantise(x16, fmt):
    """x16 fp16 [block][dim]: the numbers its codes stand for before the scale, and the scale (float32)."""
    x = x16.astype(np.float64)
    if not np.isfinite(x).all():
        return np.zeros_like(x), np.float32(np.nan)
    top = np.abs(x).max()
    if top == 0.0:
        return np.zeros_like(x), np.float32(0.0)
    if fmt == "int8":
        scale = np.float32(top) * (np.float32(1.0) / np.float32(127.0))
        return np.round(x / np.float64(scale)), scale
    k = int(np.ceil(np.log2(top / 448.0)))
    while top / 2.0 ** k > 448.0:
        k += 1
    while top / 2.0 ** (k - 1) <= 448.0:
        k -= 1
    return to_e4m3(x / 2.0 ** k), np.float32(2.0 ** k)


def visible(p, window, sinks):
    j = np.arange(p + 1)
    return j[(p - j < window) | (j < sinks)]


def attend(q, keys, values, f16=False, single=False):
    """q [d] over keys, values [n][d]: (the result, a bound of the error).

    q enters as an fp16 pair: off by 2^-22 of itself or 2^-39 of the largest, so a score by 2^-22 |q| |k|; its d
    products and sums round d + 8 times, scales and powers of two 8 times more: of |q| |k| each. A term
    2^(s - m) is off by that of its score, twice (its own and the maximum's do not cancel in rounding), and by
    2^-21 (1 + |s|) for the subtraction and the power. Terms enter as pairs, off by 2^-22 of themselves
    or 2^-39 of the largest; sums of n terms round n times and 64 more where records merge.
    single: terms enter as one fp16, off by 2^-11 of themselves. f16: the result is rounded to fp16 (2^-11, or
    2^-25 among its subnormals)."""
    n, d = keys.shape
    if n == 0:
        return np.zeros(d), np.zeros(d)
    q, keys, values = (np.asarray(x, np.float64) for x in (q, keys, values))
    s = keys @ q / np.sqrt(d)
    size = np.abs(keys) @ np.abs(q) / np.sqrt(d)
    with np.errstate(invalid="ignore", over="ignore"):
        e = np.exp(s - s.max())
        p = e / e.sum()
        out = p @ values
        delta = (2.0 ** -22 + (d + 16) * 2.0 ** -24) * size.max() + 2.0 ** -21 * (1.0 + np.abs(s).max())
        spread = p @ np.abs(values)
        tol = (2.0 * delta + (n + 64) * 2.0 ** -24 + (2.0 ** -11 if single else 2.0 ** -22)) * spread
        tol = tol + 2.0 ** -39 * n * np.abs(np.where(np.isfinite(values), values, 0.0)).max() + 1e-37
        if f16:
            tol = tol + 2.0 ** -11 * (np.abs(out) + tol) + 2.0 ** -25
    return out, tol


class Model:
    """What an 8-bit cache holds, as tokens come: the numbers of codes, scales and tails, with the pages as the
    table has them (an entry outside the cache: dropped)."""

    def __init__(self, table, n_pages, kv, page, dim, block, fmt):
        self.table, self.n_pages, self.kv, self.page, self.dim, self.block, self.fmt = table, n_pages, kv, page, dim, block, fmt
        self.capacity = table.shape[1] * page
        self.codes = [np.zeros((n_pages, kv, page, dim)) for _ in range(2)]
        self.scale = [np.zeros((n_pages, kv, page // block), np.float32) for _ in range(2)]
        self.tail = [np.zeros((table.shape[0], kv, block, dim), np.float16) for _ in range(2)]

    def at(self, s, p):
        t = int(self.table[s, p // self.page])
        return (t, p % self.page) if 0 <= t < self.n_pages else None

    def append(self, s, pos, new):
        """new: (k, v) [n][kv][dim], from position pos on."""
        with np.errstate(over="ignore"):
            new = [x.astype(np.float16) for x in new]
        end = min(pos + len(new[0]), self.capacity)
        for first in range(pos // self.block * self.block, end, self.block):
            lo, hi = max(first, pos), min(first + self.block, end)
            for i in range(2):
                x = self.tail[i][s].copy()
                x[:, lo - first:hi - first] = new[i][lo - pos:hi - pos].transpose(1, 0, 2)
                if hi < first + self.block:
                    self.tail[i][s, :, lo - first:hi - first] = x[:, lo - first:hi - first]
                    continue
                at = self.at(s, first)
                for g in range(self.kv if at else 0):
                    c, sc = quantise(x[g], self.fmt)
                    self.codes[i][at[0], g, at[1]:at[1] + self.block] = c
                    self.scale[i][at[0], g, at[1] // self.block] = sc

    def value(self, i, s, g, p, held):
        """Position p of a sequence that holds `held`, of k (i 0) or v: float64 [dim], or None."""
        if p >= held // self.block * self.block:
            return self.tail[i][s, g, p % self.block].astype(np.float64)
        at = self.at(s, p)
        if at is None:
            return None
        return self.codes[i][at[0], g, at[1]] * np.float64(self.scale[i][at[0], g, at[1] // self.block])
