"""Plain float64 forms of the paged-cache operators (include/rtxllm/paged_kv.h), on
numpy arrays, one row and one head at a time."""

from __future__ import annotations

import numpy as np

NONE = 0xFFFFFFFF
H_MAX = 65504.0


def row(table, r, one):
    return table[0] if one else table[r]


def at(table_row, n_pages, page_size, slot):
    """(physical page, place in it) of a slot, or None."""
    if slot // page_size >= len(table_row):
        return None
    p = int(table_row[slot // page_size])
    return (p, slot % page_size) if 0 <= p < n_pages else None


def filled(last, capacity):
    return 0 if last == NONE else min(last + 1, capacity)


def norm_rope(x, weight, pos, theta, eps, rotary, halves):
    """(the rotated head, |a| + |b| of the pair behind each of its values)."""
    x = x.astype(np.float64)
    y = x / np.sqrt((x * x).mean() + eps) * (1.0 if weight is None else weight.astype(np.float64))
    out, size = y.copy(), np.abs(y)
    for i in range(rotary // 2):
        a, b = (i, i + rotary // 2) if halves else (2 * i, 2 * i + 1)
        angle = float(pos) * float(theta) ** (-2.0 * i / rotary)
        c, s = np.cos(angle), np.sin(angle)
        out[a], out[b] = y[a] * c - y[b] * s, y[a] * s + y[b] * c
        size[a] = size[b] = abs(y[a]) + abs(y[b])
    return out, size


def bounds_of(keys):
    """[2][head_dim] of the filled keys [n][head_dim] of a page."""
    k = keys.astype(np.float64)
    hi = np.where(np.isnan(k), -H_MAX, k).max(0).clip(-H_MAX, H_MAX)
    lo = np.where(np.isnan(k), H_MAX, k).min(0).clip(-H_MAX, H_MAX)
    return np.stack([hi, lo])


def select(q, bounds, table_row, n_pages, used, n_first, n_last, n_select):
    """q [group][d], bounds [n_pages][2][d] of one kv head: the listed logical pages."""
    ranked = []
    for t in range(used):
        p = int(table_row[t])
        if not 0 <= p < n_pages:
            continue
        b = bounds[p].astype(np.float64)
        s = [float(np.maximum(h.astype(np.float64) * b[0], h.astype(np.float64) * b[1]).sum()) for h in q]
        s = [v for v in s if not np.isnan(v)]
        forced = t < n_first or t + n_last >= used
        ranked.append((not forced, -max(s) if s else np.inf, t))
    return sorted(t for _, _, t in sorted(ranked)[:n_select])


def attend(q, keys, values):
    """q [d] over keys, values [n][d]: (softmax weights, result, bound of the error).

    The bound: q enters as an fp16 pair of 2^-23 of the largest |q| each; an fp32 sum
    of d products rounds at most d + 8 times; s - m and 2^s round to 2^-22 of 1 + |s|; the
    sums over n positions round at most once a tile of 16 (in tiles the matrix cores
    add in steps of 4) and some 40 times where records merge."""
    n, d = keys.shape
    if n == 0:
        return np.zeros(0), np.zeros(d), np.zeros(d), np.zeros(0)
    q, keys, values = q.astype(np.float64), keys.astype(np.float64), values.astype(np.float64)
    s = keys @ q / np.sqrt(d)
    e = np.exp(s - s.max())
    p = e / e.sum()
    delta = (2.0 ** -23 * np.abs(q).max() * np.abs(keys).sum(1) + (d + 8) * 2.0 ** -24 * (np.abs(keys) @ np.abs(q))) / np.sqrt(d)
    delta = delta.max() + 2.0 ** -21 * (1.0 + np.abs(s).max())
    sums = (n / 4 + 40) * 2.0 ** -24
    return p, p @ values, (2.0 * delta + sums) * (p @ np.abs(values)) + 1e-37, p * (2.0 * delta + sums) + 2.0 ** -40


def evict(length, newest, keep, n_first, n_recent, weight, slot_pos):
    """Source slot of each slot below keep (one kv head), or None: nothing leaves."""
    if length <= keep:
        return None
    def rank(i):
        p, w = int(slot_pos[i]), float(weight[i])
        protected = p < n_first or p + n_recent > newest
        if protected:  # all alike
            return (0, 0.0, i)
        return (2, 0.0, i) if np.isnan(w) else (1, -w, i)
    kept = set(sorted(range(length), key=rank)[:keep])
    late = iter(sorted(i for i in kept if i >= keep))
    return [i if i in kept else next(late) for i in range(keep)]
