"""The paged-cache operators (include/rtxllm/paged_kv.h) where their definitions are decided by
the last bit, by an infinity or by a page that is not there."""

from __future__ import annotations

from fractions import Fraction

import numpy as np
import paged_ref as ref
import pytest

torch = pytest.importorskip("torch")

from rtxllm_amd import paged  # noqa: E402
from test_gpu_paged import DEV, Setup, dev, u32  # noqa: E402

pytestmark = pytest.mark.gpu


# ---- page scores ------------------------------------------------------------------


def listed_pages(s, bounds, q, select):
    n = s.lens[0]
    return paged.select_pages(s.cache, dev(bounds), dev(q), u32([n - 1]), select, 0, 0).cpu().numpy()[0]


@pytest.mark.parametrize("group", [1, 4, 5])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("other", ["any", "clamped", "mixed"])
def test_pages_of_one_score_are_equal(group, dim, other):
    """300 pages whose counted extremes are the same and whose others are not: one score, so the
    lowest pages are listed. The queries' sizes span some 2^40 where an extreme is at the clamp; heads of a group share their signs,
    so that each page's counted extreme is one."""
    s = Setup(31 * group + dim, [300], 2, dim, 1)
    rng = s.rng
    sign = rng.choice([-1.0, 1.0], (2, 1, dim))
    size = np.exp(4.0 * rng.standard_normal((2, group, dim))) if other != "any" else np.abs(rng.standard_normal((2, group, dim)))
    q = (sign * size).astype(np.float32)
    hi, lo = (np.sort(rng.standard_normal((2, 2, dim)), axis=0)[::-1]).astype(np.float16)  # [kv][dim] each
    unused = np.abs(rng.standard_normal((s.n_pages, 2, dim)))
    if other != "any":
        unused[rng.random(unused.shape) < (0.02 if other == "mixed" else 0.9)] = ref.H_MAX
    up = q[:, 0] >= 0
    bounds = np.empty((s.n_pages, 2, 2, dim), np.float16)
    bounds[:, :, 0] = np.where(up, hi, np.minimum(lo + unused, ref.H_MAX))
    bounds[:, :, 1] = np.where(up, np.maximum(hi - unused, -ref.H_MAX), lo)
    q = q.reshape(1, 2 * group, dim)
    for select in (1, 7, 150, 299):
        assert listed_pages(s, bounds, q, select).tolist() == [list(range(select))] * 2


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_close_scores_in_their_exact_order(dim):
    """Scores apart by some 2^-24 of their terms, beside unused extremes at the clamp: the order
    of the exact sums. A sum of dim exact products in 64 bits is off by at most dim 2^-53 of
    the terms' magnitudes, and no two scores lie closer than 2^-40 of them."""
    s = Setup(7 + dim, [200], 1, dim, 1)
    rng = s.rng
    q = rng.standard_normal(dim).astype(np.float32)
    q[5], q[6] = np.float32(2.0 ** -12), np.float32(-(2.0 ** -12))
    up = q >= 0
    used = np.broadcast_to(rng.standard_normal(dim).astype(np.float16), (s.n_pages, dim)).copy()
    used[:, 5] = (1.0 + rng.permutation(s.n_pages) / 1024).astype(np.float16)  # steps of 2^-10, exact
    far = rng.random((s.n_pages, dim)) < 0.5
    bounds = np.empty((s.n_pages, 1, 2, dim), np.float16)
    bounds[:, 0, 0] = np.where(up, used, np.where(far, ref.H_MAX, used + np.float16(1.0)))
    bounds[:, 0, 1] = np.where(up, np.where(far, -ref.H_MAX, used - np.float16(1.0)), used)
    pages = s.table[0]
    score = [sum(Fraction(float(a)) * Fraction(float(b)) for a, b in zip(q, used[p])) for p in pages]
    terms = sum(abs(Fraction(float(a)) * Fraction(float(b))) for a, b in zip(q, used[pages[0]]))
    order = sorted(range(200), key=lambda t: (-score[t], t))
    assert min(score[a] - score[b] for a, b in zip(order, order[1:])) > terms / 2 ** 40
    for select in (1, 60, 199):
        got = listed_pages(s, bounds, q.reshape(1, 1, dim), select)
        assert got[0].tolist() == sorted(order[:select])


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("value", [np.inf, -np.inf])
def test_infinite_queries_rank_by_the_definition(dim, value):
    """+inf times an extreme of the query's sign is +inf and ranks first, -inf ranks behind every
    finite score, 0 times an infinity counts for nothing and ranks last."""
    s = Setup(3 + dim, [6], 1, dim, 1)
    q = np.ones((1, 2, dim), np.float32)
    q[0, 0, 9] = value
    q[0, 1] = np.nan  # does not count
    bounds = np.zeros((s.n_pages, 1, 2, dim), np.float16)
    bounds[:, 0, 0] = 1.0
    pairs = [(0.0, -3.0), (-1.0, -2.0), (1.0, -3.0), (2.0, 2.0), (5.0, 1.0), (0.0, 0.0)]
    first = [2, 3, 4]  # of a positive infinity
    if value < 0:
        pairs = [(-b, -a) for a, b in pairs]
    for t, (a, b) in enumerate(pairs):
        bounds[s.table[0, t], 0, :, 9] = a, b
    for select, want in ((1, [2]), (3, first), (4, [1, 2, 3, 4]), (5, [0, 1, 2, 3, 4])):
        assert listed_pages(s, bounds, q, select)[0].tolist() == want


def test_reversed_bounds_count_both_ways():
    """A page of NaN keys alone has its bounds in reverse order, and scores as the largest."""
    s = Setup(4, [9], 1, 64, 1)
    bounds = np.zeros((s.n_pages, 1, 2, 64), np.float16)
    bounds[:, 0, 0], bounds[:, 0, 1] = 3.0, -3.0
    bounds[s.table[0, 6], 0, 0], bounds[s.table[0, 6], 0, 1] = -ref.H_MAX, ref.H_MAX
    q = s.rng.standard_normal((1, 3, 64)).astype(np.float32)
    assert listed_pages(s, bounds, q, 1)[0].tolist() == [6]
