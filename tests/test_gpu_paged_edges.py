"""The paged-cache operators (include/rtxllm/paged_kv.h) where their definitions are decided by
the last bit, by an infinity or by a page that is not there."""

from __future__ import annotations

from fractions import Fraction

import numpy as np
import paged_ref as ref
import pytest

torch = pytest.importorskip("torch")

from rtxllm_amd import paged  # noqa: E402
from test_gpu_paged import DEV, Setup, check_attention, dev, u32  # noqa: E402

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


# ---- eviction from a table with holes ------------------------------------------------


def evict_around_holes(there, length, newest, keep, n_first, n_recent, weight, slot_pos):
    """Source slot of each slot below keep: slots in no page stay below keep and leave behind it,
    the others fill what is left of keep by rank."""
    def rank(i):
        p, w = int(slot_pos[i]), float(weight[i])
        if p < n_first or p + n_recent > newest:
            return (0, 0.0, i)
        return (2, 0.0, i) if np.isnan(w) else (1, -w, i)

    fixed = {i for i in range(keep) if not there[i]}
    kept = fixed | set(sorted((i for i in range(length) if there[i]), key=rank)[:keep - len(fixed)])
    late = iter(sorted(i for i in kept if i >= keep))
    return [i if i in kept else next(late) for i in range(keep)]


# (slots, keep, page): moves in the choosing workgroup and apart, more table entries than one
# round of a workgroup's loads, more slots than the LDS holds, four waves of many short sequences
@pytest.mark.parametrize("n,keep,page,count,dim", [
    (130, 100, 7, 3, 64), (130, 100, 7, 3, 256), (130, 100, 1, 3, 128), (600, 300, 16, 2, 64), (600, 300, 16, 2, 256),
    (2112, 2048, 64, 2, 128), (9000, 5000, 1, 1, 64), (33000, 20000, 24, 1, 64), (200, 150, 8, 130, 64), (200, 150, 8, 130, 256)])
@pytest.mark.parametrize("place", ["apart", "in-place"])
@pytest.mark.parametrize("where", ["below", "behind", "both", "all-behind", "all-below"])
def test_evict_around_holes(n, keep, page, count, dim, place, where):
    """No key or value of a page that is not there counts: what stays is read back key by key."""
    kv = 2
    s = Setup(n + keep + page, [n] * count, kv, dim, page)
    rng = s.rng
    first_behind = -(-keep // page)
    for row in s.table:
        low, high = np.arange(0, keep // page), np.arange(first_behind, s.entries)
        some = {"below": rng.permutation(low)[:max(1, len(low) // 3)], "behind": rng.permutation(high)[:max(1, len(high) // 3)],
                "all-behind": high, "all-below": low}
        some["both"] = np.concatenate([some["below"], some["behind"]])
        row[some[where]] = rng.choice([-1, s.n_pages, 2 ** 31 - 1], len(some[where]))
    s.cache.block_table.copy_(dev(s.table))
    weight = (rng.integers(0, 50, (count, kv, s.capacity)) / 8).astype(np.float32)
    weight[:, :, ::5] = np.nan
    slot_pos = np.stack([[rng.permutation(s.capacity) for _ in range(kv)] for _ in range(count)]).astype(np.uint32)
    newest = [int(p[:, :n].max()) for p in slot_pos]
    wd, sd, ld = dev(weight), u32(slot_pos), u32([n] * count)
    apart = place == "apart"
    wo, so, lo = (torch.full_like(t, 7) for t in (wd, sd, ld)) if apart else (wd, sd, ld)
    paged.evict(s.cache, ld, u32(newest), keep, wd, sd, 3, 20, wo if apart else None, so if apart else None,
                lo if apart else None)
    gw, gp, gk, gv = wo.cpu().numpy(), so.cpu().numpy().view(np.uint32), s.kd.cpu().numpy(), s.vd.cpu().numpy()
    assert lo.cpu().tolist() == [keep] * count
    k_want, v_want = s.k.copy(), s.v.copy()
    for i in range(count):
        place_of = np.array([ref.at(s.table[i], s.n_pages, page, t) or (-1, -1) for t in range(n)])
        there = place_of[:, 0] >= 0
        for g in range(kv):
            src = np.array(evict_around_holes(there, n, newest[i], keep, 3, 20, weight[i, g], slot_pos[i, g]))
            np.testing.assert_array_equal(gw[i, g, :keep], weight[i, g, src])
            np.testing.assert_array_equal(gp[i, g, :keep], slot_pos[i, g, src])
            to = np.flatnonzero(src != np.arange(keep))
            assert there[to].all() and there[src[to]].all()
            (p, o), (p2, o2) = place_of[to].T, place_of[src[to]].T
            k_want[p, g, o], v_want[p, g, o] = s.k[p2, g, o2], s.v[p2, g, o2]
    np.testing.assert_array_equal(gk.view(np.uint16), k_want.view(np.uint16))
    np.testing.assert_array_equal(gv.view(np.uint16), v_want.view(np.uint16))


# ---- attention: queries of very different sizes in one head ---------------------------


@pytest.mark.parametrize("group", [1, 4, 8, 12, 16])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("large", [1e4, 1e5, 1e7])
def test_attention_beside_a_large_query(group, dim, large):
    """One element of a query is some powers of ten above the others, where the keys are 0. Each
    element enters as an fp16 pair: off by 2^-22 of itself or 2^-39 of the head's largest.
    The rest of the bound is that of paged_ref.attend."""
    s = Setup(group + dim, [150, 70], 2, dim, 16)
    rng = s.rng
    at = rng.integers(0, dim)
    s.k[..., at] = 0.0
    s.kd.copy_(dev(s.k))
    q = rng.standard_normal((2, 2 * group, dim)).astype(np.float32)
    q[..., at] = large
    weight = torch.zeros(2, 2, s.capacity, device=DEV)
    pages = torch.arange(s.entries, dtype=torch.int32, device=DEV).expand(2, 2, -1).contiguous()
    listed = paged.attn_pages(s.cache, dev(q), pages, u32(s.last())).cpu().numpy()
    dense = paged.attn_weights(s.cache, dev(q), u32(s.last()), weight).cpu().numpy()
    gathered = weight.cpu().numpy()
    for i, n in enumerate(s.lens):
        for g in range(2):
            keys, values, _ = s.rows(i, g, range(n))
            keys, values = keys.astype(np.float64), values.astype(np.float64)
            total, slack = np.zeros(n), np.zeros(n)
            for h in range(g * group, (g + 1) * group):
                x = q[i, h].astype(np.float64)
                score = keys @ x / np.sqrt(dim)
                p = np.exp(score - score.max())
                p /= p.sum()
                size = np.abs(keys) @ np.abs(x)
                delta = ((2.0 ** -22 + (dim + 8) * 2.0 ** -24) * size +
                         2.0 ** -39 * np.abs(x).max() * np.abs(keys).sum(1)).max() / np.sqrt(dim)
                bound = 2.0 * (delta + 2.0 ** -21 * (1.0 + np.abs(score).max())) + (n / 4 + 40) * 2.0 ** -24
                for got in (listed, dense):
                    assert (np.abs(got[i, h] - p @ values) <= bound * (p @ np.abs(values)) + 1e-37).all(), (i, h)
                total += p
                slack += p * bound + 2.0 ** -40
            assert (np.abs(gathered[i, g, :n] - total) <= slack + (group + 1) * 2.0 ** -24 * total).all(), (i, g)


@pytest.mark.parametrize("group", [1, 5, 12])
@pytest.mark.parametrize("large", [1e3, 1e7, 1e20])
def test_gathered_weights_of_large_scores(group, large):
    """Scores of thousands and more: what is gathered is the softmax itself, 1 for each head in all.
    Two positions of each head lie a few units apart, all others far below; products and sums
    are exact (one nonzero dimension, keys of few bits)."""
    s = Setup(group + 2, [200], 1, 64, 16)
    p, o = np.array(s.seen[0]).T
    s.k[:] = 0.0
    s.k[p, 0, o, 3] = s.rng.integers(0, 64, 200) / np.float16(64.0)
    s.k[p[[7, 150]], 0, o[[7, 150]], 3] = 2.0
    s.k[p[7], 0, o[7], 4] = 1.0
    s.kd.copy_(dev(s.k))
    q = np.zeros((1, group, 64), np.float32)
    q[0, :, 3] = large
    q[0, :, 4] = np.arange(group) / 2.0
    weight = torch.zeros(1, 1, s.capacity, device=DEV)
    paged.attn_weights(s.cache, dev(q), u32([199]), weight)
    got = weight.cpu().numpy()[0, 0]
    # the scores round to fp32 at 2 large / 8 (log2(e) in), where they lie apart by half a unit a head
    score = 2.0 * large / 8.0 * 1.4427
    want = np.zeros(s.capacity)
    apart = q[0, :, 4].astype(np.float64) / 8.0
    want[7], want[150] = (1.0 / (1.0 + np.exp(-apart))).sum(), (1.0 / (1.0 + np.exp(apart))).sum()
    slack = group * min(1.0, 2.0 * score * 2.0 ** -22) + 1e-6
    assert abs(got.sum() - group) <= group * 16 * 2.0 ** -24
    assert (np.abs(got - want) <= slack).all()


@pytest.mark.parametrize("group", [1, 12])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_attention_with_the_largest_queries(group, dim):
    """Finite queries up to the largest fp32 number, over keys so small that the scores are finite:
    the position with the largest score takes all (the others lie 10^28 and more below)."""
    s = Setup(group + dim + 1, [90], 1, dim, 16)
    rng = s.rng
    s.k[:] = 0.0
    p, o = np.array(s.seen[0]).T
    steps = rng.permutation(90)
    s.k[p, 0, o, 7] = steps * np.float16(2.0 ** -24)  # exact subnormals
    s.kd.copy_(dev(s.k))
    q = np.zeros((1, group, dim), np.float32)
    q[..., 7] = np.where(np.arange(group) % 2, -1.0, 1.0) * np.finfo(np.float32).max
    weight = torch.zeros(1, 1, s.capacity, device=DEV)
    pages = torch.arange(s.entries, dtype=torch.int32, device=DEV).reshape(1, 1, -1)
    for got in (paged.attn_pages(s.cache, dev(q), pages, u32([89])), paged.attn_weights(s.cache, dev(q), u32([89]), weight)):
        for h, row in enumerate(got.cpu().numpy()[0]):
            top = int(np.argmin(steps) if h % 2 else np.argmax(steps))
            np.testing.assert_allclose(row, s.v[p[top], 0, o[top]], rtol=1e-6)
    assert float(weight.sum()) == group


# ---- the wrapper's numbers --------------------------------------------------------------


def test_numbers_are_not_cut_to_32_bits():
    """What the C-ABI's unsigned arguments cannot hold is refused, not taken for its low bits."""
    k = torch.zeros(1, 1, 65536, 64, dtype=torch.float16, device=DEV)
    for entries in (65537, 257, 65536):  # 2^32 + 65536, just above 2^24 and 2^32 positions
        with pytest.raises(ValueError):
            paged.PagedKV(k, k, torch.zeros(entries, dtype=torch.int32, device=DEV))
            pytest.fail(f"{entries} entries were not refused")
    paged.PagedKV(k, k, torch.zeros(256, dtype=torch.int32, device=DEV))
    for shape in ((0, 1, 8, 64), (1, 0, 8, 64), (1, 1, 0, 64), (1, 1, 8, 0)):
        none = torch.zeros(shape, dtype=torch.float16, device=DEV)
        with pytest.raises(ValueError):
            paged.PagedKV(none, none, torch.zeros(4, dtype=torch.int32, device=DEV))
            pytest.fail(f"{shape} was not refused")
    s = Setup(1, [20, 20], 2, 64, 8)
    c, pos = s.cache, u32([3, 4])
    q, kn = torch.zeros(2, 4, 64, device=DEV), torch.zeros(2, 2, 64, device=DEV)
    bounds = torch.zeros(s.n_pages, 2, 2, 64, dtype=torch.float16, device=DEV)
    state = torch.zeros(2, 2, s.capacity, device=DEV)
    over = 1 << 32
    before = [t.clone() for t in (s.kd, s.vd, bounds, state)]
    bad = [lambda: paged.qk_norm_rope_append(c, q, kn, kn, None, None, pos, theta=1e4, rotary_dim=over + 64),
           lambda: paged.page_bounds(c, pos, bounds, span=over + 1),
           lambda: paged.select_workspace(c, over + 1),
           lambda: paged.select_pages(c, bounds, q, pos, over + 3),
           lambda: paged.select_pages(c, bounds, q, pos, 3, n_first=over),
           lambda: paged.select_pages(c, bounds, q, pos, 3, n_last=-over),
           lambda: paged.attn_pages_workspace(c, over + 4, 3, 2),
           lambda: paged.attn_pages_workspace(c, 4, over + 3, 2),
           lambda: paged.attn_weights_workspace(c, 4, over + 2),
           lambda: paged.evict_workspace(c, over + 4, 2),
           lambda: paged.evict(c, pos, pos, over + 4, state, state.int()),
           lambda: paged.evict(c, pos, pos, 4, state, state.int(), n_first=over),
           lambda: paged.evict(c, pos, pos, 4, state, state.int(), n_recent=-1)]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was not refused")
    for t, b in zip((s.kd, s.vd, bounds, state), before):
        torch.testing.assert_close(t, b, rtol=0, atol=0, equal_nan=True)


# ---- eviction and selection of one cache --------------------------------------------------


def test_selection_after_an_eviction():
    """Rows move into other pages: with the bounds of the kept slots' pages computed anew the
    selection and its attention are those of what the slots hold now."""
    s = Setup(23, [200, 150], 2, 128, 16)
    group, keep, select = 3, 100, 4
    weight = s.rng.random((2, 2, s.capacity)).astype(np.float32)
    slot_pos = np.broadcast_to(np.arange(s.capacity, dtype=np.uint32), weight.shape)
    length, pos = u32(s.lens), u32(s.last())
    bounds = torch.zeros(s.n_pages, 2, 2, 128, dtype=torch.float16, device=DEV)
    zero = torch.zeros_like(pos)
    paged.page_bounds(s.cache, pos, bounds, zero, s.entries)
    paged.evict(s.cache, length, pos, keep, dev(weight), u32(slot_pos), 2, 10)
    last = u32([keep - 1] * 2)
    paged.page_bounds(s.cache, last, bounds, zero, s.entries)
    q = s.rng.standard_normal((2, 2 * group, 128)).astype(np.float32)
    pages = paged.select_pages(s.cache, bounds, dev(q), last, select, 1, 1)
    out = paged.attn_pages(s.cache, dev(q), pages, last).cpu().numpy()
    s.k, s.v = s.kd.cpu().numpy(), s.vd.cpu().numpy()
    gb, gp = bounds.cpu().numpy(), pages.cpu().numpy()
    for i in range(2):
        for g in range(2):
            for t in range(-(-keep // 16)):
                p = s.table[i, t]
                np.testing.assert_array_equal(gb[p, g], ref.bounds_of(s.k[p, g, :min(16, keep - 16 * t)]))
            want = ref.select(q[i, g * group:(g + 1) * group], gb[:, g], s.table[i], s.n_pages, 7, 1, 1, select)
            assert gp[i, g].tolist() == want
            check_attention(s, out, q, i, g, group, [x for t in want for x in range(16 * t, min(keep, 16 * t + 16))])
