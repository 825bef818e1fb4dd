"""The paged-cache operators (include/rtxllm/paged_kv.h) against float64 (paged_ref.py):
append with norm and rotation, page bounds, page selection, attention over listed
pages, attention that gathers weights, eviction. What lies behind a context is NaN or
infinite throughout, tables are shuffled and may have holes."""

from __future__ import annotations

import numpy as np
import paged_ref as ref
import pytest

torch = pytest.importorskip("torch")

from rtxllm_amd import paged  # noqa: E402

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def u32(values) -> torch.Tensor:
    return torch.from_numpy(np.asarray(values, np.uint32).view(np.int32).copy()).to(DEV)


def dev(a) -> torch.Tensor:
    return torch.from_numpy(np.ascontiguousarray(a)).to(DEV)


class Setup:
    """A cache of len(lens) sequences; slots behind each length hold NaN and inf."""

    def __init__(self, seed, lens, kv, dim, page, entries=None, hole=False, one=False, spare=3, stride=None):
        rng = self.rng = np.random.default_rng(seed)
        self.kv, self.dim, self.page, self.lens, self.one = kv, dim, page, lens, one
        self.entries = entries or max(1, max(-(-n // page) for n in lens))
        self.capacity = self.entries * page
        self.n_pages = len(lens) * self.entries + spare
        shape = (self.n_pages, kv, page, dim)
        self.k = (0.9 * rng.standard_normal(shape) + 0.5 * rng.standard_normal((self.n_pages, kv, 1, dim))).astype(np.float16)
        self.v = rng.standard_normal(shape).astype(np.float16)
        self.table = rng.permutation(self.n_pages)[:len(lens) * self.entries].astype(np.int32).reshape(len(lens), -1)
        self.seen = [[ref.at(self.table[i], self.n_pages, page, s) for s in range(n)] for i, n in enumerate(lens)]
        poison = np.ones((self.n_pages, page), bool)
        for row in self.seen:
            for p, o in row:
                poison[p, o] = False
        for a, bad in ((self.k, np.nan), (self.v, np.inf)):
            a[np.broadcast_to(poison[:, None, :, None], shape)] = bad
            a[::2][np.broadcast_to(poison[::2, None, :, None], a[::2].shape)] = -np.inf
        if hole:  # a page in the middle of the longest sequence is not there
            i = int(np.argmax(lens))
            t = max(0, -(-lens[i] // page) // 2)
            self.table[i, t] = -1 if hole is True else hole
            self.seen[i] = [ref.at(self.table[i], self.n_pages, page, s) for s in range(lens[i])]
        self.kd, self.vd = dev(self.k), dev(self.v)
        wide = np.full((len(lens), stride or self.entries), -7, np.int32)  # rows further apart than they are long
        wide[:, :self.entries] = self.table
        td = dev(wide)[:, :self.entries]
        self.cache = paged.PagedKV(self.kd, self.vd, td[0].contiguous() if one else td)

    def rows(self, i, g, slots):
        """(keys, values, the slots that are there)."""
        there = [s for s in slots if self.seen[i][s] is not None]
        pick = [self.seen[i][s] for s in there]
        p, o = np.array([x for x, _ in pick], int), np.array([x for _, x in pick], int)
        return self.k[p, g, o], self.v[p, g, o], there

    def last(self):
        return [n - 1 if n else ref.NONE for n in self.lens]


def close(got, want, tol, what):
    bad = ~(np.abs(got.astype(np.float64) - want) <= tol)
    assert not bad.any(), (what, np.argwhere(bad)[:4].tolist(), got[bad][:4], want[bad][:4], np.broadcast_to(tol, want.shape)[bad][:4])


# ---- append --------------------------------------------------------------------

# (query heads, kv heads, head_dim, page, rotary, pairing)
APPEND = [(32, 8, 128, 64, 128, "halves"), (3, 1, 64, 5, 8, "adjacent"), (10, 2, 256, 24, 256, "halves"),
          (7, 7, 128, 16, 64, "adjacent"), (16, 1, 256, 48, 72, "halves"), (1, 1, 64, 1, 64, "adjacent")]


@pytest.mark.parametrize("shape", APPEND, ids=str)
@pytest.mark.parametrize("mode", ["batch", "one-row", "prompt", "stacked-slots"])
def test_append(shape, mode):
    heads, kv, dim, page, rotary, pairing = shape
    one = mode == "prompt"
    count = {"batch": 5, "one-row": 1, "prompt": 37, "stacked-slots": 4}[mode]
    s = Setup(heads + dim, [41] if one else [41] * count, kv, dim, page, one=one, hole=True, stride=60)
    rng = s.rng
    slot = np.arange(2, 2 + count) if one else rng.integers(0, 41, count)
    pos = slot.astype(np.uint32)
    if mode == "batch":
        pos[3] = ref.NONE
        pos[4] = s.capacity + 9  # no such slot: q alone
    if mode == "stacked-slots":
        pos = np.array([0, 131071, 4095, 2 ** 31 + 12345], np.uint32)
        wide = rng.standard_normal((count, (heads + 2 * kv) * dim + 3)).astype(np.float32) * np.float32(20.0)
        wide[0] *= np.float32(1e-6)
        src = dev(wide)[:, 1:]
        qd, kd, vd = src[:, :-2].split([heads * dim, kv * dim, kv * dim], 1)
        x = wide[:, 1:-2]
        q, k, v = (a.reshape(count, -1, dim) for a in np.split(x, [heads * dim, (heads + kv) * dim], 1))
        qd, kd, vd = (t.unflatten(1, (-1, dim)) for t in (qd, kd, vd))
    else:
        q, k, v = (rng.standard_normal((count, h, dim)).astype(np.float32) for h in (heads, kv, kv))
        qd, kd, vd = dev(q), dev(k), dev(v)
    qw = (1.0 + 0.1 * rng.standard_normal(dim)).astype(np.float32)
    kw = None if mode == "one-row" else (1.0 + 0.1 * rng.standard_normal(dim)).astype(np.float32)
    nseq = len(s.lens)
    slot_pos = rng.integers(0, 99, (nseq, kv, s.capacity)).astype(np.uint32)
    weight = rng.random((nseq, kv, s.capacity)).astype(np.float32)
    spd, wd = u32(slot_pos), dev(weight)
    out = torch.full((count, heads, dim), 7.0, device=DEV)
    use_slot = mode == "stacked-slots"
    paged.qk_norm_rope_append(s.cache, qd, kd, vd, dev(qw), None if kw is None else dev(kw), u32(pos), theta=500000.0,
                              eps=1e-6, rotary_dim=rotary, pairing=pairing, slot=u32(slot) if use_slot else None,
                              q_out=out, slot_pos=spd, slot_weight=wd)
    got, gk, gv = out.cpu().numpy(), s.kd.cpu().numpy(), s.vd.cpu().numpy()
    k_want, v_want = s.k.copy(), s.v.copy()
    # fp32: 8 products and 5 steps of the sum of squares, halved by the root, the mean, eps,
    # root, quotient and two products; the angle's fraction and its sine; product and sum
    eps32 = 24 * 2.0 ** -24
    touched = np.zeros(s.k.shape, bool)
    for r in range(count):
        if pos[r] == ref.NONE:
            assert np.all(got[r] == 7.0)
            continue
        for h in range(heads):
            want, size = ref.norm_rope(q[r, h], qw, pos[r], 500000.0, 1e-6, rotary, pairing == "halves")
            close(got[r, h], want, eps32 * size, (r, h))
        sl = int(slot[r]) if use_slot else int(pos[r])
        i = 0 if one else r
        if sl >= s.capacity:
            continue
        slot_pos[i, :, sl], weight[i, :, sl] = pos[r], 0.0
        place = ref.at(s.table[i], s.n_pages, page, sl)
        if place is None:
            continue
        p, o = place
        for g in range(kv):
            want, size = ref.norm_rope(k[r, g], kw, pos[r], 500000.0, 1e-6, rotary, pairing == "halves")
            close(gk[p, g, o], want, 2.0 ** -11 * np.abs(want) + 2 * eps32 * size + 2.0 ** -25, ("k", r, g))
            v_want[p, g, o] = v[r, g].astype(np.float16)
            touched[p, g, o] = True
    np.testing.assert_array_equal(gk.view(np.uint16)[~touched], k_want.view(np.uint16)[~touched])
    np.testing.assert_array_equal(gv.view(np.uint16), v_want.view(np.uint16))
    np.testing.assert_array_equal(spd.cpu().numpy().view(np.uint32), slot_pos)
    np.testing.assert_array_equal(wd.cpu().numpy(), weight)


def test_append_in_place_and_extremes():
    """q in place gives the bits of q apart; a zero head stays 0, one with a NaN is NaN,
    a value beyond fp16 is stored as an infinity."""
    s = Setup(3, [9, 9, 9], 2, 128, 4)
    q, k, v = (s.rng.standard_normal((3, h, 128)).astype(np.float32) for h in (6, 2, 2))
    q[0, 1], q[1, 2, 5], k[2, 0], v[2, 1, 3] = 0.0, np.nan, 0.0, 1e6
    pos = u32([8, 3, 0])
    qd = dev(q)
    args = (dev(k), dev(v), None, None, pos)
    apart = paged.qk_norm_rope_append(s.cache, qd, *args, theta=1e4).cpu().numpy()
    paged.qk_norm_rope_append(s.cache, qd, *args, theta=1e4, q_out=qd)
    np.testing.assert_array_equal(qd.cpu().numpy(), apart)
    assert np.all(apart[0, 1] == 0.0) and np.isnan(apart[1, 2]).all() and not np.isnan(apart[1, 1]).any()
    p = int(s.table[2, 0])
    assert np.all(s.kd[p, 0, 0].cpu().numpy() == 0.0) and np.isinf(s.vd[p, 1, 0, 3].item())


# ---- bounds and selection --------------------------------------------------------

POOL = [(4, 128, 64), (2, 64, 16), (1, 256, 24), (3, 128, 7), (8, 64, 1)]


# (a wave, a part of one or four waves a page, by its size and by the pages of a call)
@pytest.mark.parametrize("kv,dim,page", POOL + [(16, 128, 64), (2, 128, 21), (1, 128, 300), (3, 64, 130)])
def test_page_bounds(kv, dim, page):
    lens = [page * 9 + 1, 0, 1, page * 4, page * 6 + page // 2 + 1]
    s = Setup(dim + page, lens, kv, dim, page, hole=True, stride=31)
    p, o = s.seen[0][0]
    s.k[p, 0, o, 3], s.k[p, 0, o, 5] = np.inf, -np.inf
    s.k[p, :, :min(page, lens[0]), 7] = np.nan
    s.kd.copy_(dev(s.k))
    for first in (None, [0] * 5, [page + 1, 5, 0, page * 4, 0]):
        span = 1 if first is None else 7
        want = s.rng.standard_normal((s.n_pages, kv, 2, dim)).astype(np.float16)
        bd = dev(want)
        paged.page_bounds(s.cache, u32(s.last()), bd, None if first is None else u32(first), span)
        for i, n in enumerate(lens):
            f = n - 1 if first is None else first[i]
            for t in range(f // page, min(f // page + span, -(-n // page))) if n and f < n else ():
                page_at = int(s.table[i, t])
                if page_at >= 0:
                    for g in range(kv):
                        want[page_at, g] = ref.bounds_of(s.k[page_at, g, :min(page, n - t * page)])
        np.testing.assert_array_equal(bd.cpu().numpy(), want)


@pytest.mark.parametrize("group", [1, 3, 8, 16])
@pytest.mark.parametrize("kv,dim,page", POOL)
@pytest.mark.parametrize("first,last,select", [(1, 1, 5), (0, 0, 1), (2, 3, 5), (0, 1, 64), (1, 2, 1000)])
def test_select_pages(group, kv, dim, page, first, last, select):
    lens = [page * 70 + 1, 0, 1, page * 4, page * 20]
    s = Setup(dim + page + group, lens, kv, dim, page, hole=s_hole(select))
    bounds = np.sort(s.rng.standard_normal((s.n_pages, kv, 2, dim)).astype(np.float16), axis=2)[:, :, ::-1]
    for a, b in ((3, 9), (9, 30), (11, 12)):  # equal scores: the lower page
        bounds[s.table[0, a]] = bounds[s.table[0, b]]
    q = s.rng.standard_normal((5, group * kv, dim)).astype(np.float32)
    q[4, 0, 1] = np.nan
    pages = torch.full((5, kv, select), -9, dtype=torch.int32, device=DEV)
    paged.select_pages(s.cache, dev(bounds), dev(q), u32(s.last()), select, first, last, pages=pages)
    got = pages.cpu().numpy()
    assert np.all(got[1] == -9)  # a padded row
    for i, n in enumerate(lens):
        for g in range(kv if n else 0):
            want = ref.select(q[i, g * group:(g + 1) * group], bounds[:, g], s.table[i], s.n_pages, -(-n // page), first,
                              last, select)
            assert got[i, g].tolist() == want + [-1] * (select - len(want)), (i, g)


def s_hole(select):
    return select != 64


@pytest.mark.parametrize("n", [5000, 16384, 16385, 33000])
def test_select_many_pages_with_ties(n):
    """Thousands of pages of few distinct scores: ties across the whole radix, lowest
    first; more pages than a workgroup holds at once."""
    s = Setup(1, [n], 2, 64, 1)
    levels = s.rng.standard_normal((6, 2, 2, 64)).astype(np.float16)
    bounds = levels[s.rng.integers(0, 6, s.n_pages)]
    q = s.rng.standard_normal((1, 4, 64)).astype(np.float32)
    for select in (1, 700, 2049, n - 1, n, n + 1000):
        f, l = (3, 2) if select >= 5 else (0, 1)
        got = paged.select_pages(s.cache, dev(bounds), dev(q), u32([n - 1]), select, f, l).cpu().numpy()
        for g in range(2):
            want = ref.select(q[0, 2 * g:2 * g + 2], bounds[:, g], s.table[0], s.n_pages, n, f, l, select)
            assert got[0, g].tolist() == want + [-1] * (select - len(want))


# ---- attention over listed pages ---------------------------------------------------

ATTN = [(4, 8, 128, 64), (1, 2, 64, 16), (8, 1, 256, 24), (16, 2, 128, 7), (5, 3, 64, 1), (3, 1, 256, 40), (12, 1, 64, 128),
        (16, 1, 256, 16)]


def check_attention(s, got, q, i, g, group, slots, weight=None):
    keys, values, there = s.rows(i, g, slots)
    total = np.zeros(len(slots))
    tol_w = np.zeros(len(slots))
    index = {}
    for j, sl in enumerate(slots):
        index.setdefault(sl, []).append(j)
    for h in range(g * group, (g + 1) * group):
        p, o, tol, ptol = ref.attend(q[i, h], keys, values)
        close(got[i, h], o, tol, (i, h))
        for t, sl in enumerate(there):
            total[index[sl][0]] += p[t]
            tol_w[index[sl][0]] += ptol[t]
    return total, tol_w


@pytest.mark.parametrize("group,kv,dim,page", ATTN)
@pytest.mark.parametrize("select", [1, 6, 33])
def test_attn_pages(group, kv, dim, page, select):
    lens = [page * 40 + page // 2 + 1, 0, 1, page * 3, page + 1]
    s = Setup(group + dim + page, lens, kv, dim, page, hole=10 ** 6)
    q = s.rng.standard_normal((5, group * kv, dim)).astype(np.float32)
    q[0] *= np.float32(3.0)
    q[3] *= np.float32(1e-7)
    pages = np.full((5, kv, select), -1, np.int32)
    for i, n in enumerate(lens):
        used = -(-n // page)
        for g in range(kv if n else 0):
            some = s.rng.permutation(used)[:select]  # any order, and entries that name nothing between
            pages[i, g, s.rng.permutation(select)[:len(some)]] = some
            pages[i, g][(pages[i, g] < 0) & (s.rng.random(select) < 0.5)] = s.entries + 3
    out = torch.full((5, group * kv, dim), 7.0, device=DEV)
    paged.attn_pages(s.cache, dev(q), dev(pages), u32(s.last()), out=out)
    got = out.cpu().numpy()
    assert np.all(got[1] == 7.0)
    for i, n in enumerate(lens):
        for g in range(kv if n else 0):
            listed = [t for t in pages[i, g] if 0 <= t < s.entries]
            check_attention(s, got, q, i, g, group, [x for t in listed for x in range(t * page, min(n, t * page + page))])
    over = dev(q)  # the queries make way for the results
    paged.attn_pages(s.cache, over, dev(pages), u32(s.last()), out=over)
    got[1] = q[1]
    np.testing.assert_array_equal(over.cpu().numpy(), got)


@pytest.mark.parametrize("group,kv,dim", [(4, 2, 64), (1, 8, 128), (8, 1, 256), (12, 2, 128), (2, 16, 128)])
@pytest.mark.parametrize("select", [60, 600])
def test_attn_pages_lists_longer_than_the_context(group, kv, dim, select):
    """Room for far more pages than are listed: rows of few tiles, one of many whose list
    names pages again and again to its end."""
    page, lens = 16, [700, 0, 1, 90, 130]
    s = Setup(group + dim + select, lens, kv, dim, page)
    q = s.rng.standard_normal((5, group * kv, dim)).astype(np.float32)
    pages = np.full((5, kv, select), -1, np.int32)
    for i, n in enumerate(lens):
        used = -(-n // page)
        pages[i, :, :used] = s.rng.permutation(used)
    pages[4, :, ::2] = s.rng.integers(0, 9, (kv, -(-select // 2)))
    got = paged.attn_pages(s.cache, dev(q), dev(pages), u32(s.last())).cpu().numpy()
    for i, n in enumerate(lens):
        for g in range(kv if n else 0):
            listed = [t for t in pages[i, g] if 0 <= t < s.entries]
            check_attention(s, got, q, i, g, group, [x for t in listed for x in range(t * page, min(n, t * page + page))])


def test_attn_pages_empty_twice_and_extremes():
    s = Setup(5, [64, 64, 64, 64, 64], 1, 128, 16)
    q = s.rng.standard_normal((5, 2, 128)).astype(np.float32)
    q[3, 0] *= np.float32(1e30)  # one position takes all
    q[4, 1, 9] = np.nan
    pages = np.array([[-1, -1, -1], [2, 2, 0], [3, -1, 99], [0, 1, 2], [0, 1, 2]], np.int32)[:, None]
    got = paged.attn_pages(s.cache, dev(q), dev(pages), u32([63] * 5)).cpu().numpy()
    assert np.all(got[0] == 0.0)  # nothing listed
    check_attention(s, got, q, 1, 0, 2, [*range(32, 48), *range(32, 48), *range(16)])
    check_attention(s, got, q, 2, 0, 2, range(48, 64))
    keys, values, _ = s.rows(3, 0, range(48))
    np.testing.assert_allclose(got[3, 0], values[np.argmax(keys.astype(np.float64) @ q[3, 0])], rtol=1e-6)
    assert np.isnan(got[4, 1]).all() and np.isfinite(got[4, 0]).all()
    # a sequence whose table names no page at all
    s.cache.block_table[1] = -1
    assert np.all(paged.attn_pages(s.cache, dev(q), dev(pages), u32([63] * 5)).cpu().numpy()[1] == 0.0)


# ---- attention that gathers weights, eviction ----------------------------------------


@pytest.mark.parametrize("group,kv,dim,page", ATTN)
@pytest.mark.parametrize("place", ["apart", "in-place"])
def test_attn_weights(group, kv, dim, page, place):
    lens = [page * 17 + page // 3 + 1, 0, 1, page * 3, page + 1, 2]
    s = Setup(group + dim + page, lens, kv, dim, page, entries=19, hole=True)
    q = s.rng.standard_normal((6, group * kv, dim)).astype(np.float32)
    weight = s.rng.random((6, kv, s.capacity)).astype(np.float32)
    wd = dev(weight)
    wo = None if place == "in-place" else torch.full_like(wd, 7.0)
    out = torch.full((6, group * kv, dim), 7.0, device=DEV)
    paged.attn_weights(s.cache, dev(q), u32(s.last()), wd, wo, out)
    got, gw = out.cpu().numpy(), (wd if wo is None else wo).cpu().numpy()
    behind = weight if wo is None else np.full_like(weight, 7.0)
    for i, n in enumerate(lens):
        np.testing.assert_array_equal(gw[i, :, n:], behind[i, :, n:])
        for g in range(kv if n else 0):
            total, tol = check_attention(s, got, q, i, g, group, list(range(n)))
            want = weight[i, g, :n] + total
            close(gw[i, g, :n], want, tol + (group + 1) * 2.0 ** -24 * want, ("weight", i, g))
    assert np.all(got[1] == 7.0)


@pytest.mark.parametrize("group,kv,dim", [(4, 2, 64), (1, 3, 128), (7, 2, 128), (16, 2, 128), (3, 1, 256)])
def test_attn_weights_in_a_large_cache(group, kv, dim):
    """Room for 11200 slots a sequence: a full one, and shorter ones beside it."""
    page, lens = 16, [11200, 0, 1500, 17, 2900]
    s = Setup(group + dim, lens, kv, dim, page)
    q = s.rng.standard_normal((5, group * kv, dim)).astype(np.float32)
    weight = s.rng.random((5, kv, s.capacity)).astype(np.float32)
    wd = dev(weight)
    got = paged.attn_weights(s.cache, dev(q), u32(s.last()), wd).cpu().numpy()
    gw = wd.cpu().numpy()
    for i, n in enumerate(lens):
        np.testing.assert_array_equal(gw[i, :, n:], weight[i, :, n:])
        for g in range(kv if n else 0):
            total, tol = check_attention(s, got, q, i, g, group, list(range(n)))
            want = weight[i, g, :n] + total
            close(gw[i, g, :n], want, tol + (group + 1) * 2.0 ** -24 * want, ("weight", i, g))


def test_attn_weights_long():
    """Many splits, several rounds of tiles a wave, a chunk boundary of the gathering."""
    s = Setup(2, [9000, 2049], 1, 128, 64)
    q = s.rng.standard_normal((2, 4, 128)).astype(np.float32)
    weight = np.zeros((2, 1, s.capacity), np.float32)
    wd = dev(weight)
    got = paged.attn_weights(s.cache, dev(q), u32(s.last()), wd).cpu().numpy()
    for i, n in enumerate(s.lens):
        total, tol = check_attention(s, got, q, i, 0, 4, list(range(n)))
        close(wd.cpu().numpy()[i, 0, :n], total, tol + 5 * 2.0 ** -24 * total, i)
        assert abs(float(wd[i, 0].sum()) - 4.0) < 1e-4


@pytest.mark.parametrize("kv,dim,page", POOL)
@pytest.mark.parametrize("keep,first,recent", [(1, 0, 0), (30, 2, 9), (30, 30, 0), (64, 0, 64), (100, 3, 20)])
@pytest.mark.parametrize("place", ["apart", "in-place"])
def test_evict(kv, dim, page, keep, first, recent, place):
    lens = [130, 0, 1, keep, keep + 1, 97, 111]
    entries = -(-(130 + keep) // page)
    s = Setup(dim + page + keep, lens, kv, dim, page, entries=entries)
    rng, n_rows = s.rng, len(lens)
    weight = (rng.integers(0, 9, (n_rows, kv, s.capacity)) / 8).astype(np.float32)  # many ties
    weight[0, :, ::7], weight[0, :, 3], weight[5, :, 5] = np.nan, np.inf, -0.0
    slot_pos = np.stack([[rng.permutation(s.capacity) for _ in range(kv)] for _ in range(n_rows)]).astype(np.uint32)
    pos = [int(slot_pos[i, :, :n].max()) if n else 0 for i, n in enumerate(lens)]
    pos[6] = ref.NONE
    length = np.array([ref.NONE if i == 0 else n for i, n in enumerate(lens)], np.uint32)  # more than capacity: capacity
    lens[0] = s.capacity
    s.seen[0] = [ref.at(s.table[0], s.n_pages, page, sl) for sl in range(s.capacity)]
    pos[0] = int(slot_pos[0].max())
    wd, sd, ld = dev(weight), u32(slot_pos), u32(length)
    outs = dict(weight_out=None, slot_pos_out=None, length_out=None) if place == "in-place" else dict(
        weight_out=torch.full_like(wd, 7.0), slot_pos_out=torch.full_like(sd, 5), length_out=torch.full_like(ld, 3))
    paged.evict(s.cache, ld, u32(pos), keep, wd, sd, first, recent, **outs)
    gw = (outs["weight_out"] if outs["weight_out"] is not None else wd).cpu().numpy()
    gp = (outs["slot_pos_out"] if outs["slot_pos_out"] is not None else sd).cpu().numpy().view(np.uint32)
    gl = (outs["length_out"] if outs["length_out"] is not None else ld).cpu().numpy().view(np.uint32)
    k_want, v_want = s.k.copy(), s.v.copy()
    w_want, p_want = (weight.copy(), slot_pos.copy()) if place == "in-place" else (np.full_like(weight, 7.0),
                                                                                 np.full_like(slot_pos, 5))
    l_want = length.copy() if place == "in-place" else np.full_like(length, 3)
    for i, n in enumerate(lens):
        if pos[i] == ref.NONE:
            continue
        l_want[i] = min(n, keep)
        for g in range(kv):
            src = ref.evict(n, pos[i], keep, first, recent, weight[i, g], slot_pos[i, g])
            src = list(range(n)) if src is None else src
            w_want[i, g, :len(src)], p_want[i, g, :len(src)] = weight[i, g, src], slot_pos[i, g, src]
            for to, of in enumerate(src):
                if to != of:
                    (p, o), (p2, o2) = s.seen[i][to], s.seen[i][of]
                    k_want[p, g, o], v_want[p, g, o] = s.k[p2, g, o2], s.v[p2, g, o2]
    np.testing.assert_array_equal(gl, l_want)
    np.testing.assert_array_equal(gp, p_want)
    np.testing.assert_array_equal(gw, w_want)
    np.testing.assert_array_equal(s.kd.cpu().numpy().view(np.uint16), k_want.view(np.uint16))
    np.testing.assert_array_equal(s.vd.cpu().numpy().view(np.uint16), v_want.view(np.uint16))


@pytest.mark.parametrize("newest", [0, 6, 80, 2**32 - 2])
@pytest.mark.parametrize("first,recent", [(0, 0), (5, 0), (0, 7), (20, 30)])
def test_evict_protected_positions(newest, first, recent):
    """Newest positions below n_recent, between the slots' own, and the largest one."""
    s = Setup(newest % 97 + first, [100], 2, 64, 8)
    weight = s.rng.standard_normal((1, 2, s.capacity)).astype(np.float32)
    at = [0, 1, 4, 5, 6, 7, 50, 51, 73, 74, 80, 81, 2**31, 2**32 - 10, 2**32 - 9, 2**32 - 2, 2**32 - 1]
    slot_pos = s.rng.choice(at, (1, 2, s.capacity)).astype(np.uint32)
    wd, sd = dev(weight), u32(slot_pos)
    paged.evict(s.cache, u32([100]), u32([newest]), 60, wd, sd, first, recent)
    for g in range(2):
        src = ref.evict(100, newest, 60, first, recent, weight[0, g], slot_pos[0, g])
        np.testing.assert_array_equal(wd.cpu().numpy()[0, g, :60], weight[0, g, src])
        np.testing.assert_array_equal(sd.cpu().numpy()[0, g, :60].view(np.uint32), slot_pos[0, g, src])


@pytest.mark.parametrize("n,keep", [(32768, 100), (32769, 32768), (70001, 40000)])
@pytest.mark.parametrize("levels", [1, 5, 0])
def test_evict_long(n, keep, levels):
    """More slots than a workgroup holds at once; equal weights, few distinct ones, all distinct."""
    s = Setup(n, [n], 2, 64, 7)
    weight = s.rng.standard_normal((1, 2, s.capacity)).astype(np.float32)
    if levels:
        weight = np.floor(weight % 1 * levels)
    slot_pos = np.stack([[s.rng.permutation(s.capacity) for _ in range(2)]]).astype(np.uint32)
    wd, sd, ld = dev(weight), u32(slot_pos), u32([n])
    newest = int(slot_pos[0, :, :n].max())
    paged.evict(s.cache, ld, u32([newest]), keep, wd, sd, 3, 50)
    assert ld.cpu().tolist() == [keep]
    kd, vd = s.kd.cpu().numpy(), s.vd.cpu().numpy()
    place = np.array(s.seen[0])
    for g in range(2):
        src = np.array(ref.evict(n, newest, keep, 3, 50, weight[0, g], slot_pos[0, g]))
        np.testing.assert_array_equal(wd.cpu().numpy()[0, g], np.concatenate([weight[0, g, src], weight[0, g, keep:]]))
        np.testing.assert_array_equal(sd.cpu().numpy()[0, g, :keep].view(np.uint32), slot_pos[0, g, src])
        to, of = place[:keep], place[src]
        for got, was in ((kd, s.k), (vd, s.v)):
            np.testing.assert_array_equal(got[to[:, 0], g, to[:, 1]], was[of[:, 0], g, of[:, 1]])
            rest = place[keep:]
            np.testing.assert_array_equal(got[rest[:, 0], g, rest[:, 1]], was[rest[:, 0], g, rest[:, 1]])


# ---- used together, captured, on streams, far offsets ---------------------------------


def heads(rng, count, n, dim):
    return rng.standard_normal((count, n, dim)).astype(np.float32)


class Decoder:
    """A layer's decode loop over fixed buffers: append, gather weights, evict; and the
    float64 form of the same, which carries the cache of the GPU's fp16 values along."""

    def __init__(self, seed, lens, group, kv, dim, page, keep, room):
        self.s = s = Setup(seed, lens, kv, dim, page, entries=-(-room // page))
        self.group, self.keep, self.count = group, keep, len(lens)
        rng = s.rng
        self.slot_pos = np.zeros((self.count, kv, s.capacity), np.uint32)
        self.slot_pos[:] = np.arange(s.capacity)
        self.weight = rng.random((self.count, kv, s.capacity)).astype(np.float32)
        self.length = np.array(lens, np.uint32)
        self.pos = np.array([n - 1 if n else ref.NONE for n in lens], np.uint32)
        self.qw, self.kw = ((1 + 0.1 * rng.standard_normal(dim)).astype(np.float32) for _ in range(2))
        self.d = {n: u32(getattr(self, n)) for n in ("slot_pos", "length", "pos")}
        self.d.update(weight=dev(self.weight), qw=dev(self.qw), kw=dev(self.kw), slot=u32(self.length))
        for n, h in (("q", group * kv), ("k", kv), ("v", kv)):
            self.d[n] = torch.zeros(self.count, h, dim, device=DEV)
        self.out, self.q_out = torch.full_like(self.d["q"], 7.0), torch.full_like(self.d["q"], 7.0)
        self.work = paged.attn_weights_workspace(s.cache, group * kv, self.count)
        self.work2 = paged.evict_workspace(s.cache, keep, self.count)

    def feed(self):
        """The next token's projections, positions and slots into the fixed buffers."""
        s = self.s
        self.live = self.pos != ref.NONE
        self.pos[self.live] += 1
        self.x = {n: heads(s.rng, self.count, h, s.dim) for n, h in (("q", self.group * s.kv), ("k", s.kv), ("v", s.kv))}
        for n, a in self.x.items():
            self.d[n].copy_(dev(a))
        self.d["pos"].copy_(u32(self.pos))
        slot = self.length.copy()
        slot[~self.live] = ref.NONE
        self.slot = slot
        self.d["slot"].copy_(u32(slot))
        length = np.where(self.live, self.length + 1, 0).astype(np.uint32)
        self.d["length"].copy_(u32(length))

    def step(self):
        d, c = self.d, self.s.cache
        paged.qk_norm_rope_append(c, d["q"], d["k"], d["v"], d["qw"], d["kw"], d["pos"], theta=1e4, slot=d["slot"],
                                  q_out=self.q_out, slot_pos=d["slot_pos"], slot_weight=d["weight"])
        paged.attn_weights(c, self.q_out, d["slot"], d["weight"], out=self.out, workspace=self.work)
        paged.evict(c, d["length"], d["pos"], self.keep, d["weight"], d["slot_pos"], 2, 4, workspace=self.work2)

    def check(self):
        s = self.s
        gk, gv = s.kd.cpu().numpy(), s.vd.cpu().numpy()
        gq, go, gw = self.q_out.cpu().numpy(), self.out.cpu().numpy(), self.d["weight"].cpu().numpy()
        gp, gl = (self.d[n].cpu().numpy().view(np.uint32) for n in ("slot_pos", "length"))
        for i in range(self.count):
            if not self.live[i]:
                assert np.all(go[i] == 7.0) and np.all(gq[i] == 7.0)
                continue
            n = int(self.length[i]) + 1
            assert gl[i] == min(n, self.keep)
            s.seen[i] = [ref.at(s.table[i], s.n_pages, s.page, t) for t in range(s.capacity)]
            p, o = s.seen[i][n - 1]
            for g in range(s.kv):
                want, size = ref.norm_rope(self.x["k"][i, g], self.kw, self.pos[i], 1e4, 1e-6, s.dim, True)
                got = want.astype(np.float16)
                s.v[p, g, o] = self.x["v"][i, g].astype(np.float16)
                self.slot_pos[i, g, n - 1], self.weight[i, g, n - 1] = self.pos[i], 0.0
                # the new key as the GPU stored it, wherever the eviction left it
                where = [t for t in range(min(n, self.keep)) if gp[i, g, t] == self.pos[i]]
                assert len(where) == 1  # the newest position is protected
                pw, ow = s.seen[i][where[0]]
                stored = gk[pw, g, ow]
                close(stored, want, 2.0 ** -11 * np.abs(want) + 48 * 2.0 ** -24 * size + 2.0 ** -25, ("k", i, g))
                s.k[p, g, o] = stored
                total, tol = check_attention(s, go, gq, i, g, self.group, list(range(n)))
                w = self.weight[i, g, :n] + total
                # the eviction by the GPU's own sums, which the attention's bound ties to w
                kept = ref.evict(n, int(self.pos[i]), self.keep, 2, 4, w, self.slot_pos[i, g])
                src = list(range(n)) if kept is None else kept
                by_pos = {int(q): t for t, q in enumerate(self.slot_pos[i, g, :n])}
                mine = [by_pos[int(q)] for q in gp[i, g, :len(src)]]
                if mine != src:  # only where two weights lie within the bound of one another
                    gap = np.abs(np.sort(w[sorted(set(src) ^ set(mine))]))
                    assert np.ptp(gap) <= 2 * tol.max() + 1e-6, (i, g)
                close(gw[i, g, :len(src)], w[mine], tol[mine] + 20 * 2.0 ** -24 * w[mine], ("weight", i, g))
                keys, values = (np.stack([a[s.seen[i][t][0], g, s.seen[i][t][1]] for t in mine]) for a in (s.k, s.v))
                for t in range(len(src)):
                    pt, ot = s.seen[i][t]
                    np.testing.assert_array_equal(gk[pt, g, ot], keys[t])
                    np.testing.assert_array_equal(gv[pt, g, ot], values[t])
                self.slot_pos[i, g], self.weight[i, g] = gp[i, g], gw[i, g]
            self.length[i] = gl[i]
        s.k, s.v = gk.copy(), gv.copy()


@pytest.mark.parametrize("captured", [False, True], ids=["eager", "graph"])
def test_decode_with_eviction(captured):
    """Ten steps of three live sequences and a padded one, into and past their budget, eager
    or one graph replayed on another stream with eager work between the replays."""
    d = Decoder(11, [37, 20, 0, 41], 3, 2, 64, 7, 40, 48)
    step = d.step
    if captured:
        d.feed()
        before = [t.clone() for t in (*d.d.values(), d.s.kd, d.s.vd, d.out, d.q_out)]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            d.step()
        for t, b in zip((*d.d.values(), d.s.kd, d.s.vd, d.out, d.q_out), before):
            torch.testing.assert_close(t, b, rtol=0, atol=0, equal_nan=True)  # (a capture runs nothing)
        d.pos[d.live] -= 1

        def step():
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                graph.replay()
            torch.cuda.current_stream().wait_stream(side)

    for _ in range(10):
        d.feed()
        step()
        d.check()


def test_decode_over_selected_pages():
    """Append, the newest page's bounds, selection and attention, step by step: the bounds
    stay those of the filled positions and the listed pages are the float64 choice."""
    s = Setup(12, [61, 5, 100], 2, 128, 8, entries=16)
    group, select = 4, 5
    bounds = torch.zeros(s.n_pages, s.kv, 2, s.dim, dtype=torch.float16, device=DEV)
    paged.page_bounds(s.cache, u32(s.last()), bounds, u32([0, 0, 0]), s.entries)
    pos = np.array(s.last(), np.uint32)
    for _ in range(9):
        pos += 1
        q, k, v = (heads(s.rng, 3, n, s.dim) for n in (group * s.kv, s.kv, s.kv))
        turned = paged.qk_norm_rope_append(s.cache, dev(q), dev(k), dev(v), None, None, u32(pos), theta=1e6,
                                           pairing="adjacent", rotary_dim=64)
        paged.page_bounds(s.cache, u32(pos), bounds)
        pages = paged.select_pages(s.cache, bounds, turned, u32(pos), select, 1, 2)
        out = paged.attn_pages(s.cache, turned, pages, u32(pos)).cpu().numpy()
        s.k, s.v = s.kd.cpu().numpy(), s.vd.cpu().numpy()
        gb, gp, gq = bounds.cpu().numpy(), pages.cpu().numpy(), turned.cpu().numpy()
        for i in range(3):
            n = int(pos[i]) + 1
            s.seen[i] = [ref.at(s.table[i], s.n_pages, s.page, t) for t in range(n)]
            for g in range(s.kv):
                for t in range(-(-n // s.page)):
                    at = s.table[i, t]
                    np.testing.assert_array_equal(gb[at, g], ref.bounds_of(s.k[at, g, :min(s.page, n - t * s.page)]))
                want = ref.select(gq[i, g * group:(g + 1) * group], gb[:, g], s.table[i], s.n_pages, -(-n // s.page), 1, 2,
                                  select)
                assert gp[i, g].tolist() == want + [-1] * (select - len(want))
                check_attention(s, out, gq, i, g, group,
                                [x for t in want for x in range(t * s.page, min(n, t * s.page + s.page))])


def test_all_pages_agree_with_dense_attention():
    """Every page listed, over the cache that rtxllm_attn_decode_gqa_f16 reads: both within
    their error of one another (each within 1e-5 of the largest value of a row)."""
    from rtxllm_amd import ops
    from rtxllm_amd._lib import lib

    s = Setup(13, [300, 512, 1], 8, 128, 64, entries=8)
    q = dev(heads(s.rng, 3, 32, 128))
    pos = u32(s.last())
    pages = torch.arange(8, dtype=torch.int32, device=DEV).expand(3, 8, 8).contiguous()
    got = paged.attn_pages(s.cache, q, pages, pos)
    out = torch.empty_like(q)
    table = dev(s.table)
    need = int(lib().rtxllm_attn_decode_workspace(32, 8, 512, 3))
    ws = torch.empty(need, dtype=torch.uint8, device=DEV)
    assert lib().rtxllm_attn_decode_gqa_f16(ops.ptr(q), ops.ptr(s.kd), ops.ptr(s.vd), ops.ptr(table), 8, 32, 8, 64, 512,
                                            ops.ptr(pos), 3, ops.ptr(out), ops.ptr(ws), need, ops.stream()) == 0
    for r in range(3):
        assert float((got[r] - out[r]).abs().max()) <= 2e-5 * float(out[r].abs().max())


def test_offsets_past_32_bits():
    """Pages whose rows lie more than 2^32 values into the cache (9 GB of keys)."""
    kv, dim, page = 8, 128, 64
    n_pages = (1 << 32) // (kv * dim * page) + 40
    k = torch.empty(n_pages, kv, page, dim, dtype=torch.float16, device=DEV)
    v = torch.empty_like(k)
    far = n_pages - 1 - torch.randperm(12, generator=torch.Generator().manual_seed(3))
    small = Setup(14, [12 * page - 5], kv, dim, page)
    table = far.to(torch.int32).reshape(1, 12)
    for t in range(12):
        k[far[t]], v[far[t]] = small.kd[small.table[0, t]], small.vd[small.table[0, t]]
    cache = paged.PagedKV(k, v, table.to(DEV))
    rng = small.rng
    q, kn, vn = (dev(heads(rng, 1, n, dim)) for n in (4 * kv, kv, kv))
    pos, slot_pos = u32(small.last()), u32(rng.permutation(12 * page)).expand(1, kv, 12 * page).contiguous()
    weight = dev(rng.random((1, kv, 12 * page)).astype(np.float32))
    answers = []
    for c, kk, vv, tab in ((cache, k, v, far), (small.cache, small.kd, small.vd, torch.from_numpy(small.table[0]).long())):
        w, sp = weight.clone(), slot_pos.clone()
        turned = paged.qk_norm_rope_append(c, q, kn, vn, None, None, pos, theta=1e4)
        bounds = torch.zeros(kk.shape[0], kv, 2, dim, dtype=torch.float16, device=DEV)
        paged.page_bounds(c, pos, bounds, torch.zeros_like(pos), 12)
        pages = paged.select_pages(c, bounds, turned, pos, 5)
        some = paged.attn_pages(c, turned, pages, pos)
        out = paged.attn_weights(c, turned, pos, w)
        paged.evict(c, pos + 1, u32([12 * page]), 600, w, sp, 3, 9)
        answers.append([turned, bounds[tab.to(DEV)], pages, some, out, w, sp, kk[tab.to(DEV)], vv[tab.to(DEV)]])
    for a, b in zip(*answers):
        assert torch.equal(a.view(torch.int16) if a.dtype == torch.float16 else a,
                           b.view(torch.int16) if b.dtype == torch.float16 else b)


def test_two_streams_and_repeats_give_the_same_bits():
    """Two calls at once on streams of their own, each with its workspace, repeatedly: the
    bits of a call alone."""
    s = Setup(15, [3000, 900], 4, 128, 64)
    q = [dev(heads(s.rng, 2, 20, 128)) for _ in range(2)]
    pos = u32(s.last())
    bounds = torch.zeros(s.n_pages, 4, 2, 128, dtype=torch.float16, device=DEV)
    paged.page_bounds(s.cache, pos, bounds, torch.zeros_like(pos), s.entries)
    weight = torch.zeros(2, 4, s.capacity, device=DEV)

    def run(x):
        pages = paged.select_pages(s.cache, bounds, x, pos, 9)
        w = torch.empty_like(weight).fill_(-1.0)
        return pages, paged.attn_pages(s.cache, x, pages, pos), paged.attn_weights(s.cache, x, pos, weight, w), w

    alone = [run(x) for x in q]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        got = []
        for x, st in zip(q, streams):
            with torch.cuda.stream(st):
                got.append(run(x))
        torch.cuda.synchronize()
        for a, b in zip(alone, got):
            assert all(torch.equal(m, n) for m, n in zip(a, b))


def test_wrapper_refusals():
    s = Setup(16, [20, 20], 2, 64, 8)
    c, pos = s.cache, u32([3, 4])
    q, k = torch.zeros(2, 4, 64, device=DEV), torch.zeros(2, 2, 64, device=DEV)
    bounds = torch.zeros(s.n_pages, 2, 2, 64, dtype=torch.float16, device=DEV)
    state = torch.zeros(2, 2, s.capacity, device=DEV)
    pages = torch.zeros(2, 2, 3, dtype=torch.int32, device=DEV)
    from rtxllm_amd import HipError

    bad = [
        lambda: paged.PagedKV(s.kd.float(), s.vd, c.block_table),
        lambda: paged.PagedKV(s.kd, s.vd[:1], c.block_table),
        lambda: paged.PagedKV(s.kd, s.vd, c.block_table.long()),
        lambda: paged.PagedKV(s.kd.cpu(), s.vd.cpu(), c.block_table.cpu()),
        lambda: paged.PagedKV(s.kd, s.vd, c.block_table[:1].expand(2, -1)),
        lambda: paged.qk_norm_rope_append(c, q, k, k, None, None, u32([1, 2, 3]), theta=1e4),
        lambda: paged.qk_norm_rope_append(c, q, k[:, :1], k, None, None, pos, theta=1e4),
        lambda: paged.qk_norm_rope_append(c, q.transpose(1, 2), k, k, None, None, pos, theta=1e4),
        lambda: paged.qk_norm_rope_append(c, q, k, k, None, None, pos, theta=1e4, pairing="both"),
        lambda: paged.qk_norm_rope_append(c, q, k, k, q[0, 0, :32], None, pos, theta=1e4),
        lambda: paged.qk_norm_rope_append(c, q, k, k, None, None, pos.long(), theta=1e4),
        lambda: paged.qk_norm_rope_append(c, q, k, k, None, None, pos, theta=1e4, slot_weight=state[:1]),
        lambda: paged.page_bounds(c, pos, bounds[:2]),
        lambda: paged.select_pages(c, bounds, q[:, :3], pos, 3),
        lambda: paged.select_pages(c, bounds, q, pos, 3, workspace=torch.zeros(8, dtype=torch.uint8, device=DEV)),
        lambda: paged.attn_pages(c, q, pages[:, :1], pos),
        lambda: paged.attn_pages(c, q, pages, pos, out=torch.zeros(2, 4, 64)),
        lambda: paged.attn_weights(c, q, pos, state[..., :-1]),
        lambda: paged.evict(c, pos, pos, 0, state, state.int()),
        lambda: paged.evict(c, pos, pos, 4, state, state),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was not refused")
    for call in (lambda: paged.qk_norm_rope_append(c, q, k, k, None, None, pos, theta=1e4, rotary_dim=12),
                 lambda: paged.select_pages(c, bounds, q, pos, 3, 2, 2),
                 lambda: paged.evict(c, pos, pos, 4, state, state.int(), 3, 2),
                 lambda: paged.page_bounds(c, pos, bounds, span=0)):
        with pytest.raises(HipError):
            call()


@pytest.mark.parametrize("heads,kv,dim,page,rotary,pairing", [(32, 8, 128, 64, 128, "halves"), (40, 2, 64, 24, 16, "adjacent"),
                                                              (8, 1, 64, 16, 64, "halves")])
def test_append_long_prompt(heads, kv, dim, page, rotary, pairing):
    """1100 rows of one sequence (the kernel of long prompts where a row has more heads than a
    workgroup holds), some of them padded, against float64."""
    count = 1100
    s = Setup(17, [count], kv, dim, page, one=True)
    q, k, v = (s.rng.standard_normal((count, h, dim)).astype(np.float32) for h in (heads, kv, kv))
    w = (1.0 + 0.1 * s.rng.standard_normal(dim)).astype(np.float32)
    pos = s.rng.permutation(count).astype(np.uint32)  # any order
    pad = s.rng.random(count) < 0.05
    given = np.where(pad, ref.NONE, pos).astype(np.uint32)
    out = torch.full((count, heads, dim), 7.0, device=DEV)
    paged.qk_norm_rope_append(s.cache, dev(q), dev(k), dev(v), dev(w), dev(w), u32(given), theta=1e5, rotary_dim=rotary,
                              pairing=pairing, q_out=out)
    gk, gv, got = s.kd.cpu().numpy(), s.vd.cpu().numpy(), out.cpu().numpy()
    i = np.arange(rotary // 2)
    a, b = (i, i + rotary // 2) if pairing == "halves" else (2 * i, 2 * i + 1)
    angle = pos[:, None].astype(np.float64) * 1e5 ** (-2.0 * i / rotary)

    def form(x):
        y = x.astype(np.float64)
        y = y / np.sqrt((y * y).mean(-1, keepdims=True) + 1e-6) * w.astype(np.float64)
        z, size = y.copy(), np.abs(y)
        c, sn = np.cos(angle)[:, None], np.sin(angle)[:, None]
        z[..., a], z[..., b] = y[..., a] * c - y[..., b] * sn, y[..., a] * sn + y[..., b] * c
        size[..., a] = size[..., b] = np.abs(y[..., a]) + np.abs(y[..., b])
        return z, size

    want, size = form(q)
    live = ~pad
    close(got[live], want[live], 24 * 2.0 ** -24 * size[live], "q")
    assert np.all(got[pad] == 7.0)
    want, size = form(k)
    place = np.array(s.seen[0])[pos]
    k_want, v_want = s.k.copy(), s.v.copy()
    p, o = place[live, 0], place[live, 1]
    close(gk[p, :, o], want[live], 2.0 ** -11 * np.abs(want[live]) + 48 * 2.0 ** -24 * size[live] + 2.0 ** -25, "k")
    k_want[p, :, o], v_want[p, :, o] = gk[p, :, o], v[live].astype(np.float16)
    np.testing.assert_array_equal(gk.view(np.uint16), k_want.view(np.uint16))
    np.testing.assert_array_equal(gv.view(np.uint16), v_want.view(np.uint16))


@pytest.mark.parametrize("group,dim,n", [(16, 64, 300001), (5, 256, 270000)])
def test_attention_of_very_long_contexts(group, dim, n):
    """More splits than one round of the merge holds; and the scores that a split keeps in
    the LDS stay of one size. float64 on the GPU, the bounds of paged_ref.attend."""
    page = 128
    entries = -(-n // page) + 1
    g = torch.Generator(device=DEV).manual_seed(n)
    k, v = (torch.randn(entries, 1, page, dim, generator=g, device=DEV).half() for _ in range(2))
    table = torch.randperm(entries, generator=g, device=DEV).int().reshape(1, -1)
    cache = paged.PagedKV(k, v, table)
    q = torch.randn(1, group, dim, generator=g, device=DEV)
    weight = torch.zeros(1, 1, cache.capacity, device=DEV)
    pos = u32([n - 1])
    out = paged.attn_weights(cache, q, pos, weight)[0].double()
    pages = torch.arange(entries, dtype=torch.int32, device=DEV).reshape(1, 1, -1).contiguous()
    listed = paged.attn_pages(cache, q, pages, pos)[0].double()
    keys, values = (x[table[0].long(), 0].reshape(-1, dim)[:n].double() for x in (k, v))
    total = torch.zeros(n, dtype=torch.float64, device=DEV)
    for h in range(group):
        s = keys @ q[0, h].double() / dim ** 0.5
        p = torch.softmax(s, 0)
        delta = (2.0 ** -23 * q[0, h].abs().max() * keys.abs().sum(1).max() +
                 (dim + 8) * 2.0 ** -24 * (keys.abs() @ q[0, h].abs().double()).max()) / dim ** 0.5
        bound = 2.0 * (delta + 2.0 ** -21 * (1.0 + s.abs().max())) + (n / 4 + 40) * 2.0 ** -24
        for got in (out[h], listed[h]):
            assert bool(((got - p @ values).abs() <= bound * (p @ values.abs())).all())
        total += p
    assert bool(((weight[0, 0, :n].double() - total).abs() <= bound * total).all())
    assert float(weight[0, 0, n:].abs().max()) == 0.0


def test_queries_of_one_sequence():
    """Rows that share one block table: a prompt's last positions, each over its own past."""
    s = Setup(18, [150], 2, 64, 16, one=True)
    count, group = 9, 3
    pos = np.array([149, 0, 15, 16, ref.NONE, 77, 148, 31, 2 ** 31], np.uint32)  # (past the capacity: all of it)
    q = heads(s.rng, count, group * s.kv, s.dim)
    bounds = torch.zeros(s.n_pages, s.kv, 2, s.dim, dtype=torch.float16, device=DEV)
    paged.page_bounds(s.cache, u32([149]), bounds, u32([0]), 10)
    pages = torch.full((count, s.kv, 4), -9, dtype=torch.int32, device=DEV)
    paged.select_pages(s.cache, bounds, dev(q), u32(pos), 4, 1, 1, pages=pages)
    out = torch.full((count, group * s.kv, s.dim), 7.0, device=DEV)
    paged.attn_pages(s.cache, dev(q), pages, u32(pos), out=out)
    got, gp, gb = out.cpu().numpy(), pages.cpu().numpy(), bounds.cpu().numpy()
    assert np.all(got[4] == 7.0) and np.all(gp[4] == -9)
    s.seen = [s.seen[0] + [ref.at(s.table[0], s.n_pages, s.page, t) for t in range(150, s.capacity)]] * count
    for i in (0, 1, 2, 3, 5, 6, 7):
        n = int(pos[i]) + 1
        for g in range(s.kv):
            want = ref.select(q[i, g * group:(g + 1) * group], gb[:, g], s.table[0], s.n_pages, -(-n // s.page), 1, 1, 4)
            assert gp[i, g].tolist() == want + [-1] * (4 - len(want))
            check_attention(s, got, q, i, g, group, [x for t in want for x in range(t * 16, min(n, t * 16 + 16))])
    assert gp[8].max() == 9  # 160 slots are 10 pages


def off(a, floats=1):
    """a on the GPU, its data `floats` values past a 16-byte boundary."""
    t = torch.from_numpy(np.ascontiguousarray(a))
    big = torch.zeros(t.numel() + 8, dtype=t.dtype, device=DEV)
    view = big[floats:floats + t.numel()].view(t.shape)
    view.copy_(t)
    return view


def test_unaligned_buffers():
    """Queries, results, weights, positions and lists at any 4-byte alignment, odd capacity."""
    s = Setup(19, [63, 40], 3, 64, 7, entries=11)  # capacity 77
    q = heads(s.rng, 2, 6, 64)
    weight = s.rng.random((2, 3, 77)).astype(np.float32)
    slot_pos = np.stack([[s.rng.permutation(77) for _ in range(3)] for _ in range(2)]).astype(np.int32)
    bounds = torch.zeros(s.n_pages, 3, 2, 64, dtype=torch.float16, device=DEV)
    pos = u32(s.last())
    paged.page_bounds(s.cache, pos, bounds, torch.zeros_like(pos), 11)
    answers = []
    for place in (dev, off):
        lists, out, out2 = place(np.full((2, 3, 5), -9, np.int32)), place(np.zeros_like(q)), place(np.zeros_like(q))
        w, sp, ln = place(weight), place(slot_pos), place(np.array([63, 40], np.int32))
        k, v = s.kd.clone(), s.vd.clone()
        cache = paged.PagedKV(k, v, s.cache.block_table)
        at = place(np.array([n - 1 for n in s.lens], np.int32))
        paged.select_pages(cache, bounds, place(q), at, 5, 1, 1, pages=lists)
        paged.attn_pages(cache, place(q), lists, at, out=out)
        paged.attn_weights(cache, place(q), at, w, out=out2)
        paged.evict(cache, ln, place(np.array([76, 76], np.int32)), 33, w, sp, 2, 5)
        answers.append([lists, out, out2, w, sp, ln, k.view(torch.int16), v.view(torch.int16)])
    for a, b in zip(*answers):
        assert torch.equal(a, b)


def test_smallest_cache():
    """One page of one slot, one head: every operator."""
    s = Setup(20, [1], 1, 64, 1, spare=0)
    assert s.capacity == 1 and s.n_pages == 1
    q, k, v = (heads(s.rng, 1, 1, 64) for _ in range(3))
    pos = u32([0])
    turned = paged.qk_norm_rope_append(s.cache, dev(q), dev(k), dev(v), None, None, pos, theta=1e4)
    bounds = paged.page_bounds(s.cache, pos, torch.zeros(1, 1, 2, 64, dtype=torch.float16, device=DEV))
    assert torch.equal(bounds[0, 0, 0], s.kd[0, 0, 0]) and torch.equal(bounds[0, 0, 1], s.kd[0, 0, 0])
    pages = paged.select_pages(s.cache, bounds, turned, pos, 2)
    assert pages.flatten().tolist() == [0, -1]
    weight = torch.zeros(1, 1, 1, device=DEV)
    value = s.vd[0, 0, 0].float()
    for out in (paged.attn_pages(s.cache, turned, pages, pos), paged.attn_weights(s.cache, turned, pos, weight)):
        assert torch.equal(out[0, 0], value)  # one term: 2^15 v / 2^15
    assert weight.item() == 1.0
    length, slot_pos = u32([1]), u32([[[0]]])
    paged.evict(s.cache, length, pos, 1, weight, slot_pos)
    assert length.item() == 1 and slot_pos.item() == 0 and weight.item() == 1.0
