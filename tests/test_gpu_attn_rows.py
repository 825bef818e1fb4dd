"""Attention of new rows with a window and sinks (rtxllm_attn_window_f16, rtxllm_attn_kv8) against float64
(rows_ref.py): one token a sequence, drafts, prompts; fp16 pages and 8-bit codes. What lies where no row looks is
NaN or infinite, tables are shuffled and may have holes."""

from __future__ import annotations

import numpy as np
import pytest
import rows_ref as ref

torch = pytest.importorskip("torch")

from rtxllm_amd import kv8, paged  # noqa: E402

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
DTYPE = dict(int8=torch.int8, e4m3=torch.float8_e4m3fn)
ALL = 1 << 24


def dev(a) -> torch.Tensor:
    return torch.from_numpy(np.ascontiguousarray(a)).to(DEV)


def u32(values) -> torch.Tensor:
    return dev(np.asarray(values, np.uint32).view(np.int32))


class Setup:
    """Sequences of held[s] positions, the last lens[s] of them the call's rows (held NONE: a padded one)."""

    def __init__(self, seed, fmt, held, lens, kv, group, dim, page, block=16, hole=None, f16=False, more=0, size=1.0):
        rng = self.rng = np.random.default_rng(seed)
        self.fmt, self.held, self.lens, self.kv, self.group, self.dim, self.f16 = fmt, held, lens, kv, group, dim, f16
        n_seq = len(held)
        most = max([h for h in held if h != ref.NONE] + [1])
        entries = -(-most // page) + more
        n_pages = n_seq * entries + 3
        table = rng.permutation(n_pages)[:n_seq * entries].astype(np.int32).reshape(n_seq, entries)
        self.real = table.copy()
        if hole:
            table[hole[0], hole[1]] = hole[2]
        self.table, self.n_pages, self.page, self.capacity = table, n_pages, page, entries * page
        drift = 0.45 * rng.standard_normal((n_seq, entries, kv, dim))
        self.x = []
        for i in range(2):
            x = size * rng.standard_normal((n_seq, entries * page, kv, dim))
            if i == 0:
                x = 0.9 * x + size * np.repeat(drift, page, axis=1)
            self.x.append(x.astype(np.float16))
        self.pos = [ref.NONE if h == ref.NONE else h - n for h, n in zip(held, lens)]
        self.rows = sum(lens)
        self.q = rng.standard_normal((self.rows, kv * group, dim)).astype(np.float16 if f16 else np.float32)
        if fmt == "f16":
            arrays = []
            for i, bad in ((0, np.nan), (1, np.inf)):
                a = np.full((n_pages, kv, page, dim), bad, np.float16)
                for s, h in enumerate(held):
                    for p in range(h if h != ref.NONE else 0):
                        a[self.real[s, p // page], :, p % page] = self.x[i][s, p]
                arrays.append(dev(a))
            self.cache = paged.PagedKV(*arrays, dev(table))
        else:
            self.cache = kv8.PagedKV8.empty(n_pages, kv, page, dim, block, dev(table), DTYPE[fmt])
            c = self.cache
            for x in (c.k, c.v):
                x.view(torch.uint8).fill_(0x7F)  # e4m3: NaN
            for x in (c.k_scale, c.v_scale, c.k_tail, c.v_tail):
                x.fill_(float("nan"))
            self.m = ref.Model(table, n_pages, kv, page, dim, block, fmt)
            live = [(s, h) for s, h in enumerate(held) if h != ref.NONE and h > 0]
            new = [np.concatenate([self.x[i][s, :h] for s, h in live]) for i in range(2)] if live else None
            if live:
                start = np.cumsum([0] + [0 if h == ref.NONE else h for h in held])
                kv8.append(c, dev(new[0]), dev(new[1]), u32([0] * n_seq), u32(start))
                for s, h in live:
                    self.m.append(s, 0, [self.x[i][s, :h] for i in range(2)])

    def value(self, i, s, g, p):
        if self.fmt == "f16":
            t = int(self.table[s, p // self.page])
            return self.x[i][s, p, g] if 0 <= t < self.n_pages else None
        return self.m.value(i, s, g, p, self.held[s])

    def call(self, window, sinks, single=False, out=None, start=None, **more):
        run = paged.attn_window if self.fmt == "f16" else kv8.attn
        start = None if single else u32(np.cumsum([0] + list(self.lens))) if start is None else start
        return run(self.cache, dev(self.q), u32(self.pos), start, window=window, sinks=sinks, out=out, **more)

    def check(self, got, window, sinks, sample=None, single=False):
        """Rows (all, or every `sample`-th and the last of each sequence) against float64."""
        got = got.cpu().numpy()
        row = 0
        for s, n in enumerate(self.lens):
            for r in range(n):
                here, row = row, row + 1
                if self.pos[s] == ref.NONE:
                    assert not got[here].any()
                    continue
                if sample and r % sample and r != n - 1:
                    continue
                p = min(self.pos[s] + r, self.capacity - 1)
                j = ref.visible(p, window, sinks)
                for g in range(self.kv):
                    kvs = [[self.value(i, s, g, int(t)) for t in j] for i in range(2)]
                    kvs = [np.array([x for x in v if x is not None]).reshape(-1, self.dim) for v in kvs]
                    for h in range(g * self.group, (g + 1) * self.group):
                        want, tol = ref.attend(self.q[here, h], kvs[0], kvs[1], self.f16, single)
                        with np.errstate(invalid="ignore"):
                            bad = ~(np.abs(got[here, h].astype(np.float64) - want) <= tol)
                        bad &= ~(np.isnan(want) & np.isnan(got[here, h]))  # (an infinity: that or NaN)
                        bad &= ~(np.isinf(want) & ~np.isfinite(got[here, h]))
                        assert not bool(bad.any()), (s, r, p, h, np.argwhere(bad)[:3].tolist(), got[here, h][bad][:3], want[bad][:3],
                                               tol[bad][:3] if tol.shape else tol)


FORMATS = ["f16", "int8", "e4m3"]
# (kv heads, query heads a kv head, head_dim, page, block)
SHAPES = [(8, 4, 128, 64, 16), (2, 1, 64, 16, 8), (1, 16, 128, 32, 32), (2, 5, 256, 48, 8), (3, 3, 64, 64, 64), (1, 12, 256, 64, 64)]


@pytest.mark.parametrize("window,sinks", [(ALL, 0), (1, 0), (37, 3), (100, 70), (64, 64)])
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_one_token_each(shape, fmt, window, sinks):
    kv, group, dim, page, block = shape
    held = [301, 1, ref.NONE, 64, 2 * page, 33]
    s = Setup(dim + kv, fmt, held, [1] * 6, kv, group, dim, page, block, f16=window == 37)
    got = s.call(window, sinks, single=True)
    s.check(got, window, sinks)


@pytest.mark.parametrize("window,sinks", [(ALL, 0), (1, 1), (29, 5), (130, 40)])
@pytest.mark.parametrize("f16", [False, True], ids=["f32", "half"])
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_drafts_and_prompts(shape, fmt, f16, window, sinks):
    """Ragged rows: drafts over a long context, a prompt from nothing, an empty sequence, a padded one with rows."""
    kv, group, dim, page, block = shape
    held = [350, 75, 90, ref.NONE, 3]
    s = Setup(dim + group, fmt, held, [5, 75, 0, 4, 1], kv, group, dim, page, block, f16=f16)
    got = s.call(window, sinks)
    s.check(got, window, sinks, sample=9, single=f16)


@pytest.mark.parametrize("window,sinks", [(ALL, 0), (1, 0), (70, 5), (64, 64), (200, 130)])
@pytest.mark.parametrize("f16", [False, True], ids=["f32", "half"])
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_prompts(shape, fmt, f16, window, sinks):
    """Prompts long enough for tiles that many rows share: from nothing, over a held context, beside a few rows."""
    kv, group, dim, page, block = shape
    s = Setup(dim + 3 * group, fmt, [330, 400, ref.NONE, 3], [330, 250, 2, 3], kv, group, dim, page, block, f16=f16)
    got = s.call(window, sinks)
    s.check(got, window, sinks, sample=41, single=f16)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_prompts_over_long_contexts(fmt, dim):
    """Few tiles of rows over a long context: its tiles of positions in splits."""
    for f16 in (False, True):
        s = Setup(18, fmt, [2900, 700], [70, 61], 1, 6, dim, 64, 32, f16=f16)
        for window, sinks in ((ALL, 0), (900, 100)):
            s.check(s.call(window, sinks), window, sinks, sample=35, single=f16)


@pytest.mark.parametrize("page", [1, 5, 7, 30])
def test_pages_of_any_size(page):
    s = Setup(page, "f16", [97, 60], [20, 1], 2, 3, 128, page)
    for window, sinks in ((ALL, 0), (33, 7)):
        s.check(s.call(window, sinks), window, sinks, sample=6)


@pytest.mark.parametrize("fmt", FORMATS)
def test_pages_that_are_not_there(fmt):
    """A hole is passed over; a row that sees nothing but holes is 0."""
    for bad in (-1, 2 ** 31 - 1):
        s = Setup(5, fmt, [150, 40], [6, 40], 2, 4, 128, 32, 16, hole=(0, 1, bad))
        for window, sinks in ((ALL, 0), (20, 40)):
            s.check(s.call(window, sinks), window, sinks)
    s = Setup(6, fmt, [64, 64], [64, 1], 1, 2, 64, 64, 8, hole=(0, 0, -1))
    got = s.call(ALL, 0)
    assert not got[:64].any() and got[64].any()
    s.check(got, ALL, 0, sample=16)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dim", [64, 128])
def test_late_rows_do_not_reach_earlier_ones(fmt, dim):
    """Infinities and NaN in a prompt's keys and values: rows before them, and rows whose window has passed them, are
    numbers (and right); rows that attend them are NaN where they enter."""
    for f16 in (False, True):
        s = Setup(8, fmt, [140, 70], [90, 70], 2, 4 if dim == 128 else 3, dim, 32, 8, f16=f16)
        bad_v, bad_k = 77, 93  # of sequence 0
        for i, p, d, x in ((1, bad_v, 5, np.nan), (1, bad_v + 1, 6, np.inf), (0, bad_k, 3, np.nan), (1, 139, 7, np.nan)):
            s.x[i][0, p, 1, d] = x
        if fmt == "f16":
            for i, c in enumerate((s.cache.k, s.cache.v)):
                for p in (bad_v, bad_v + 1, bad_k, 139):
                    c[int(s.real[0, p // 32]), :, p % 32] = dev(s.x[i][0, p])
        else:
            kv8.append(s.cache, dev(s.x[0][0, :140]), dev(s.x[1][0, :140]), u32([0, ref.NONE]), u32([0, 140, 140]))
            s.m.append(0, 0, [s.x[i][0, :140] for i in range(2)])
        for window, sinks in ((ALL, 0), (11, 3)):
            got = s.call(window, sinks)
            s.check(got, window, sinks, single=f16)
            heads = got[:90, s.group:].isnan()
            assert not got[:90, :s.group].isnan().any() and not got[90:].isnan().any()
            first = bad_v // 8 * 8 if fmt != "f16" else bad_v  # (of an 8-bit block, all of it)
            assert not heads[:first - 50].any() and heads[bad_v - 50:].any()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("f16", [False, True], ids=["f32", "half"])
@pytest.mark.parametrize("rows", [30, 130])
def test_queries_that_are_not_finite(fmt, rows, f16):
    s = Setup(9, fmt, [180, 40], [rows, 1], 2, 4, 128, 64, 16, f16=f16)
    s.q[3, 5, 7], s.q[20, 0, 0] = np.nan, np.inf
    got = s.call(50, 2)
    bad = got.isnan()
    assert bad[3, 5].all() and bad[20, 0].all() and int(bad.any(-1).sum()) == 2
    s.q[3, 5, 7], s.q[20, 0, 0] = 0.0, 0.0
    want = s.call(50, 2)
    keep = ~bad.any(-1)
    assert torch.equal(got[keep], want[keep])


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("size", [1e-6, 3e-3, 300.0])
def test_sizes_of_keys_and_values(fmt, size):
    """Values from fp16's subnormals to its largest: softmax terms and scales keep their bits."""
    s = Setup(10, fmt, [200, 90], [1, 1], 2, 4, 128, 64, 8, size=size)
    s.q = (s.q / max(size, 1e-3) * 0.5).astype(np.float32)
    s.check(s.call(ALL, 0, single=True), ALL, 0)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_scales_over_many_powers_of_ten(fmt):
    """Blocks whose values differ by up to 1e9 in size, the large ones where the weight is small and where it is not."""
    s = Setup(11, fmt, [256, 256], [1, 9], 1, 4, 128, 64, 8)
    scale = 10.0 ** s.rng.uniform(-5, 4, (1, 32, 1, 1, 1))
    x = (s.x[1][:, :256].reshape(2, 32, 8, 1, 128).astype(np.float64) * scale).astype(np.float16)
    s.x[1][:, :256] = x.reshape(2, 256, 1, 128)
    for i in range(2):
        kv8.append(s.cache, dev(s.x[0][i, :256]), dev(s.x[1][i, :256]), u32([0 if j == i else ref.NONE for j in range(2)]),
                   u32([0, 256 * (1 - i), 256]))
        s.m.append(i, 0, [s.x[j][i, :256] for j in range(2)])
    s.check(s.call(ALL, 0), ALL, 0)
    s.check(s.call(40, 8), 40, 8)


@pytest.mark.parametrize("fmt", FORMATS)
def test_positions_at_and_behind_the_capacity(fmt):
    """Such rows attend as the last position does."""
    s = Setup(12, fmt, [128, 128], [1, 1], 2, 2, 64, 64, 16)
    a = s.call(30, 2, single=True)
    s.pos = [128, 2 ** 32 - 2]
    b = s.call(30, 2, single=True)
    assert torch.equal(a, b)
    start = u32([0, 1, 2])
    c = s.call(30, 2, start=start)
    s.check(b, 30, 2), s.check(c, 30, 2)


def test_one_table_row_for_all():
    """table_stride 0: rows of one sequence at any positions, and sequences that share every page."""
    s = Setup(13, "f16", [200], [1], 2, 4, 128, 32)
    cache = paged.PagedKV(s.cache.k, s.cache.v, s.cache.block_table[0].contiguous())
    q = s.rng.standard_normal((5, 8, 128)).astype(np.float32)
    pos = [199, 0, 77, ref.NONE, 150]
    got = paged.attn_window(cache, dev(q), u32(pos), window=60, sinks=4)
    for i, p in enumerate(pos):
        s.q, s.pos, s.lens, s.held = q[i:i + 1], [p], [1], [200]
        s.check(got[i:i + 1], 60, 4)


@pytest.mark.parametrize("fmt", FORMATS)
def test_rows_outside_every_sequence(fmt):
    s = Setup(14, fmt, [70, 50, 60], [12, 0, 9], 1, 3, 64, 32, 8)
    pad = np.full((30, 3, 64), np.nan, np.float32)
    pad[5:17], pad[17:26] = s.q[:12], s.q[12:]
    want = s.call(40, 2)
    out = torch.full((30, 3, 64), 7.0, device=DEV)
    s.q = pad
    s.call(40, 2, start=u32([5, 17, 17, 26]), out=out)
    assert torch.equal(out[5:26], want) and (out[:5] == 7.0).all() and (out[26:] == 7.0).all()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("f16", [False, True], ids=["f32", "half"])
@pytest.mark.parametrize("rows", [40, 150])
def test_unaligned_and_in_place(fmt, f16, rows):
    s = Setup(15, fmt, [190, 33], [rows, 1], 2, 4, 128, 64, 8, f16=f16)
    want = s.call(50, 3)
    flat = torch.zeros(s.q.size + 1, dtype=want.dtype, device=DEV)
    q = flat[1:].view(want.shape)
    q.copy_(dev(s.q))
    run = paged.attn_window if fmt == "f16" else kv8.attn
    got = run(s.cache, q, u32(s.pos), u32([0, rows, rows + 1]), window=50, sinks=3, out=q)
    assert got.data_ptr() == q.data_ptr() and torch.equal(got, want) and flat[0] == 0.0


@pytest.mark.parametrize("fmt", FORMATS)
def test_long_contexts_in_splits(fmt):
    """Contexts long enough for many splits, some of them empty at the shorter sequences."""
    s = Setup(16, fmt, [5003, 40, 2600], [1, 1, 1], 2, 4, 128, 64, 16)
    s.check(s.call(ALL, 0, single=True), ALL, 0)
    s = Setup(17, fmt, [4000, 900], [3, 40], 1, 4, 64, 64, 16)
    for window, sinks in ((ALL, 0), (1500, 100)):
        s.check(s.call(window, sinks), window, sinks, sample=8)
