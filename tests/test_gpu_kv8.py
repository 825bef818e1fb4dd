"""The paged cache in 8 bits (include/rtxllm/kv8.h): codes, scales and tails as its rule has them, bit
for bit, however the tokens come; positions read back; what is not written stays."""

from __future__ import annotations

import numpy as np
import pytest
import rows_ref as ref

torch = pytest.importorskip("torch")

from rtxllm_amd import kv8  # noqa: E402

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
DTYPE = dict(int8=torch.int8, e4m3=torch.float8_e4m3fn)
MARK = 0x55  # what lies in codes that nothing writes


def dev(a) -> torch.Tensor:
    return torch.from_numpy(np.ascontiguousarray(a)).to(DEV)


def u32(values) -> torch.Tensor:
    return dev(np.asarray(values, np.uint32).view(np.int32))


class Setup:
    """An empty cache of `count` sequences with a shuffled table, and its model."""

    def __init__(self, seed, count, entries, kv, dim, page, block, fmt, hole=None, stride=None):
        rng = self.rng = np.random.default_rng(seed)
        n_pages = count * entries + 2
        table = rng.permutation(n_pages)[:count * entries].astype(np.int32).reshape(count, entries)
        if hole:
            table[hole[0], hole[1]] = hole[2]
        wide = np.full((count, stride or entries), -9, np.int32)
        wide[:, :entries] = table
        self.cache = kv8.PagedKV8.empty(n_pages, kv, page, dim, block, dev(wide)[:, :entries], DTYPE[fmt])
        for x in (self.cache.k, self.cache.v):
            x.view(torch.uint8).fill_(MARK)
        self.m = ref.Model(table, n_pages, kv, page, dim, block, fmt)
        mark = float(torch.tensor([MARK], dtype=torch.uint8).view(DTYPE[fmt]).float())
        for c in self.m.codes:
            c.fill(mark)
        self.fmt, self.kv, self.dim = fmt, kv, dim

    def check(self):
        c, m = self.cache, self.m
        for i, (codes, scale, tail) in enumerate(((c.k, c.k_scale, c.k_tail), (c.v, c.v_scale, c.v_tail))):
            assert bool(np.array_equal(scale.cpu().numpy(), m.scale[i], equal_nan=True)), i
            assert np.array_equal(codes.float().cpu().numpy().astype(np.float64), m.codes[i]), i
            assert np.array_equal(tail.cpu().numpy().view(np.uint16), m.tail[i].view(np.uint16)), i

    def tokens(self, n, dtype=np.float32):
        """k and v rows, of sizes over some powers of ten."""
        size = 10.0 ** self.rng.uniform(-3, 2, (n, 1, 1))
        return [(size * self.rng.standard_normal((n, self.kv, self.dim))).astype(dtype) for _ in range(2)]

    def append(self, lens, pos, new, gaps=0, dtype=np.float32, single=False):
        """lens rows from pos on, of each sequence; the rows of the stacked projection lie `gaps` values further apart."""
        for s, (n, p) in enumerate(zip(lens, pos)):
            a = sum(lens[:s])
            if p != ref.NONE and n:
                self.m.append(s, p, [x[a:a + n].astype(dtype) for x in new])
        rows, width = sum(lens), self.kv * self.dim
        wide = np.full((rows, 2 * width + gaps), np.nan, dtype)
        wide[:, gaps // 2:gaps // 2 + width] = new[0].reshape(rows, -1)
        wide[:, gaps // 2 + width:gaps // 2 + 2 * width] = new[1].reshape(rows, -1)
        w = dev(wide)
        parts = [w[:, gaps // 2 + i * width:gaps // 2 + (i + 1) * width].unflatten(1, (self.kv, self.dim)) for i in range(2)]
        start = None if single else u32(np.cumsum([0] + list(lens)))
        kv8.append(self.cache, *parts, u32(pos), start)


# (kv heads, head_dim, page, block)
SHAPES = [(8, 128, 64, 16), (1, 64, 8, 8), (2, 256, 48, 8), (3, 128, 64, 64), (2, 64, 96, 32), (1, 256, 64, 64)]


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_prompts_and_tokens(shape, fmt):
    """A ragged batch of prompts, then tokens one at a time, then drafts over block borders."""
    kv, dim, page, block = shape
    entries = max(3, -(-150 // page))
    s = Setup(dim + block, 4, entries, kv, dim, page, block, fmt, stride=entries + 3)
    lens = [block * 2 + 3, 1, 0, min(99, s.m.capacity - 9)]
    s.append(lens, [0, 0, 5, 0], s.tokens(sum(lens)), gaps=6)
    s.check()
    pos = list(lens)
    for i in range(block + 2):
        at = [p if j != 2 else ref.NONE for j, p in enumerate(pos)]
        s.append([1] * 4, at, s.tokens(4), single=True)
        pos = [p + 1 for p in pos]
    s.check()
    pos[2] = 0
    for lens in ([5, 3, block + 1, 2], [1, 2 * block, 7, 0], [3, 1, 1, 9]):
        s.append(lens, pos, s.tokens(sum(lens)))
        s.check()
        pos = [min(p + n, s.m.capacity) for p, n in zip(pos, lens)]


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("block", [8, 64])
def test_one_by_one_is_the_prompt(block, fmt):
    """The cache is the same whether tokens come one at a time, in uneven chunks or at once, in fp32 or fp16."""
    n, one, chunks, whole, half = 3 * block + 5, *(Setup(7, 1, 4, 2, 128, 64, block, fmt) for _ in range(4))
    new = [x.astype(np.float16).astype(np.float32) for x in one.tokens(n)]
    for i in range(n):
        one.append([1], [i], [x[i:i + 1] for x in new], single=True)
    at = 0
    while at < n:
        step = min(n - at, int(chunks.rng.integers(1, 2 * block)))
        chunks.append([step], [at], [x[at:at + step] for x in new])
        at += step
    whole.append([n], [0], new)
    half.append([n], [0], new, dtype=np.float16, gaps=3)
    whole.check()
    for x in (one, chunks, half):
        x.check()
        for a, b in ((x.cache.k, whole.cache.k), (x.cache.v, whole.cache.v)):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
        assert torch.equal(x.cache.k_scale, whole.cache.k_scale) and torch.equal(x.cache.v_scale, whole.cache.v_scale)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_every_fp16_value(fmt):
    """All finite fp16 values, a power of two and its sign to a block, so that codes meet every tie and every
    subnormal; blocks of zeros, of the largest value, of infinities, of NaN."""
    s = Setup(1, 1, 80, 1, 128, 64, 16, fmt)
    bits = np.arange(0x7C00, dtype=np.uint16)
    x = np.concatenate([bits, bits | 0x8000]).view(np.float16)
    x = np.concatenate([x, np.zeros(2048, np.float16)])
    odd = np.zeros((6, 2048), np.float16)
    odd[0, 7], odd[1, 2000], odd[2, 5], odd[3], odd[4, 9], odd[5, 2047] = np.inf, -np.inf, np.nan, -65504.0, 2.0 ** -24, -0.0
    x = np.concatenate([x, odd.reshape(-1)])
    k = x.reshape(-1, 1, 128)
    v = s.rng.permutation(x[:0x7C00 * 2]).reshape(-1, 1, 128)
    v = np.concatenate([v, np.zeros((len(k) - len(v), 1, 128), np.float16)])
    s.append([len(k)], [0], [k.astype(np.float32), v.astype(np.float32)])
    s.check()
    held = u32([len(k)])
    gk, gv = kv8.read(s.cache, u32([0]), held, u32([0, len(k)]), rows=len(k))
    want = s.m.codes[0], s.m.scale[0]
    for p in range(len(k)):
        at = s.m.at(0, p)
        with np.errstate(invalid="ignore"):
            x = (want[0][at[0], 0, at[1]].astype(np.float32) * want[1][at[0], 0, at[1] // 16])
        assert np.array_equal(gk[p, 0].cpu().numpy(), x, equal_nan=True), p


def test_ties_and_near_ties():
    """Quotients at halves and one step of fp16 beside them, over scales whose quotient by 127 is not exact."""
    s = Setup(2, 1, 8, 1, 64, 64, 8, "int8")
    x = np.zeros((512, 1, 64), np.float32)
    for b in range(64):
        top = np.float16(1.0 + b / 64.0 + 2.0 ** -10 * (b % 7))
        scale = np.float64(np.float32(top) * (np.float32(1.0) / np.float32(127.0)))
        n = s.rng.integers(-126, 126, 512)
        h = ((n + 0.5) * scale).astype(np.float16)
        h = (h.view(np.uint16).astype(np.int64) + s.rng.integers(-1, 2, 512)).astype(np.uint16).view(np.float16)
        h[0] = top
        x[8 * b:8 * b + 8, 0] = np.clip(h, -top, top).reshape(8, 64)
    s.append([512], [0], [x, x[::-1].copy()])
    s.check()


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_beyond_fp16_and_not_finite(fmt):
    s = Setup(3, 1, 1, 2, 64, 64, 16, fmt)
    new = s.tokens(60)
    new[0][3, 0, 5], new[0][20, 1, 0], new[1][40, 0, 63] = 1e6, np.inf, np.nan
    new[1][50, 1, 2] = np.nan  # stays in the tail
    s.append([60], [0], new)
    s.check()
    assert np.isnan(s.m.scale[0][s.m.table[0, 0], 0, 0]) and np.isfinite(s.m.scale[0][s.m.table[0, 0], 0, 1])


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("bad", [-1, 2 ** 31 - 1, 10])
def test_pages_that_are_not_there(fmt, bad):
    s = Setup(4, 2, 4, 2, 64, 32, 16, fmt, hole=(0, 1, bad if bad != 10 else 10))
    assert s.m.n_pages == 10
    lens = [100, 31]
    s.append(lens, [0, 0], s.tokens(131))
    s.append([40, 2], [100, 31], s.tokens(42))  # over the capacity of 128
    s.check()
    s.append([3, 1], [128, 2 ** 32 - 2], s.tokens(4))  # behind it
    s.append([1, 1], [127, ref.NONE], s.tokens(2), single=True)  # the last position, from a tail of old ones
    s.check()


def test_rows_outside_every_sequence():
    """Starts need not begin at 0 nor end at the last row; rows outside are not read (they are NaN) nor written."""
    s = Setup(5, 3, 2, 1, 128, 64, 8, "int8")
    new = s.tokens(50)
    for x in new:
        x[:4], x[40:] = np.nan, np.nan
    for i, (a, b) in enumerate(((4, 20), (20, 20), (20, 40))):
        s.m.append(i, 0, [x[a:b] for x in new])
    kv8.append(s.cache, dev(new[0]), dev(new[1]), u32([0, 0, 0]), u32([4, 20, 20, 40]))
    s.check()
    out = [torch.full((50, 1, 128), 7.0, device=DEV) for _ in range(2)]
    kv8.read(s.cache, u32([3, 0, 1]), u32([16, 0, 20]), u32([4, 20, 20, 40]), k_out=out[0], v_out=out[1])
    for i, o in enumerate(out):
        got = o.cpu().numpy()
        for r in range(50):
            q, p, held = (0, 3 + r - 4, 16) if 4 <= r < 20 else (2, 1 + r - 20, 20) if 20 <= r < 40 else (0, 99, 0)
            want = np.full(128, 7.0) if p >= held else s.m.value(i, q, 0, p, held)
            assert np.array_equal(got[r, 0], want.astype(np.float32)), (i, r)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16], ids=["f32", "f16"])
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_read(shape, fmt, dtype):
    """Positions as rows: whole blocks, the open one, single rows, holes, unaligned outputs; one product, rounded once."""
    kv, dim, page, block = shape
    entries = max(3, -(-150 // page))
    s = Setup(dim + page, 3, entries, kv, dim, page, block, fmt, hole=(0, 1, -1))
    held = [min(2 * page + block // 2 + 1, s.m.capacity), 5, 0]
    s.append(held, [0, 0, 0], s.tokens(sum(held)))
    lens, pos = [held[0] + 4, 3, 2], [0, 2, ref.NONE]
    rows = sum(lens)
    flat = [torch.full((rows * kv * dim + 1,), 9.0, dtype=dtype, device=DEV) for _ in range(2)]
    out = [f[1:].view(rows, kv, dim) for f in flat]
    kv8.read(s.cache, u32(pos), u32(held), u32(np.cumsum([0] + lens)), k_out=out[0], v_out=out[1])
    one = kv8.read(s.cache, u32([held[0] - 1, 4, ref.NONE]), u32(held), dtype=dtype)
    for i in range(2):
        got, single = out[i].cpu().numpy(), one[i].cpu().numpy()
        assert flat[i][0] == 9.0
        row = 0
        for q, n in enumerate(lens):
            for r in range(n):
                p = pos[q] + r
                for g in range(kv):
                    x = s.m.value(i, q, g, p, held[q]) if pos[q] != ref.NONE and p < held[q] else None
                    want = np.full(dim, 9.0) if x is None else x.astype(np.float32)
                    assert np.array_equal(got[row, g], want.astype(got.dtype)), (i, q, p, g)
                    if x is not None and p == (held[0] - 1, 4, -1)[q]:
                        assert np.array_equal(single[q, g], want.astype(got.dtype))
                row += 1
        assert not single[2].any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16], ids=["f32", "f16"])
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_long_reads(dim, fmt, dtype):
    """Reads of many positions, which a lane takes several of, are those of few: ragged, a hole, open blocks, rows behind."""
    kv, page = 8 if dim == 64 else 4, 96
    lens, held = [5001, 3, 0, 4099], [5000, 77, 40, 4096]
    n_pages = 200
    rng = np.random.default_rng(dim)
    table = rng.integers(0, n_pages, (4, 53)).astype(np.int32)
    table[0, 7] = -1
    cache = kv8.PagedKV8.empty(n_pages, kv, page, dim, 32, dev(table), DTYPE[fmt])
    g = torch.Generator(device=DEV)
    g.manual_seed(dim)
    for x in (cache.k, cache.v):
        x.copy_(torch.randint(-100, 100, x.shape, device=DEV, generator=g).to(torch.float32).to(x.dtype))
    for x in (cache.k_scale, cache.v_scale, cache.k_tail, cache.v_tail):
        x.copy_(torch.rand(x.shape, device=DEV, generator=g))
    start = np.cumsum([0] + lens)
    pos = [0, 70, 5, 0]
    rows = int(start[-1]) + 5
    many = [torch.full((rows, kv, dim), 7.0, dtype=dtype, device=DEV) for _ in range(2)]
    kv8.read(cache, u32(pos), u32(held), u32(start), k_out=many[0], v_out=many[1])
    few = [torch.full((rows, kv, dim), 7.0, dtype=dtype, device=DEV) for _ in range(2)]
    for i, n in enumerate(lens):
        for a in range(0, n, 300):
            b = min(n, a + 300)
            part = [x[start[i] + a:start[i] + b] for x in few]
            at = [ref.NONE] * 4
            at[i] = pos[i] + a
            kv8.read(cache, u32(at), u32(held), u32([0] * (i + 1) + [b - a] * (4 - i)), k_out=part[0], v_out=part[1])
    assert torch.equal(many[0], few[0]) and torch.equal(many[1], few[1])
    assert bool((many[0][-5:] == 7.0).all()) and bool((many[0][5000] == 7.0).all()) and bool((many[0][7 * 96:8 * 96] == 7.0).all())
    assert rows * kv * (dim // 8) >= 393216


def test_v_alone_and_both():
    s = Setup(9, 1, 2, 2, 64, 32, 8, "int8")
    s.append([40], [0], s.tokens(40))
    k, v = kv8.read(s.cache, u32([0]), u32([40]), u32([0, 40]), rows=40)
    only = torch.zeros_like(v)
    from rtxllm_amd._lib import lib

    start, pos, held = u32([0, 40]), u32([0]), u32([40])
    assert lib().rtxllm_kv8_read(s.cache.ref, held.data_ptr(), start.data_ptr(), pos.data_ptr(), 1, 40, 0, None, only.data_ptr(), None) == 0
    assert torch.equal(only, v) and not torch.equal(k, v)


def test_many_sequences():
    """More sequences than a launch's workgroups take in one round, most of them empty."""
    count = 700
    s = Setup(11, count, 1, 1, 64, 16, 8, "int8")
    lens = [int(s.rng.integers(1, 17)) if i % 7 == 0 else 0 for i in range(count)]
    s.append(lens, [0] * count, s.tokens(sum(lens)))
    s.check()


def test_past_32_bit_offsets():
    """Codes behind 4 GiB of the cache, and behind 2^32 of its bytes in one sequence's pages."""
    page, kv, dim, block = 1024, 8, 256, 64
    n_pages = (1 << 32) // (page * kv * dim) + 3
    table = torch.tensor([[n_pages - 1, 0, n_pages - 2]], dtype=torch.int32, device=DEV)
    cache = kv8.PagedKV8.empty(n_pages, kv, page, dim, block, table)
    rng = np.random.default_rng(6)
    new = [rng.standard_normal((2048 + 200, kv, dim)).astype(np.float32) for _ in range(2)]
    rows = len(new[0])
    kv8.append(cache, dev(new[0]), dev(new[1]), u32([0]), u32([0, rows]))
    got = kv8.read(cache, u32([0]), u32([rows]), u32([0, rows]), rows=rows)
    for x, y in zip(new, got):
        y = y.cpu().numpy()
        for p in range(0, rows // block * block, block):
            for g in (0, kv - 1):
                c, sc = ref.quantise(x[p:p + block, g].astype(np.float16), "int8")
                assert np.array_equal(y[p:p + block, g], c.astype(np.float32) * sc), (p, g)
