"""What the attention of new rows (rtxllm_attn_window_f16, rtxllm_attn_kv8) keeps of its terms and of its rows, against
float64 (rows_ref.py) with bounds of each row's own attended values."""

from __future__ import annotations

import numpy as np
import pytest
import rows_ref as ref

torch = pytest.importorskip("torch")

from test_gpu_attn_rows import ALL, DTYPE, FORMATS, Setup, dev, u32  # noqa: E402

from rtxllm_amd import kv8, paged  # noqa: E402

pytestmark = pytest.mark.gpu


def bound(q, keys, values, f16, codes, lift, tops=None):
    """(the result, a bound of its error): that of rows_ref.attend, with terms as pairs of which the smaller half ends at
    2^-25 where the largest term is at least 2^(lift - 2): 2^(-23 - lift) of the largest attended value, n times. codes: a
    scale may enter a term and the sum as its logarithm, off by 2^-19 each. f16: rounded once (2^-11).
    tops: over codes, the largest |value| of each position's block. A term times the scale is what enters as a pair, to the
    largest such: 2^(-23 - lift) of the largest weight times scale, n codes; a scale times the format's largest code
    is at most twice the block's largest value (e4m3: 224 / scale or more). And no logarithms."""
    out, _ = ref.attend(q, keys, values)
    n, d = keys.shape
    q, keys, values = (np.asarray(x, np.float64) for x in (q, keys, values))
    s = keys @ q / np.sqrt(d)
    p = np.exp(s - s.max())
    p /= p.sum()
    size = np.abs(keys) @ np.abs(q) / np.sqrt(d)
    delta = (2.0 ** -22 + (d + 16) * 2.0 ** -24) * size.max() + 2.0 ** -21 * (1.0 + np.abs(s).max())
    tol = (2.0 * delta + (n + 64) * 2.0 ** -24 + 2.0 ** -22 + (2.0 ** -18 if codes and tops is None else 0.0)) * (p @ np.abs(values))
    tol = tol + 2.0 ** (-23 - lift) * n * (np.abs(values).max() if tops is None else 2.0 * (p * tops).max()) + 1e-37
    if f16:
        tol = tol + 2.0 ** -11 * (np.abs(out) + tol) + 2.0 ** -25
    return out, tol


def tiles(s, window, sinks):
    """Whether a call takes the tiles of many rows (csrc/attn_rows.h, rows_prompt)."""
    columns, wide = s.rows * s.group, {64: 512 if s.f16 else 128, 128: 256, 256: 128}[s.dim]
    near = min(window + sinks, s.capacity)
    return columns >= (40 if s.dim == 256 else 192) * len(s.lens) and columns * near >= 6144 * wide and s.page % 4 == 0


def rows_within(s, got, window, sinks, lift, sample=1):
    """Every sample-th row of a Setup's call within `bound`."""
    got, row = got.cpu().numpy().astype(np.float64), 0
    for i, n in enumerate(s.lens):
        for r in range(n):
            here, row = row, row + 1
            if s.pos[i] == ref.NONE:
                assert not got[here].any()
                continue
            if r % sample and r != n - 1:
                continue
            p = s.pos[i] + r
            j = ref.visible(p, window, sinks)
            for g in range(s.kv):
                k, v = (np.stack([s.value(c, i, g, int(t)) for t in j]) for c in range(2))
                for h in range(g * s.group, (g + 1) * s.group):
                    want, tol = bound(s.q[here, h], k, v, s.f16, s.fmt != "f16", lift)
                    assert bool((np.abs(got[here, h] - want) <= tol).all()), (i, r, p, h, float((np.abs(got[here, h] - want) / tol).max()))


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_terms_of_fp16_prompts_keep_their_bits(dim, fmt):
    """fp16 queries of many rows: softmax terms are held as finely as in the form for few rows, so that the result's own
    rounding is what an element of any size is off by."""
    s = Setup(21, fmt, [1300, 1050], [1300, 1000], 1, 16, dim, 64, 16, f16=True)
    for window, sinks in ((84, 3), (ALL, 0)):
        assert tiles(s, window, sinks)
        rows_within(s, s.call(window, sinks), window, sinks, 11, sample=97)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("wave", range(4))
def test_every_wave_hands_on_what_it_left_out(wave, fmt):
    """A value that is not finite in a tile that rows see in part is left out of the products and given to its rows at the
    end, whichever of a workgroup's waves met it: tile `wave` of the sinks, and the newest positions."""
    s = Setup(22, fmt, [420], [4], 1, 4, 128, 32, 8)
    at = 32 * wave + 3
    if fmt == "f16":
        s.cache.v[int(s.real[0, at // 32]), 0, at % 32, 9] = float("inf")
    else:
        s.cache.v_scale[int(s.real[0, at // 32]), 0, at % 32 // 8] = float("nan")
    bad = s.call(5, 32 * wave + 5).isfinite().logical_not()
    assert bad[..., 9].all() and (bad.all() if fmt != "f16" else int(bad.sum()) == 16)
    assert s.call(5, 32 * wave).isfinite().all()
    if fmt != "f16":  # the tail's two tiles are the last
        s = Setup(23, fmt, [380 + 32 * wave], [4], 1, 4, 128, 64, 64)
        s.cache.v_tail[0, 0, (s.held[0] - 2) % 64, 9] = float("inf")
        bad = s.call(ALL, 0).isfinite().logical_not()
        assert bad[2:, :, 9].all() and int(bad.sum()) == 8


@pytest.mark.parametrize("bad", [1e-44, 1e-38, 1e-30, 3e38, -1.0, float("inf")])
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dim,rows,f16", [(128, 1200, True), (128, 1200, False), (64, 2000, True), (256, 700, True), (128, 3, True), (128, 1, False)])
def test_scales_that_no_row_sees(dim, rows, f16, fmt, bad):
    """Scales of blocks that are not held, of pages in no table (page 0 among them, whose first row stands in for what is not
    there) and of positions that every window has passed: any number, and the results are the same bits."""
    held = [rows + 310, 290]
    pages = 2 * -(-held[0] // 32)
    seed = next(i for i in range(999) if 0 not in np.random.default_rng(i).permutation(pages + 3)[:pages])  # (the table's draw)
    s = Setup(seed, fmt, held, [rows, min(rows, 60)], 1, 16, dim, 32, 8, f16=f16)
    assert s.n_pages == pages + 3 and 0 not in s.table and tiles(s, 97, 3) == (rows > 3)
    seen, passed = np.zeros((s.n_pages, 4), bool), np.zeros((s.n_pages, 4), bool)
    for i, h in enumerate(s.held):
        for b in range(h // 8):
            seen[s.table[i, b // 4], b % 4] = True
            passed[s.table[i, b // 4], b % 4] = 8 <= 8 * b and 8 * b + 8 <= s.pos[i] - 97
    assert passed.any()
    want = s.call(97, 3)
    assert bool(want.isfinite().all())
    for x in (s.cache.k_scale, s.cache.v_scale):
        x[dev(~seen | passed)[:, None]] = bad
    assert torch.equal(s.call(97, 3), want)


@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
@pytest.mark.parametrize("which", ["k_scale", "v_scale"])
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dim,rows,f16", [(64, 4, False), (128, 4, True), (256, 4, False), (128, 700, False), (128, 700, True)])
def test_scales_that_some_rows_see(dim, rows, f16, fmt, which, bad):
    """A scale that is not finite, of a block that the window of the first row reaches and no other's, of a prompt the first
    half's: those rows are not finite, the others the same bits."""
    s = Setup(24, fmt, [rows + 160], [rows], 1, 4 if rows == 4 else 16, dim, 32, 8, f16=f16)
    first = s.pos[0] if rows == 4 else 487
    window = 9 if rows == 4 else 150
    block = (first + 1 - window) // 8  # its last position is the row's first
    window += first + 1 - window - (8 * block + 7)
    sees = [s.pos[0] + i - window < 8 * block + 7 and s.pos[0] + i >= 8 * block for i in range(rows)]
    want = s.call(window, 0)
    assert tiles(s, window, 0) == (rows > 4)
    assert bool(want.isfinite().all()) and 0 < sum(sees) < rows and (rows > 4 or sees == [True, False, False, False])
    getattr(s.cache, which)[int(s.table[0, block // 4]), 0, block % 4] = bad
    got = s.call(window, 0)
    hit = torch.tensor(sees, device=got.device)
    assert torch.equal(got[~hit], want[~hit])
    if which == "v_scale":
        assert not got[hit].isfinite().any()
    else:  # (an infinite score of -infinity weighs nothing, every other row has NaN)
        assert bad == float("inf") or got[hit].isnan().all()


def tops_of(s, i, g, j):
    """The largest |value| of the blocks of positions j; of those in the tail, the largest of them that is attended."""
    x, block = np.abs(s.x[1][i, :, g].astype(np.float64)).max(-1), s.m.block
    whole = s.held[i] // block * block
    tops = np.array([x[t // block * block:t // block * block + block].max() for t in j])
    tops[j >= whole] = x[j[j >= whole]].max(initial=0.0)
    return tops


# where the large values are, for 4 rows and for many: (positions held, the first, the one behind the last)
LARGE = dict(passed=((235, 40, 48), (675, 104, 112)), little=((235, 96, 104), (675, 96, 104)),
             later=((233, 230, 232), (675, 400, 408)), tail=((235, 234, 235), (675, 674, 675)))


@pytest.mark.parametrize("where", sorted(LARGE))
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_large_values_that_do_not_count_few_rows(dim, fmt, where):
    large_values(dim, fmt, where, 4, False)


@pytest.mark.parametrize("where", sorted(LARGE))
@pytest.mark.parametrize("f16", [False, True], ids=["f32", "half"])
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_large_values_that_do_not_count_prompts(dim, fmt, f16, where):
    large_values(dim, fmt, where, 500, f16)


def large_values(dim, fmt, where, rows, f16):
    """Values of one size, but 6e4 in a few positions: those that the windows of a unit's later rows have passed, that weigh
    nothing by their scores, that only later rows see, in whole blocks and in the tail. Each row is as exact as its own
    attended and weighted values are large."""
    held, lo, hi = LARGE[where][rows > 4]
    s = Setup(25, fmt, [held], [rows], 1, 4 if rows == 4 else 16, dim, 32, 8, f16=f16)
    size = 1e-3 if f16 else 1e-5
    s.x[1][0] = (size * s.rng.standard_normal(s.x[1][0].shape)).astype(np.float16)
    s.x[1][0, lo:hi] = (6e4 * np.sign(s.rng.standard_normal(s.x[1][0, lo:hi].shape))).astype(np.float16)
    s.q = (s.q * 0.1 + 1.0).astype(s.q.dtype)
    if where == "little":
        s.x[0][0, lo:hi] = -6.0
    kv8.append(s.cache, dev(s.x[0][0, :held]), dev(s.x[1][0, :held]), u32([0]), u32([0, held]))
    s.m.append(0, 0, [s.x[i][0, :held] for i in range(2)])
    window = ALL if where != "passed" else s.pos[0] - 44 if rows == 4 else 400
    assert tiles(s, window, 0) == (rows > 4)
    got, seen = s.call(window, 0).cpu().numpy().astype(np.float64), []
    for r in range(4) if rows == 4 else {*range(0, rows, 17), *(r for r in range(lo - s.pos[0] - 9, lo - s.pos[0], 4) if r >= 0)}:
        p = s.pos[0] + r
        j = ref.visible(p, window, 0)
        seen.append(bool(((j >= lo) & (j < hi)).any()))
        k, v = (np.stack([s.value(c, 0, 0, int(t)) for t in j]) for c in range(2))
        for h in range(0, s.group, 1 if rows == 4 else 5):
            want, tol = bound(s.q[r, h], k, v, f16, True, 15 if rows == 4 or not f16 else 11, tops_of(s, 0, 0, j))
            off = np.abs(got[r, h] - want) / tol
            assert bool((off <= 1.0).all()), (r, p, h, float(off.max()), float(np.abs(want).max()))
    assert all(seen) if where == "little" else not all(seen)


@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("rows,f16", [(1, False), (4, True), (300, False), (300, True)])
def test_scales_that_every_row_sees(rows, f16, fmt, bad):
    """A value scale that is not finite, of a block in a tile that all rows see whole: none of its head's rows is a number,
    the other head's are the same bits."""
    s = Setup(27, fmt, [430], [rows], 2, 4 if rows < 5 else 16, 128, 32, 8, f16=f16)
    assert tiles(s, ALL, 0) == (rows > 4)
    want = s.call(ALL, 0)
    s.cache.v_scale[int(s.table[0, 1]), 1, 2] = bad
    got = s.call(ALL, 0)
    assert not got[:, s.group:].isfinite().any() and torch.equal(got[:, :s.group], want[:, :s.group]) and bool(want.isfinite().all())


@pytest.mark.parametrize("fmt", FORMATS)
def test_terms_of_few_fp16_rows_keep_their_bits(fmt):
    """fp16 queries of one row and of drafts: terms as pairs, so that nothing but the result's rounding is fp16's."""
    for lens in ([1, 1], [4, 3]):
        s = Setup(28, fmt, [330, 250], lens, 2, 4, 128, 64, 16, f16=True)
        for window, sinks in ((12, 2), (ALL, 0)):
            rows_within(s, s.call(window, sinks), window, sinks, 15)


@pytest.mark.parametrize("f16", [False, True], ids=["f32", "half"])
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("lens", [[700, 1], [1, 1300, 1, 1], [40, 1, 5]], ids=str)
def test_prompts_beside_tokens(lens, fmt, f16):
    """One call of a prompt and of single tokens, and drafts, of far longer contexts, in either form."""
    held = [n if n > 5 else 3000 + 500 * n for n in lens]
    s = Setup(29, fmt, held, lens, 1, 4, 128, 64, 16, f16=f16)
    for window, sinks in ((ALL, 0), (900, 70)):
        rows_within(s, s.call(window, sinks), window, sinks, 11 if f16 else 15, sample=60)


WINDOWS = [(ALL, 0), (70, 5), (64, 64), (200, 130), (20, 60)]


@pytest.mark.parametrize("f16", [False, True], ids=["f32", "half"])
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dim,group", [(64, 16), (128, 16), (256, 12)])
def test_prompts_in_tiles(dim, group, fmt, f16):
    """Calls that the tiles of many rows take: prompts from nothing and over a held context, a padded sequence, a few rows,
    windows that end inside tiles and inside the sinks."""
    s = Setup(30, fmt, [1500, 1700, ref.NONE, 3], [1500, 1200, 2, 3], 1, group, dim, 64, 16, f16=f16)
    for window, sinks in WINDOWS:
        assert tiles(s, window, sinks)
        rows_within(s, s.call(window, sinks), window, sinks, 11 if f16 else 15, sample=173)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dim,f16", [(64, False), (128, True), (256, False)])
def test_tiles_with_a_window_of_one(dim, f16, fmt):
    """A row that sees itself alone gives its value."""
    rows = 6144 * {64: 128, 128: 256, 256: 128}[dim] // 16
    entries = rows // 64
    table = torch.randperm(entries, device="cuda:0", generator=torch.Generator("cuda:0").manual_seed(dim)).to(torch.int32).reshape(1, -1)
    x = [torch.randn(rows, 1, dim, device="cuda:0").half() for _ in range(2)]
    start, zero = u32([0, rows]), u32([0])
    if fmt == "f16":
        parts = [torch.empty(entries, 1, 64, dim, dtype=torch.float16, device="cuda:0") for _ in range(2)]
        for part, y in zip(parts, x):
            part[table[0].long()] = y.view(entries, 64, 1, dim).transpose(1, 2)
        cache, want, run = paged.PagedKV(*parts, table), x[1].float(), paged.attn_window
    else:
        cache = kv8.PagedKV8.empty(entries, 1, 64, dim, 16, table, DTYPE[fmt])
        kv8.append(cache, *x, zero, start)
        want, run = kv8.read(cache, zero, u32([rows]), start, rows=rows)[1], kv8.attn
    q = torch.randn(rows, 16, dim, device="cuda:0").to(torch.float16 if f16 else torch.float32)
    got = run(cache, q, zero, start, window=1, sinks=0).float()
    # p = 1 in units of the sum, exact; the value or code times a scale rounds thrice (scale, product, quotient)
    assert torch.allclose(got, want.expand_as(got), rtol=2.0 ** -11 if f16 else 2.0 ** -21, atol=2.0 ** -24 if f16 else 0.0)


@pytest.mark.parametrize("f16", [False, True], ids=["f32", "half"])
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_values_and_keys_that_are_not_finite_in_tiles(dim, fmt, f16):
    """Infinities and NaN among a prompt's values and keys, in the pages and in the tail: the rows that see them are not
    finite where they enter, all others are the same bits."""
    held, rows, window = 1523, 1500, 140
    s = Setup(31, fmt, [held], [rows], 1, 16, dim, 64, 16, f16=f16)
    assert tiles(s, window, 0)
    want = s.call(window, 0)
    assert bool(want.isfinite().all())
    block = 1 if fmt == "f16" else 16  # (a block with such a value is NaN as a whole)
    for which, at, d, x in ((1, 700, 5, np.inf), (1, 1001, 6, np.nan), (0, 400, 3, np.nan), (1, held - 3, 9, -np.inf), (1, 64, 0, np.nan)):
        old = s.x[which][0, at, 0, d]
        s.x[which][0, at, 0, d] = x
        if fmt == "f16":
            c = s.cache.v if which else s.cache.k
            c[int(s.real[0, at // 64]), 0, at % 64, d] = float(x)
        else:
            kv8.append(s.cache, dev(s.x[0][0, :held]), dev(s.x[1][0, :held]), u32([0]), u32([0, held]))
        got = s.call(window, 0)
        tail = fmt != "f16" and at >= held // 16 * 16
        lo, hi = (at, at) if block == 1 or tail else (at // 16 * 16, at // 16 * 16 + 15)
        p = np.arange(rows) + s.pos[0]
        sees = torch.tensor((p >= lo) & (p - hi < window), device=got.device)
        assert torch.equal(got[~sees], want[~sees]), (which, at)
        hit = ~got[sees].isfinite()
        if which == 0 or block > 1 and not tail:
            assert bool(hit.all()), (which, at)
        else:
            assert bool(hit[..., d].all()) and int(hit.sum()) == int(sees.sum()) * 16, (which, at)
        s.x[which][0, at, 0, d] = old
        if fmt == "f16":
            c[int(s.real[0, at // 64]), 0, at % 64, d] = float(old)
        else:
            kv8.append(s.cache, dev(s.x[0][0, :held]), dev(s.x[1][0, :held]), u32([0]), u32([0, held]))


@pytest.mark.parametrize("f16", [False, True], ids=["f32", "half"])
@pytest.mark.parametrize("fmt", FORMATS)
def test_holes_strides_and_rows_outside_in_tiles(fmt, f16):
    """Pages that are not there, q and out the same unaligned rows, and rows outside every sequence, of calls in tiles."""
    s = Setup(32, fmt, [900, 640], [800, 600], 1, 16, 128, 32, 8, hole=(0, 3, -1), f16=f16)
    assert tiles(s, 150, 40)
    want = s.call(150, 40)
    got = want.cpu().numpy().astype(np.float64)
    for r in (0, 10, 130, 140, 300):  # beside the hole (positions 96 .. 127), and one far behind it
        p = s.pos[0] + r
        j = ref.visible(p, 150, 40)
        k, v = (np.array([x for x in (s.value(c, 0, 0, int(t)) for t in j) if x is not None]) for c in range(2))
        for h in (0, 15):
            out, tol = bound(s.q[r, h], k, v, f16, fmt != "f16", 11 if f16 else 15)
            assert bool((np.abs(got[r, h] - out) <= tol).all()), (p, h)
    flat = torch.zeros(want.numel() + 1 + 16 * 128 * 20, dtype=want.dtype, device="cuda:0")
    q = flat[1:].view(1420, 16, 128)
    q.fill_(float("nan"))
    q[7:1407] = dev(s.q)
    run = paged.attn_window if fmt == "f16" else kv8.attn
    run(s.cache, q, u32(s.pos), u32([7, 807, 1407]), window=150, sinks=40, out=q)
    assert torch.equal(q[7:1407], want) and bool(q[:7].isnan().all()) and bool(q[1407:].isnan().all())


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("f16", [False, True], ids=["f32", "half"])
def test_queries_that_are_not_finite_in_tiles(fmt, f16):
    s = Setup(33, fmt, [800, 40], [750, 1], 1, 16, 128, 64, 16, f16=f16)
    assert tiles(s, 170, 2)
    want = s.call(170, 2)
    s.q[3, 5, 7], s.q[700, 0, 0] = np.nan, np.inf
    bad = s.call(170, 2)
    hit = bad.isnan().any(-1)
    assert bool(bad[3, 5].isnan().all()) and bool(bad[700, 0].isnan().all()) and int(hit.sum()) == 2
    assert torch.equal(bad[~hit], want[~hit])
