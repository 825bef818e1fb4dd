"""The entry points on ragged rows (include/rtxllm/kv8.h, the windowed attention of include/rtxllm/paged_kv.h) refuse
what their kernels do not take before any launch (no GPU is needed for a refusal), size their workspaces, and share
rows out to units of work as documented; rows.h and attn_rows.h on the CPU."""

from __future__ import annotations

import ctypes
import re
import shutil
import subprocess
from pathlib import Path

import numpy as np
import pytest
import rows_ref as ref
import torch

from rtxllm_amd import kv8, paged
from rtxllm_amd._lib import PagedKV8Struct, PagedKVStruct

REPO = Path(__file__).resolve().parent.parent
INVALID = 1
BASE = 1 << 24  # an address that no refused call reads


def ptr(i):
    return (16 + i) * BASE


def cache16(**change):
    f = dict(k=BASE, v=2 * BASE, block_table=3 * BASE, table_stride=8, n_pages=64, n_kv_heads=2, head_dim=128,
             page_size=16, capacity=128)
    f.update(change)
    return PagedKVStruct(*(f[n] for n, _ in PagedKVStruct._fields_))


def cache8(**change):
    f = dict(k=BASE, v=2 * BASE, k_scale=4 * BASE, v_scale=5 * BASE, k_tail=6 * BASE, v_tail=7 * BASE, block_table=3 * BASE,
             table_stride=8, n_pages=64, n_kv_heads=2, head_dim=128, page_size=16, capacity=128, block=16, format=0)
    f.update(change)
    return PagedKV8Struct(*(f[n] for n, _ in PagedKV8Struct._fields_))


ATTN = dict(q=ptr(0), type=0, n_heads=4, start=ptr(1), pos=ptr(2), sequences=2, rows=9, window=100, sinks=4, out=ptr(3),
            workspace=ptr(4), workspace_bytes=1 << 20)
CALLS = {
    "rtxllm_kv8_append": dict(k=ptr(0), k_stride=256, v=ptr(1), v_stride=300, type=0, start=ptr(2), pos=ptr(3), sequences=2, rows=9),
    "rtxllm_kv8_read": dict(held=ptr(0), start=ptr(1), pos=ptr(2), sequences=2, rows=9, type=0, k_out=ptr(3), v_out=ptr(4)),
    "rtxllm_attn_kv8": ATTN,
    "rtxllm_attn_window_f16": ATTN,
}
BAD_PAGES = [dict(k=None), dict(v=None), dict(block_table=None), dict(k=BASE + 8), dict(v=BASE + 2), dict(block_table=BASE + 2),
             dict(n_pages=0), dict(n_pages=1 << 31), dict(n_kv_heads=0), dict(n_kv_heads=4097), dict(head_dim=96),
             dict(page_size=0), dict(capacity=0), dict(capacity=120), dict(capacity=(1 << 24) + 16), dict(table_stride=7)]
BAD_KV8 = [dict(k_scale=None), dict(v_scale=None), dict(k_tail=None), dict(v_tail=None), dict(k_scale=BASE + 2), dict(v_scale=BASE + 1),
           dict(k_tail=BASE + 8), dict(v_tail=BASE + 8), dict(block=0), dict(block=4), dict(block=12), dict(block=128), dict(block=32),
           dict(format=2), dict(format=-1), dict(table_stride=0)]
ROWS = [dict(pos=None), dict(pos=ptr(9) + 2), dict(start=ptr(9) + 1), dict(sequences=0), dict(sequences=65536), dict(rows=0),
        dict(rows=(1 << 20) + 1), dict(start=None), dict(type=2), dict(type=-1)]
BAD_ATTN = [dict(q=None), dict(out=None), dict(workspace=None), dict(q=ptr(0) + 2), dict(out=ptr(3) + 1), dict(workspace=ptr(4) + 128),
            dict(workspace_bytes=16), dict(n_heads=0), dict(n_heads=3), dict(n_heads=34), dict(window=0), dict(out=ptr(0) + 512),
            dict(out=ptr(0) - 512), dict(out=ptr(2)), dict(out=ptr(1) - 256), dict(out=ptr(4)), dict(out=BASE + 64), dict(out=2 * BASE),
            dict(out=3 * BASE), dict(workspace=ptr(0)), dict(workspace=BASE), dict(workspace=ptr(2)), dict(q=ptr(0) + 1, type=1)]
BAD = {
    "rtxllm_kv8_append": [dict(k=None), dict(v=None), dict(k=ptr(0) + 2), dict(v=ptr(1) + 1, type=1), dict(k_stride=255), dict(v_stride=0),
                          dict(k_stride=(1 << 30) + 1), dict(k=BASE + 64), dict(v=4 * BASE), dict(pos=6 * BASE), dict(start=2 * BASE)],
    "rtxllm_kv8_read": [dict(held=None), dict(held=ptr(0) + 2), dict(k_out=None, v_out=None), dict(k_out=ptr(3) + 2), dict(v_out=ptr(4) + 1),
                        dict(k_out=ptr(4)), dict(v_out=ptr(3) + 512), dict(k_out=ptr(0)), dict(v_out=ptr(2)), dict(k_out=ptr(1)),
                        dict(k_out=BASE), dict(v_out=4 * BASE), dict(v_out=7 * BASE), dict(k_out=3 * BASE)],
    "rtxllm_attn_kv8": BAD_ATTN + [dict(out=4 * BASE), dict(out=6 * BASE), dict(workspace=5 * BASE)],
    "rtxllm_attn_window_f16": BAD_ATTN,
}


def call(rlib, name, c, **change):
    args = dict(CALLS[name])
    args.update(change)
    return getattr(rlib, name)(None if c is None else ctypes.addressof(c), *args.values(), None)


@pytest.mark.parametrize("name", sorted(CALLS))
def test_refusals(rlib, name):
    make = cache16 if name == "rtxllm_attn_window_f16" else cache8
    assert call(rlib, name, None) == INVALID
    for change in BAD_PAGES + (BAD_KV8 if make is cache8 else []):
        assert call(rlib, name, make(**change)) == INVALID, change
    for change in ROWS + BAD[name]:
        assert call(rlib, name, make(), **change) == INVALID, change


def test_arrays_of_a_cache_lie_apart(rlib):
    for change in (dict(k=2 * BASE), dict(k_scale=BASE + 64), dict(k_tail=7 * BASE), dict(v_tail=BASE), dict(block_table=6 * BASE)):
        assert call(rlib, "rtxllm_kv8_append", cache8(**change)) == INVALID, change


def test_workspaces(rlib):
    a, b = cache16(), cache8()
    for ws, c in ((rlib.rtxllm_attn_window_workspace, a), (rlib.rtxllm_attn_kv8_workspace, b)):
        p = ctypes.addressof(c)
        assert ws(p, 4, 2, 9, 100, 4) > 0
        for bad in ((3, 2, 9, 100, 4), (0, 2, 9, 100, 4), (34, 2, 9, 100, 4), (4, 0, 9, 100, 4), (4, 65536, 9, 100, 4), (4, 2, 0, 100, 4),
                    (4, 2, (1 << 20) + 1, 100, 4), (4, 2, 9, 0, 4)):
            assert ws(p, *bad) == 0, bad
        assert ws(None, 4, 2, 9, 100, 4) == 0
    # a window needs no more room than the whole context
    long = cache16(capacity=1 << 20, table_stride=1 << 16)
    whole = rlib.rtxllm_attn_window_workspace(ctypes.addressof(long), 4, 1, 1, 1 << 24, 0)
    assert 0 < rlib.rtxllm_attn_window_workspace(ctypes.addressof(long), 4, 1, 1, 100, 4) <= whole < 1 << 24


def build(tmp_path, body):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("g++ not available")
    (tmp_path / "t.cpp").write_text('#include <hip/hip_runtime_api.h>\n#include <cstdio>\n#include <vector>\n'
                                    '#include "attn_rows.h"\nusing namespace rtxllm;\n' + body)
    exe = tmp_path / "t"
    subprocess.run([gxx, "-std=c++17", "-Wall", "-O1", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include", "-I", str(REPO / "include"), "-I",
                    str(REPO / "local-ai-gpu-acceleration_amd" / "csrc"), str(tmp_path / "t.cpp"), "-o", str(exe)], check=True, timeout=120)
    return subprocess.run([exe], check=True, capture_output=True, text=True).stdout.split("\n")


def test_units_reach_every_row_once(tmp_path):
    """Units of up to `per` rows (attention) and of blocks (append): each row in one unit of its own sequence, whatever the
    starts; none out of range where starts do not ascend."""
    rng = np.random.default_rng(3)
    starts = [[0, 5], [0, 0, 0, 7, 7, 40], [3, 3, 9], [0, 1, 2, 3], [9, 2, 30, 4], [50, 60], [0, 2 ** 32 - 1], [7, 7]]
    starts += [list(np.cumsum(rng.integers(0, 20, 12))) for _ in range(6)]
    lines = []
    for s in starts:
        for per in (1, 3, 16, 32):
            lines.append("{{%s}, %uu}" % (", ".join(f"{x}u" for x in s), per))
    body = ("struct C { std::vector<std::uint32_t> start; std::uint32_t per; };\nint main() {\n  std::vector<C> cs = {%s};\n"
            "  std::vector<std::uint32_t> pos(64, 5u);\n  for (const C& c : cs) {\n"
            "    const CallRows r{c.start.data(), pos.data(), static_cast<std::uint32_t>(c.start.size() - 1), 41u};\n"
            "    const std::uint32_t units = units_of(r.sequences, r.rows, c.per, 1u);\n"
            "    for (std::uint32_t w = 0; w < units; ++w) {\n      std::uint32_t base;\n      const std::uint32_t s = unit_sequence(r, w, c.per, 1u, base);\n"
            "      const SeqRows q = seq_rows(r, s);\n      if (w < base || (w - base) > q.n / c.per || (w - base) * c.per >= q.n) continue;\n"
            "      const std::uint32_t i0 = (w - base) * c.per, n = q.n - i0 < c.per ? q.n - i0 : c.per;\n"
            "      for (std::uint32_t i = 0; i < n; ++i) std::printf(\"%%u:%%u \", s, q.row + i0 + i);\n    }\n    std::printf(\"\\n\");\n  }\n}\n"
            % ", ".join(lines))
    got = build(tmp_path, body)
    i = 0
    for s in starts:
        ascends = all(a <= b for a, b in zip(s, s[1:]))
        for _ in range(4):
            pairs = [tuple(map(int, x.split(":"))) for x in got[i].split()]
            i += 1
            assert all(r < 41 for _, r in pairs)
            if ascends:
                want = [(k, r) for k, (a, b) in enumerate(zip(s, s[1:])) for r in range(a, min(b, 41))]
                assert sorted(pairs) == want, s


@pytest.mark.parametrize("tile", [32, 64])
def test_tiles_cover_what_rows_see(tmp_path, tile):
    """Every position that some row of a unit sees lies in exactly one of its tiles, in the pages below code_end, in the tail
    from there on; no tile is without one that could be seen but for the edges of the window."""
    cases = [(pos, n, cap, window, sinks, shift) for pos in (0, 1, 31, 64, 100, 250, 255, 256, 4000000000) for n in (1, 5, 40)
             for cap in (256,) for window in (1, 2, 33, 64, 256) for sinks in (0, 1, 33, 70, 256) for shift in (0, 3, 6)]
    body = ("int main() {\n  static const std::uint32_t c[][6] = {%s};\n  for (const auto& x : c) {\n    const std::uint32_t start[2] = {0u, x[1]};\n"
            "    const CallRows r{start, &x[0], 1u, x[1]};\n    RowsCache kv{};\n    kv.p.capacity = x[2], kv.block_shift = x[5];\n"
            "    const std::uint32_t tq = 7u;\n    for (std::uint32_t w = 0; w < units_of(1u, x[1], tq, 1u); ++w) {\n"
            "      const RowSpan s = row_span(r, kv, w, tq, x[3], x[4], %uu);\n      if (s.nq == 0u) continue;\n"
            "      std::printf(\"%%u %%u %%u %%u %%u\", s.row, s.nq, s.code_end, s.tail, s.total);\n"
            "      for (std::uint32_t u = 0; u < s.total; ++u) std::printf(\" %%u\", u < s.ncode ? span_position(s, u, %uu) : s.tail + (u - s.ncode) * %uu);\n"
            "      std::printf(\"|\");\n    }\n    std::printf(\"\\n\");\n  }\n}\n"
            % (", ".join("{" + ", ".join(f"{v}u" for v in c) + "}" for c in cases), tile, tile, tile))
    got = build(tmp_path, body)
    for line, (pos, n, cap, window, sinks, shift) in zip(got, cases):
        end = min(pos + n, cap)
        whole = end >> shift << shift if shift else None
        rows = 0
        for unit in line.split("|")[:-1]:
            row, nq, code_end, tail, total, *tiles = map(int, unit.split())
            assert row == rows and len(tiles) == total and nq >= 1
            rows += nq
            seen = set()
            for i in range(nq):
                seen |= set(ref.visible(min(pos + row + i, cap - 1), window, sinks).tolist())
            last = max(seen)
            want_end = last + 1 if whole is None else min(whole, last + 1)
            assert code_end == want_end and (tail == code_end or tail > last)
            covered = []
            for t in tiles:
                here = [j for j in range(t, t + tile) if (j < code_end if t < code_end and t % tile == 0 and t != tail else j >= tail)]
                covered += here
            assert len(covered) == len(set(covered)) and seen <= set(covered), (pos, n, window, sinks, shift, unit)
        assert rows == n


def test_a_cache_of_the_other_kind_is_refused():
    """fp16 pages and a cache in 8 bits are different structs: neither reaches the other's functions."""
    pages, codes = object.__new__(paged.PagedKV), object.__new__(kv8.PagedKV8)
    x, pos = torch.zeros(1, 2, 128), torch.zeros(1, dtype=torch.int32)
    for call in (lambda: kv8.append(pages, x, x, pos), lambda: kv8.read(pages, pos, pos), lambda: kv8.attn(pages, x, pos),
                 lambda: kv8.attn_workspace(pages, 2, 1, 1)):
        with pytest.raises(ValueError, match="expected a PagedKV8"):
            call()
    names = set(re.findall(r'_call\("(rtxllm_\w+)"', Path(paged.__file__).read_text())) | {"rtxllm_attn_window_f16"}
    assert len(names) >= 6
    for name in names:
        with pytest.raises(ValueError, match="not a cache in 8 bits"):
            codes._call(name)
