"""The paged-cache entry points refuse what their kernels do not take before any
launch (no GPU is needed for a refusal), size their workspaces, and address the
cache's rows as documented, pages that are not there included."""

from __future__ import annotations

import ctypes
import shutil
import subprocess
from pathlib import Path

import pytest

from rtxllm_amd._lib import PagedKVStruct

REPO = Path(__file__).resolve().parent.parent
INVALID = 1
BASE = 1 << 20  # an address that no refused call reads


def cache(**change):
    f = dict(k=BASE, v=2 * BASE, block_table=BASE + 4096, table_stride=8, n_pages=64, n_kv_heads=2, head_dim=128,
             page_size=16, capacity=128)
    f.update(change)
    return PagedKVStruct(*(f[n] for n, _ in PagedKVStruct._fields_))


def ptr(i):
    return (16 + i) * BASE


# entry point -> arguments behind the cache, by name, in order
CALLS = {
    "rtxllm_qk_norm_rope_append_f16": dict(q=ptr(0), q_stride=512, k=ptr(1), k_stride=256, v=ptr(2), v_stride=256,
                                           q_weight=None, k_weight=None, n_heads=4, rotary_dim=128, pairing=1,
                                           theta=1e4, eps=1e-6, pos=ptr(3), slot=None, count=2, q_out=ptr(4),
                                           slot_pos=None, slot_weight=None),
    "rtxllm_kv_page_bounds_f16": dict(first=None, last=ptr(0), count=2, span=1, bounds=ptr(1)),
    "rtxllm_attn_select_pages": dict(bounds=ptr(0), q=ptr(1), n_heads=4, pos=ptr(2), count=2, n_first=1, n_last=1,
                                     n_select=4, pages=ptr(3), workspace=ptr(4), workspace_bytes=1 << 18),
    "rtxllm_attn_decode_pages_gqa_f16": dict(q=ptr(0), n_heads=4, pages=ptr(1), n_select=4, pos=ptr(2), count=2,
                                             out=ptr(3), workspace=ptr(4), workspace_bytes=1 << 19),
    "rtxllm_attn_decode_weights_gqa_f16": dict(q=ptr(0), n_heads=4, last=ptr(1), count=2, out=ptr(2), weight=ptr(3),
                                               weight_out=ptr(4), workspace=ptr(5), workspace_bytes=1 << 19),
    "rtxllm_kv_evict_f16": dict(length=ptr(0), pos=ptr(1), count=2, keep=64, n_first=2, n_recent=8, weight=ptr(2),
                                slot_pos=ptr(3), weight_out=ptr(4), slot_pos_out=ptr(5), length_out=ptr(6),
                                workspace=ptr(7), workspace_bytes=1 << 18),
}

BAD_CACHE = [dict(k=None), dict(v=None), dict(block_table=None), dict(k=BASE + 8), dict(v=BASE + 2),
             dict(block_table=BASE + 2), dict(n_pages=0), dict(n_pages=1 << 31), dict(n_kv_heads=0),
             dict(n_kv_heads=4097), dict(head_dim=96), dict(head_dim=0), dict(page_size=0), dict(capacity=0),
             dict(capacity=120), dict(capacity=(1 << 24) + 16), dict(table_stride=7), dict(n_pages=(1 << 31) - 1, page_size=128)]

BAD = {
    "rtxllm_qk_norm_rope_append_f16": [
        dict(q=None), dict(k=None), dict(v=None), dict(pos=None), dict(q_out=None), dict(q=ptr(0) + 2), dict(slot=ptr(9) + 1),
        dict(slot_pos=ptr(9) + 2), dict(count=0), dict(count=(1 << 20) + 1), dict(n_heads=0), dict(n_heads=4095),
        dict(rotary_dim=0), dict(rotary_dim=12), dict(rotary_dim=136), dict(pairing=2), dict(pairing=-1),
        dict(theta=0.0), dict(theta=float("nan")), dict(theta=float("inf")), dict(eps=-1.0), dict(eps=float("nan")),
        dict(q_stride=511), dict(k_stride=0), dict(v_stride=255), dict(q_stride=1 << 40),
        dict(q_out=ptr(0), q_stride=600), dict(q_out=ptr(0) + 512), dict(q_out=ptr(1)), dict(q_out=ptr(2) - 512)],
    "rtxllm_kv_page_bounds_f16": [dict(last=None), dict(bounds=None), dict(bounds=ptr(1) + 8), dict(last=ptr(0) + 2),
                                  dict(first=ptr(5) + 1), dict(count=0), dict(count=65536), dict(span=0),
                                  dict(span=(1 << 20) + 1), dict(last=ptr(0) + 1)],
    "rtxllm_attn_select_pages": [
        dict(bounds=None), dict(q=None), dict(pos=None), dict(pages=None), dict(workspace=None), dict(bounds=ptr(0) + 8),
        dict(q=ptr(1) + 1), dict(workspace=ptr(4) + 16), dict(workspace_bytes=0), dict(n_heads=3), dict(n_heads=0),
        dict(n_heads=34), dict(count=0), dict(count=65536), dict(n_select=0), dict(n_select=65537), dict(n_first=4),
        dict(n_first=0xFFFFFFFF), dict(n_last=4)],
    "rtxllm_attn_decode_pages_gqa_f16": [
        dict(q=None), dict(pages=None), dict(pos=None), dict(out=None), dict(workspace=None), dict(out=ptr(3) + 2),
        dict(workspace=ptr(4) + 8), dict(workspace_bytes=1024), dict(n_heads=5), dict(n_heads=34), dict(count=0),
        dict(count=65536), dict(n_select=0), dict(n_select=65537), dict(out=ptr(0) + 512), dict(out=ptr(0) - 512)],
    "rtxllm_attn_decode_weights_gqa_f16": [
        dict(q=None), dict(last=None), dict(out=None), dict(weight=None), dict(weight_out=None), dict(workspace=None),
        dict(weight_out=ptr(3) + 4), dict(weight=ptr(3) + 1), dict(out=ptr(0) + 512), dict(workspace_bytes=4096), dict(n_heads=7), dict(count=0)],
    "rtxllm_kv_evict_f16": [
        dict(length=None), dict(pos=None), dict(weight=None), dict(slot_pos=None), dict(weight_out=None),
        dict(slot_pos_out=None), dict(length_out=None), dict(workspace=None), dict(workspace_bytes=16),
        dict(workspace=ptr(7) + 4), dict(keep=0), dict(keep=129), dict(n_first=60), dict(n_recent=0xFFFFFFFF),
        dict(weight_out=ptr(2) + 16), dict(weight_out=ptr(3)), dict(slot_pos_out=ptr(2)), dict(slot_pos_out=ptr(4)),
        dict(length_out=ptr(1)), dict(length_out=ptr(0) + 4), dict(length_out=ptr(2)), dict(length_out=ptr(5) + 8), dict(pos=ptr(1) + 1), dict(count=0), dict(count=65536)],
}


def call(rlib, name, c, **change):
    args = dict(CALLS[name])
    args.update(change)
    return getattr(rlib, name)(None if c is None else ctypes.addressof(c), *args.values(), None)


@pytest.mark.parametrize("name", sorted(CALLS))
def test_refusals(rlib, name):
    assert call(rlib, name, None) == INVALID
    for change in BAD_CACHE:
        assert call(rlib, name, cache(**change)) == INVALID, change
    c = cache()
    for change in BAD[name]:
        assert call(rlib, name, c, **change) == INVALID, change


@pytest.mark.parametrize("name", ["rtxllm_attn_decode_weights_gqa_f16", "rtxllm_kv_evict_f16"])
def test_gathered_state_is_one_row_a_sequence(rlib, name):
    assert call(rlib, name, cache(table_stride=0)) == INVALID


def test_workspaces(rlib):
    c = cache()
    ref = ctypes.addressof(c)
    assert rlib.rtxllm_attn_select_workspace(ref, 3) == 8 * 3 * 2 * 8 + 128
    assert rlib.rtxllm_kv_evict_workspace(ref, 100, 2) == 1024  # 2 x 2 (1 + 2 x 28) words
    assert rlib.rtxllm_kv_evict_workspace(ref, 128, 1) == 256
    for n in (rlib.rtxllm_attn_select_workspace(ref, 0), rlib.rtxllm_attn_select_workspace(None, 1),
              rlib.rtxllm_attn_pages_workspace(ref, 5, 4, 1), rlib.rtxllm_attn_pages_workspace(ref, 4, 0, 1),
              rlib.rtxllm_attn_pages_workspace(None, 4, 4, 1), rlib.rtxllm_attn_weights_workspace(ref, 34, 1),
              rlib.rtxllm_attn_weights_workspace(None, 4, 1), rlib.rtxllm_kv_evict_workspace(ref, 129, 1),
              rlib.rtxllm_kv_evict_workspace(None, 1, 1)):
        assert n == 0
    assert rlib.rtxllm_attn_weights_workspace(ref, 4, 2) >= rlib.rtxllm_attn_pages_workspace(ref, 4, 8, 2) + 4 * 2 * 4 * 128


def test_row_addresses(tmp_path):
    """paged.h on the CPU: rows of pages that are there, none for pages and slots that are not."""
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("g++ not available")
    src = tmp_path / "t.cpp"
    src.write_text('#include "paged.h"\n#include <cstdio>\nusing namespace rtxllm;\nint main() {\n'
                   "  const std::int32_t table[4] = {2, -1, 7, 6};\n"
                   "  const rtxllm_paged_kv d{reinterpret_cast<std::uint16_t*>(16), reinterpret_cast<std::uint16_t*>(16), table, 4, 7, 3, 64, 5, 20};\n"
                   "  const PagedView c = paged_view(&d);\n"
                   "  for (std::uint32_t p : {1u, 2u, 3u, 5u, 7u, 24u, 64u, 100u, 4095u, 65537u, (1u << 24) - 1u}) {\n"
                   "    rtxllm_paged_kv e = d;\n    e.page_size = p, e.capacity = p;\n    const PagedView v = paged_view(&e);\n"
                   "    for (std::uint64_t x = 0; x < (1ull << 31); x += 1 + x / 97)\n"
                   "      for (std::uint64_t y : {x, x / p * p, x / p * p + p - 1})\n"
                   "        if (y < (1ull << 31) && page_of(v, static_cast<std::uint32_t>(y)) != y / p) return 1;\n  }\n"
                   "  for (std::uint32_t s = 0; s < 22; ++s) std::printf(\"%u \", paged_slot_row(c, table, 2, s));\n"
                   "  std::printf(\"%u %u %u %u\", paged_filled(c, 0xFFFFFFFFu), paged_filled(c, 0), paged_filled(c, 19),\n"
                   "              paged_filled(c, 4000000000u));\n}\n")
    exe = tmp_path / "t"
    subprocess.run([gxx, "-std=c++17", "-Wall", "-Werror", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include", "-I",
                    str(REPO / "include"), "-I", str(REPO / "local-ai-gpu-acceleration_amd" / "csrc"), str(src), "-o",
                    str(exe)], check=True, timeout=120)
    got = [int(x) for x in subprocess.run([exe], check=True, capture_output=True, text=True).stdout.split()]
    none = 0xFFFFFFFF
    want = [(2 * 3 + 2) * 5 + i for i in range(5)] + [none] * 10 + [(6 * 3 + 2) * 5 + i for i in range(5)] + [none] * 2
    assert got == want + [0, 1, 20, 20]


def test_attention_sizes(rlib):
    """A split's scores have one size in the LDS at any capacity (no launch asks for more LDS
    than there is), and sizes beyond a launch's threads are refused."""
    for capacity in (1 << 18, 1 << 20, 1 << 24):
        c = cache(capacity=capacity, table_stride=1 << 20, page_size=256)
        need = rlib.rtxllm_attn_weights_workspace(ctypes.addressof(c), 32, 1)
        splits = capacity // (64 * 16)
        assert need == 8 * 32 * splits + 4 * 32 * splits * 128 + 4 * 32 * capacity
    c = cache(n_kv_heads=4096, n_pages=1024, page_size=256, capacity=1 << 24, table_stride=1 << 16)
    assert rlib.rtxllm_attn_weights_workspace(ctypes.addressof(c), 4096, 1) == 0
    assert rlib.rtxllm_attn_pages_workspace(ctypes.addressof(c), 4096, 65536, 1) == 0
    c = cache(page_size=16384 * 2, capacity=1 << 16, n_pages=2)
    assert rlib.rtxllm_attn_pages_workspace(ctypes.addressof(c), 4, 65536, 1) == 0  # 2^31 positions
