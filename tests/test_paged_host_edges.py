"""Refusals of the paged-cache entry points beyond those of test_paged_host.py (no GPU is
needed for a refusal), and the rules that choose a kernel's form."""

from __future__ import annotations

import shutil
import subprocess

import paged_forms as forms
import pytest

from test_paged_host import CALLS, INVALID, REPO, cache, call, ptr


# ends and starts of one array inside another: a row of 2 x 4 heads of 128 fp32 values is 4096
# bytes, gathered state of 2 x 2 x 128 slots 2048
@pytest.mark.parametrize("name,change", [
    ("rtxllm_attn_decode_weights_gqa_f16", dict(out=ptr(3) + 2044)),
    ("rtxllm_attn_decode_weights_gqa_f16", dict(out=ptr(3) - 4092)),
    ("rtxllm_attn_decode_weights_gqa_f16", dict(out=ptr(4))),
    ("rtxllm_attn_decode_weights_gqa_f16", dict(weight_out=ptr(1) - 2044)),
    ("rtxllm_attn_decode_weights_gqa_f16", dict(out=ptr(1) + 4)),
    ("rtxllm_attn_decode_pages_gqa_f16", dict(out=ptr(1) + 60)),
    ("rtxllm_attn_decode_pages_gqa_f16", dict(out=ptr(2) - 4092)),
    ("rtxllm_kv_evict_f16", dict(weight_out=ptr(0) - 2044)),
    ("rtxllm_kv_evict_f16", dict(weight_out=ptr(1) + 4)),
    ("rtxllm_kv_evict_f16", dict(slot_pos_out=ptr(0) + 4)),
    ("rtxllm_kv_evict_f16", dict(slot_pos_out=ptr(1) - 2044)),
])
def test_outputs_inside_other_arrays(rlib, name, change):
    assert set(change) <= set(CALLS[name])
    assert call(rlib, name, cache(), **change) == INVALID


RULES = r"""
#include "paged.h"
#include <cstdio>
#include <cstring>
using namespace rtxllm;
int main() {
  char kind[8];
  unsigned long long a, b, c;
  while (std::scanf("%7s %llu %llu %llu", kind, &a, &b, &c) == 4) {
    if (kind[0] == 'a') std::puts(append_row_a_workgroup(a, b, c) ? "row" : "parts");
    if (kind[0] == 'b') {
      const BoundsForm f = bounds_form(a, b);
      std::puts(f == BoundsForm::kFourWaves ? "four-waves" : f == BoundsForm::kLanes ? "lanes" : "wave");
    }
    if (kind[0] == 's') std::puts(score_four_steps(a, b) ? "four-steps" : "one-step");
    if (kind[0] == 'e') std::printf("%s %s\n", evict_four_waves(a, b) ? "four-waves" : "sixteen", c <= kEvictMovesHere ? "here" : "apart");
  }
}
"""


def test_every_form_has_its_calls(tmp_path):
    """The listed calls take the forms they are listed for, for every width of a head."""
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("g++ not available")
    lines, want, dims = [], [], {}

    def add(line, form, dim):
        lines.append(line)
        want.append(form)
        dims.setdefault(form, set()).add(dim)

    for form, calls in forms.APPEND.items():
        for heads, kv, dim, rows in calls:
            add(f"a {rows} {heads + 2 * kv} {2048 // dim}", form, dim)
    for form, calls in forms.BOUNDS.items():
        for kv, dim, page, filled, span in calls:
            add(f"b {min(span, forms.entries(page, filled)) * kv * len(filled)} {page // (2048 // dim)} 0", form, dim)
    for form, calls in forms.SCORE.items():
        for group, kv, dim, filled in calls:
            add(f"s {len(filled) * kv * -(-max(filled) // (512 // dim))} {group} 0", form, dim)
    for form, calls in forms.EVICT.items():
        for count, kv, dim, page, slots, keep in calls:
            capacity = -(-slots // page) * page
            add(f"e {capacity} {count * kv} {min(keep, capacity - keep)}", " ".join(form), dim)
    assert all(dims[form] == {64, 128, 256} for form in dims if form != "parts"), dims
    src, exe = tmp_path / "t.cpp", tmp_path / "t"
    src.write_text(RULES)
    subprocess.run([gxx, "-std=c++17", "-Wall", "-Werror", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include", "-I",
                    str(REPO / "include"), "-I", str(REPO / "local-ai-gpu-acceleration_amd" / "csrc"), str(src), "-o",
                    str(exe)], check=True, timeout=120)
    got = subprocess.run([exe], input="\n".join(lines) + "\n", check=True, capture_output=True, text=True).stdout.splitlines()
    assert got == want, [(a, b, c) for a, b, c in zip(lines, got, want) if b != c]
