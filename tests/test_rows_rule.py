"""Which form of the attention of new rows takes a call (csrc/attn_rows.h, rows_prompt), on the CPU: the one that was
measured faster, but for a few calls next to the rule's border."""

from __future__ import annotations

import pytest
from test_rows_host import build

# (head_dim, sequences, rows, query heads a kv head, positions that a row can see): us of 16 columns and of tiles,
# over int8 codes of 8 kv heads, of fp32 rows and of fp16 ones
MEASURED = [
    ((128, 1, 32, 4, 1024), (17.7, 28.2), (17.0, 21.9)),
    ((128, 8, 225, 4, 16000), (201.9, 389.3), (204.2, 278.8)),
    ((128, 1, 64, 4, 1024), (22.7, 37.9), (21.9, 29.5)),
    ((128, 1, 64, 4, 1088), (22.2, 36.4), (21.7, 29.5)),  # a window of 1024 over 4000
    ((128, 1, 64, 4, 4032), (38.3, 43.0), (38.0, 35.8)),
    ((128, 1, 64, 4, 16000), (90.2, 95.6), (90.1, 71.7)),
    ((128, 1, 256, 4, 1024), (25.4, 46.3), (25.1, 37.5)),
    ((128, 1, 256, 4, 4032), (80.7, 69.7), (81.9, 55.8)),
    ((128, 8, 576, 4, 128), (19.5, 31.5), (18.9, 27.8)),
    ((128, 1, 1000, 4, 16000), (905.0, 573.6), (905.4, 414.8)),
    ((64, 1, 64, 4, 16000), (65.3, 64.7), (60.1, 47.9)),
    ((64, 1, 512, 4, 1024), (27.8, 34.1), (27.3, 44.9)),
    ((64, 1, 128, 4, 1024), (13.8, 21.3), (13.7, 37.4)),
    ((64, 1, 1000, 4, 4032), (157.6, 136.8), (158.1, 99.7)),
    ((256, 1, 16, 4, 16000), (61.2, 53.1), (61.4, 44.4)),
    ((256, 1, 128, 4, 1024), (27.0, 45.4), (27.0, 38.5)),
    ((256, 1, 512, 4, 1024), (85.0, 72.1), (83.2, 60.9)),
]
BORDER = {(64, 1, 512, 4, 1024)}


@pytest.fixture(scope="module")
def rule(tmp_path_factory):
    def choose(cases):
        body = ("int main() {\n  static const std::uint32_t c[][6] = {%s};\n  for (const auto& x : c)\n"
                "    std::printf(\"%%d\\n\", rows_prompt(x[1], x[2], x[3], x[0], 64u, x[5] != 0u, x[4]) ? 1 : 0);\n}\n"
                % ", ".join("{" + ", ".join(f"{v}u" for v in c) + "}" for c in cases))
        return [int(x) for x in build(tmp_path_factory.mktemp("rule"), body) if x]
    return choose


def test_the_faster_form(rule):
    cases = [(*shape, f32) for shape, _, _ in MEASURED for f32 in (1, 0)]
    for (*shape, f32), tiles in zip(cases, rule(cases)):
        us = next((a if f32 else b) for s, a, b in MEASURED if s == tuple(shape))
        if tuple(shape) not in BORDER:
            assert us[tiles] <= 1.1 * min(us), (shape, f32, us, tiles)


def test_large_calls_take_tiles_and_small_ones_never(rule):
    for dim in (64, 128, 256):
        for f32 in (0, 1):
            assert rule([(dim, 1, 8192, 4, 8192, f32), (dim, 1, 8000, 4, 2052, f32), (dim, 1, 1 << 20, 16, 1 << 24, f32)]) == [1, 1, 1]
            assert rule([(dim, 1, 1, 16, 1 << 24, f32), (dim, 65535, 65535, 16, 1 << 24, f32), (dim, 1, 8, 4, 1 << 24, f32),
                         (dim, 1, 1 << 16, 1, 1, f32)]) == [0, 0, 0, 0]
