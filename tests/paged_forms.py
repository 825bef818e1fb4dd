"""Calls that reach each form of the paged-cache kernels (the rules are in csrc/paged.h): run
against float64 by test_gpu_paged_forms.py, held to the rules by test_paged_host_edges.py, so
that a rule that changes names the forms that lost their test."""

from __future__ import annotations

# (query heads, kv heads, head_dim, rows): a workgroup a row, or several
APPEND = {"row": [(16, 2, 256, 1100), (30, 2, 128, 1024), (40, 4, 64, 1025)],
          "parts": [(16, 2, 256, 1023), (4, 2, 256, 1100), (12, 2, 128, 1100)]}

# (kv heads, head_dim, page, filled positions of each row, pages of the call)
BOUNDS = {
    "four-waves": [(2, 64, 64, (200, 0, 64), 4), (3, 128, 40, (130, 1), 4), (2, 256, 24, (100, 99), 5), (1, 256, 16, (16,), 1)],
    "lanes": [(3, 64, 31, (130, 0, 31), 5), (2, 128, 5, (77, 1), 16), (2, 256, 5, (41, 40, 0), 9), (5, 256, 7, (3,), 1)],
    "wave": [(2, 64, 40, (400, 1, 81), 10), (2, 128, 21, (100, 40), 5), (3, 256, 8, (90, 0, 8), 12), (2, 256, 13, (100,), 8),
             (8, 64, 64, (4000, 64, 3999), 63), (9, 256, 24, (1000, 980, 3), 42)],
}

# (heads a kv head, kv heads, head_dim, filled pages of each row): pages of one position
SCORE = {"one-step": [(1, 4, 128, (2000, 2000, 40, 2000)), (5, 3, 256, (2100, 7, 300)), (12, 2, 64, (2100, 100))],
         "four-steps": [(2, 8, 64, (2300, 17, 0, 2301, 2302, 2300, 640, 8)), (5, 8, 64, (2100, 2100, 9, 700, 0, 2099, 2100, 2085)),
                        (1, 4, 128, (2100, 40, 2099, 700)), (5, 8, 128, (2100, 4, 2098, 1500)),
                        (12, 8, 128, (2100, 0, 17, 2100, 2097, 800)), (1, 4, 256, (2100, 41)), (5, 4, 256, (2100, 3, 2099, 1000)),
                        (12, 4, 256, (2100, 1, 2100, 500, 0, 2099))]}

# (sequences, kv heads, head_dim, page, slots, keep): four waves or 16, moves in the choosing
# workgroup or in a launch of their own
EVICT = {("four-waves", "here"): [(40, 8, 64, 7, 200, 150), (40, 8, 128, 16, 1024, 960), (33, 8, 256, 5, 100, 60)],
         ("four-waves", "apart"): [(40, 8, 64, 16, 600, 300), (33, 8, 128, 7, 500, 200), (129, 2, 256, 8, 400, 200)],
         ("sixteen", "here"): [(3, 8, 64, 7, 1029, 1000), (2, 2, 128, 16, 200, 150), (32, 8, 256, 5, 100, 60)],
         ("sixteen", "apart"): [(2, 3, 64, 9, 1026, 400), (3, 2, 128, 16, 2000, 1000), (2, 2, 256, 8, 1200, 200)]}


def entries(page, filled):
    return max(1, max(-(-n // page) for n in filled))
