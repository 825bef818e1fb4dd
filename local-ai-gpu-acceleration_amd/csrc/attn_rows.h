// What the kernels of attention over new rows (attn_rows.hip, attn_prompt.hip) share:
// the call, and which positions a tile of query rows sees.
#pragma once

#include "rows.h"

namespace rtxllm {

constexpr std::uint32_t kRowTile = 32;     // positions of a tile of attn_rows.hip's form,
constexpr std::uint32_t kPromptTile = 64;  // of attn_prompt.hip's

// attn_prompt.hip: waves of a workgroup and blocks of 16 columns (query rows times query heads) of a wave.
constexpr int kPromptWaves = 8;
constexpr int prompt_blocks(int head_dim, bool f32) { return head_dim == 256 ? 1 : head_dim == 128 ? 2 : f32 ? 1 : 4; }
inline std::uint32_t prompt_columns(std::uint32_t head_dim, bool f32) {
  return 16u * kPromptWaves * static_cast<std::uint32_t>(prompt_blocks(static_cast<int>(head_dim), f32));
}

// Whether tiles of many rows (attn_prompt.hip) take a call, or attn_rows.hip's 16 columns (rows times query heads): by the
// columns that a sequence has on average, and by the work, the call's columns times the positions that a row can see
// (`near`), of which tiles need many before their fewer workgroups fill the card. us of 16 columns / tiles over int8 codes,
// 8 kv heads of 128, fp32 and fp16 rows:
//   128 columns over one context of 1000      18 /  28    17 /  22
//   128 over one of 16000                     60 /  52    57 /  40   (16 columns all the same)
//   112 over each of eight of up to 16000    202 / 389   204 / 279
//   256 over one of 1000                      23 /  38    22 /  30
//   256 over one of 4000                      38 /  43    38 /  36
//   256 over one of 16000                     90 /  96    90 /  72   tiles
//   1024 over one of 1000                     25 /  46    25 /  38
//   1024 over one of 4000                     81 /  70    82 /  56   tiles
//   4000, a prompt of 1000                    55 /  69    53 /  54   tiles
//   288 each, eight prompts of up to 128      20 /  32    19 /  28
//   675 each, eight prompts of up to 300      40 /  43    37 /  31   tiles
//   4000 over one of 16000                   905 / 574   905 / 415   tiles
// Over 258 such calls (heads of 64, 128 and 256, fp16 pages too) the choice is 3 % behind the faster form on average; by the
// columns alone it was 14 %. Heads of 256, where 16 columns fill the registers: 64 columns over 16000 61 / 53, 61 / 44 and
// 2048, 512 rows over 1000, 85 / 72, 83 / 61 are tiles', 512 over 1000 27 / 45, 27 / 38 are not. The averages are the
// call's: a long prompt beside many single tokens is better off in a call of its own.
inline bool rows_prompt(std::uint32_t sequences, std::uint32_t rows, std::uint32_t group, std::uint32_t head_dim,
                        std::uint32_t page_size, bool f32, std::uint64_t near) {
  const std::uint64_t columns = static_cast<std::uint64_t>(rows) * group, enough = head_dim == 256u ? 40u : 192u;
  return columns >= enough * sequences && columns * near >= 6144ull * prompt_columns(head_dim, f32) && page_size % 4u == 0u;
}

// Splits of a unit's tiles (at most `tiles`) in attn_rows.hip: the largest of 64 to 4 tiles a workgroup that make as
// many workgroups as run at once (512; 256 where registers leave room for two of fp16 heads of 128 or one of 256 a CU), not a
// few more than those, and at most twice as many, which long contexts of different lengths need. us of 1024 / 512 / 256
// workgroups: eight contexts to 65500 in 8 bits 113 / 140 / 223 (of 256 dimensions 220 / 211 / 317), one of 65000
// 42 / 36 / 42, one of 16001 - / 15.7 / 16.3, of 4000 - / 12.3 / 10.5 (32 of 8 tiles or of 4), four of 4000 - / 13.4 /
// 15.4; windows of 1024 over fp16 pages, eight 320 workgroups 17.0, 256 14.0, 32 sequences 41 / 35 / 27. A split's tiles
// are whole rounds of its four waves (span_per), so some splits may get none: of those 256, with 33 tiles in 4 splits of 12,
// 192 have work.
inline std::uint32_t rows_splits(std::uint64_t items, std::uint64_t tiles, bool codes, std::uint32_t head_dim) {
  const std::uint64_t slots = head_dim == 64u || (codes && head_dim == 128u) ? 512u : 256u;
  std::uint64_t per = 64u;
  while (per > 4u && items * ((tiles + per - 1u) / per) < slots) per /= 2u;
  std::uint64_t splits = (tiles + per - 1u) / per;
  if (items * splits > 2u * slots) splits = (2u * slots + items - 1u) / items;
  if (items * splits > slots && 2u * items * splits < 3u * slots) splits = slots / items != 0u ? slots / items : 1u;
  return static_cast<std::uint32_t>(splits);
}

struct AttnRows {
  const void* q;
  void* out;
  float2* ml;   // [unit][kv head][column][split]: maximum (in log2), sum
  float* part;  // [unit][kv head][column][split][head_dim], not divided by the sum
  std::uint32_t f16, group, tq, window, sinks, splits, units;  // tq: query rows of a unit
};

// A unit: up to tq query rows of one sequence. The tiles of positions that one of them sees, in the
// order they are taken: sink tiles before the window, the window's in the pages, the tail's.
struct RowSpan {
  std::uint32_t s, row, nq;      // sequence, first row, rows (0: none)
  std::uint32_t p0, plast, pos;  // positions of the first and last row (below the capacity); of row i: row_pos
  std::uint32_t code_end;        // positions below it are read from the pages,
  std::uint32_t tail;            // those from here on (a block's start) from the tail
  std::uint32_t ns, lo_tile, ncode, total;  // sink tiles, the window's first tile, tiles in the pages, all
};

RTXLLM_HD std::uint32_t row_pos(std::uint32_t pos, std::uint32_t i, std::uint32_t capacity) {
  return pos >= capacity || i >= capacity - pos ? capacity - 1u : pos + i;
}

RTXLLM_HD RowSpan row_span(const CallRows& c, const RowsCache& kv, std::uint32_t w, std::uint32_t tq, std::uint32_t window,
                           std::uint32_t sinks, std::uint32_t tile) {
  RowSpan r{};
  std::uint32_t base = w;
  r.s = w;
  if (c.start != nullptr) r.s = unit_sequence(c, w, tq, 1u, base);
  const SeqRows q = seq_rows(c, r.s);
  const std::uint32_t t = w - base;
  if (w < base || t > q.n / tq || t * tq >= q.n) return r;
  const std::uint32_t i0 = t * tq, cap = kv.p.capacity;
  r.row = q.row + i0;
  r.nq = q.n - i0 < tq ? q.n - i0 : tq;
  r.pos = q.pos >= cap ? cap : q.pos + i0;
  r.p0 = row_pos(r.pos, 0u, cap);
  r.plast = row_pos(r.pos, r.nq - 1u, cap);
  r.code_end = r.plast + 1u;
  r.tail = r.plast + 1u;
  if (kv.block_shift != 0u) {
    const std::uint32_t whole = held_end(q.pos, q.n, cap) >> kv.block_shift << kv.block_shift;
    if (whole < r.code_end) r.code_end = r.tail = whole;
  }
  r.lo_tile = (r.p0 + 1u > window ? r.p0 + 1u - window : 0u) / tile;
  const std::uint32_t front = sinks < r.code_end ? sinks : r.code_end, nf = (front + tile - 1u) / tile;
  const std::uint32_t end_tile = (r.code_end + tile - 1u) / tile;
  r.ns = nf < r.lo_tile ? nf : r.lo_tile;
  r.ncode = r.ns + (end_tile > r.lo_tile ? end_tile - r.lo_tile : 0u);
  r.total = r.ncode + (r.plast + 1u - r.tail + tile - 1u) / tile;
  return r;
}

// The first position of tile u of a unit that lies in the pages.
RTXLLM_HD std::uint32_t span_position(const RowSpan& r, std::uint32_t u, std::uint32_t tile) {
  return (u < r.ns ? u : u - r.ns + r.lo_tile) * tile;
}

// Tiles of a split when `splits` may share them, of whole rounds of the workgroup's waves.
RTXLLM_HD std::uint32_t span_per(std::uint32_t total, std::uint32_t splits, std::uint32_t round) {
  return ((total + splits - 1u) / splits + round - 1u) / round * round;
}

#if defined(__HIPCC__)
hipError_t attn_prompt(Cached kind, std::uint32_t head_dim, const AttnRows& a, const CallRows& rows, const RowsCache& kv,
                       hipStream_t stream);
#endif

}  // namespace rtxllm
