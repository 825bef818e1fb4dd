// What the operators on ragged rows share (kv8.hip, attn_rows.hip, attn_prompt.hip): the
// rows of a call, a paged cache of fp16 values or of 8-bit codes as the kernels see it, and the
// host's checks. Index arithmetic is plain C++, so that a CPU build can test it.
#pragma once

#include "paged.h"
#include "rtxllm/kv8.h"

namespace rtxllm {

enum class Cached { kF16, kInt8, kE4m3 };

// The pages as PagedView has them (k and v as bytes), the scales and the tails.
struct RowsCache {
  PagedView p;  // p.k, p.v: not used
  const std::uint8_t *k, *v;
  const float *ks, *vs;         // [row >> block_shift], the rows of paged_row
  const std::uint16_t *kt, *vt;
  std::uint32_t block_shift;
};

struct CallRows {
  const std::uint32_t* start;  // null: row s is sequence s
  const std::uint32_t* pos;
  std::uint32_t sequences, rows;
};

// A sequence's rows: none (n 0), or the first of them and its position.
struct SeqRows {
  std::uint32_t row, n, pos;
};

RTXLLM_HD SeqRows seq_rows(const CallRows& c, std::uint32_t s) {
  SeqRows r{s, 1u, c.pos[s]};
  if (c.start != nullptr) {
    r.row = c.start[s];
    const std::uint32_t end = c.start[s + 1u] < c.rows ? c.start[s + 1u] : c.rows;
    r.n = r.row < end ? end - r.row : 0u;
  }
  if (r.pos == RTXLLM_NO_POSITION) r.n = 0u;
  return r;
}

// Positions of [pos, pos + n) below the capacity: the end of them.
RTXLLM_HD std::uint32_t held_end(std::uint32_t pos, std::uint32_t n, std::uint32_t capacity) {
  return pos >= capacity || n >= capacity - pos ? capacity : pos + n;
}

// Units of a call, of which each sequence has up to n / per + more for its n rows: sequence
// s's start at start[s] / per + more * s, as floor(a + n) >= floor(a) + floor(n). The
// sequence that unit w belongs to; its first unit goes to `base`.
RTXLLM_HD std::uint32_t unit_base(const CallRows& c, std::uint32_t s, std::uint32_t per, std::uint32_t more) {
  const std::uint32_t at = c.start[s] < c.rows ? c.start[s] : c.rows;
  return at / per + more * s;
}
RTXLLM_HD std::uint32_t unit_sequence(const CallRows& c, std::uint32_t w, std::uint32_t per, std::uint32_t more,
                                      std::uint32_t& base) {
  std::uint32_t lo = 0u, hi = c.sequences;  // the last s in [lo, hi) whose base is not above w
  while (hi - lo > 1u) {
    const std::uint32_t mid = lo + (hi - lo) / 2u;
    if (unit_base(c, mid, per, more) <= w)
      lo = mid;
    else
      hi = mid;
  }
  base = unit_base(c, lo, per, more);
  return lo;
}
inline std::uint32_t units_of(std::uint32_t sequences, std::uint32_t rows, std::uint32_t per, std::uint32_t more) {
  return rows / per + more * sequences;
}

inline bool rows_ok(const std::uint32_t* start, const std::uint32_t* pos, std::uint32_t sequences, std::uint32_t rows) {
  return pos != nullptr && aligned_to(pos, 4u) && aligned_to(start, 4u) && sequences >= 1u && sequences <= 65535u &&
         rows >= 1u && rows <= (1u << 20) && (start != nullptr || rows == sequences);
}

// Append: a block of 8 rounds (16 bytes a lane of fp16) or more is four waves', which keeps all of them from waiting for
// their last read and then computing at once (us of one wave / four, 64 positions of 8 heads: 8192 of 128 in fp32 20.0 /
// 17.2, in e4m3 17.1 / 16.9, from fp16 14.2 / 11.9, 1024 of 128 10.4 / 7.0, 4096 of 256 26.7 / 19.4; of 4 rounds, 16
// positions of 128, 17.1 / 17.3).
constexpr bool append_shared(int rounds) { return rounds >= 8; }

// Read: positions of a head that a lane takes where there are many (units: positions times heads), one where there are
// few. us of one / many, 8 heads of 128: 2000 positions as fp16 4.9 / 5.3, as fp32 7.6 / 8.8; 4000 9.0 / 8.4, 12.7 / 12.1;
// 32000 65.6 / 45.0, 88.7 / 69.5.
constexpr int read_units(bool f16) { return f16 ? 4 : 8; }
inline bool read_many(std::uint64_t units, std::uint32_t lanes, bool f16) { return units * lanes >= 393216u; }

inline bool type_ok(int type) { return type == RTXLLM_F32 || type == RTXLLM_F16; }
inline std::size_t type_bytes(int type) { return type == RTXLLM_F32 ? 4u : 2u; }

// The pages' part of an 8-bit cache, for the checks of paged.h.
inline rtxllm_paged_kv kv8_pages(const rtxllm_paged_kv8* c) {
  return rtxllm_paged_kv{reinterpret_cast<std::uint16_t*>(c->k), reinterpret_cast<std::uint16_t*>(c->v),
                         c->block_table,  c->table_stride, c->n_pages,  c->n_kv_heads,
                         c->head_dim,     c->page_size,    c->capacity};
}

inline std::uint32_t kv8_block_shift(std::uint32_t block) {
  return block == 8u ? 3u : block == 16u ? 4u : block == 32u ? 5u : block == 64u ? 6u : 0u;
}

inline bool kv8_cache_ok(const rtxllm_paged_kv8* c, std::uint32_t sequences) {
  if (c == nullptr || c->k_scale == nullptr || c->v_scale == nullptr || c->k_tail == nullptr || c->v_tail == nullptr ||
      (c->format != RTXLLM_KV8_INT8 && c->format != RTXLLM_KV8_E4M3) || kv8_block_shift(c->block) == 0u ||
      c->page_size % c->block != 0u || (c->table_stride == 0u && sequences > 1u))
    return false;
  const rtxllm_paged_kv pages = kv8_pages(c);
  return paged_cache_ok(&pages, sequences) && aligned_to(c->k_scale, 4u) && aligned_to(c->v_scale, 4u) &&
         aligned_to(c->k_tail, 16u) && aligned_to(c->v_tail, 16u);
}

// The arrays of a cache and their bytes, the tails of `sequences`.
struct Kv8Ranges {
  const void* at[6];
  std::uint64_t n[6];
};
inline Kv8Ranges kv8_ranges(const rtxllm_paged_kv8* c, std::uint32_t sequences) {
  const std::uint64_t rows = static_cast<std::uint64_t>(c->n_pages) * c->n_kv_heads * c->page_size;
  const std::uint64_t codes = rows * c->head_dim, scales = rows / c->block * 4u;
  const std::uint64_t tails = 2ull * sequences * c->n_kv_heads * c->block * c->head_dim;
  return Kv8Ranges{{c->k, c->v, c->k_scale, c->v_scale, c->k_tail, c->v_tail}, {codes, codes, scales, scales, tails, tails}};
}
inline bool apart(const Kv8Ranges& r, const void* p, std::uint64_t n) {
  for (int i = 0; i < 6; ++i)
    if (overlap(r.at[i], r.n[i], p, n)) return false;
  return true;
}

inline RowsCache kv8_view(const rtxllm_paged_kv8* c) {
  const rtxllm_paged_kv pages = kv8_pages(c);
  return RowsCache{paged_view(&pages), c->k, c->v, c->k_scale, c->v_scale, c->k_tail, c->v_tail, kv8_block_shift(c->block)};
}

inline Cached kv8_kind(const rtxllm_paged_kv8* c) { return c->format == RTXLLM_KV8_E4M3 ? Cached::kE4m3 : Cached::kInt8; }

inline RowsCache f16_view(const rtxllm_paged_kv* c) {
  return RowsCache{paged_view(c), reinterpret_cast<const std::uint8_t*>(c->k), reinterpret_cast<const std::uint8_t*>(c->v),
                   nullptr,       nullptr, nullptr, nullptr, 0u};
}

}  // namespace rtxllm
