// What the paged-cache operators (paged_append.hip, paged_attn.hip,
// paged_select.hip) share: the cache as the kernels see it, the address of a
// slot, and the host's checks. The address arithmetic is plain C++, so that a
// CPU build can test it.
#pragma once

#include <cstddef>
#include <cstdint>

#include "rtxllm/paged_kv.h"

#if defined(__HIPCC__)
#define RTXLLM_HD __host__ __device__ __forceinline__
#else
#define RTXLLM_HD inline
#endif

namespace rtxllm {

constexpr std::uint32_t kNoRow = 0xFFFFFFFFu;
constexpr std::uint32_t kMaxQueryGroup = 16;

struct PagedView {
  std::uint16_t* k;
  std::uint16_t* v;
  const std::int32_t* table;
  std::uint32_t table_stride, n_pages, n_kv, page_size, capacity, entries;
  std::uint32_t page_mul, page_shift;  // page_of
};

// x / page_size for x < 2^31, as the high word of a product: with s = ceil(log2 d) and M =
// ceil(2^(31 + s) / d), M d exceeds 2^(31 + s) by less than d <= 2^s, so x M / 2^(31 + s) lies
// less than 1 / d above x / d.
RTXLLM_HD std::uint32_t page_of(const PagedView& c, std::uint32_t x) {
  return static_cast<std::uint32_t>(static_cast<std::uint64_t>(2u * x) * c.page_mul >> 32) >> c.page_shift;
}

// Number of the cache row (head_dim values of one position of one kv head) of
// place `in_page` of physical page `page`, or kNoRow for a page that is not
// there. paged_cache_ok keeps every row number below kNoRow.
RTXLLM_HD std::uint32_t paged_row(const PagedView& c, std::int32_t page, std::uint32_t head, std::uint32_t in_page) {
  if (static_cast<std::uint32_t>(page) >= c.n_pages) return kNoRow;
  return (static_cast<std::uint32_t>(page) * c.n_kv + head) * c.page_size + in_page;
}

// The row of slot `slot` through a table row, or kNoRow.
RTXLLM_HD std::uint32_t paged_slot_row(const PagedView& c, const std::int32_t* table, std::uint32_t head,
                                       std::uint32_t slot) {
  if (slot >= c.capacity) return kNoRow;
  const std::uint32_t page = page_of(c, slot);
  return paged_row(c, table[page], head, slot - page * c.page_size);
}

// Filled positions of a row whose newest is `last`: 0 for a padded row, at most
// the capacity.
RTXLLM_HD std::uint32_t paged_filled(const PagedView& c, std::uint32_t last) {
  if (last == RTXLLM_NO_POSITION) return 0u;
  return last < c.capacity ? last + 1u : c.capacity;
}

inline bool paged_cache_ok(const rtxllm_paged_kv* c, std::uint32_t count) {
  if (c == nullptr || c->k == nullptr || c->v == nullptr || c->block_table == nullptr || c->n_pages == 0u ||
      c->n_kv_heads == 0u || c->n_kv_heads > 4096u || c->page_size == 0u || c->capacity == 0u ||
      c->capacity > (1u << 24) || c->capacity % c->page_size != 0u || c->n_pages > 0x7FFFFFFFu)
    return false;
  if (c->head_dim != 64u && c->head_dim != 128u && c->head_dim != 256u) return false;
  if (c->table_stride != 0u && count > 1u && c->table_stride < c->capacity / c->page_size) return false;
  if (((reinterpret_cast<std::uintptr_t>(c->k) | reinterpret_cast<std::uintptr_t>(c->v)) % 16u) != 0u ||
      (reinterpret_cast<std::uintptr_t>(c->block_table) % 4u) != 0u)
    return false;
  const unsigned __int128 rows = static_cast<unsigned __int128>(c->n_pages) * c->n_kv_heads * c->page_size;
  return rows < kNoRow;
}

inline PagedView paged_view(const rtxllm_paged_kv* c) {
  std::uint32_t shift = 0;
  while ((std::uint64_t{1} << shift) < c->page_size) ++shift;
  const std::uint64_t mul = ((std::uint64_t{1} << (31u + shift)) + c->page_size - 1u) / c->page_size;
  return PagedView{c->k,          c->v,        c->block_table,              c->table_stride, c->n_pages, c->n_kv_heads,
                   c->page_size,  c->capacity, c->capacity / c->page_size, static_cast<std::uint32_t>(mul), shift};
}

// Query heads per kv head, or 0 if the heads do not fit the cache.
inline std::uint32_t paged_group(const rtxllm_paged_kv* c, std::uint32_t n_heads) {
  if (n_heads == 0u || n_heads % c->n_kv_heads != 0u) return 0u;
  const std::uint32_t g = n_heads / c->n_kv_heads;
  return g <= kMaxQueryGroup ? g : 0u;
}

// ---- which form of a kernel takes a call ----------------------------------------

// Append: one workgroup a row saves the row's angles and the others' starts where rows alone
// fill the chip (us of one / several a row: 32 + 2 x 8 heads of 128 at 512 rows 7.6 /
// 6.8, 1024 11.7 / 11.9, 4001 32.5 / 34.2; 16 + 2 x 2 of 256 at 4001 27.8 / 30.7; rows that
// one workgroup holds at once, 8 + 2 x 1 of 64 at 4001, 8.8 / 7.9). units: heads of a row, per: of a
// workgroup.
inline bool append_row_a_workgroup(std::uint32_t count, std::uint32_t units, std::uint32_t per) {
  return count >= 1024u && units > per;
}

// Page bounds: three ways to share the pages out, by the units (a page of a head) and by the
// rounds of 256 / L keys (L = head_dim / 8 lanes a key) that a wave reads one at a page of them.
// Few units: a page's rounds go to the four waves of a workgroup (8 heads of 128, us of one wave / four:
// 256 keys at 8000 positions 12.5 / 5.9 and at 24000 15.0 / 10.9, 128 at 16000 9.1 / 8.7
// and at 32000 13.0 / 13.2, 64 at 4000 5.4 / 4.4 and at 8000 5.6 / 6.2, 32 at 2000 3.4 / 3.7; the newest page
// alone of 256 keys 6.2 / 3.4, of 16, one round, 2.8 / 3.1). The keys stay in the
// caches then: a newest page alone is attended next.
// Pages of less than a round: L lanes take a page each (60000 positions of 8 heads, us of
// a wave / L lanes: 8 keys of 128 38.2 / 29.0, 16 of 64 30.1 / 19.6, 16 of 128 26.6 / 27.3).
// Everything else: a wave a page, streamed past the caches, which hold nothing of it for
// long.
enum class BoundsForm { kFourWaves, kLanes, kWave };
inline BoundsForm bounds_form(std::uint64_t units, std::uint32_t rounds) {
  if (rounds >= 2u && units <= 128u * rounds && units <= 1024u) return BoundsForm::kFourWaves;
  return rounds == 0u ? BoundsForm::kLanes : BoundsForm::kWave;
}

// Page scores: four steps a wave from where single steps, whose sums grow with the heads, fill
// the chip more than once (us of the selection with four / one: 504 waves of 4 heads 9.7 / 8.1, 4096
// 10.9 / 10.6, 8192 13.2 / 14.2, 12000 15.6 / 17.1; of 8 heads 8192 18.8 / 19.1, 12000 23.5 / 24.2; of 12
// 4096 16.2 / 14.8, 12000 28.3 / 28.6; of 16 12000 33.3 / 33.1). waves: of single steps.
inline bool score_four_steps(std::uint64_t waves, std::uint32_t group) {
  return waves > 8192u * ((group + 3u) / 4u);
}

// Eviction: a workgroup of 16 waves, but of four where short sequences give each CU several
// (us of four / 16: 1024 slots of 8 x 8 8.8 / 8.4, of 64 x 8 16.2 / 20.5, 2112 of 8 x 8
// 14.9 / 9.4). pairs: of a sequence and a kv head.
inline bool evict_four_waves(std::uint32_t capacity, std::uint64_t pairs) { return capacity <= 1024u && pairs > 256u; }

// Moves that the choosing workgroup makes itself, at most (us of here / in a launch of
// their own: 64 of 2112 slots 9.3 / 10.6, 96 of 4096 10.6 / 11.1, 256 of 2304 13.5 / 12.4, 512 of
// 2560 18.3 / 14.4).
constexpr std::uint32_t kEvictMovesHere = 128;

inline bool aligned_to(const void* p, std::size_t bytes) { return reinterpret_cast<std::uintptr_t>(p) % bytes == 0u; }
// Whether two ranges of bytes share memory.
inline bool overlap(const void* a, std::size_t an, const void* b, std::size_t bn) {
  const auto x = reinterpret_cast<std::uintptr_t>(a), y = reinterpret_cast<std::uintptr_t>(b);
  return x < y + bn && y < x + an;
}
inline std::size_t round_256(std::size_t b) { return (b + 255u) & ~std::size_t{255}; }

}  // namespace rtxllm
