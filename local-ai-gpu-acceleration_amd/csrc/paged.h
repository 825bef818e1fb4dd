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

inline bool aligned_to(const void* p, std::size_t bytes) { return reinterpret_cast<std::uintptr_t>(p) % bytes == 0u; }
// Whether two ranges of bytes share memory.
inline bool overlap(const void* a, std::size_t an, const void* b, std::size_t bn) {
  const auto x = reinterpret_cast<std::uintptr_t>(a), y = reinterpret_cast<std::uintptr_t>(b);
  return x < y + bn && y < x + an;
}
inline std::size_t round_256(std::size_t b) { return (b + 255u) & ~std::size_t{255}; }

}  // namespace rtxllm
