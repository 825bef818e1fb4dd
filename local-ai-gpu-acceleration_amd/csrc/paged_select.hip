// The two choices over a paged cache: the pages worth attending, and the slots
// worth keeping. Both rank up to some ten thousand keys per (sequence, kv head) and
// take the best k of them, the lower index between equals: a radix selection in
// one workgroup, exact in every bit of the keys.
#include "common.h"
#include "layer_common.cuh"
#include "paged.h"

namespace rtxllm {
namespace {

constexpr std::uint32_t kThreads = 256;
constexpr std::uint32_t kSelThreads = 1024, kSelWaves = kSelThreads / 64u;

__device__ __forceinline__ double lane_xor_d(double v, int mask) { return __shfl_xor(v, mask, 64); }

// A score as an unsigned key of the same order: 1 for NaN, so that 0 is left for
// "no candidate".
__device__ __forceinline__ unsigned long long score_key(double s) {
  if (s != s) return 1ull;
  const unsigned long long b = __builtin_bit_cast(unsigned long long, s + 0.0);  // -0 -> +0
  return (b >> 63) != 0ull ? ~b : b | (1ull << 63);
}

// Scores of 64 / L pages a wave, L = head_dim / 8 lanes a page, 8 dimensions a
// lane. With c = (hi + lo) / 2 and w = |hi - lo| / 2, max(q hi, q lo) = q c + |q| w;
// here both are doubled, which changes no order. Products of fp32 and fp16 values are
// exact in 64 bits, and the sums' 2^-53 keep two pages apart whose scores differ at all.
template <int L>
__global__ __launch_bounds__(kThreads) void page_score_kernel(PagedView kv, const std::uint16_t* __restrict__ bounds,
                                                              const float* __restrict__ q, std::uint32_t group,
                                                              const std::uint32_t* __restrict__ pos,
                                                              std::uint32_t n_first, std::uint32_t n_last,
                                                              unsigned long long* __restrict__ keys) {
  constexpr std::uint32_t D = 8u * L, kPages = 64u / L;
  typedef _Float16 half8 __attribute__((ext_vector_type(8)));
  const std::uint32_t g = blockIdx.y, r = blockIdx.z, lane = threadIdx.x & 63u, t = lane % L;
  const std::uint32_t used = (paged_filled(kv, pos[r]) + kv.page_size - 1u) / kv.page_size;
  const std::uint32_t p = (blockIdx.x * (kThreads / 64u) + (threadIdx.x >> 6)) * kPages + lane / L;
  if (__builtin_amdgcn_readfirstlane(p) >= used) return;
  const std::uint32_t pc = p < used ? p : used - 1u;
  const std::int32_t page = kv.table[static_cast<std::size_t>(r) * kv.table_stride + pc];
  const bool there = static_cast<std::uint32_t>(page) < kv.n_pages;
  const half8* b = reinterpret_cast<const half8*>(
                       bounds + (static_cast<std::size_t>(there ? page : 0) * kv.n_kv + g) * 2u * D) + t;
  const half8 hi = b[0], lo = b[L];
  double c[8], w[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const double x = static_cast<double>(static_cast<float>(hi[i])), y = static_cast<double>(static_cast<float>(lo[i]));
    c[i] = x + y;
    w[i] = x - y;
  }
  const float* qr = q + (static_cast<std::size_t>(r) * kv.n_kv + g) * group * D + 8u * t;
  double best = 0.0;
  for (std::uint32_t h = 0; h < group; ++h) {
    const f32x4_any qa = *reinterpret_cast<const f32x4_any*>(qr + h * D), qb = *reinterpret_cast<const f32x4_any*>(qr + h * D + 4u);
    double s = 0.0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const double x = static_cast<double>(i < 4 ? qa[i & 3] : qb[i & 3]);
      s = fma(x, c[i], s);
      s = fma(fabs(x), fabs(w[i]), s);
    }
#pragma unroll
    for (int m = 1; m < L; m *= 2) s += lane_xor_d(s, m);
    best = h == 0u || s > best || best != best ? s : best;  // a head's NaN gives way to a number
  }
  if (t != 0u || p >= used) return;
  const bool forced = p < n_first || p + n_last >= used;
  keys[(static_cast<std::size_t>(r) * kv.n_kv + g) * kv.entries + p] = !there ? 0ull : forced ? ~0ull : score_key(best);
}

// The best k of n keys: those >= `least`, of those equal to it only the first
// `ties` in index order.
template <class K>
struct Choice {
  K least;
  std::uint32_t ties;
};

struct SelectShared {
  std::uint32_t hist[4096];
  std::uint32_t wave[kSelWaves], bin, above, count;
};

// Radix selection from the top, 12 bits a pass: the workgroup counts the keys
// that share the digits found so far by their next digit, and takes the digit in
// which the k-th largest lies. It ends early once all keys of that digit are
// wanted. key(i) is read anew in every pass (its array stays in the L2).
template <class K, class Key>
__device__ Choice<K> radix_choice(SelectShared& sh, std::uint32_t n, std::uint32_t k, Key key) {
  constexpr int kBits = static_cast<int>(8u * sizeof(K));
  const std::uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6;
  if (k >= n) return Choice<K>{0, 0xFFFFFFFFu};
  K prefix = 0;
  int shift = kBits;
  for (;;) {
    const int bits = shift < 12 ? shift : 12;
    const int next = shift - bits;
    for (std::uint32_t i = tid; i < 4096u; i += kSelThreads) sh.hist[i] = 0u;
    __syncthreads();
    for (std::uint32_t i = tid; i < n; i += kSelThreads) {
      const K x = key(i);
      if (shift == kBits || (x >> shift) == prefix) atomicAdd(&sh.hist[static_cast<std::uint32_t>(x >> next) & ((1u << bits) - 1u)], 1u);
    }
    __syncthreads();
    // thread t holds the four digits 4 (1023 - t) .. + 3: sums from the largest digit down
    const uint4 d = reinterpret_cast<const uint4*>(sh.hist)[kSelThreads - 1u - tid];
    const std::uint32_t mine = d.x + d.y + d.z + d.w;
    std::uint32_t sum = mine;
#pragma unroll
    for (int m = 1; m < 64; m *= 2) {
      const std::uint32_t o = __shfl_up(sum, m, 64);
      sum += lane >= static_cast<std::uint32_t>(m) ? o : 0u;
    }
    if (lane == 63u) sh.wave[wave] = sum;
    __syncthreads();
    std::uint32_t before = sum - mine;
    for (std::uint32_t w = 0; w < wave; ++w) before += sh.wave[w];
    if (before < k && k <= before + mine) {
      const std::uint32_t c[4] = {d.w, d.z, d.y, d.x};
      std::uint32_t j = 0;
      while (before + c[j] < k) before += c[j++];
      sh.bin = 4u * (kSelThreads - 1u - tid) + 3u - j;
      sh.above = before;
      sh.count = c[j];
    }
    __syncthreads();
    prefix = (prefix << bits) | static_cast<K>(sh.bin);
    k -= sh.above;
    const std::uint32_t count = sh.count;
    shift = next;
    __syncthreads();
    if (count == k) return Choice<K>{static_cast<K>(prefix << shift), 0xFFFFFFFFu};
    if (shift == 0) return Choice<K>{prefix, k};
  }
}

// Walks keys 0..n-1 in order, 1024 at a time: body(i, chosen, rank), rank the
// number of chosen keys before i. Every thread calls body for its own i < n.
template <class K, class Key, class Body>
__device__ void for_chosen(SelectShared& sh, std::uint32_t n, const Choice<K>& ch, Key key, Body body) {
  const std::uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6;
  std::uint32_t base_over = 0, base_tie = 0;
  for (std::uint32_t i0 = 0; i0 < n; i0 += kSelThreads) {
    const std::uint32_t i = i0 + tid;
    const K x = i < n ? key(i) : 0;
    const bool all = ch.ties == 0xFFFFFFFFu;
    const bool over = i < n && (all ? x >= ch.least : x > ch.least), tie = i < n && !all && x == ch.least;
    const unsigned long long bo = __ballot(over), bt = __ballot(tie), below = (1ull << lane) - 1ull;
    if (lane == 0u) sh.wave[wave] = static_cast<std::uint32_t>(__popcll(bo)) << 16 | static_cast<std::uint32_t>(__popcll(bt));
    __syncthreads();
    std::uint32_t no = 0, nt = 0, total_o = 0, total_t = 0;
    for (std::uint32_t w = 0; w < kSelWaves; ++w) {
      const std::uint32_t v = sh.wave[w];
      no += w < wave ? v >> 16 : 0u, nt += w < wave ? v & 0xFFFFu : 0u;
      total_o += v >> 16, total_t += v & 0xFFFFu;
    }
    no += base_over + static_cast<std::uint32_t>(__popcll(bo & below));
    nt += base_tie + static_cast<std::uint32_t>(__popcll(bt & below));
    if (i < n) body(i, over || (tie && nt < ch.ties), no + (nt < ch.ties ? nt : ch.ties));
    base_over += total_o, base_tie += total_t;
    __syncthreads();
  }
}

__global__ __launch_bounds__(kSelThreads) void page_choice_kernel(PagedView kv, const std::uint32_t* __restrict__ pos,
                                                                  const unsigned long long* __restrict__ keys,
                                                                  std::uint32_t n_select,
                                                                  std::int32_t* __restrict__ pages) {
  __shared__ __align__(16) SelectShared sh;
  __shared__ std::uint32_t listed;
  const std::uint32_t g = blockIdx.x, r = blockIdx.y;
  const std::uint32_t used = (paged_filled(kv, pos[r]) + kv.page_size - 1u) / kv.page_size;
  if (used == 0u) return;  // a padded row
  const unsigned long long* const row = keys + (static_cast<std::size_t>(r) * kv.n_kv + g) * kv.entries;
  std::int32_t* const out = pages + (static_cast<std::size_t>(r) * kv.n_kv + g) * n_select;
  auto key = [&](std::uint32_t i) { return row[i]; };
  Choice<unsigned long long> ch = radix_choice<unsigned long long>(sh, used, n_select, key);
  if (ch.least == 0ull) ch = Choice<unsigned long long>{1ull, 0xFFFFFFFFu};  // every candidate, and no page that is not there
  if (threadIdx.x == 0u) listed = 0u;
  __syncthreads();
  for_chosen(sh, used, ch, key, [&](std::uint32_t i, bool chosen, std::uint32_t rank) {
    if (chosen && rank < n_select) out[rank] = static_cast<std::int32_t>(i);
    if (i + 1u == used) listed = rank + (chosen ? 1u : 0u);
  });
  for (std::uint32_t i = listed + threadIdx.x; i < n_select; i += kSelThreads) out[i] = -1;
}

// A weight as an unsigned key of the same order, 0 for NaN; protected slots above
// every weight.
__device__ __forceinline__ std::uint32_t weight_key(float w, std::uint32_t p, std::uint32_t newest,
                                                    std::uint32_t n_first, std::uint32_t n_recent) {
  if (p < n_first || static_cast<std::uint64_t>(p) + n_recent > newest) return 0xFFFFFFFFu;
  if (w != w) return 0u;
  const std::uint32_t b = __float_as_uint(w + 0.0f);
  return (b >> 31) != 0u ? ~b : b | 0x80000000u;
}

// The moves of one (sequence, kv head): moves[0] of them, then their destination
// and source slots in `most` places each.
struct EvictArgs {
  const std::uint32_t *length, *pos;
  const float* weight;
  const std::uint32_t* slot_pos;
  float* weight_out;
  std::uint32_t* slot_pos_out;
  std::uint32_t* moves;
  std::uint32_t keep, n_first, n_recent, most;
};

__global__ __launch_bounds__(kSelThreads) void evict_choice_kernel(PagedView kv, EvictArgs a) {
  __shared__ __align__(16) SelectShared sh;
  __shared__ std::uint32_t below;
  const std::uint32_t g = blockIdx.x, r = blockIdx.y, tid = threadIdx.x;
  const std::size_t gr = static_cast<std::size_t>(r) * kv.n_kv + g;
  std::uint32_t* const moves = a.moves + gr * (1u + 2u * static_cast<std::size_t>(a.most));
  const std::uint32_t newest = a.pos[r];
  std::uint32_t n = a.length[r];
  n = n < kv.capacity ? n : kv.capacity;
  if (newest == RTXLLM_NO_POSITION || n == 0u) {
    if (tid == 0u) moves[0] = 0u;
    return;
  }
  const float* const w = a.weight + gr * kv.capacity;
  const std::uint32_t* const p = a.slot_pos + gr * kv.capacity;
  float* const wo = a.weight_out + gr * kv.capacity;
  std::uint32_t* const po = a.slot_pos_out + gr * kv.capacity;
  const std::uint32_t stay = n < a.keep ? n : a.keep;
  if (n <= a.keep) {
    for (std::uint32_t i = tid; i < stay; i += kSelThreads) wo[i] = w[i], po[i] = p[i];
    if (tid == 0u) moves[0] = 0u;
    return;
  }
  auto key = [&](std::uint32_t i) { return weight_key(w[i], p[i], newest, a.n_first, a.n_recent); };
  const Choice<std::uint32_t> ch = radix_choice<std::uint32_t>(sh, n, a.keep, key);
  if (tid == 0u) below = 0u;
  __syncthreads();
  std::uint32_t* const to = moves + 1u;
  std::uint32_t* const from = to + a.most;
  for_chosen(sh, n, ch, key, [&](std::uint32_t i, bool chosen, std::uint32_t rank) {
    if (i < a.keep && !chosen && i - rank < a.most) to[i - rank] = i;
    if (i + 1u == a.keep) below = rank + (chosen ? 1u : 0u);
  });
  __syncthreads();
  const std::uint32_t kept_below = below, n_moves = a.keep - kept_below < a.most ? a.keep - kept_below : a.most;
  for_chosen(sh, n, ch, key, [&](std::uint32_t i, bool chosen, std::uint32_t rank) {
    if (i >= a.keep && chosen && rank - kept_below < a.most) from[rank - kept_below] = i;
  });
  if (tid == 0u) moves[0] = n_moves;
  __threadfence_block();
  __syncthreads();
  // every slot that is written lies below keep, every moved one at or behind it: in
  // place, no read meets a write of another thread
  if (wo != w)
    for (std::uint32_t i = tid; i < stay; i += kSelThreads) wo[i] = w[i];
  if (po != p)
    for (std::uint32_t i = tid; i < stay; i += kSelThreads) po[i] = p[i];
  __syncthreads();
  for (std::uint32_t m = tid; m < n_moves; m += kSelThreads) {
    wo[to[m]] = w[from[m]];
    po[to[m]] = p[from[m]];
  }
}

// L = head_dim / 8 lanes a row: 16 bytes a lane of its key and of its value.
template <int L>
__global__ __launch_bounds__(kThreads) void evict_move_kernel(PagedView kv, const std::uint32_t* moves_all,
                                                              std::uint32_t most, std::uint32_t keep,
                                                              const std::uint32_t* pos, const std::uint32_t* length,
                                                              std::uint32_t* length_out) {
  const std::uint32_t g = blockIdx.y, r = blockIdx.z;
  if (blockIdx.x == 0u && g == 0u && threadIdx.x == 0u && pos[r] != RTXLLM_NO_POSITION) {
    std::uint32_t n = length[r];
    n = n < kv.capacity ? n : kv.capacity;
    length_out[r] = n < keep ? n : keep;
  }
  const std::uint32_t* const moves =
      moves_all + (static_cast<std::size_t>(r) * kv.n_kv + g) * (1u + 2u * static_cast<std::size_t>(most));
  const std::uint32_t m = blockIdx.x * (kThreads / L) + threadIdx.x / L, t = threadIdx.x % L;
  if (m >= moves[0]) return;
  const std::int32_t* const table = kv.table + static_cast<std::size_t>(r) * kv.table_stride;
  const std::uint32_t to = paged_slot_row(kv, table, g, moves[1u + m]);
  const std::uint32_t from = paged_slot_row(kv, table, g, moves[1u + most + m]);
  if (to == kNoRow || from == kNoRow) return;
  const uint4 x = reinterpret_cast<const uint4*>(kv.k)[static_cast<std::size_t>(from) * L + t];
  const uint4 y = reinterpret_cast<const uint4*>(kv.v)[static_cast<std::size_t>(from) * L + t];
  reinterpret_cast<uint4*>(kv.k)[static_cast<std::size_t>(to) * L + t] = x;
  reinterpret_cast<uint4*>(kv.v)[static_cast<std::size_t>(to) * L + t] = y;
}

std::uint32_t most_moves(const rtxllm_paged_kv* c, std::uint32_t keep) {
  const std::uint32_t behind = c->capacity - keep;
  return keep < behind ? keep : behind;
}

}  // namespace
}  // namespace rtxllm

using namespace rtxllm;

extern "C" size_t rtxllm_attn_select_workspace(const rtxllm_paged_kv* cache, uint32_t count) {
  if (!paged_cache_ok(cache, count) || count == 0u || count > 65535u) return 0u;
  return round_256(8u * static_cast<std::size_t>(count) * cache->n_kv_heads * (cache->capacity / cache->page_size));
}

extern "C" hipError_t rtxllm_attn_select_pages(const rtxllm_paged_kv* cache, const uint16_t* bounds, const float* q,
                                               uint32_t n_heads, const uint32_t* pos, uint32_t count,
                                               uint32_t n_first, uint32_t n_last, uint32_t n_select, int32_t* pages,
                                               void* workspace, size_t workspace_bytes, hipStream_t stream) {
  const std::size_t need = rtxllm_attn_select_workspace(cache, count);
  if (need == 0u || bounds == nullptr || q == nullptr || pos == nullptr || pages == nullptr || workspace == nullptr ||
      workspace_bytes < need || n_select == 0u || n_select > 65536u ||
      static_cast<std::uint64_t>(n_first) + n_last > n_select || !aligned_to(bounds, 16u) || !aligned_to(q, 4u) ||
      !aligned_to(pos, 4u) || !aligned_to(pages, 4u) || !aligned_to(workspace, 256u))
    return hipErrorInvalidValue;
  const std::uint32_t group = paged_group(cache, n_heads);
  if (group == 0u) return hipErrorInvalidValue;
  const PagedView view = paged_view(cache);
  auto* keys = static_cast<unsigned long long*>(workspace);
  const std::uint32_t per = (kThreads / 64u) * (512u / cache->head_dim);
  const dim3 grid((view.entries + per - 1u) / per, view.n_kv, count);
  if (cache->head_dim == 64u)
    hipLaunchKernelGGL(page_score_kernel<8>, grid, dim3(kThreads), 0, stream, view, bounds, q, group, pos, n_first, n_last, keys);
  else if (cache->head_dim == 128u)
    hipLaunchKernelGGL(page_score_kernel<16>, grid, dim3(kThreads), 0, stream, view, bounds, q, group, pos, n_first, n_last, keys);
  else
    hipLaunchKernelGGL(page_score_kernel<32>, grid, dim3(kThreads), 0, stream, view, bounds, q, group, pos, n_first, n_last, keys);
  hipError_t rc = hipGetLastError();
  if (rc != hipSuccess) return rc;
  hipLaunchKernelGGL(page_choice_kernel, dim3(view.n_kv, count), dim3(kSelThreads), 0, stream, view, pos, keys, n_select, pages);
  return hipGetLastError();
}

extern "C" size_t rtxllm_kv_evict_workspace(const rtxllm_paged_kv* cache, uint32_t keep, uint32_t count) {
  if (!paged_cache_ok(cache, count) || count == 0u || count > 65535u || keep == 0u || keep > cache->capacity) return 0u;
  return round_256(4u * static_cast<std::size_t>(count) * cache->n_kv_heads *
                   (1u + 2u * static_cast<std::size_t>(most_moves(cache, keep))));
}

extern "C" hipError_t rtxllm_kv_evict_f16(const rtxllm_paged_kv* cache, const uint32_t* length, const uint32_t* pos,
                                          uint32_t count, uint32_t keep, uint32_t n_first, uint32_t n_recent,
                                          const float* weight, const uint32_t* slot_pos, float* weight_out,
                                          uint32_t* slot_pos_out, uint32_t* length_out, void* workspace,
                                          size_t workspace_bytes, hipStream_t stream) {
  const std::size_t need = rtxllm_kv_evict_workspace(cache, keep, count);
  if (need == 0u || length == nullptr || pos == nullptr || weight == nullptr || slot_pos == nullptr ||
      weight_out == nullptr || slot_pos_out == nullptr || length_out == nullptr || workspace == nullptr ||
      workspace_bytes < need || static_cast<std::uint64_t>(n_first) + n_recent > keep ||
      (cache->table_stride == 0u && count > 1u) || !aligned_to(workspace, 256u))
    return hipErrorInvalidValue;
  for (const void* p : {static_cast<const void*>(length), static_cast<const void*>(pos), static_cast<const void*>(weight),
                        static_cast<const void*>(slot_pos), static_cast<const void*>(weight_out),
                        static_cast<const void*>(slot_pos_out), static_cast<const void*>(length_out)})
    if (!aligned_to(p, 4u)) return hipErrorInvalidValue;
  // an output is one of the inputs or shares no memory with any: another workgroup
  // may still be reading
  const std::size_t n = 4u * static_cast<std::size_t>(count) * cache->n_kv_heads * cache->capacity;
  if ((weight_out != weight && overlap(weight_out, n, weight, n)) || overlap(weight_out, n, slot_pos, n) ||
      (slot_pos_out != slot_pos && overlap(slot_pos_out, n, slot_pos, n)) || overlap(slot_pos_out, n, weight, n) ||
      overlap(weight_out, n, slot_pos_out, n) || (length_out != length && overlap(length_out, 4u * count, length, 4u * count)) ||
      overlap(length_out, 4u * count, pos, 4u * count))
    return hipErrorInvalidValue;
  const PagedView view = paged_view(cache);
  const std::uint32_t most = most_moves(cache, keep), per = kThreads / (cache->head_dim / 8u);
  const EvictArgs a{length, pos, weight, slot_pos, weight_out, slot_pos_out, static_cast<std::uint32_t*>(workspace),
                    keep,   n_first, n_recent, most};
  hipLaunchKernelGGL(evict_choice_kernel, dim3(view.n_kv, count), dim3(kSelThreads), 0, stream, view, a);
  hipError_t rc = hipGetLastError();
  if (rc != hipSuccess) return rc;
  const dim3 grid(most > 0u ? (most + per - 1u) / per : 1u, view.n_kv, count);
  if (cache->head_dim == 64u)
    hipLaunchKernelGGL(evict_move_kernel<8>, grid, dim3(kThreads), 0, stream, view, a.moves, most, keep, pos, length, length_out);
  else if (cache->head_dim == 128u)
    hipLaunchKernelGGL(evict_move_kernel<16>, grid, dim3(kThreads), 0, stream, view, a.moves, most, keep, pos, length, length_out);
  else
    hipLaunchKernelGGL(evict_move_kernel<32>, grid, dim3(kThreads), 0, stream, view, a.moves, most, keep, pos, length, length_out);
  return hipGetLastError();
}
