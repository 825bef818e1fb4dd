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

typedef std::uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(4)));

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

constexpr std::uint32_t kAllTies = 0xFFFFFFFFu;
constexpr int kDigit = 11;  // bits of a pass
constexpr std::uint32_t kBins = 1u << kDigit;
static_assert(kBins == 2u * kSelThreads, "two bins a thread");

struct SelectShared {
  std::uint32_t hist[2][kBins];
  std::uint32_t wave[3][kSelWaves];
  std::uint32_t bin, above, count;
};

// Inclusive sum over the lanes below and the lane itself, by DPP.
__device__ __forceinline__ std::uint32_t wave_scan(std::uint32_t v) {
  auto add = [&](auto ctrl, auto rows) {
    v += static_cast<std::uint32_t>(
        __builtin_amdgcn_update_dpp(0, static_cast<int>(v), decltype(ctrl)::value, decltype(rows)::value, 0xF, false));
  };
  constexpr std::integral_constant<int, 0xF> all{};
  add(std::integral_constant<int, 0x111>{}, all);  // row_shr:1, 2, 4, 8
  add(std::integral_constant<int, 0x112>{}, all);
  add(std::integral_constant<int, 0x114>{}, all);
  add(std::integral_constant<int, 0x118>{}, all);
  // a row's last lane into the next row (rows 1, 3), then of row 1 into rows 2 and 3
  add(std::integral_constant<int, 0x142>{}, std::integral_constant<int, 0xA>{});
  add(std::integral_constant<int, 0x143>{}, std::integral_constant<int, 0xC>{});
  return v;
}

// Sum of the waves' words before this wave, and of all.
__device__ __forceinline__ uint2 waves_before(const std::uint32_t* words, std::uint32_t wave) {
  uint2 s = make_uint2(0u, 0u);
#pragma unroll
  for (std::uint32_t w = 0; w < kSelWaves; w += 4u) {
    const uint4 x = *reinterpret_cast<const uint4*>(words + w);
    s.x += (w < wave ? x.x : 0u) + (w + 1u < wave ? x.y : 0u) + (w + 2u < wave ? x.z : 0u) + (w + 3u < wave ? x.w : 0u);
    s.y += (x.x + x.y) + (x.z + x.w);
  }
  return s;
}

// The keys of a workgroup: a wave's part contiguous, four keys a lane and round, so
// that loads are wide and ranks follow from ballots. Up to `room` keys are read
// once and stay in the LDS, each thread's own where it alone reads them; of more,
// every pass reads all again (from the L2). The loops are rolled: each runs a few
// rounds once, and unrolled code with the keys in registers took longer to fetch
// (32 keys a thread: 92 us for 32768 keys). load(i, x): keys i..i + 3, i % 4 == 0.
template <class K, class Load>
struct Keys {
  struct alignas(16) Four {
    K k[4];
  };
  const Load& load;
  Four* held;
  std::uint32_t n, rounds, first;  // rounds of a wave, first key of its own
  bool in_lds;

  __device__ __forceinline__ Keys(const Load& l, void* lds, std::uint32_t count, std::uint32_t room)
      : load(l), held(static_cast<Four*>(lds) + threadIdx.x), n(count), in_lds(count <= room) {
    rounds = (n + 4u * kSelThreads - 1u) / (4u * kSelThreads);
    first = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) * 256u * rounds;
    if (in_lds)
      for (std::uint32_t j = 0; j < rounds && first + 256u * j < n; ++j) load(place(j), held[kSelThreads * j].k);
  }
  __device__ __forceinline__ std::uint32_t place(std::uint32_t j) const {
    return first + 256u * j + 4u * (threadIdx.x & 63u);
  }
  // body(four keys, index of the first) for each round of the wave
  template <class Body>
  __device__ __forceinline__ void each(Body body) const {
    for (std::uint32_t j = 0; j < rounds && first + 256u * j < n; ++j) {
      Four f;
      if (in_lds)
        f = held[kSelThreads * j];
      else
        load(place(j), f.k);
      body(f.k, place(j));
    }
  }
};

// Radix selection from the top, 11 bits a pass: the workgroup counts the keys that
// share the digits found so far by their next digit, and takes the digit in which
// the k-th largest lies. It ends early once all keys of that digit are wanted,
// after two or three passes where keys are spread. Lanes that all count the same
// digit (equal keys) add once, as one address takes one addition at a time.
template <class K, class Load>
__device__ Choice<K> radix_choice(SelectShared& sh, const Keys<K, Load>& keys, std::uint32_t k) {
  constexpr int kBits = static_cast<int>(8u * sizeof(K));
  const std::uint32_t tid = threadIdx.x, lane = tid & 63u, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  if (k >= keys.n) return Choice<K>{0, kAllTies};
  reinterpret_cast<uint2*>(sh.hist[0])[tid] = make_uint2(0u, 0u);
  __syncthreads();
  K prefix = 0;
  int shift = kBits;
  for (std::uint32_t turn = 0;; turn ^= 1u) {
    const int bits = shift < kDigit ? shift : kDigit, next = shift - bits;
    std::uint32_t* const hist = sh.hist[turn];
    keys.each([&](const K (&x)[4], std::uint32_t i) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const bool match = i + e < keys.n && (shift == kBits || (x[e] >> shift) == prefix);
        const std::uint32_t digit = static_cast<std::uint32_t>(x[e] >> next) & ((1u << bits) - 1u);
        const unsigned long long who = __ballot(match);
        if (who == 0ull) continue;
        const std::uint32_t one = __builtin_amdgcn_readlane(digit, static_cast<int>(__builtin_ctzll(who)));
        if (__ballot(match && digit == one) == who) {
          if (lane == 0u) atomicAdd(&hist[one], static_cast<std::uint32_t>(__popcll(who)));
        } else if (match) {
          atomicAdd(&hist[digit], 1u);
        }
      }
    });
    __syncthreads();
    // thread t: bins 2047 - 2 t and 2046 - 2 t, sums from the largest digit down
    const uint2 c = reinterpret_cast<const uint2*>(hist)[kSelThreads - 1u - tid];
    reinterpret_cast<uint2*>(sh.hist[turn ^ 1u])[tid] = make_uint2(0u, 0u);
    const std::uint32_t sum = wave_scan(c.x + c.y);
    if (lane == 63u) sh.wave[0][wave] = sum;
    __syncthreads();
    const std::uint32_t before = waves_before(sh.wave[0], wave).x + sum - (c.x + c.y);
    if (before < k && k <= before + c.x + c.y) {
      const bool upper = k <= before + c.y;
      sh.bin = 2u * (kSelThreads - 1u - tid) + (upper ? 1u : 0u);
      sh.above = upper ? before : before + c.y;
      sh.count = upper ? c.y : c.x;
    }
    __syncthreads();
    prefix = (prefix << bits) | static_cast<K>(sh.bin);
    k -= sh.above;
    shift = next;
    if (sh.count == k) return Choice<K>{static_cast<K>(prefix << shift), kAllTies};
    if (shift == 0) return Choice<K>{prefix, k};
  }
}

// Walks the keys in two classes: kind(i, chosen) is 0 (neither), 1 or 2, put(kind, i,
// rank) gets a place of a class with the number of those of the class before it.
// Returns the sizes of both.
template <class K, class Load, class Kind, class Put>
__device__ uint2 for_chosen(SelectShared& sh, const Keys<K, Load>& keys, const Choice<K>& ch, Kind kind, Put put) {
  const std::uint32_t tid = threadIdx.x, lane = tid & 63u, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const unsigned long long below = (1ull << lane) - 1ull;
  const bool all = ch.ties == kAllTies;
  std::uint32_t ties_before = 0;
  if (!all) {
    std::uint32_t mine = 0;
    keys.each([&](const K (&x)[4], std::uint32_t i) {
#pragma unroll
      for (int e = 0; e < 4; ++e) mine += static_cast<std::uint32_t>(__popcll(__ballot(i + e < keys.n && x[e] == ch.least)));
    });
    if (lane == 0u) sh.wave[0][wave] = mine;
    __syncthreads();
    ties_before = waves_before(sh.wave[0], wave).x;
  }
  // the classes of a round's four places, 2 bits each; `ties`: equal keys before the round
  auto classes = [&](const K (&x)[4], std::uint32_t i, std::uint32_t& ties) {
    std::uint32_t c = 0u;
    unsigned long long tie[4];
    std::uint32_t at = ties;
    if (!all) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        tie[e] = __ballot(i + e < keys.n && x[e] == ch.least);
        at += static_cast<std::uint32_t>(__popcll(tie[e] & below));
        ties += static_cast<std::uint32_t>(__popcll(tie[e]));
      }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      bool chosen = x[e] >= ch.least;
      if (!all && x[e] == ch.least) chosen = at++ < ch.ties;
      c |= i + e < keys.n ? static_cast<std::uint32_t>(kind(i + e, chosen)) << (2 * e) : 0u;
    }
    return c;
  };
  std::uint32_t n1 = 0, n2 = 0, ties = ties_before;
  keys.each([&](const K (&x)[4], std::uint32_t i) {
    const std::uint32_t c = classes(x, i, ties);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      n1 += static_cast<std::uint32_t>(__popcll(__ballot((c >> (2 * e) & 3u) == 1u)));
      n2 += static_cast<std::uint32_t>(__popcll(__ballot((c >> (2 * e) & 3u) == 2u)));
    }
  });
  if (lane == 0u) sh.wave[1][wave] = n1, sh.wave[2][wave] = n2;
  __syncthreads();
  const uint2 w1 = waves_before(sh.wave[1], wave), w2 = waves_before(sh.wave[2], wave);
  std::uint32_t at1 = w1.x, at2 = w2.x;
  ties = ties_before;
  keys.each([&](const K (&x)[4], std::uint32_t i) {
    const std::uint32_t c = classes(x, i, ties);
    std::uint32_t r1 = at1, r2 = at2;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const unsigned long long b1 = __ballot((c >> (2 * e) & 3u) == 1u), b2 = __ballot((c >> (2 * e) & 3u) == 2u);
      r1 += static_cast<std::uint32_t>(__popcll(b1 & below)), at1 += static_cast<std::uint32_t>(__popcll(b1));
      r2 += static_cast<std::uint32_t>(__popcll(b2 & below)), at2 += static_cast<std::uint32_t>(__popcll(b2));
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const std::uint32_t k = c >> (2 * e) & 3u;
      if (k == 1u) put(1, i + e, r1++);
      if (k == 2u) put(2, i + e, r2++);
    }
  });
  return make_uint2(w1.y, w2.y);
}

// LDS bytes for n keys of `width` bytes, up to 128 KB, in whole rounds of a workgroup.
std::size_t held_bytes(std::uint32_t n, std::size_t width) {
  const std::size_t round = 4u * kSelThreads * width, rounds = (n * width + round - 1u) / round;
  return round * rounds < (128u << 10) ? round * rounds : 128u << 10;
}

typedef unsigned long long u64x4 __attribute__((ext_vector_type(4), aligned(8)));

__global__ __launch_bounds__(kSelThreads) void page_choice_kernel(PagedView kv, const std::uint32_t* __restrict__ pos,
                                                                  const unsigned long long* __restrict__ row_keys,
                                                                  std::uint32_t room, std::uint32_t n_select,
                                                                  std::int32_t* __restrict__ pages) {
  __shared__ __align__(16) SelectShared sh;
  extern __shared__ __align__(16) std::uint8_t lds[];
  const std::uint32_t g = blockIdx.x, r = blockIdx.y;
  const std::uint32_t used = (paged_filled(kv, pos[r]) + kv.page_size - 1u) / kv.page_size;
  if (used == 0u) return;  // a padded row
  const unsigned long long* const row = row_keys + (static_cast<std::size_t>(r) * kv.n_kv + g) * kv.entries;
  std::int32_t* const out = pages + (static_cast<std::size_t>(r) * kv.n_kv + g) * n_select;
  auto load = [&](std::uint32_t i, unsigned long long (&x)[4]) {
    if (i + 4u <= used) {
      const u64x4 v = *reinterpret_cast<const u64x4*>(row + i);
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = v[e];
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = i + e < used ? row[i + e] : 0ull;
    }
  };
  const Keys<unsigned long long, decltype(load)> keys(load, lds, used, room);
  Choice<unsigned long long> ch = radix_choice(sh, keys, n_select);
  if (ch.least == 0ull) ch = Choice<unsigned long long>{1ull, kAllTies};  // every candidate, and no page that is not there
  const std::uint32_t listed = for_chosen(
      sh, keys, ch, [](std::uint32_t, bool chosen) { return chosen ? 1 : 0; },
      [&](int, std::uint32_t i, std::uint32_t rank) {
        if (rank < n_select) out[rank] = static_cast<std::int32_t>(i);
      }).x;
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
  std::uint32_t keep, n_first, n_recent, most, room;
};

__global__ __launch_bounds__(kSelThreads) void evict_choice_kernel(PagedView kv, EvictArgs a) {
  __shared__ __align__(16) SelectShared sh;
  extern __shared__ __align__(16) std::uint8_t lds[];
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
  auto load = [&](std::uint32_t i, std::uint32_t (&x)[4]) {
    f32x4_any wv = {0.0f, 0.0f, 0.0f, 0.0f};
    u32x4_any pv = {0u, 0u, 0u, 0u};
    if (i + 4u <= n) {
      wv = *reinterpret_cast<const f32x4_any*>(w + i);
      pv = *reinterpret_cast<const u32x4_any*>(p + i);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (i + e < n) wv[e] = w[i + e], pv[e] = p[i + e];
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = weight_key(wv[e], pv[e], newest, a.n_first, a.n_recent);
  };
  const Keys<std::uint32_t, decltype(load)> keys(load, lds, n, a.room);
  const Choice<std::uint32_t> ch = radix_choice(sh, keys, a.keep);
  std::uint32_t* const to = moves + 1u;
  std::uint32_t* const from = to + a.most;
  const std::uint32_t holes = for_chosen(
      sh, keys, ch,
      [&](std::uint32_t i, bool chosen) { return i < a.keep ? (chosen ? 0 : 1) : (chosen ? 2 : 0); },
      [&](int kind, std::uint32_t i, std::uint32_t m) {
        if (m < a.most) (kind == 1 ? to : from)[m] = i;
      }).x;
  const std::uint32_t n_moves = holes < a.most ? holes : a.most;
  if (tid == 0u) moves[0] = n_moves;
  // every slot that is written lies below keep, every moved one at or behind it: in
  // place, no read meets a write of another thread
  if (wo != w)
    for (std::uint32_t i = tid; i < stay; i += kSelThreads) wo[i] = w[i];
  if (po != p)
    for (std::uint32_t i = tid; i < stay; i += kSelThreads) po[i] = p[i];
  __threadfence_block();
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
  const std::size_t held = held_bytes(view.entries, 8u);
  hipLaunchKernelGGL(page_choice_kernel, dim3(view.n_kv, count), dim3(kSelThreads), held, stream, view, pos, keys,
                     static_cast<std::uint32_t>(held / 8u), n_select, pages);
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
  const std::size_t held = held_bytes(view.capacity, 4u);
  const EvictArgs a{length, pos, weight, slot_pos, weight_out, slot_pos_out, static_cast<std::uint32_t*>(workspace),
                    keep,   n_first, n_recent, most, static_cast<std::uint32_t>(held / 4u)};
  hipLaunchKernelGGL(evict_choice_kernel, dim3(view.n_kv, count), dim3(kSelThreads), held, stream, view, a);
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
