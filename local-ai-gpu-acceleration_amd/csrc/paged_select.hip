// The two choices over a paged cache: the pages worth attending, and the slots
// worth keeping. Both rank up to some ten thousand keys per (sequence, kv head) and
// take the best k of them, the lower index between equals: a radix selection in
// one workgroup, exact in every bit of the keys.
#include <type_traits>

#include "common.h"
#include "layer_common.cuh"
#include "paged.h"

namespace rtxllm {
namespace {

constexpr std::uint32_t kThreads = 256;

typedef std::uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(4)));

// lane_xor of a 64-bit value.
template <int M>
__device__ __forceinline__ double lane_xor_d(double v) {
  const uint2 u = __builtin_bit_cast(uint2, v);
  return __builtin_bit_cast(double, make_uint2(__float_as_uint(lane_xor<M>(__uint_as_float(u.x))),
                                               __float_as_uint(lane_xor<M>(__uint_as_float(u.y)))));
}

// A score as an unsigned key of the same order: 1 for NaN, so that 0 is left for
// "no candidate".
__device__ __forceinline__ unsigned long long score_key(double s) {
  if (s != s) return 1ull;
  const unsigned long long b = __builtin_bit_cast(unsigned long long, s + 0.0);  // -0 -> +0
  return (b >> 63) != 0ull ? ~b : b | (1ull << 63);
}

// Keys of the pages of one (row, kv head): a wave scores kSteps times 64 / L pages, L =
// head_dim / 8 lanes a page, 8 dimensions a lane. max(q hi, q lo) is q times the larger
// extreme where q >= 0, the smaller one where it is not: chosen by the sign, two dimensions
// at a time as fp16 pairs, so that the other extreme enters nothing (with an infinite q it would
// make a NaN, and equal scores would differ by the roundings of what cancels). Products of fp32 and fp16 values are exact in 64 bits; their sums take one
// order for every page. Four heads at a time: two halving exchanges
// leave each lane one head's part, so that four heads take one head's further steps.
// What bounds it is the chain of reads (table and q, then bounds): the position is
// needed last, a wave's table entries are one load, and the next step's bounds are
// read before this step's sums.
template <int L, int kSteps>
__global__ __launch_bounds__(kThreads) void page_score_kernel(PagedView kv, const std::uint16_t* __restrict__ bounds,
                                                              const float* __restrict__ q, std::uint32_t group,
                                                              const std::uint32_t* __restrict__ pos,
                                                              std::uint32_t n_first, std::uint32_t n_last,
                                                              unsigned long long* __restrict__ keys) {
  constexpr std::uint32_t D = 8u * L, kPages = 64u / L, kOwn = kPages * kSteps;
  static_assert(kOwn <= 64u, "a lane a page of the wave");
  typedef _Float16 half2 __attribute__((ext_vector_type(2)));
  typedef _Float16 half8 __attribute__((ext_vector_type(8)));
  typedef short short2_t __attribute__((ext_vector_type(2)));
  typedef std::uint32_t u32x4 __attribute__((ext_vector_type(4)));
  const std::uint32_t g = blockIdx.y, r = blockIdx.z, lane = threadIdx.x & 63u, t = lane % L;
  const std::size_t gr = static_cast<std::size_t>(r) * kv.n_kv + g;
  // step s of a wave lies s * stride pages on: where few pages are filled, waves take a step each
  const std::uint32_t p0 = __builtin_amdgcn_readfirstlane(blockIdx.x * (kThreads / 64u) + (threadIdx.x >> 6)) * kPages;
  const std::uint32_t stride = gridDim.x * (kThreads / 64u) * kPages;
  if (p0 >= kv.entries) return;
  const std::uint32_t mine = p0 + lane % kOwn / kPages * stride + lane % kPages;
  const std::int32_t entry =
      kv.table[static_cast<std::size_t>(r) * kv.table_stride + (mine < kv.entries ? mine : kv.entries - 1u)];
  const std::uint32_t filled = paged_filled(kv, pos[r]), used = (filled + kv.page_size - 1u) / kv.page_size;
  const float* const qr = q + gr * group * D + 8u * t;
  double qd[4][8];
  std::uint32_t below[4][4];  // all ones in the half of a dimension whose q is below 0
  auto load_q = [&](std::uint32_t h0) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const std::uint32_t h = h0 + k < group ? h0 + k : group - 1u;  // a head twice changes no maximum
      const f32x4_any a = *reinterpret_cast<const f32x4_any*>(qr + h * D), b = *reinterpret_cast<const f32x4_any*>(qr + h * D + 4u);
#pragma unroll
      for (int i = 0; i < 8; ++i) qd[k][i] = static_cast<double>(i < 4 ? a[i & 3] : b[i & 3]);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const f32x4_any& v = i < 2 ? a : b;
        const short2_t top = {static_cast<short>(__float_as_uint(v[2 * i & 3]) >> 16),
                              static_cast<short>(__float_as_uint(v[(2 * i & 3) + 1]) >> 16)};
        below[k][i] = __builtin_bit_cast(std::uint32_t, top >> static_cast<short>(15));
      }
    }
  };
  half8 hi[2], lo[2];
  bool there[2];
  auto load_bounds = [&](int s) {
    const std::int32_t page = __shfl(entry, static_cast<int>(kPages * s + lane / L), 64);
    there[s & 1] = static_cast<std::uint32_t>(page) < kv.n_pages;
    const half8* b = reinterpret_cast<const half8*>(
                         bounds + (static_cast<std::size_t>(there[s & 1] ? page : 0) * kv.n_kv + g) * 2u * D) + t;
    hi[s & 1] = b[0], lo[s & 1] = b[L];
  };
  if (p0 >= used) return;
  load_bounds(0);
  load_q(0u);
  const bool odd = (lane & 1u) != 0u, odd2 = (lane & 2u) != 0u;
#pragma unroll
  for (int s = 0; s < kSteps; ++s) {
    if (p0 + stride * s >= used) break;
    if (s + 1 < kSteps) load_bounds(s + 1);
    double best = __builtin_nan("");
    // (a page of NaN keys alone has them in reverse order)
    const u32x4 large = __builtin_bit_cast(u32x4, __builtin_elementwise_max(hi[s & 1], lo[s & 1]));
    const u32x4 small = __builtin_bit_cast(u32x4, __builtin_elementwise_min(hi[s & 1], lo[s & 1]));
    for (std::uint32_t h0 = 0; h0 < group; h0 += 4u) {
      if (group > 4u) load_q(h0);
      double sum[4] = {0.0, 0.0, 0.0, 0.0};
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const half2 x = __builtin_bit_cast(half2, (below[k][i] & small[i]) | (~below[k][i] & large[i]));
          sum[k] = fma(qd[k][2 * i], static_cast<double>(static_cast<float>(x[0])), sum[k]);
          sum[k] = fma(qd[k][2 * i + 1], static_cast<double>(static_cast<float>(x[1])), sum[k]);
        }
      const double x0 = odd ? sum[2] : sum[0], x1 = odd ? sum[3] : sum[1];
      const double y0 = odd ? sum[0] : sum[2], y1 = odd ? sum[1] : sum[3];
      const double v0 = x0 + lane_xor_d<1>(y0), v1 = x1 + lane_xor_d<1>(y1);
      double v = (odd2 ? v1 : v0) + lane_xor_d<2>(odd2 ? v0 : v1);
      v += lane_xor_d<4>(v);
      if constexpr (L > 8) v += lane_xor_d<8>(v);
      if constexpr (L > 16) v += lane_xor_d<16>(v);
      v = fmax(v, lane_xor_d<1>(v));  // fmax: a head's NaN gives way to a number
      best = fmax(best, fmax(v, lane_xor_d<2>(v)));
    }
    const std::uint32_t p = p0 + stride * s + lane / L;
    const bool forced = p < n_first || p + n_last >= used;
    if (t == 0u && p < used) keys[gr * kv.entries + p] = !there[s & 1] ? 0ull : forced ? ~0ull : score_key(best);
  }
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

template <std::uint32_t T>  // threads
struct SelectShared {
  std::uint32_t hist[2][kBins];
  std::uint32_t wave[3][T / 64u];
  std::uint32_t bin, above, count;
};

// Inclusive sum over the lanes below and the lane itself (of its row of 16), by DPP.
template <int LANES = 64>
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
  if constexpr (LANES == 16) return v;
  // a row's last lane into the next row (rows 1, 3), then of row 1 into rows 2 and 3
  add(std::integral_constant<int, 0x142>{}, std::integral_constant<int, 0xA>{});
  add(std::integral_constant<int, 0x143>{}, std::integral_constant<int, 0xC>{});
  return v;
}

// Lanes of a mask below this one.
__device__ __forceinline__ std::uint32_t lanes_below(unsigned long long mask) {
  return __builtin_amdgcn_mbcnt_hi(static_cast<std::uint32_t>(mask >> 32),
                                   __builtin_amdgcn_mbcnt_lo(static_cast<std::uint32_t>(mask), 0u));
}

// Sum of the waves' words before this wave, and of all: a lane a wave (at most 16, one
// row of lanes), every wave for itself.
template <std::uint32_t T>
__device__ __forceinline__ uint2 waves_before(const std::uint32_t (&words)[T / 64u], std::uint32_t wave) {
  constexpr std::uint32_t kWaves = T / 64u;
  const std::uint32_t lane = threadIdx.x & 63u;
  const std::uint32_t own = lane < kWaves ? words[lane] : 0u, sum = wave_scan<16>(own);
  return make_uint2(__builtin_amdgcn_readlane(sum - own, wave), __builtin_amdgcn_readlane(sum, kWaves - 1u));
}

// Counts four keys a lane by a digit, those that match.
template <class Digit>
__device__ __forceinline__ void count_digits(std::uint32_t* hist, Digit digit_of) {
  std::uint32_t digit[4], others = 0u;  // kBins: no match
#pragma unroll
  for (int e = 0; e < 4; ++e) digit[e] = digit_of(e);
  const std::uint32_t one = __builtin_amdgcn_readfirstlane(digit[0]);
#pragma unroll
  for (int e = 0; e < 4; ++e) others |= digit[e] ^ one;
  if (__ballot(others != 0u) == 0ull) {
    if ((threadIdx.x & 63u) == 0u && one != kBins) atomicAdd(&hist[one], 256u);
    return;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (digit[e] != kBins) atomicAdd(&hist[digit[e]], 1u);
}

// The keys of a workgroup: a wave's part contiguous, four keys a lane and round, so
// that loads are wide and ranks follow from ballots; 0 behind the last key. Up to
// `room` keys are read once and stay in the LDS, each thread's own where it alone
// reads them; of more, every pass reads all again (from the L2). The loops over them are
// rolled: each runs a few rounds once, and unrolled code with the keys in registers
// took longer to fetch (32 keys a thread: 92 us for 32768 keys). src.raw(i) loads what
// keys i..i + 3 (i % 4 == 0) are made of, src.keys(i, raw, x) makes them (<true>: all four
// are there), src.seen(i, raw) is called for each once, where they go into the LDS;
// src.begin() comes before all of them, behind a barrier.
template <class K, class Source, std::uint32_t T>
struct Keys {
  struct alignas(16) Four {
    K k[4];
  };
  Source& src;
  Four* held;
  std::uint32_t n, rounds, first;  // rounds of this wave, its first key
  bool in_lds;

  // `hist` gets the counts of the keys' first digit where they are read into the LDS.
  __device__ __forceinline__ Keys(Source& s, void* lds, std::uint32_t* hist, std::uint32_t count, std::uint32_t room)
      : src(s), held(static_cast<Four*>(lds) + threadIdx.x), n(count), in_lds(count <= room) {
    const std::uint32_t most = (n + 4u * T - 1u) / (4u * T);
    first = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) * 256u * most;
    const std::uint32_t own = first < n ? (n - first + 255u) / 256u : 0u;
    rounds = own < most ? own : most;
    for (std::uint32_t i = 4u * threadIdx.x; i < kBins; i += 4u * T)
      *reinterpret_cast<uint4*>(hist + i) = make_uint4(0u, 0u, 0u, 0u);
    __syncthreads();
    src.begin();
    if (!in_lds) return;
    using Raw = decltype(src.template raw<true>(0u));
    auto take = [&](auto full, std::uint32_t round, const Raw& v) {
      const std::uint32_t at = place(round);
      Four f;
      src.seen(at, v);
      src.template keys<decltype(full)::value>(at, v, f.k);
      held[T * round] = f;
      count_digits(hist, [&](int e) { return static_cast<std::uint32_t>(f.k[e] >> (8 * sizeof(K) - kDigit)); });
    };
    std::uint32_t j = 0;
    for (; j + 4u <= rounds && first + 256u * (j + 4u) <= n; j += 4u) {  // four rounds' loads in flight
      Raw v[4];
#pragma unroll
      for (std::uint32_t u = 0; u < 4u; ++u) v[u] = src.template raw<true>(place(j + u));
#pragma unroll
      for (std::uint32_t u = 0; u < 4u; ++u) take(std::true_type{}, j + u, v[u]);
    }
    for (; j < rounds; ++j) take(std::false_type{}, j, src.template raw<false>(place(j)));
  }
  __device__ __forceinline__ std::uint32_t place(std::uint32_t j) const {
    return first + 256u * j + 4u * (threadIdx.x & 63u);
  }
  // body(four keys, index of the first) for each round of the wave
  template <class Body>
  __device__ __forceinline__ void each(Body body) const {
    for (std::uint32_t j = 0; j < rounds; ++j) {
      Four f;
      if (in_lds)
        f = held[T * j];
      else
        src.template keys<false>(place(j), src.template raw<false>(place(j)), f.k);
      body(f.k, place(j));
    }
  }
};

// Radix selection from the top, 11 bits a pass: the workgroup counts the keys that
// share the digits found so far by their next digit, and takes the digit in which
// the k-th largest lies. It ends early once all keys of that digit are wanted,
// after two or three passes where keys are spread. 256 keys of one digit are one
// addition, as an address takes one at a time (equal weights, protected slots). k is at
// most the number of keys: the zeros behind the last one are never among the best,
// since of equal keys the first count.
template <class K, class Source, std::uint32_t T>
__device__ Choice<K> radix_choice(SelectShared<T>& sh, const Keys<K, Source, T>& keys, std::uint32_t k) {
  constexpr int kBits = static_cast<int>(8u * sizeof(K));
  const std::uint32_t tid = threadIdx.x, lane = tid & 63u, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  K prefix = 0;
  int shift = kBits;
  for (std::uint32_t turn = 0;; turn ^= 1u) {
    const int bits = shift < kDigit ? shift : kDigit, next = shift - bits;
    std::uint32_t* const hist = sh.hist[turn];
    if (shift < kBits || !keys.in_lds)
      keys.each([&](const K (&x)[4], std::uint32_t) {
        count_digits(hist, [&](int e) {
          const bool match = shift == kBits || (x[e] >> shift) == prefix;
          return match ? static_cast<std::uint32_t>(x[e] >> next) & ((1u << bits) - 1u) : kBins;
        });
      });
    __syncthreads();
    if (wave == 0u) {
      // lane l sums the 32 bins below 2048 - 32 l; in the lane whose sums pass k, the bins
      // again, one a lane, from the largest digit down
      constexpr std::uint32_t kOwn = kBins / 64u;
      const uint4* own = reinterpret_cast<const uint4*>(hist + kBins - kOwn * (lane + 1u));
      std::uint32_t mine = 0;
#pragma unroll
      for (std::uint32_t i = 0; i < kOwn / 4u; ++i) {
        const uint4 v = own[(i + lane) % (kOwn / 4u)];  // turned by the lane: no two of eight in one bank
        mine += (v.x + v.y) + (v.z + v.w);
      }
      const std::uint32_t upto = wave_scan(mine);
      const auto l = static_cast<std::uint32_t>(__builtin_ctzll(__ballot(upto >= k)));
      const std::uint32_t before = __builtin_amdgcn_readlane(upto - mine, l);
      const std::uint32_t bin = kBins - kOwn * l - 1u - (lane & (kOwn - 1u));
      const std::uint32_t c = lane < kOwn ? hist[bin] : 0u, sum = before + wave_scan(c);
      if (lane == static_cast<std::uint32_t>(__builtin_ctzll(__ballot(sum >= k)))) {
        sh.bin = bin;
        sh.above = sum - c;
        sh.count = c;
      }
    } else {
      for (std::uint32_t i = 4u * (tid - 64u); i < kBins; i += 4u * (T - 64u))
        *reinterpret_cast<uint4*>(&sh.hist[turn ^ 1u][i]) = make_uint4(0u, 0u, 0u, 0u);
    }
    __syncthreads();
    prefix = (prefix << bits) | static_cast<K>(sh.bin);
    k -= sh.above;
    shift = next;
    if (sh.count == k) return Choice<K>{static_cast<K>(prefix << shift), kAllTies};
    if (shift == 0) return Choice<K>{prefix, k};
  }
}

// A list of indices, `most` at most (a round that would pass them, which keys that change
// meanwhile could make, is dropped whole).
struct Places {
  std::uint32_t* to;
  std::uint32_t most;
};

// Walks the choice: the keys below `split` that are not chosen go into `freed`, the chosen ones
// at or behind it into `kept`, both in order. Returns the number of both.
template <class K, class Source, std::uint32_t T>
__device__ uint2 for_choice(SelectShared<T>& sh, const Keys<K, Source, T>& keys, const Choice<K>& ch, std::uint32_t split,
                            Places freed, Places kept) {
  const std::uint32_t tid = threadIdx.x, lane = tid & 63u, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const bool all = ch.ties == kAllTies;
  std::uint32_t ties_before = 0;
  if (!all) {
    std::uint32_t mine = 0;
    keys.each([&](const K (&x)[4], std::uint32_t) {
#pragma unroll
      for (int e = 0; e < 4; ++e) mine += static_cast<std::uint32_t>(__popcll(__ballot(x[e] == ch.least)));
    });
    if (lane == 0u) sh.wave[0][wave] = mine;
    __syncthreads();
    ties_before = waves_before<T>(sh.wave[0], wave).x;
  }
  // a lane's four places of either kind, a bit each; `ties`: equal keys before the round
  struct Kinds {
    std::uint32_t freed, kept;
  };
  auto kinds = [&](const K (&x)[4], std::uint32_t i, std::uint32_t& ties) {
    std::uint32_t chosen = 0u;
    if (all) {
#pragma unroll
      for (int e = 0; e < 4; ++e) chosen |= x[e] >= ch.least ? 1u << e : 0u;
    } else {
      std::uint32_t at = ties;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const unsigned long long b = __ballot(x[e] == ch.least);
        at += lanes_below(b);
        ties += static_cast<std::uint32_t>(__popcll(b));
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) chosen |= x[e] > ch.least || (x[e] == ch.least && at++ < ch.ties) ? 1u << e : 0u;
    }
    const std::uint32_t low = i >= split ? 0u : split - i >= 4u ? 15u : (1u << (split - i)) - 1u;
    return Kinds{low & ~chosen, chosen & ~low};
  };
  std::uint32_t nf = 0, nk = 0, ties = ties_before;  // of the lane
  keys.each([&](const K (&x)[4], std::uint32_t i) {
    const Kinds s = kinds(x, i, ties);
    nf += static_cast<std::uint32_t>(__popc(s.freed));
    nk += static_cast<std::uint32_t>(__popc(s.kept));
  });
  const std::uint32_t sum_f = wave_scan(nf), sum_k = wave_scan(nk);
  if (lane == 63u) sh.wave[1][wave] = sum_f, sh.wave[2][wave] = sum_k;
  __syncthreads();
  const uint2 wf = waves_before<T>(sh.wave[1], wave), wk = waves_before<T>(sh.wave[2], wave);
  std::uint32_t at_f = wf.x, at_k = wk.x;
  ties = ties_before;
  auto put = [&](std::uint32_t bits, std::uint32_t i, std::uint32_t& at, const Places& list) {
    if (__ballot(bits != 0u) == 0ull) return;
    const std::uint32_t own = static_cast<std::uint32_t>(__popc(bits)), upto = wave_scan(own);
    std::uint32_t rank = at + upto - own;
    at += __builtin_amdgcn_readlane(upto, 63);
    if (at > list.most) return;
#pragma unroll
    for (std::uint32_t e = 0; e < 4u; ++e)
      if ((bits >> e & 1u) != 0u) list.to[rank++] = i + e;
  };
  keys.each([&](const K (&x)[4], std::uint32_t i) {
    const Kinds s = kinds(x, i, ties);
    put(s.freed, i, at_f, freed);
    put(s.kept, i, at_k, kept);
  });
  return make_uint2(wf.y, wk.y);
}

// LDS bytes for n keys of `width` bytes, up to 128 KB, in whole rounds of a workgroup.
std::size_t held_bytes(std::uint32_t n, std::size_t width, std::uint32_t threads) {
  const std::size_t round = 4u * threads * width, rounds = (n * width + round - 1u) / round;
  return round * rounds < (128u << 10) ? round * rounds : 128u << 10;
}

typedef unsigned long long u64x4 __attribute__((ext_vector_type(4), aligned(8)));

struct KeyRow {
  const unsigned long long* row;
  std::uint32_t n;
  template <bool FULL>
  __device__ __forceinline__ u64x4 raw(std::uint32_t i) const {
    u64x4 v = {0ull, 0ull, 0ull, 0ull};
    if (FULL || i + 4u <= n) {
      v = *reinterpret_cast<const u64x4*>(row + i);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (i + e < n) v[e] = row[i + e];
    }
    return v;
  }
  __device__ __forceinline__ void begin() const {}
  __device__ __forceinline__ void seen(std::uint32_t, const u64x4&) const {}
  template <bool>
  __device__ __forceinline__ void keys(std::uint32_t, const u64x4& v, unsigned long long (&x)[4]) const {
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = v[e];
  }
};

template <std::uint32_t T>
__global__ __launch_bounds__(T) void page_choice_kernel(PagedView kv, const std::uint32_t* __restrict__ pos,
                                                        const unsigned long long* __restrict__ row_keys,
                                                        std::uint32_t room, std::uint32_t n_select,
                                                        std::int32_t* __restrict__ pages) {
  __shared__ __align__(16) SelectShared<T> sh;
  extern __shared__ __align__(16) std::uint8_t lds[];
  const std::uint32_t g = blockIdx.x, r = blockIdx.y;
  const std::uint32_t used = (paged_filled(kv, pos[r]) + kv.page_size - 1u) / kv.page_size;
  if (used == 0u) return;  // a padded row
  const std::size_t gr = static_cast<std::size_t>(r) * kv.n_kv + g;
  KeyRow src{row_keys + gr * kv.entries, used};
  const Keys<unsigned long long, KeyRow, T> keys(src, lds, sh.hist[0], used, room);
  std::int32_t* const out = pages + gr * n_select;
  // 1 and more: every page that is there
  Choice<unsigned long long> ch{1ull, kAllTies};
  if (n_select < used) ch = radix_choice(sh, keys, n_select);
  if (ch.least == 0ull) ch = Choice<unsigned long long>{1ull, kAllTies};
  const std::uint32_t listed =
      for_choice(sh, keys, ch, 0u, Places{nullptr, 0u}, Places{reinterpret_cast<std::uint32_t*>(out), n_select}).y;
  for (std::uint32_t i = listed + threadIdx.x; i < n_select; i += T) out[i] = -1;
}

// A weight as an unsigned key of the same order, 1 for NaN; protected slots above every
// weight. 0 and kStays are left for slots in no page (SlotKeys). The positions from n_first on
// that are not protected are `open` many.
constexpr std::uint32_t kStays = 0xFFFFFFFFu;
__device__ __forceinline__ std::uint32_t weight_key(float w, std::uint32_t p, std::uint32_t n_first, std::uint32_t open) {
  const std::uint32_t b = __float_as_uint(w + 0.0f);
  const std::uint32_t key = b ^ (static_cast<std::uint32_t>(static_cast<std::int32_t>(b) >> 31) | 0x80000000u);
  return p - n_first >= open ? kStays - 1u : w != w ? 1u : key;
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

// A slot in no page holds no key or value that could move, and takes none: below keep it
// stays whatever it weighs, behind it it leaves. (There are enough others: those below keep
// alone make up the number.) Such slots are looked for once, in the table.
struct SlotKeys {
  const float* w;
  const std::uint32_t* p;
  float* wo;
  std::uint32_t* po;
  std::uint32_t n, stay, n_first, open;
  const PagedView& kv;
  const std::int32_t* table;
  const std::uint32_t* wave_holes;  // in the LDS: whether a wave has found one
  std::uint32_t waves;
  bool holes;
  __device__ __forceinline__ void begin() {
    const std::uint32_t lane = threadIdx.x & 63u;
    holes = __ballot(lane < waves && wave_holes[lane] != 0u) != 0ull;
  }
  struct Raw {
    f32x4_any w;
    u32x4_any p;
  };
  template <bool FULL>
  __device__ __forceinline__ Raw raw(std::uint32_t i) const {
    Raw v{{0.0f, 0.0f, 0.0f, 0.0f}, {0u, 0u, 0u, 0u}};
    if (FULL || i + 4u <= n) {
      v.w = *reinterpret_cast<const f32x4_any*>(w + i);
      v.p = *reinterpret_cast<const u32x4_any*>(p + i);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (i + e < n) v.w[e] = w[i + e], v.p[e] = p[i + e];
    }
    return v;
  }
  template <bool FULL>
  __device__ __forceinline__ void keys(std::uint32_t i, const Raw& v, std::uint32_t (&x)[4]) const {
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = weight_key(v.w[e], v.p[e], n_first, open);
    if (holes) {
#pragma unroll
      for (std::uint32_t e = 0; e < 4u; ++e)
        if (i + e < n && static_cast<std::uint32_t>(table[page_of(kv, i + e)]) >= kv.n_pages) x[e] = i + e < stay ? kStays : 0u;
    }
    if (FULL || __ballot(i + 4u > n) == 0ull) return;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (i + e >= n) x[e] = 0u;
  }
  // copies the slots below `stay`, unless they lie there already
  __device__ __forceinline__ void seen(std::uint32_t i, const Raw& v) const {
    if (__ballot(i < stay) == 0ull) return;
    if (i + 4u <= stay) {
      if (wo != w) *reinterpret_cast<f32x4_any*>(wo + i) = v.w;
      if (po != p) *reinterpret_cast<u32x4_any*>(po + i) = v.p;
    } else {
#pragma unroll
      for (std::uint32_t e = 0; e < 4u; ++e)
        if (i + e < stay) wo[i + e] = v.w[e], po[i + e] = v.p[e];
    }
  }
};

// One move: the row's key and value by L = head_dim / 8 lanes, 16 bytes each of
// both, its weight and position by the first two of them. Every slot that is written
// lies below keep, every moved one at or behind it: no read meets a write.
template <int L>
__device__ __forceinline__ void move_row(const PagedView& kv, const EvictArgs& a, std::uint32_t r, std::uint32_t g,
                                         std::uint32_t to_slot, std::uint32_t from_slot, std::uint32_t t) {
  if (to_slot >= kv.capacity || from_slot >= kv.capacity) return;  // (weights that changed meanwhile)
  const std::int32_t* const table = kv.table + static_cast<std::size_t>(r) * kv.table_stride;
  const std::size_t state = (static_cast<std::size_t>(r) * kv.n_kv + g) * kv.capacity;
  const std::uint32_t to = paged_slot_row(kv, table, g, to_slot), from = paged_slot_row(kv, table, g, from_slot);
  if (t == 0u) a.weight_out[state + to_slot] = a.weight[state + from_slot];
  if (t == 1u) a.slot_pos_out[state + to_slot] = a.slot_pos[state + from_slot];
  if (to == kNoRow || from == kNoRow) return;
  const uint4 x = reinterpret_cast<const uint4*>(kv.k)[static_cast<std::size_t>(from) * L + t];
  const uint4 y = reinterpret_cast<const uint4*>(kv.v)[static_cast<std::size_t>(from) * L + t];
  reinterpret_cast<uint4*>(kv.k)[static_cast<std::size_t>(to) * L + t] = x;
  reinterpret_cast<uint4*>(kv.v)[static_cast<std::size_t>(to) * L + t] = y;
}

// L: 0, or the moves follow in the same workgroup, L lanes a row (and the length, of
// which then no other workgroup's copy is overwritten).
template <std::uint32_t T, int L>
__global__ __launch_bounds__(T) void evict_choice_kernel(PagedView kv, EvictArgs a, std::uint32_t* length_out) {
  __shared__ __align__(16) SelectShared<T> sh;
  extern __shared__ __align__(16) std::uint8_t lds[];
  const std::uint32_t g = blockIdx.x, r = blockIdx.y, tid = threadIdx.x;
  const std::size_t gr = static_cast<std::size_t>(r) * kv.n_kv + g;
  std::uint32_t* const moves = a.moves + gr * (1u + 2u * static_cast<std::size_t>(a.most));
  const std::int32_t* const table = kv.table + static_cast<std::size_t>(r) * kv.table_stride;
  const std::int32_t entry = table[tid < kv.entries ? tid : 0u];  // (with the length in flight)
  const std::uint32_t newest = a.pos[r];
  std::uint32_t n = a.length[r];
  n = n < kv.capacity ? n : kv.capacity;
  if (newest == RTXLLM_NO_POSITION) {
    if (tid == 0u) moves[0] = 0u;
    return;
  }
  if (L != 0 && g == 0u && tid == 0u) length_out[r] = n < a.keep ? n : a.keep;
  const std::uint32_t recent = newest >= a.n_recent ? newest - a.n_recent + 1u : 0u;  // the first such position
  SlotKeys src{a.weight + gr * kv.capacity, a.slot_pos + gr * kv.capacity, a.weight_out + gr * kv.capacity,
               a.slot_pos_out + gr * kv.capacity, n, n < a.keep ? n : a.keep, a.n_first,
               recent > a.n_first ? recent - a.n_first : 0u, kv, table, sh.wave[0], T / 64u, false};
  if (n <= a.keep || n > a.room)
    for (std::uint32_t i = 4u * tid; i < src.stay; i += 4u * T) src.seen(i, src.raw<false>(i));
  if (n <= a.keep) {
    if (tid == 0u) moves[0] = 0u;
    return;
  }
  const std::uint32_t used = page_of(kv, n - 1u) + 1u;
  bool hole = tid < used && static_cast<std::uint32_t>(entry) >= kv.n_pages;
  for (std::uint32_t t = T + 4u * tid; t < used; t += 4u * T)
#pragma unroll
    for (std::uint32_t e = 0; e < 4u; ++e)  // past the last: read again
      hole |= static_cast<std::uint32_t>(table[t + e < used ? t + e : used - 1u]) >= kv.n_pages;
  if (const unsigned long long b = __ballot(hole); (tid & 63u) == 0u) sh.wave[0][tid >> 6] = b != 0ull ? 1u : 0u;
  const Keys<std::uint32_t, SlotKeys, T> keys(src, lds, sh.hist[0], n, a.room);
  const Choice<std::uint32_t> ch = radix_choice(sh, keys, a.keep);
  std::uint32_t* const to = moves + 1u;
  std::uint32_t* const from = to + a.most;
  const std::uint32_t freed = for_choice(sh, keys, ch, a.keep, Places{to, a.most}, Places{from, a.most}).x;
  const std::uint32_t n_moves = freed < a.most ? freed : a.most;
  if constexpr (L == 0) {
    if (tid == 0u) moves[0] = n_moves;
  } else {
    __threadfence_block();
    __syncthreads();
    for (std::uint32_t m = tid / L; m < n_moves; m += T / L) move_row<L>(kv, a, r, g, to[m], from[m], tid % L);
  }
}

template <int L>
__global__ __launch_bounds__(kThreads) void evict_move_kernel(PagedView kv, EvictArgs a, std::uint32_t* length_out) {
  const std::uint32_t g = blockIdx.y, r = blockIdx.z;
  if (blockIdx.x == 0u && g == 0u && threadIdx.x == 0u && a.pos[r] != RTXLLM_NO_POSITION) {
    std::uint32_t n = a.length[r];
    n = n < kv.capacity ? n : kv.capacity;
    length_out[r] = n < a.keep ? n : a.keep;
  }
  const std::uint32_t* const moves =
      a.moves + (static_cast<std::size_t>(r) * kv.n_kv + g) * (1u + 2u * static_cast<std::size_t>(a.most));
  const std::uint32_t m = blockIdx.x * (kThreads / L) + threadIdx.x / L;
  if (m >= a.most) return;
  const std::uint32_t to = moves[1u + m], from = moves[1u + a.most + m];  // read with the count: used below it
  if (m < moves[0]) move_row<L>(kv, a, r, g, to, from, threadIdx.x % L);
}

template <int L>
hipError_t launch_select(const PagedView& view, const std::uint16_t* bounds, const float* q, std::uint32_t group,
                         const std::uint32_t* pos, std::uint32_t count, std::uint32_t n_first, std::uint32_t n_last,
                         std::uint32_t n_select, unsigned long long* keys, std::int32_t* pages, hipStream_t stream) {
  const dim3 choices(view.n_kv, count);
  auto score = [&](auto steps) {
    constexpr int kSteps = decltype(steps)::value;
    constexpr std::uint32_t kPer = kSteps * kThreads / L;  // pages of a workgroup
    hipLaunchKernelGGL((page_score_kernel<L, kSteps>), dim3((view.entries + kPer - 1u) / kPer, view.n_kv, count),
                       dim3(kThreads), 0, stream, view, bounds, q, group, pos, n_first, n_last, keys);
  };
  const std::uint64_t waves = static_cast<std::uint64_t>(count) * view.n_kv * ((view.entries + 64u / L - 1u) / (64u / L));
  if (score_four_steps(waves, group))
    score(std::integral_constant<int, 4>{});
  else
    score(std::integral_constant<int, 1>{});
  const hipError_t rc = hipGetLastError();
  if (rc != hipSuccess) return rc;
  // four waves up to 1024 pages, whose barriers cost less (us of both launches, four / 16
  // waves: 250 pages of 8 heads 7.9 / 8.3, 1024 8.6 / 8.9, 2047 11.8 / 11.0, 4094 18.7 / 16.3)
  const std::uint32_t threads = view.entries <= 1024u ? 256u : 1024u;
  const std::size_t held = held_bytes(view.entries, 8u, threads);
  const auto room = static_cast<std::uint32_t>(held / 8u);
  if (threads == 256u)
    hipLaunchKernelGGL(page_choice_kernel<256>, choices, dim3(256), held, stream, view, pos, keys, room, n_select, pages);
  else
    hipLaunchKernelGGL(page_choice_kernel<1024>, choices, dim3(1024), held, stream, view, pos, keys, room, n_select, pages);
  return hipGetLastError();
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
  return cache->head_dim == 64u    ? launch_select<8>(view, bounds, q, group, pos, count, n_first, n_last, n_select, keys, pages, stream)
         : cache->head_dim == 128u ? launch_select<16>(view, bounds, q, group, pos, count, n_first, n_last, n_select, keys, pages, stream)
                                   : launch_select<32>(view, bounds, q, group, pos, count, n_first, n_last, n_select, keys, pages, stream);
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
      overlap(length_out, 4u * count, pos, 4u * count) || overlap(length_out, 4u * count, weight, n) ||
      overlap(length_out, 4u * count, slot_pos, n) || overlap(length_out, 4u * count, weight_out, n) ||
      overlap(length_out, 4u * count, slot_pos_out, n) || overlap(weight_out, n, length, 4u * count) ||
      overlap(weight_out, n, pos, 4u * count) || overlap(slot_pos_out, n, length, 4u * count) ||
      overlap(slot_pos_out, n, pos, 4u * count))
    return hipErrorInvalidValue;
  const PagedView view = paged_view(cache);
  const std::uint32_t most = most_moves(cache, keep), per = kThreads / (cache->head_dim / 8u);
  const bool small = evict_four_waves(view.capacity, static_cast<std::uint64_t>(count) * view.n_kv);
  const std::size_t held = held_bytes(view.capacity, 4u, small ? 256u : 1024u);
  const EvictArgs a{length, pos, weight, slot_pos, weight_out, slot_pos_out, static_cast<std::uint32_t*>(workspace),
                    keep,   n_first, n_recent, most, static_cast<std::uint32_t>(held / 4u)};
  auto choose = [&](auto lanes) {
    constexpr int L = decltype(lanes)::value;
    if (small)
      hipLaunchKernelGGL((evict_choice_kernel<256, L>), dim3(view.n_kv, count), dim3(256), held, stream, view, a, length_out);
    else
      hipLaunchKernelGGL((evict_choice_kernel<1024, L>), dim3(view.n_kv, count), dim3(1024), held, stream, view, a, length_out);
  };
  // In place, a kv head's workgroup may read the length after another has written it.
  if (most <= kEvictMovesHere && length_out != length) {
    if (cache->head_dim == 64u)
      choose(std::integral_constant<int, 8>{});
    else if (cache->head_dim == 128u)
      choose(std::integral_constant<int, 16>{});
    else
      choose(std::integral_constant<int, 32>{});
    return hipGetLastError();
  }
  choose(std::integral_constant<int, 0>{});
  hipError_t rc = hipGetLastError();
  if (rc != hipSuccess) return rc;
  const dim3 grid(most > 0u ? (most + per - 1u) / per : 1u, view.n_kv, count);
  if (cache->head_dim == 64u)
    hipLaunchKernelGGL(evict_move_kernel<8>, grid, dim3(kThreads), 0, stream, view, a, length_out);
  else if (cache->head_dim == 128u)
    hipLaunchKernelGGL(evict_move_kernel<16>, grid, dim3(kThreads), 0, stream, view, a, length_out);
  else
    hipLaunchKernelGGL(evict_move_kernel<32>, grid, dim3(kThreads), 0, stream, view, a, length_out);
  return hipGetLastError();
}
