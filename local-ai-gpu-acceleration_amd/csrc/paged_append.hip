// New keys and values enter the paged cache: the norm of every query and key
// head, its rotation and the store into the page slot in one pass over the
// projections' output; and the bounds of a page's keys, which the selection of
// pages reads.
#include <type_traits>

#include "common.h"
#include "layer_common.cuh"
#include "paged.h"

namespace rtxllm {
namespace {

constexpr std::uint32_t kThreads = 256;

struct AppendArgs {
  const float *q, *k, *v, *qw, *kw;
  std::size_t q_stride, k_stride, v_stride;
  const std::uint32_t *pos, *slot;
  float* q_out;
  std::uint32_t* slot_pos;
  float* slot_weight;
  double log2_theta;
  float eps;
  std::uint32_t n_heads, rotary, halves;
};

// Sum over aligned groups of L lanes; every lane receives it.
template <int L>
__device__ __forceinline__ float group_sum(float v) {
  v += lane_xor<1>(v);
  v += lane_xor<2>(v);
  v += lane_xor<4>(v);
  if constexpr (L > 8) v += lane_xor<8>(v);
  if constexpr (L > 16) v += lane_xor<16>(v);
  return v;
}

// L = head_dim / 8 lanes hold a head, 8 values each: the two values of a pair
// lie in one lane (halves: 4 values and the 4 half a rotation on; adjacent: 8 in
// a row), so a rotation needs no exchange, and in place is safe. The row's
// (cos, sin) go through LDS, one thread a pair: revolutions pos theta^(-2i/R) /
// 2 pi in 64 bits, of which the nearest whole number is dropped; the rest, at
// most half a turn, is exact enough in fp32 for sincospif's last bit. ROW: a workgroup
// takes every head of its row in turn, else 2048 / head_dim of them. Bound by bytes from
// some hundred rows on: 4001 rows of 32 + 2 x 8 heads of 128 (180 MB) 32.3 us, 5.6 TB/s (a
// 1 GiB copy: 5.2); one row 2.8 us, a launch.
template <int L, bool ROW>
__global__ __launch_bounds__(kThreads) void append_kernel(AppendArgs a, PagedView kv) {
  constexpr std::uint32_t D = 8u * L, kUnits = kThreads / L;
  __shared__ float2 cs[128];
  const std::uint32_t r = blockIdx.x, pos = a.pos[r];
  if (pos == RTXLLM_NO_POSITION) return;
  const std::uint32_t half = a.rotary / 2u;
  if (threadIdx.x < half) {
    const double inv = exp2(static_cast<double>(threadIdx.x) / static_cast<double>(half) * -a.log2_theta);
    const double turns = static_cast<double>(pos) * inv * 0.15915494309189535;  // 1 / (2 pi)
    float s, c;
    sincospif(static_cast<float>(2.0 * (turns - rint(turns))), &s, &c);
    cs[threadIdx.x] = make_float2(c, s);
  }
  __syncthreads();
  const std::uint32_t units = a.n_heads + 2u * kv.n_kv;
  const std::uint32_t t = threadIdx.x % L;
  const std::uint32_t slot = a.slot != nullptr ? a.slot[r] : pos;
  auto head = [&](std::uint32_t u) {
    const std::uint32_t h = u < units ? u : units - 1u;  // past the last: computed, not stored
    const bool is_q = h < a.n_heads, is_v = h >= a.n_heads + kv.n_kv;
    const float* src = is_q   ? a.q + r * a.q_stride + h * D
                       : is_v ? a.v + r * a.v_stride + (h - a.n_heads - kv.n_kv) * D
                              : a.k + r * a.k_stride + (h - a.n_heads) * D;
    const bool rot = 8u * t < a.rotary && !is_v;
    const bool split = a.halves != 0u && 8u * t < a.rotary;
    const std::uint32_t ia = split ? 4u * t : 8u * t, ib = split ? ia + half : ia + 4u;
    // read once: past the caches (4001 rows 32.3 us, through them 37.1)
    f32x4_any xa = __builtin_nontemporal_load(reinterpret_cast<const f32x4_any*>(src + ia));
    f32x4_any xb = __builtin_nontemporal_load(reinterpret_cast<const f32x4_any*>(src + ib));
    float ss = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) ss = fmaf(xa[i], xa[i], ss);
#pragma unroll
    for (int i = 0; i < 4; ++i) ss = fmaf(xb[i], xb[i], ss);
    ss = group_sum<L>(ss);
    if (!is_v) {
      const float inv = 1.0f / sqrtf(ss / static_cast<float>(D) + a.eps);
      const float* w = is_q ? a.qw : a.kw;
      f32x4_any wa = {1.0f, 1.0f, 1.0f, 1.0f}, wb = wa;
      if (w != nullptr) {
        wa = *reinterpret_cast<const f32x4_any*>(w + ia);
        wb = *reinterpret_cast<const f32x4_any*>(w + ib);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        xa[i] = xa[i] * inv * wa[i];
        xb[i] = xb[i] * inv * wb[i];
      }
    }
    if (rot) {
      if (split) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 t2 = cs[ia + i];
          const float x = xa[i], y = xb[i];
          xa[i] = x * t2.x - y * t2.y;
          xb[i] = x * t2.y + y * t2.x;
        }
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 t2 = cs[4u * t + i];
          const float x = i < 2 ? xa[2 * i] : xb[2 * i - 4], y = i < 2 ? xa[2 * i + 1] : xb[2 * i - 3];
          const float e = x * t2.x - y * t2.y, o = x * t2.y + y * t2.x;
          if (i < 2) {
            xa[2 * i] = e, xa[2 * i + 1] = o;
          } else {
            xb[2 * i - 4] = e, xb[2 * i - 3] = o;
          }
        }
      }
    }
    if (u >= units) return;
    if (is_q) {
      float* dst = a.q_out + (static_cast<std::size_t>(r) * a.n_heads + h) * D;
      *reinterpret_cast<f32x4_any*>(dst + ia) = xa;
      *reinterpret_cast<f32x4_any*>(dst + ib) = xb;
      return;
    }
    const std::uint32_t g = is_v ? h - a.n_heads - kv.n_kv : h - a.n_heads;
    if (slot >= kv.capacity) return;
    const std::uint32_t row = paged_slot_row(kv, kv.table + static_cast<std::size_t>(r) * kv.table_stride, g, slot);
    if (row != kNoRow) {
      std::uint16_t* dst = (is_v ? kv.v : kv.k) + static_cast<std::size_t>(row) * D;
      auto pack = [](const f32x4_any& x) {
        return make_uint2(f2h(x[0]) | static_cast<std::uint32_t>(f2h(x[1])) << 16,
                          f2h(x[2]) | static_cast<std::uint32_t>(f2h(x[3])) << 16);
      };
      *reinterpret_cast<uint2*>(dst + ia) = pack(xa);
      *reinterpret_cast<uint2*>(dst + ib) = pack(xb);
    }
    if (!is_v && t == 0u) {
      const std::size_t i = (static_cast<std::size_t>(kv.table_stride != 0u ? r : 0u) * kv.n_kv + g) * kv.capacity + slot;
      if (a.slot_pos != nullptr) a.slot_pos[i] = pos;
      if (a.slot_weight != nullptr) a.slot_weight[i] = 0.0f;
    }
  };
  if constexpr (ROW)
    for (std::uint32_t u0 = 0; u0 < units; u0 += kUnits) head(u0 + threadIdx.x / L);
  else
    head(blockIdx.y * kUnits + threadIdx.x / L);
}

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
constexpr _Float16 kHalfMax = static_cast<_Float16>(65504.0f);

// The w-th (page, kv head) of row r's pages from first[r] on: its first cache row, its
// filled keys (0: there is none), its place among the bounds.
struct PageUnit {
  std::uint32_t row, keys;
  std::size_t at;
};
__device__ __forceinline__ PageUnit page_unit(const PagedView& kv, const std::uint32_t* first, const std::uint32_t* last,
                                              std::uint32_t r, std::uint32_t w, std::uint32_t span) {
  const PageUnit none{kNoRow, 0u, 0u};
  const std::uint32_t n = paged_filled(kv, last[r]);
  if (n == 0u || w / kv.n_kv >= span) return none;
  const std::uint32_t from = first != nullptr ? first[r] : n - 1u;
  if (from >= n) return none;
  const std::uint32_t lp = page_of(kv, from) + w / kv.n_kv, g = w % kv.n_kv;
  if (lp >= kv.entries || lp * kv.page_size >= n) return none;
  const std::int32_t page = kv.table[static_cast<std::size_t>(r) * kv.table_stride + lp];
  const std::uint32_t row = paged_row(kv, page, g, 0u), rest = n - lp * kv.page_size;
  if (row == kNoRow) return none;
  return PageUnit{row, rest < kv.page_size ? rest : kv.page_size, static_cast<std::size_t>(page) * kv.n_kv + g};
}

template <int L>
__device__ __forceinline__ void store_bounds(std::uint16_t* bounds, std::size_t at, std::uint32_t t, half8 hi, half8 lo) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    hi[i] = hi[i] > kHalfMax ? kHalfMax : hi[i];
    lo[i] = lo[i] < -kHalfMax ? -kHalfMax : lo[i];
  }
  half8* dst = reinterpret_cast<half8*>(bounds) + at * 2u * L + t;
  dst[0] = hi;
  dst[L] = lo;
}

// One wave a (page, kv head), or W of a workgroup whose extremes meet in LDS: L = head_dim
// / 8 lanes a key, 64 / L keys at a time. Repeating a filled key changes neither extreme, so the last step reads
// its last key again instead of masking. Bound by bytes: 1024 pages of 64 keys of 8
// heads of 128 (138 MB) 24.0 us, 5.8 TB/s, streamed past the caches (28.4 through them).
template <int L, int W>
__global__ __launch_bounds__(kThreads) void page_bounds_kernel(PagedView kv, const std::uint32_t* first,
                                                               const std::uint32_t* last, std::uint32_t span,
                                                               std::uint16_t* bounds) {
  constexpr std::uint32_t D = 8u * L, kKeys = 64u / L;
  const std::uint32_t r = blockIdx.y, lane = threadIdx.x & 63u;
  const std::uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), part = wave % W;
  const PageUnit u = page_unit(kv, first, last, r, blockIdx.x * (kThreads / 64u / W) + wave / W, span);
  if (u.keys == 0u) return;  // (W > 1: the whole workgroup)
  const half8* src = reinterpret_cast<const half8*>(kv.k + static_cast<std::size_t>(u.row) * D) + lane % L;
  half8 hi = half8{} - kHalfMax, lo = half8{} + kHalfMax;
  for (std::uint32_t k0 = 4u * kKeys * part; k0 < u.keys; k0 += 4u * kKeys * W) {
    const std::uint32_t i0 = k0 + lane / L;
    half8 x[4];
#pragma unroll
    for (std::uint32_t j = 0; j < 4u; ++j) {
      const std::uint32_t i = i0 + kKeys * j;
      const half8* at = src + static_cast<std::size_t>(i < u.keys ? i : u.keys - 1u) * L;
      x[j] = W == 1 ? __builtin_nontemporal_load(at) : *at;
    }
#pragma unroll
    for (std::uint32_t j = 0; j < 4u; ++j) {
      hi = __builtin_elementwise_max(hi, x[j]);  // a NaN operand gives the other one
      lo = __builtin_elementwise_min(lo, x[j]);
    }
  }
  auto fold = [&](auto mask) {
    constexpr int M = decltype(mask)::value;
    uint4 a = __builtin_bit_cast(uint4, hi), b = __builtin_bit_cast(uint4, lo);
    auto move = [](std::uint32_t& v) { v = __float_as_uint(lane_xor<M>(__uint_as_float(v))); };
    move(a.x), move(a.y), move(a.z), move(a.w);
    move(b.x), move(b.y), move(b.z), move(b.w);
    hi = __builtin_elementwise_max(hi, __builtin_bit_cast(half8, a));
    lo = __builtin_elementwise_min(lo, __builtin_bit_cast(half8, b));
  };
  if constexpr (L <= 8) fold(std::integral_constant<int, 8>{});
  if constexpr (L <= 16) fold(std::integral_constant<int, 16>{});
  fold(std::integral_constant<int, 32>{});
  if constexpr (W > 1) {
    __shared__ half8 parts[W][2][L];
    if (lane < static_cast<std::uint32_t>(L)) parts[wave][0][lane] = hi, parts[wave][1][lane] = lo;
    __syncthreads();
    if (wave != 0u || lane >= static_cast<std::uint32_t>(L)) return;
#pragma unroll
    for (int k = 1; k < W; ++k) {
      hi = __builtin_elementwise_max(hi, parts[k][0][lane]);
      lo = __builtin_elementwise_min(lo, parts[k][1][lane]);
    }
  }
  if (lane >= static_cast<std::uint32_t>(L)) return;
  store_bounds<L>(bounds, u.at, lane, hi, lo);
}

// Small pages of a prompt: each L lanes take a (page, kv head) of their own, all its
// keys one after the other, eight in flight. No exchange between lanes, which is most of
// the work above where a page has few keys.
template <int L>
__global__ __launch_bounds__(kThreads) void prompt_bounds_kernel(PagedView kv, const std::uint32_t* first,
                                                                 const std::uint32_t* last, std::uint32_t span,
                                                                 std::uint16_t* bounds) {
  constexpr std::uint32_t D = 8u * L;
  const std::uint32_t r = blockIdx.y, t = threadIdx.x % L;
  const std::uint32_t w = blockIdx.x * (kThreads / L) + threadIdx.x / L;
  const PageUnit u = page_unit(kv, first, last, r, w, span);
  if (u.keys == 0u) return;
  const half8* src = reinterpret_cast<const half8*>(kv.k + static_cast<std::size_t>(u.row) * D) + t;
  half8 hi = half8{} - kHalfMax, lo = half8{} + kHalfMax;
  for (std::uint32_t i0 = 0; i0 < u.keys; i0 += 8u) {
    half8 x[8];
#pragma unroll
    for (std::uint32_t j = 0; j < 8u; ++j) {
      const std::uint32_t i = i0 + j < u.keys ? i0 + j : u.keys - 1u;
      x[j] = __builtin_nontemporal_load(src + static_cast<std::size_t>(i) * L);
    }
#pragma unroll
    for (std::uint32_t j = 0; j < 8u; ++j) {
      hi = __builtin_elementwise_max(hi, x[j]);
      lo = __builtin_elementwise_min(lo, x[j]);
    }
  }
  store_bounds<L>(bounds, u.at, t, hi, lo);
}

}  // namespace
}  // namespace rtxllm

using namespace rtxllm;

extern "C" hipError_t rtxllm_qk_norm_rope_append_f16(const rtxllm_paged_kv* cache, const float* q, size_t q_stride,
                                                     const float* k, size_t k_stride, const float* v, size_t v_stride,
                                                     const float* q_weight, const float* k_weight, uint32_t n_heads,
                                                     uint32_t rotary_dim, int pairing, float theta, float eps,
                                                     const uint32_t* pos, const uint32_t* slot, uint32_t count,
                                                     float* q_out, uint32_t* slot_pos, float* slot_weight,
                                                     hipStream_t stream) {
  if (!paged_cache_ok(cache, count) || q == nullptr || k == nullptr || v == nullptr || pos == nullptr ||
      q_out == nullptr || count == 0u || count > (1u << 20) || n_heads == 0u ||
      n_heads > 4096u || n_heads + 2u * cache->n_kv_heads > 4096u || rotary_dim < 8u ||
      rotary_dim > cache->head_dim || rotary_dim % 8u != 0u ||
      (pairing != RTXLLM_PAIR_ADJACENT && pairing != RTXLLM_PAIR_HALVES) || !(theta > 0.0f) || theta > 3.0e38f ||
      !(eps >= 0.0f))
    return hipErrorInvalidValue;
  for (const void* p : {static_cast<const void*>(q), static_cast<const void*>(k), static_cast<const void*>(v),
                        static_cast<const void*>(q_weight), static_cast<const void*>(k_weight),
                        static_cast<const void*>(pos), static_cast<const void*>(slot),
                        static_cast<const void*>(q_out), static_cast<const void*>(slot_pos),
                        static_cast<const void*>(slot_weight)})
    if (!aligned_to(p, 4u)) return hipErrorInvalidValue;
  const std::size_t d = cache->head_dim, q_row = n_heads * d, kv_row = cache->n_kv_heads * d;
  constexpr std::size_t kMaxStride = std::size_t{1} << 36;
  if (q_stride > kMaxStride || k_stride > kMaxStride || v_stride > kMaxStride ||
      (count > 1u && (q_stride < q_row || k_stride < kv_row || v_stride < kv_row)))
    return hipErrorInvalidValue;
  // in place means the very same rows: a row's heads are read by other workgroups
  const std::size_t out_n = 4u * count * q_row;
  if ((overlap(q_out, out_n, q, 4u * ((count - 1u) * q_stride + q_row)) && !(q_out == q && (q_stride == q_row || count == 1u))) ||
      overlap(q_out, out_n, k, 4u * ((count - 1u) * k_stride + kv_row)) ||
      overlap(q_out, out_n, v, 4u * ((count - 1u) * v_stride + kv_row)))
    return hipErrorInvalidValue;
  const AppendArgs a{q,    k,    v,     q_weight, k_weight, q_stride,    k_stride,
                     v_stride, pos, slot, q_out, slot_pos, slot_weight, log2(static_cast<double>(theta)),
                     eps,  n_heads, rotary_dim, pairing == RTXLLM_PAIR_HALVES ? 1u : 0u};
  const PagedView view = paged_view(cache);
  const std::uint32_t units = n_heads + 2u * cache->n_kv_heads, per = kThreads / static_cast<std::uint32_t>(d / 8u);
  auto launch = [&](auto row) {
    constexpr bool kRow = decltype(row)::value;
    const dim3 grid(count, kRow ? 1u : (units + per - 1u) / per);
    if (d == 64u)
      hipLaunchKernelGGL((append_kernel<8, kRow>), grid, dim3(kThreads), 0, stream, a, view);
    else if (d == 128u)
      hipLaunchKernelGGL((append_kernel<16, kRow>), grid, dim3(kThreads), 0, stream, a, view);
    else
      hipLaunchKernelGGL((append_kernel<32, kRow>), grid, dim3(kThreads), 0, stream, a, view);
  };
  if (append_row_a_workgroup(count, units, per))
    launch(std::true_type{});
  else
    launch(std::false_type{});
  return hipGetLastError();
}

extern "C" hipError_t rtxllm_kv_page_bounds_f16(const rtxllm_paged_kv* cache, const uint32_t* first,
                                                const uint32_t* last, uint32_t count, uint32_t span,
                                                uint16_t* bounds, hipStream_t stream) {
  if (!paged_cache_ok(cache, count) || last == nullptr || bounds == nullptr || count == 0u || count > 65535u ||
      span == 0u || span > (1u << 20) || !aligned_to(first, 4u) || !aligned_to(last, 4u) || !aligned_to(bounds, 16u))
    return hipErrorInvalidValue;
  const PagedView view = paged_view(cache);
  const std::uint32_t pages = span < view.entries ? span : view.entries;
  const std::uint64_t waves = static_cast<std::uint64_t>(pages) * view.n_kv;
  if (waves > (1ull << 24)) return hipErrorInvalidValue;  // the launch's thread count
  const dim3 grid(static_cast<std::uint32_t>((waves + 3u) / 4u), count);
  auto launch = [&](auto lanes) {
    constexpr int L = decltype(lanes)::value;
    const std::uint32_t per = kThreads / L, rounds = view.page_size / (256u / L);
    const std::uint64_t units = waves * count;
    const BoundsForm form = bounds_form(units, rounds);
    if (form == BoundsForm::kFourWaves)
      hipLaunchKernelGGL((page_bounds_kernel<L, 4>), dim3(static_cast<std::uint32_t>(waves), count), dim3(kThreads), 0,
                         stream, view, first, last, pages, bounds);
    else if (form == BoundsForm::kLanes)
      hipLaunchKernelGGL(prompt_bounds_kernel<L>, dim3(static_cast<std::uint32_t>((waves + per - 1u) / per), count),
                         dim3(kThreads), 0, stream, view, first, last, pages, bounds);
    else
      hipLaunchKernelGGL((page_bounds_kernel<L, 1>), grid, dim3(kThreads), 0, stream, view, first, last, pages, bounds);
  };
  if (cache->head_dim == 64u)
    launch(std::integral_constant<int, 8>{});
  else if (cache->head_dim == 128u)
    launch(std::integral_constant<int, 16>{});
  else
    launch(std::integral_constant<int, 32>{});
  return hipGetLastError();
}
