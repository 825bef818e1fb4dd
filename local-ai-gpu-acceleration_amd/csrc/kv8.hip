// The paged cache in 8 bits: codes and scales of new keys and values, and
// positions read back.
#include "common.h"
#include "layer_common.cuh"
#include "rows.h"

namespace rtxllm {
namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef std::uint16_t u16x2 __attribute__((ext_vector_type(2)));
typedef std::uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 half8_any __attribute__((ext_vector_type(8), aligned(2)));

constexpr std::uint32_t kThreads = 256, kWaves = kThreads / 64u;

struct Kv8Append {
  const void *x[2];  // k, v
  std::size_t stride[2];
  std::uint8_t* codes[2];
  float* scale[2];
  std::uint16_t* tail[2];
  std::uint32_t units, block;
};

template <bool F16>
__device__ __forceinline__ half8 load8(const void* x, std::size_t at) {
  half8 h;
  if constexpr (F16) {
    h = half8(__builtin_nontemporal_load(reinterpret_cast<const half8_any*>(static_cast<const _Float16*>(x) + at)));
  } else {
    const float* f = static_cast<const float*>(x) + at;
    const f32x4_any a = __builtin_nontemporal_load(reinterpret_cast<const f32x4_any*>(f));
    const f32x4_any b = __builtin_nontemporal_load(reinterpret_cast<const f32x4_any*>(f + 4));
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = static_cast<_Float16>(a[i]), h[i + 4] = static_cast<_Float16>(b[i]);
  }
  return h;
}

// code(x / scale): c = round(x inv) is off by one at most, and only next to a half; x - c scale
// is exact in one fma (a multiple of scale's last bit below scale), so which side of the half x / scale
// lies on is a comparison without rounding.
__device__ __forceinline__ std::uint32_t int8_code(float x, float inv, float scale) {
  float c = rintf(x * inv);
  const float r = fmaf(-c, scale, x), two = 2.0f * fabsf(r);
  const float other = c + copysignf(1.0f, r);
  const bool odd = (static_cast<int>(c) & 1) != 0;
  c = two > scale || (two == scale && odd) ? other : c;
  return static_cast<std::uint32_t>(static_cast<int>(c)) & 0xFFu;
}

// One wave an item: a block that new rows touch, of one kv head, of k or of v. L = head_dim / 8 lanes
// hold a position, 8 values each, R = block L / 64 positions a lane. A whole block is read
// (its first positions from the tail where an earlier call brought them), its largest magnitude found
// across the wave, and its codes leave in one piece, since a block of a head lies in one piece in its
// page. Values that stay in the open block go to the tail; where the call also makes an earlier block
// whole from the same tail, that block's wave writes them, once it has read.
template <int L, int R, bool E4M3, bool F16>
__global__ __launch_bounds__(kThreads) void kv8_append_kernel(Kv8Append a, CallRows rows, RowsCache kv) {
  constexpr std::uint32_t D = 8u * L, kStep = 64u / L;  // positions of a round
  const std::uint32_t item = blockIdx.x * kWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const std::uint32_t per_unit = 2u * kv.p.n_kv, w = item / per_unit;
  if (w >= a.units) return;
  const std::uint32_t which = item % per_unit / kv.p.n_kv, g = item % kv.p.n_kv;
  std::uint32_t s = w, base = w;
  if (rows.start != nullptr) s = unit_sequence(rows, w, a.block, 2u, base);
  const SeqRows q = seq_rows(rows, s);
  if (w < base || q.n == 0u || q.pos >= kv.p.capacity) return;
  const std::uint32_t end = held_end(q.pos, q.n, kv.p.capacity), first = q.pos & ~(a.block - 1u);
  const std::uint32_t t = w - base, b0 = first + t * a.block;
  if (b0 >= end) return;
  const std::uint32_t lane = threadIdx.x & 63u, part = lane % L, in = lane / L;
  std::uint16_t* const tail = a.tail[which] + (static_cast<std::size_t>(s) * kv.p.n_kv + g) * a.block * D + 8u * part;
  const void* const x = a.x[which];
  const std::size_t stride = a.stride[which], col = g * D + 8u * part;
  auto at = [&](std::uint32_t p) { return static_cast<std::size_t>(q.row + (p - q.pos)) * stride + col; };
  auto to_tail = [&](std::uint32_t from) {
    for (std::uint32_t p = from + in; p < end; p += kStep)
      if (p >= q.pos) *reinterpret_cast<half8*>(tail + (p & (a.block - 1u)) * D) = load8<F16>(x, at(p));
  };
  const std::uint32_t open = end & ~(a.block - 1u);  // the open block's start
  if (b0 + a.block > end) {
    if (t == 0u || q.pos == first) to_tail(b0);  // (else the first block's wave)
    return;
  }
  half8 v[R];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const std::uint32_t p = b0 + in + kStep * i;
    v[i] = p < q.pos ? *reinterpret_cast<const half8*>(tail + (p & (a.block - 1u)) * D) : load8<F16>(x, at(p));
  }
  // fp16 magnitudes compare as their bits, numbers that are not finite above all
  u16x2 most = {0, 0};
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const u32x4 w = __builtin_bit_cast(u32x4, v[i]);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const std::uint32_t m = w[j] & 0x7FFF7FFFu;
      most = __builtin_elementwise_max(most, __builtin_bit_cast(u16x2, m));
    }
  }
  std::uint32_t top = most[0] > most[1] ? most[0] : most[1];
  top = lanes_reduce_exact(top, [](std::uint32_t x, std::uint32_t y) { return x > y ? x : y; });
  if (t == 0u && q.pos != first && open < end) {  // the tail has been read: no wave but this one touches it
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    to_tail(open);
  }
  const std::int32_t* const table = kv.p.table + static_cast<std::size_t>(s) * kv.p.table_stride;
  const std::uint32_t row = paged_slot_row(kv.p, table, g, b0);
  if (row == kNoRow) return;
  const bool finite = top < 0x7C00u;
  const float amax = static_cast<float>(__builtin_bit_cast(_Float16, static_cast<unsigned short>(top)));
  float scale, inv;
  if constexpr (E4M3) {  // amax = 2^e m: 448 = 1.75 2^8
    const std::uint32_t bits = __float_as_uint(amax);
    const std::uint32_t e = (bits >> 23) - 8u + ((bits & 0x7FFFFFu) > 0x600000u ? 1u : 0u);
    scale = __uint_as_float(e << 23), inv = __uint_as_float((254u - e) << 23);
  } else {
    scale = amax * (1.0f / 127.0f), inv = 1.0f / scale;
  }
  const bool some = finite && top != 0u;
  std::uint8_t* const out = a.codes[which] + static_cast<std::size_t>(row) * D + 8u * part;
#pragma unroll
  for (int i = 0; i < R; ++i) {
    uint2 c = make_uint2(0u, 0u);
    if (some) {
      if constexpr (E4M3) {
        int lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[i][0] * inv, v[i][1] * inv, 0, false);
        lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[i][2] * inv, v[i][3] * inv, lo, true);
        int hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[i][4] * inv, v[i][5] * inv, 0, false);
        hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[i][6] * inv, v[i][7] * inv, hi, true);
        c = make_uint2(static_cast<std::uint32_t>(lo), static_cast<std::uint32_t>(hi));
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          c.x |= int8_code(static_cast<float>(v[i][j]), inv, scale) << (8 * j);
          c.y |= int8_code(static_cast<float>(v[i][j + 4]), inv, scale) << (8 * j);
        }
      }
    }
    *reinterpret_cast<uint2*>(out + static_cast<std::size_t>(in + kStep * i) * D) = c;
  }
  if (lane == 0u) a.scale[which][row >> kv.block_shift] = !finite ? NAN : some ? scale : 0.0f;
}

struct Kv8Read {
  const std::uint32_t* held;
  void* out[2];
};

// L lanes a position of a head, 8 values each; the heads of a row lie next to each
// other in the result. Bound by bytes.
template <int L, bool E4M3, bool F16>
__global__ __launch_bounds__(kThreads) void kv8_read_kernel(Kv8Read a, CallRows rows, RowsCache kv) {
  constexpr std::uint32_t D = 8u * L;
  const std::uint64_t unit = static_cast<std::uint64_t>(blockIdx.x) * (kThreads / L) + threadIdx.x / L;
  const std::uint64_t r64 = unit / kv.p.n_kv;
  if (r64 >= rows.rows) return;
  const std::uint32_t r = static_cast<std::uint32_t>(r64), g = static_cast<std::uint32_t>(unit - r64 * kv.p.n_kv);
  const std::uint32_t part = threadIdx.x % L, which = blockIdx.y;
  std::uint32_t s = r, base;
  if (rows.start != nullptr) {  // the last sequence that does not start behind the row
    s = unit_sequence(rows, r, 1u, 0u, base);
  }
  const SeqRows q = seq_rows(rows, s);
  if (r < q.row || r - q.row >= q.n) return;
  const std::uint32_t held = a.held[s] < kv.p.capacity ? a.held[s] : kv.p.capacity;
  if (q.pos >= held || r - q.row >= held - q.pos) return;
  const std::uint32_t p = q.pos + (r - q.row), block = 1u << kv.block_shift;
  float x[8];
  if (p >= (held & ~(block - 1u))) {
    const half8 h = *reinterpret_cast<const half8*>((which == 0u ? kv.kt : kv.vt) +
                                                    ((static_cast<std::size_t>(s) * kv.p.n_kv + g) * block + (p & (block - 1u))) * D + 8u * part);
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = static_cast<float>(h[j]);
  } else {
    const std::uint32_t row = paged_slot_row(kv.p, kv.p.table + static_cast<std::size_t>(s) * kv.p.table_stride, g, p);
    if (row == kNoRow) return;
    const uint2 c = *reinterpret_cast<const uint2*>((which == 0u ? kv.k : kv.v) + static_cast<std::size_t>(row) * D + 8u * part);
    const float scale = (which == 0u ? kv.ks : kv.vs)[row >> kv.block_shift];
    if constexpr (E4M3) {
      auto four = [&](std::uint32_t u, float* f) {
        const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(u), false);
        const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(u), true);
        f[0] = lo[0], f[1] = lo[1], f[2] = hi[0], f[3] = hi[1];
      };
      four(c.x, x), four(c.y, x + 4);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        x[j] = static_cast<float>(static_cast<std::int8_t>(c.x >> (8 * j)));
        x[j + 4] = static_cast<float>(static_cast<std::int8_t>(c.y >> (8 * j)));
      }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] *= scale;
  }
  const std::size_t at = static_cast<std::size_t>(unit) * D + 8u * part;
  if constexpr (F16) {
    half8 h;
#pragma unroll
    for (int j = 0; j < 8; ++j) h[j] = static_cast<_Float16>(x[j]);
    __builtin_nontemporal_store(half8_any(h), reinterpret_cast<half8_any*>(static_cast<_Float16*>(a.out[which]) + at));
  } else {
    float* o = static_cast<float*>(a.out[which]) + at;
    __builtin_nontemporal_store(f32x4_any{x[0], x[1], x[2], x[3]}, reinterpret_cast<f32x4_any*>(o));
    __builtin_nontemporal_store(f32x4_any{x[4], x[5], x[6], x[7]}, reinterpret_cast<f32x4_any*>(o + 4));
  }
}

template <int L, int R>
void launch_append(bool e4m3, bool f16, std::uint32_t grid, const Kv8Append& a, const CallRows& rows, const RowsCache& kv,
                   hipStream_t stream) {
  auto run = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(grid), dim3(kThreads), 0, stream, a, rows, kv); };
  if (e4m3) {
    f16 ? run(kv8_append_kernel<L, R, true, true>) : run(kv8_append_kernel<L, R, true, false>);
  } else {
    f16 ? run(kv8_append_kernel<L, R, false, true>) : run(kv8_append_kernel<L, R, false, false>);
  }
}

template <int L>
void launch_append_block(std::uint32_t block, bool e4m3, bool f16, std::uint32_t grid, const Kv8Append& a, const CallRows& rows,
                         const RowsCache& kv, hipStream_t stream) {
  constexpr int R = L / 8;  // of a block of 8
  if (block == 8u) return launch_append<L, R>(e4m3, f16, grid, a, rows, kv, stream);
  if (block == 16u) return launch_append<L, 2 * R>(e4m3, f16, grid, a, rows, kv, stream);
  if (block == 32u) return launch_append<L, 4 * R>(e4m3, f16, grid, a, rows, kv, stream);
  launch_append<L, 8 * R>(e4m3, f16, grid, a, rows, kv, stream);
}

template <int L>
void launch_read(bool e4m3, bool f16, const Kv8Read& a, const CallRows& rows, const RowsCache& kv, hipStream_t stream) {
  const std::uint64_t units = static_cast<std::uint64_t>(rows.rows) * kv.p.n_kv, per = kThreads / L;
  // both, or k (y 0), or v alone (moved to y 0 by the caller)
  const dim3 grid(static_cast<std::uint32_t>((units + per - 1u) / per), a.out[1] != nullptr ? 2u : 1u);
  auto run = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(kThreads), 0, stream, a, rows, kv); };
  if (e4m3) {
    f16 ? run(kv8_read_kernel<L, true, true>) : run(kv8_read_kernel<L, true, false>);
  } else {
    f16 ? run(kv8_read_kernel<L, false, true>) : run(kv8_read_kernel<L, false, false>);
  }
}

}  // namespace
}  // namespace rtxllm

using namespace rtxllm;

extern "C" hipError_t rtxllm_kv8_append(const rtxllm_paged_kv8* cache, const void* k, size_t k_stride, const void* v,
                                        size_t v_stride, int type, const uint32_t* start, const uint32_t* pos,
                                        uint32_t sequences, uint32_t rows, hipStream_t stream) {
  if (!rows_ok(start, pos, sequences, rows) || !kv8_cache_ok(cache, sequences) || !type_ok(type) || k == nullptr ||
      v == nullptr || !aligned_to(k, type_bytes(type)) || !aligned_to(v, type_bytes(type)))
    return hipErrorInvalidValue;
  const std::size_t width = static_cast<std::size_t>(cache->n_kv_heads) * cache->head_dim;
  if (k_stride < width || v_stride < width || k_stride > (1u << 30) || v_stride > (1u << 30)) return hipErrorInvalidValue;
  const std::uint64_t units = start == nullptr ? sequences : units_of(sequences, rows, cache->block, 2u);
  const std::uint64_t grid = (units * 2u * cache->n_kv_heads + kWaves - 1u) / kWaves;
  if (grid * kThreads > 0xFFFFFFFFull) return hipErrorInvalidValue;
  const Kv8Ranges r = kv8_ranges(cache, sequences);
  for (int i = 0; i < 6; ++i)
    for (int j = 0; j < i; ++j)
      if (overlap(r.at[i], r.n[i], r.at[j], r.n[j])) return hipErrorInvalidValue;
  const std::uint64_t e = type_bytes(type);
  if (!apart(r, k, ((rows - 1u) * k_stride + width) * e) || !apart(r, v, ((rows - 1u) * v_stride + width) * e) ||
      !apart(r, pos, 4ull * sequences) || (start != nullptr && !apart(r, start, 4ull * sequences + 4u)) ||
      !apart(r, cache->block_table, 4ull * ((sequences - 1ull) * cache->table_stride + cache->capacity / cache->page_size)))
    return hipErrorInvalidValue;
  const Kv8Append a{{k, v}, {k_stride, v_stride}, {cache->k, cache->v}, {cache->k_scale, cache->v_scale},
                    {cache->k_tail, cache->v_tail}, static_cast<std::uint32_t>(units), cache->block};
  const CallRows call{start, pos, sequences, rows};
  const RowsCache view = kv8_view(cache);
  const bool e4m3 = cache->format == RTXLLM_KV8_E4M3, f16 = type == RTXLLM_F16;
  const auto n = static_cast<std::uint32_t>(grid);
  if (cache->head_dim == 64u)
    launch_append_block<8>(cache->block, e4m3, f16, n, a, call, view, stream);
  else if (cache->head_dim == 128u)
    launch_append_block<16>(cache->block, e4m3, f16, n, a, call, view, stream);
  else
    launch_append_block<32>(cache->block, e4m3, f16, n, a, call, view, stream);
  return hipGetLastError();
}

extern "C" hipError_t rtxllm_kv8_read(const rtxllm_paged_kv8* cache, const uint32_t* held, const uint32_t* start,
                                      const uint32_t* pos, uint32_t sequences, uint32_t rows, int type, void* k_out,
                                      void* v_out, hipStream_t stream) {
  if (!rows_ok(start, pos, sequences, rows) || !kv8_cache_ok(cache, sequences) || !type_ok(type) || held == nullptr ||
      !aligned_to(held, 4u) || (k_out == nullptr && v_out == nullptr) || !aligned_to(k_out, type_bytes(type)) ||
      !aligned_to(v_out, type_bytes(type)))
    return hipErrorInvalidValue;
  const std::uint64_t bytes = type_bytes(type) * static_cast<std::uint64_t>(rows) * cache->n_kv_heads * cache->head_dim;
  if (static_cast<std::uint64_t>(rows) * cache->n_kv_heads * (cache->head_dim / 8u) > 0xFFFFFF00ull) return hipErrorInvalidValue;
  const Kv8Ranges r = kv8_ranges(cache, sequences);
  const std::uint64_t table = 4ull * ((sequences - 1ull) * cache->table_stride + cache->capacity / cache->page_size);
  for (const void* o : {k_out, v_out})
    if (o != nullptr && (!apart(r, o, bytes) || overlap(o, bytes, held, 4ull * sequences) || overlap(o, bytes, pos, 4ull * sequences) ||
                         (start != nullptr && overlap(o, bytes, start, 4ull * sequences + 4u)) ||
                         overlap(o, bytes, cache->block_table, table)))
      return hipErrorInvalidValue;
  if (k_out != nullptr && v_out != nullptr && overlap(k_out, bytes, v_out, bytes)) return hipErrorInvalidValue;
  Kv8Read a{held, {k_out, v_out}};
  RowsCache view = kv8_view(cache);
  if (k_out == nullptr) {  // v alone
    a.out[0] = v_out, a.out[1] = nullptr;
    view.k = view.v, view.ks = view.vs, view.kt = view.vt;
  }
  const CallRows call{start, pos, sequences, rows};
  const bool e4m3 = cache->format == RTXLLM_KV8_E4M3, f16 = type == RTXLLM_F16;
  if (cache->head_dim == 64u)
    launch_read<8>(e4m3, f16, a, call, view, stream);
  else if (cache->head_dim == 128u)
    launch_read<16>(e4m3, f16, a, call, view, stream);
  else
    launch_read<32>(e4m3, f16, a, call, view, stream);
  return hipGetLastError();
}
