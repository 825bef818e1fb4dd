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
    // (through the caches: a line's halves are two reads; past them a prompt's 17.1 us are 22.2)
    const f32x4_any a = *reinterpret_cast<const f32x4_any*>(f), b = *reinterpret_cast<const f32x4_any*>(f + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = static_cast<_Float16>(a[i]), h[i + 4] = static_cast<_Float16>(b[i]);
  }
  return h;
}

// Eight codes of values x / scale, as two words. c, the integer nearest to x inv, is the code or, next to a half, one
// off; adding 1.5 2^23 rounds to it (half to even) and leaves it in the low byte. x - c scale is exact in one fma (a
// multiple of scale's last bit below scale), so twice its size against scale says without rounding on which side of
// the half the quotient lies; an odd c gives way at the half itself (scale less its last bit). No branch: one that a
// wave in thirty took made a prompt's 24 us 29, by its longest waves.
__device__ __forceinline__ uint2 int8_codes(half8 v, float inv, float scale) {
  constexpr float kMagic = 12582912.0f;
  std::uint32_t w[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float x = static_cast<float>(v[j]), t = fmaf(x, inv, kMagic), r = fmaf(kMagic - t, scale, x);
    const std::uint32_t c = __float_as_uint(t);
    const bool beyond = 2.0f * fabsf(r) > __uint_as_float(__float_as_uint(scale) - (c & 1u));
    w[j] = c + (beyond ? static_cast<std::uint32_t>(static_cast<std::int32_t>(__float_as_uint(r)) >> 31) | 1u : 0u);
  }
  auto four = [](std::uint32_t a, std::uint32_t b, std::uint32_t c, std::uint32_t d) {  // low bytes
    return __builtin_amdgcn_perm(__builtin_amdgcn_perm(d, c, 0x0C0C0400u), __builtin_amdgcn_perm(b, a, 0x0C0C0400u), 0x05040100u);
  };
  return make_uint2(four(w[0], w[1], w[2], w[3]), four(w[4], w[5], w[6], w[7]));
}

// One wave an item: a block that new rows touch, of one kv head, of k or of v. L = head_dim / 8 lanes
// hold a position, 8 values each, R = block L / 64 positions a lane. A whole block is read
// (its first positions from the tail where an earlier call brought them), its largest magnitude found
// across the wave, and its codes leave in one piece, since a block of a head lies in one piece in its
// page. Values that stay in the open block go to the tail; where the call also makes an earlier block
// whole from the same tail, that block's wave writes them, once it has read. From R = 8
// on the four waves of a workgroup share an item. Bound by bytes: 8192 tokens of 8 heads of 128 in fp32 (84 MB) as int8
// 17.2 us, 4.9 TB/s; a step of few tokens by a launch and the chain position, input, tail (3.9 us).
template <int L, int R, bool E4M3, bool F16>
__global__ __launch_bounds__(kThreads) void kv8_append_kernel(Kv8Append a, CallRows rows, RowsCache kv) {
  constexpr std::uint32_t D = 8u * L, kStep = 64u / L;  // positions of a round
  constexpr bool SHARED = append_shared(R);
  constexpr int RW = SHARED ? R / 4 : R;  // rounds of a wave
  __shared__ std::uint32_t tops[kWaves];
  const std::uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), item = SHARED ? blockIdx.x : blockIdx.x * kWaves + wave;
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
  const std::uint32_t lane = threadIdx.x & 63u, part = lane % L, col = g * D + 8u * part;
  const std::uint32_t in = (SHARED ? threadIdx.x : lane) / L, step = SHARED ? kWaves * kStep : kStep;
  std::uint16_t* const tail = a.tail[which] + (static_cast<std::size_t>(s) * kv.p.n_kv + g) * a.block * D + 8u * part;
  const void* const x = a.x[which];
  const std::size_t stride = a.stride[which];
  auto value = [&](std::uint32_t p) { return load8<F16>(x, static_cast<std::size_t>(q.row + (p - q.pos)) * stride + col); };
  auto to_tail = [&](std::uint32_t from) {
    for (std::uint32_t p = from + in; p < end; p += step)
      if (p >= q.pos) *reinterpret_cast<half8*>(tail + (p & (a.block - 1u)) * D) = value(p);
  };
  const std::uint32_t open = end & ~(a.block - 1u);  // the open block's start
  if (b0 + a.block > end) {
    if (t == 0u || q.pos == first) to_tail(b0);  // (else the first block's wave)
    return;
  }
  const std::uint32_t row = paged_slot_row(kv.p, kv.p.table + static_cast<std::size_t>(s) * kv.p.table_stride, g, b0);
  half8 v[RW];
#pragma unroll
  for (int i = 0; i < RW; ++i) {
    const std::uint32_t p = b0 + in + step * i;
    v[i] = p < q.pos ? *reinterpret_cast<const half8*>(tail + (p & (a.block - 1u)) * D) : value(p);
  }
  // fp16 magnitudes compare as their bits, numbers that are not finite above all
  u16x2 most = {0, 0};
#pragma unroll
  for (int i = 0; i < RW; ++i) {
    const u32x4 w = __builtin_bit_cast(u32x4, v[i]);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const std::uint32_t m = w[j] & 0x7FFF7FFFu;
      most = __builtin_elementwise_max(most, __builtin_bit_cast(u16x2, m));
    }
  }
  std::uint32_t top = most[0] > most[1] ? most[0] : most[1];
  top = lanes_reduce_exact(top, [](std::uint32_t x, std::uint32_t y) { return x > y ? x : y; });
  if constexpr (SHARED) {
    if (lane == 0u) tops[wave] = top;
    __syncthreads();
#pragma unroll
    for (std::uint32_t i = 0; i < kWaves; ++i) top = top > tops[i] ? top : tops[i];
  }
  if (t == 0u && q.pos != first && open < end) {  // the tail has been read: no wave but this one touches it
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    to_tail(open);
  }
  if (row == kNoRow) return;
  const bool finite = top < 0x7C00u, some = finite && top != 0u;
  const float amax = static_cast<float>(__builtin_bit_cast(_Float16, static_cast<unsigned short>(top)));
  float scale, inv;
  if constexpr (E4M3) {  // amax = 2^e m: 448 = 1.75 2^8
    const std::uint32_t bits = __float_as_uint(amax);
    const std::uint32_t e = (bits >> 23) - 8u + ((bits & 0x7FFFFFu) > 0x600000u ? 1u : 0u);
    scale = __uint_as_float(e << 23), inv = __uint_as_float((254u - e) << 23);
  } else {
    scale = amax * (1.0f / 127.0f), inv = 1.0f / scale;
  }
  std::uint8_t* const out = a.codes[which] + static_cast<std::size_t>(row) * D + 8u * part;
#pragma unroll
  for (int i = 0; i < RW; ++i) {
    uint2 c = make_uint2(0u, 0u);
    if (some) {
      if constexpr (E4M3) {
        int lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[i][0] * inv, v[i][1] * inv, 0, false);
        lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[i][2] * inv, v[i][3] * inv, lo, true);
        int hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[i][4] * inv, v[i][5] * inv, 0, false);
        hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[i][6] * inv, v[i][7] * inv, hi, true);
        c = make_uint2(static_cast<std::uint32_t>(lo), static_cast<std::uint32_t>(hi));
      } else {
        c = int8_codes(v[i], inv, scale);
      }
    }
    *reinterpret_cast<uint2*>(out + static_cast<std::size_t>(in + step * i) * D) = c;
  }
  if ((SHARED ? threadIdx.x : lane) == 0u) a.scale[which][row >> kv.block_shift] = !finite ? NAN : some ? scale : 0.0f;
}

struct Kv8Read {
  const std::uint32_t* held;
  void* out[2];
};

// L lanes a position of a head, 8 values each; the heads of a row lie next to each other in the result. A lane takes
// kUnits positions of heads a workgroup's width apart, whose reads, each behind two others (the table's and the
// sequence's), are in flight together. Bound by bytes: 65530 positions of 8 heads of 128 (134 MB of codes) as fp16 85.9 us, as
// fp32 133 (2 / 4 / 8 positions a lane: 102 / 86 / 96, 155 / 146 / 133; through the caches 89, 164).
template <int L, bool E4M3, bool F16, bool MANY>
__global__ __launch_bounds__(kThreads) void kv8_read_kernel(Kv8Read a, CallRows rows, RowsCache kv) {
  constexpr std::uint32_t D = 8u * L, kPer = kThreads / L;
  constexpr int kUnits = MANY ? read_units(F16) : 1;
  const std::uint32_t part = threadIdx.x % L, which = blockIdx.y, block = 1u << kv.block_shift;
  const std::uint32_t units = rows.rows * kv.p.n_kv;
  const std::uint8_t* const codes = which == 0u ? kv.k : kv.v;
  const float* const scales = which == 0u ? kv.ks : kv.vs;
  std::uint32_t unit[kUnits], s[kUnits], g[kUnits], p[kUnits];
  std::int32_t page[kUnits];
  bool there[kUnits], tail[kUnits];
#pragma unroll
  for (int i = 0; i < kUnits; ++i) {
    unit[i] = (blockIdx.x * kUnits + i) * kPer + threadIdx.x / L;
    const std::uint32_t u = unit[i] < units ? unit[i] : units - 1u, r = u / kv.p.n_kv;
    std::uint32_t base;
    g[i] = u - r * kv.p.n_kv;
    s[i] = rows.start == nullptr ? r : unit_sequence(rows, r, 1u, 0u, base);  // the last that does not start behind the row
    const SeqRows q = seq_rows(rows, s[i]);
    const std::uint32_t held = a.held[s[i]] < kv.p.capacity ? a.held[s[i]] : kv.p.capacity;
    there[i] = unit[i] < units && r >= q.row && r - q.row < q.n && q.pos < held && r - q.row < held - q.pos;
    p[i] = there[i] ? q.pos + (r - q.row) : 0u;
    tail[i] = there[i] && p[i] >= (held & ~(block - 1u));
    page[i] = kv.p.table[static_cast<std::size_t>(s[i]) * kv.p.table_stride + page_of(kv.p, p[i])];
  }
  uint2 c[kUnits];
  float scale[kUnits];
#pragma unroll
  for (int i = 0; i < kUnits; ++i) {
    const std::uint32_t row = paged_row(kv.p, page[i], g[i], p[i] - page_of(kv.p, p[i]) * kv.p.page_size);
    there[i] = there[i] && (tail[i] || row != kNoRow);
    const std::uint32_t at = row != kNoRow ? row : 0u;
    typedef std::uint32_t u32x2 __attribute__((ext_vector_type(2)));
    const u32x2 w = __builtin_nontemporal_load(reinterpret_cast<const u32x2*>(codes + static_cast<std::size_t>(at) * D + 8u * part));
    c[i] = make_uint2(w[0], w[1]);
    scale[i] = scales[at >> kv.block_shift];
  }
#pragma unroll
  for (int i = 0; i < kUnits; ++i) {
    float x[8];
    if constexpr (E4M3) {
      auto four = [&](std::uint32_t u, float* f) {
        const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(u), false);
        const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(u), true);
        f[0] = lo[0], f[1] = lo[1], f[2] = hi[0], f[3] = hi[1];
      };
      four(c[i].x, x), four(c[i].y, x + 4);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        x[j] = static_cast<float>(static_cast<std::int8_t>(c[i].x >> (8 * j)));
        x[j + 4] = static_cast<float>(static_cast<std::int8_t>(c[i].y >> (8 * j)));
      }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] *= scale[i];
    if (tail[i]) {
      const half8 h = *reinterpret_cast<const half8*>((which == 0u ? kv.kt : kv.vt) +
                                                      ((static_cast<std::size_t>(s[i]) * kv.p.n_kv + g[i]) * block + (p[i] & (block - 1u))) * D + 8u * part);
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = static_cast<float>(h[j]);
    }
    if (!there[i]) continue;
    const std::size_t at = static_cast<std::size_t>(unit[i]) * D + 8u * part;
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
}

template <int L, int R>
void launch_append(bool e4m3, bool f16, const Kv8Append& a, const CallRows& rows, const RowsCache& kv, hipStream_t stream) {
  const std::uint64_t items = 2ull * a.units * kv.p.n_kv;
  const dim3 grid(static_cast<std::uint32_t>(append_shared(R) ? items : (items + kWaves - 1u) / kWaves));
  auto run = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(kThreads), 0, stream, a, rows, kv); };
  if (e4m3) {
    f16 ? run(kv8_append_kernel<L, R, true, true>) : run(kv8_append_kernel<L, R, true, false>);
  } else {
    f16 ? run(kv8_append_kernel<L, R, false, true>) : run(kv8_append_kernel<L, R, false, false>);
  }
}

template <int L>
void launch_append_block(std::uint32_t block, bool e4m3, bool f16, const Kv8Append& a, const CallRows& rows,
                         const RowsCache& kv, hipStream_t stream) {
  constexpr int R = L / 8;  // of a block of 8
  if (block == 8u) return launch_append<L, R>(e4m3, f16, a, rows, kv, stream);
  if (block == 16u) return launch_append<L, 2 * R>(e4m3, f16, a, rows, kv, stream);
  if (block == 32u) return launch_append<L, 4 * R>(e4m3, f16, a, rows, kv, stream);
  launch_append<L, 8 * R>(e4m3, f16, a, rows, kv, stream);
}

template <int L>
void launch_read(bool e4m3, bool f16, const Kv8Read& a, const CallRows& rows, const RowsCache& kv, hipStream_t stream) {
  const std::uint64_t units = static_cast<std::uint64_t>(rows.rows) * kv.p.n_kv;
  const bool many = read_many(units, L, f16);
  const std::uint64_t per = (many ? read_units(f16) : 1) * kThreads / L;
  // both, or k (y 0), or v alone (moved to y 0 by the caller)
  const dim3 grid(static_cast<std::uint32_t>((units + per - 1u) / per), a.out[1] != nullptr ? 2u : 1u);
  auto run = [&](auto one, auto more) { hipLaunchKernelGGL(many ? more : one, grid, dim3(kThreads), 0, stream, a, rows, kv); };
  if (e4m3) {
    f16 ? run(kv8_read_kernel<L, true, true, false>, kv8_read_kernel<L, true, true, true>)
        : run(kv8_read_kernel<L, true, false, false>, kv8_read_kernel<L, true, false, true>);
  } else {
    f16 ? run(kv8_read_kernel<L, false, true, false>, kv8_read_kernel<L, false, true, true>)
        : run(kv8_read_kernel<L, false, false, false>, kv8_read_kernel<L, false, false, true>);
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
  if (units * 2u * cache->n_kv_heads * kThreads > 0xFFFFFFFFull) return hipErrorInvalidValue;
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
  if (cache->head_dim == 64u)
    launch_append_block<8>(cache->block, e4m3, f16, a, call, view, stream);
  else if (cache->head_dim == 128u)
    launch_append_block<16>(cache->block, e4m3, f16, a, call, view, stream);
  else
    launch_append_block<32>(cache->block, e4m3, f16, a, call, view, stream);
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
