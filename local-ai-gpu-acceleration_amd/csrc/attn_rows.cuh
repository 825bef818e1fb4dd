// Device helpers that the kernels of attention over new rows share.
#pragma once

#include "attn_rows.h"
#include "common.h"
#include "layer_common.cuh"

namespace rtxllm {

typedef std::uint16_t u16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 half2 __attribute__((ext_vector_type(2)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half4_any __attribute__((ext_vector_type(4), aligned(2)));
typedef _Float16 half8_any __attribute__((ext_vector_type(8), aligned(2)));
typedef std::uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef std::uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef std::uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ std::uint32_t from_lane(std::uint32_t v, std::uint32_t lane) {
  return static_cast<std::uint32_t>(__builtin_amdgcn_ds_bpermute(static_cast<int>(4u * lane), static_cast<int>(v)));
}

// Two values as fp16, each 1152 too large: 1024 + (code + 128) is 0x6400 | the code with its top bit turned.
__device__ __forceinline__ std::uint32_t less_1152(std::uint32_t w) {
  const half2 bias = {static_cast<_Float16>(1152.0f), static_cast<_Float16>(1152.0f)};
  return __builtin_bit_cast(std::uint32_t, __builtin_bit_cast(half2, w) - bias);
}

// Four codes of a word as fp16, exactly.
template <Cached F>
__device__ __forceinline__ uint2 codes_to_half(std::uint32_t w) {
  if constexpr (F == Cached::kInt8) {
    w ^= 0x80808080u;
    return make_uint2(less_1152(__builtin_amdgcn_perm(0x64646464u, w, 0x05010400u)),
                      less_1152(__builtin_amdgcn_perm(0x64646464u, w, 0x07030602u)));
  } else {
    return make_uint2(__builtin_bit_cast(std::uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false)),
                      __builtin_bit_cast(std::uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true)));
  }
}

// log2(e) / sqrt(head_dim)
template <int D>
constexpr float score_scale() { return 1.4426950408889634f / (D == 64 ? 8.0f : D == 128 ? 11.313708498984761f : 16.0f); }

// Four values of a result, of either type, at any alignment to an element.
__device__ __forceinline__ void store_row4(const AttnRows& a, std::size_t at, f32x4 v) {
  if (a.f16 != 0u) {
    const half4 r = {static_cast<_Float16>(v[0]), static_cast<_Float16>(v[1]), static_cast<_Float16>(v[2]), static_cast<_Float16>(v[3])};
    *reinterpret_cast<half4_any*>(static_cast<_Float16*>(a.out) + at) = half4_any(r);
  } else {
    *reinterpret_cast<f32x4_any*>(static_cast<float*>(a.out) + at) = f32x4_any(v);
  }
}

// Two fp16 values without those that are not finite; whether there were any. A tile that some rows of a unit see in
// part is taken without them (0 times them would not be 0); rows that see them get their NaN at the end.
__device__ __forceinline__ bool finite_only(std::uint32_t& w) {
  const bool lo = (w & 0x7C00u) == 0x7C00u, hi = (w & 0x7C000000u) == 0x7C000000u;
  w = lo || hi ? w & ((lo ? 0u : 0xFFFFu) | (hi ? 0u : 0xFFFF0000u)) : w;
  return lo || hi;
}

// That end: NaN where a row sees a value of tiles [u0, u1) that is not finite (SCALES: also by its scale). All threads of
// the workgroup, behind its results' writes.
template <int D, bool CODES, bool SCALES>
__device__ __forceinline__ void not_finite_rows(const AttnRows& a, const CallRows& rows, const RowsCache& kv, std::uint32_t unit,
                                                std::uint32_t g, std::uint32_t split, std::uint32_t tile, std::uint32_t round) {
  asm volatile("" : "+s"(unit));  // (all of this is found anew: nothing is kept for it)
  const RowSpan sp = row_span(rows, kv, unit, a.tq, a.window, a.sinks, tile);
  const std::uint32_t per = span_per(sp.total, a.splits, round), u0 = split * per, u1 = u0 + per < sp.total ? u0 + per : sp.total;
  const std::int32_t* const table = kv.p.table + static_cast<std::size_t>(sp.s) * kv.p.table_stride;
  const bool whole = per >= sp.total;
  __syncthreads();
#pragma unroll 1
  for (std::uint32_t u = u0; u < u1; ++u) {
    const std::uint32_t j0 = u < sp.ncode ? span_position(sp, u, tile) : sp.tail + (u - sp.ncode) * tile;
#pragma unroll 1
    for (std::uint32_t x = threadIdx.x; x < tile * D; x += blockDim.x) {
      const std::uint32_t j = j0 + x / D, d = x % D;
      if (j > sp.plast) continue;
      bool bad = false;
      if (u >= sp.ncode) {
        const std::uint32_t block = 1u << kv.block_shift;
        bad = CODES && (kv.vt[((static_cast<std::size_t>(sp.s) * kv.p.n_kv + g) * block + (j & (block - 1u))) * D + d] & 0x7C00u) == 0x7C00u;
      } else if (j < sp.code_end) {
        const std::uint32_t r = paged_slot_row(kv.p, table, g, j);
        if (r != kNoRow) {
          if constexpr (!CODES)
            bad = (reinterpret_cast<const std::uint16_t*>(kv.v)[static_cast<std::size_t>(r) * D + d] & 0x7C00u) == 0x7C00u;
          else if constexpr (SCALES)
            bad = !(fabsf(kv.vs[r >> kv.block_shift]) < INFINITY);
        }
      }
      if (!bad) continue;
#pragma unroll 1
      for (std::uint32_t i = 0; i < sp.nq; ++i) {
        const std::uint32_t p = row_pos(sp.pos, i, kv.p.capacity);
        if (j > p || !(p - j < a.window || j < a.sinks)) continue;
#pragma unroll 1
        for (std::uint32_t h = 0; h < a.group; ++h) {
          const std::size_t at = (static_cast<std::size_t>(sp.row + i) * a.group * kv.p.n_kv + g * a.group + h) * D + d;
          if (!whole)
            a.part[(((static_cast<std::size_t>(unit) * kv.p.n_kv + g) * (a.tq * a.group) + i * a.group + h) * a.splits + split) * D + d] = NAN;
          else if (a.f16 != 0u)
            static_cast<_Float16*>(a.out)[at] = static_cast<_Float16>(NAN);
          else
            static_cast<float*>(a.out)[at] = NAN;
        }
      }
    }
  }
}

}  // namespace rtxllm
