// Device helpers that the kernels of attention over new rows share.
#pragma once

#include "attn_rows.h"
#include "common.h"
#include "layer_common.cuh"

namespace rtxllm {

typedef _Float16 half2 __attribute__((ext_vector_type(2)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half4_any __attribute__((ext_vector_type(4), aligned(2)));
typedef _Float16 half8_any __attribute__((ext_vector_type(8), aligned(2)));
typedef std::uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef std::uint32_t u32x4 __attribute__((ext_vector_type(4)));
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

}  // namespace rtxllm
