// Attention of new rows over a paged cache, the form for many rows a sequence: tiles
// of keys and values in the LDS, shared by the query rows of a workgroup.
#include "attn_rows.cuh"

namespace rtxllm {
namespace {

constexpr std::uint32_t kTile = kPromptTile;  // 64 positions
constexpr int kLift = 11;          // F16: softmax terms are 2^11 times what they are to the maximum they count from,
constexpr float kSlack = 4.0f;     // which may lag 2^4 behind: 2^15 at most
constexpr int kPairLift = 15;      // F32: exact maxima, as in attn_rows.hip

// Where a row's 16-byte slots lie, so that what the lanes of one phase of an LDS access touch (16 of them for a
// 16-byte read, of two quarters and not in a row) covers its 64 banks once: 16 keys' rows of 256 bytes (of 128: two rows
// a line), dimensions' rows of 128, read 16 at a time and written four apart.
template <int D>
__device__ __forceinline__ std::uint32_t key_slot(std::uint32_t row, std::uint32_t slot) {
  return slot ^ (D == 64 ? (row >> 1) & 7u : row & 15u);
}
__device__ __forceinline__ std::uint32_t value_slot(std::uint32_t d, std::uint32_t slot) {
  return slot ^ ((d >> 1) & 7u) ^ ((d >> 4) & 1u);
}

// A barrier that waits for the LDS alone: reads of the cache stay in flight across it.
__device__ __forceinline__ void lds_barrier() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// One workgroup of eight waves per (unit, kv head, split). A unit is up to tq query rows times the kv head's query
// heads, 16 NB columns a wave; tiles of 64 positions go through the LDS as fp16, twice buffered: while a tile is
// computed the next one's codes are on their way into registers, and become fp16 once it is done.
//  * scores: S = K q^T by v_mfma_f32_16x16x32_f16, keys' rows from the LDS, q in registers (F32: an fp16 pair, lifted as
//    in attn_rows.hip); an 8-bit key enters as its code, its scale multiplies the scores of four positions at a time;
//  * terms: as fp16 pairs. F32 as in attn_rows.hip. F16: p = 2^(s - m + 11), where the m counted from may lag up to 2^4
//    behind the maximum, so that it hardly ever moves. An 8-bit value's scale over 2^E multiplies its term before it is
//    split, E the column's own as in attn_rows.hip, so that what a row does not see takes no bits from it. (8192 rows
//    over int8 codes, us: terms as one fp16 717, but off by as much as the result's own rounding, and only in calls that
//    take this form; pairs relative to the largest scale that any row of the unit had seen 842; the column's own 867.)
//  * o += V^T p, values turned when they are stored ([dimension][position], the positions in the order in which the
//    scores' layout holds their terms), so that both products read 16 bytes a lane.
// Bound by what a wave issues: at two waves a SIMD vector instructions take 67 % of the cycles and matrix ones 40 %, with
// hardly any overlap: 8192 rows over int8 codes, 32 heads over 8 kv heads of 128, 867 us, over fp16 pages 435 for 8000 rows
// with a window of 2048. Columns a wave: heads of 128 32, which fill the registers; heads of 64 64 (spills of up to 25
// registers; 48 without spills 747 us instead of 645), in fp32 16, at four waves a SIMD (765 us; five registers more, and so
// two waves, were 1126).
template <int D, Cached F, bool F32, int NB, int NW>
__global__ __launch_bounds__(64 * NW, F32 && D == 64 ? 4 : 2) void attn_prompt_kernel(AttnRows a, CallRows rows, RowsCache kv) {
  constexpr bool CODES = F != Cached::kF16;
  constexpr int BYTES = CODES ? 1 : 2, T = 64 * NW, J = D / 32, B = D / 16;
  constexpr int KC = (64 * D * BYTES / 16 + T - 1) / T;  // 16-byte pieces of keys a thread
  constexpr int VU = (4 * D + T - 1) / T;                // units of values a thread: 4 positions of 4 dimensions
  constexpr int KL = D * BYTES / 16;                     // pieces of a row
  constexpr bool AHEAD = !F32 && (D == 128 || (D == 64 && !CODES));
  typedef std::uint32_t vword __attribute__((ext_vector_type(BYTES)));
  __shared__ __align__(16) std::uint8_t keys[2][64 * D * 2];
  __shared__ __align__(16) std::uint8_t vals[2][64 * D * 2];  // [dimension][position], positions as the products take them
  // of each position: its key's scale, its value's, log2 of that in whole powers of two (-infinity: none)
  __shared__ __align__(16) float scales[2][CODES ? 64 : 1][4];
  __shared__ std::uint32_t odd;

  const std::uint32_t g = blockIdx.x % kv.p.n_kv, us = blockIdx.x / kv.p.n_kv, split = us % a.splits;
  const std::uint32_t unit = a.units - 1u - us / a.splits;  // the last rows, which see most, first
  const RowSpan sp = row_span(rows, kv, unit, a.tq, a.window, a.sinks, kTile);
  if (sp.nq == 0u) return;
  const std::uint32_t per = span_per(sp.total, a.splits, 1u), u0 = split * per;
  if (u0 >= sp.total) return;
  const std::uint32_t u1 = u0 + per < sp.total ? u0 + per : sp.total, code1 = u1 < sp.ncode ? u1 : sp.ncode;
  const std::uint32_t tid = threadIdx.x, lane = tid & 63u, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const std::uint32_t col = lane & 15u, qq = lane >> 4;
  const std::uint32_t n_heads = a.group * kv.p.n_kv, cap = kv.p.capacity;
  const std::int32_t* const table = kv.p.table + static_cast<std::size_t>(sp.s) * kv.p.table_stride;

  // The lane's columns: query row and head, the row's position; B operands of the scores.
  std::uint32_t pc[NB];
  half8 qh[NB][J], ql[F32 ? NB : 1][F32 ? J : 1];
  float qscale[NB];
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    const std::uint32_t c = (wave * NB + n) * 16u + col;
    const std::uint32_t ci = c / a.group;
    const bool mine = ci < sp.nq;
    const std::uint32_t i = mine ? ci : 0u, h = mine ? c - ci * a.group : 0u;
    pc[n] = row_pos(sp.pos, i, cap);
    const std::size_t at = (static_cast<std::size_t>(sp.row + i) * n_heads + g * a.group + h) * D + 8u * qq;
    if constexpr (F32) {
      float x[J][8], top = 0.0f;
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const float* f = static_cast<const float*>(a.q) + at + 32 * j;
        const f32x4_any lo = *reinterpret_cast<const f32x4_any*>(f), hi = *reinterpret_cast<const f32x4_any*>(f + 4);
#pragma unroll
        for (int k = 0; k < 4; ++k) x[j][k] = lo[k], x[j][k + 4] = hi[k];
#pragma unroll
        for (int k = 0; k < 8; ++k) top = fmaxf(top, fabsf(x[j][k]));
      }
      top = fmaxf(top, lane_xor<16>(top));
      top = fmaxf(top, lane_xor<32>(top));
      int e = 0;
      if (top > 0.0f && top < INFINITY) frexpf(top, &e);
      qscale[n] = ldexpf(score_scale<D>(), e - 15);
#pragma unroll
      for (int j = 0; j < J; ++j)
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          float v = mine ? ldexpf(x[j][k], 15 - e) : 0.0f;
          asm("" : "+v"(v));  // one rounded value for hi and lo
          qh[n][j][k] = static_cast<_Float16>(v);
          ql[n][j][k] = static_cast<_Float16>(v - static_cast<float>(qh[n][j][k]));
        }
    } else {
      qscale[n] = score_scale<D>();
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const half8 t = half8(*reinterpret_cast<const half8_any*>(static_cast<const _Float16*>(a.q) + at + 32 * j));
        qh[n][j] = mine ? t : half8{};
      }
    }
  }
  // positions of the wave's rows; those of a wave without rows see nothing
  const std::uint32_t c0 = wave * NB * 16u, cols = sp.nq * a.group, c1 = c0 + NB * 16u < cols ? c0 + NB * 16u : cols;
  const bool idle = c0 >= cols;
  const std::uint32_t pa = row_pos(sp.pos, idle ? 0u : c0 / a.group, cap), pb = row_pos(sp.pos, idle ? 0u : (c1 - 1u) / a.group, cap);

  float m[NB], l[NB];
  float lead[NB];  // codes: the largest log2 of a position's term times its value's scale (it may lag as m does),
  int E[NB];       // lead - m in whole powers of two, over which o is held
  f32x4 o[NB][B];
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    m[n] = -INFINITY, l[n] = 0.0f, lead[n] = -INFINITY, E[n] = 0;
#pragma unroll
    for (int b = 0; b < B; ++b) o[n][b] = f32x4{};
  }

  // ---- a tile on its way: which rows, their pieces in registers, then in the LDS ----
  u32x4 kraw[KC];
  vword vraw[VU][4];
  std::uint32_t row = 0u;  // of the lane's position
  unsigned long long seen = 0ull;
  std::int32_t page = 0;
  float ks1 = 0.0f, vs1 = 0.0f;
  auto first_of = [&](std::uint32_t u) { return u < sp.ncode ? span_position(sp, u, kTile) : sp.tail + (u - sp.ncode) * kTile; };
  auto some_row = [&](std::uint32_t j) { return j <= sp.plast && (j + a.window > sp.p0 || j < a.sinks); };
  // Unit x of a tile's values: dimensions 4 unit_dims.., positions 4 unit_quad..; neighbours take both 8-byte
  // halves of a slot.
  auto unit_dims = [](std::uint32_t x) { return x / 2u % (D / 4); };
  auto unit_quad = [](std::uint32_t x) {
    const std::uint32_t y = x / (D / 2);  // 0..7
    return (y & 3u) + 4u * (x & 1u) + 8u * (y >> 2);
  };
  auto load_page = [&](std::uint32_t u) {
    const std::uint32_t j = span_position(sp, u < code1 ? u : (code1 != 0u ? code1 - 1u : 0u), kTile) + lane;
    return table[page_of(kv.p, j < cap ? j : cap - 1u)];
  };
  auto load_tile = [&](std::uint32_t u) {  // a tile in the pages, from `page`
    const std::uint32_t j = span_position(sp, u, kTile) + lane, jc = j < cap ? j : cap - 1u;
    const std::uint32_t r = paged_row(kv.p, page, g, jc - page_of(kv.p, jc) * kv.p.page_size);
    const bool there = j < sp.code_end && r != kNoRow;
    row = there ? r : 0u;
    seen = __ballot(there && some_row(j));
#pragma unroll
    for (int i = 0; i < KC; ++i) {
      const std::uint32_t piece = tid + T * i, at = from_lane(row, (piece / KL) & 63u);
      if (64 * KL % T == 0 || piece < 64u * KL)
        kraw[i] = reinterpret_cast<const u32x4*>(kv.k + static_cast<std::size_t>(at) * (D * BYTES))[piece % KL];
    }
#pragma unroll
    for (int i = 0; i < VU; ++i) {
      const std::uint32_t x = tid + T * i, quad = unit_quad(x) & 15u, at = from_lane(row, 4u * quad);
      if (4 * D % T == 0 || x < 4u * D) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          vraw[i][e] = reinterpret_cast<const vword*>(kv.v + static_cast<std::size_t>(at + e) * (D * BYTES))[unit_dims(x)];
      }
    }
    if constexpr (CODES) {
      ks1 = kv.ks[row >> kv.block_shift];
      vs1 = kv.vs[row >> kv.block_shift];
    }
  };
  // Values of four dimensions, each four positions (one 8-byte write each)
  auto put_values = [&](int buf, std::uint32_t x, const uint2* v) {
    const std::uint32_t quad = unit_quad(x), d0 = 4u * unit_dims(x);
    const std::uint32_t slot = 4u * (quad / 8u) + (quad & 3u), half = (quad >> 2) & 1u;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      *reinterpret_cast<uint2*>(&vals[buf][(d0 + i) * 128u + 16u * value_slot(d0 + i, slot) + 8u * half]) = v[i];
  };
  auto turn_halves = [&](const u32x2* w, uint2* v) {  // w[e]: dimensions 0..3 of position e
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const std::uint32_t sel = (i & 1) != 0 ? 0x07060302u : 0x05040100u;
      v[i] = make_uint2(__builtin_amdgcn_perm(w[1][i / 2], w[0][i / 2], sel), __builtin_amdgcn_perm(w[3][i / 2], w[2][i / 2], sel));
    }
  };
  auto drop = [](u32x2& w) {
    std::uint32_t lo = w[0], hi = w[1];
    const bool bad_lo = finite_only(lo), bad_hi = finite_only(hi);
    w = u32x2{lo, hi};
    return bad_lo || bad_hi;
  };
  // Whether some row of the unit does not see all of a tile that some row sees.
  auto is_edge = [&](std::uint32_t j0, unsigned long long s) {
    return s != ~0ull || j0 + kTile - 1u > sp.p0 || !(sp.plast - j0 < a.window || j0 + kTile <= a.sinks);
  };
  auto put_scales = [&](int buf) {
    if (wave != 0u) return;
    const bool number = vs1 < INFINITY && vs1 > -INFINITY;
    if (!number && (seen >> lane & 1ull) != 0ull) odd = 1u;  // (0 times what a row does not see must stay 0)
    const float v = number ? vs1 : 0.0f;
    const f32x4 x = {ks1, v, v > 0.0f ? static_cast<float>(__builtin_amdgcn_frexp_expf(v)) : -INFINITY, 0.0f};
    *reinterpret_cast<f32x4*>(scales[buf][lane]) = x;
  };
  auto store_tile = [&](int buf, std::uint32_t j0) {
    bool bad = false;
    const bool edge = !CODES && is_edge(j0, seen);
#pragma unroll
    for (int i = 0; i < KC; ++i) {
      const std::uint32_t piece = tid + T * i, r = piece / KL, c = piece % KL;
      if (64 * KL % T == 0 || piece < 64u * KL) {
        if constexpr (CODES) {
          const uint2 x0 = codes_to_half<F>(kraw[i][0]), x1 = codes_to_half<F>(kraw[i][1]);
          const uint2 x2 = codes_to_half<F>(kraw[i][2]), x3 = codes_to_half<F>(kraw[i][3]);
          *reinterpret_cast<uint4*>(&keys[buf][r * (D * 2) + 16u * key_slot<D>(r, 2u * c)]) = make_uint4(x0.x, x0.y, x1.x, x1.y);
          *reinterpret_cast<uint4*>(&keys[buf][r * (D * 2) + 16u * key_slot<D>(r, 2u * c + 1u)]) = make_uint4(x2.x, x2.y, x3.x, x3.y);
        } else {
          *reinterpret_cast<u32x4*>(&keys[buf][r * (D * 2) + 16u * key_slot<D>(r, c)]) = kraw[i];
        }
      }
    }
#pragma unroll
    for (int i = 0; i < VU; ++i) {
      const std::uint32_t x = tid + T * i, quad = unit_quad(x) & 15u;
      if (4 * D % T == 0 || x < 4u * D) {
        const auto mask = static_cast<std::uint32_t>(seen >> (4u * quad)) & 15u;
        if (mask != 15u && F != Cached::kInt8) {  // 0 times what no row sees must stay 0
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if ((mask >> e & 1u) == 0u) vraw[i][e] = vword{};
        }
        uint2 v[4];
        if constexpr (CODES) {
          const std::uint32_t w0 = vraw[i][0][0], w1 = vraw[i][1][0], w2 = vraw[i][2][0], w3 = vraw[i][3][0];
          const std::uint32_t ab = __builtin_amdgcn_perm(w1, w0, 0x05010400u), AB = __builtin_amdgcn_perm(w1, w0, 0x07030602u);
          const std::uint32_t cd = __builtin_amdgcn_perm(w3, w2, 0x05010400u), CD = __builtin_amdgcn_perm(w3, w2, 0x07030602u);
          v[0] = codes_to_half<F>(__builtin_amdgcn_perm(cd, ab, 0x05040100u));
          v[1] = codes_to_half<F>(__builtin_amdgcn_perm(cd, ab, 0x07060302u));
          v[2] = codes_to_half<F>(__builtin_amdgcn_perm(CD, AB, 0x05040100u));
          v[3] = codes_to_half<F>(__builtin_amdgcn_perm(CD, AB, 0x07060302u));
        } else {
          u32x2 w[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) w[e] = vraw[i][e];
          if (edge) {
#pragma unroll
            for (int e = 0; e < 4; ++e) bad |= drop(w[e]);
          }
          turn_halves(w, v);
        }
        put_values(buf, x, v);
      }
    }
    if constexpr (CODES) put_scales(buf);
    if (bad) odd = 1u;
  };
  // The newest block, fp16, at once.
  auto tail_tile = [&](int buf, std::uint32_t j0) {
    if constexpr (CODES) {
      std::uint32_t tid = threadIdx.x;
      asm volatile("" : "+v"(tid));  // (its addresses are not kept over the loop)
      const std::uint32_t lane = tid & 63u;
      const std::uint32_t block = 1u << kv.block_shift;
      const std::size_t base = (static_cast<std::size_t>(sp.s) * kv.p.n_kv + g) * block * D;
      seen = __ballot(some_row(j0 + lane));
      auto place = [&](std::uint32_t i) {
        const std::uint32_t j = j0 + i < sp.plast ? j0 + i : sp.plast;
        return base + static_cast<std::size_t>(j & (block - 1u)) * D;
      };
      for (std::uint32_t x = tid; x < 64u * (D / 8); x += T) {
        const std::uint32_t r = x / (D / 8), c = x % (D / 8);
        *reinterpret_cast<u32x4*>(&keys[buf][r * (D * 2) + 16u * key_slot<D>(r, c)]) = *reinterpret_cast<const u32x4*>(kv.kt + place(r) + 8u * c);
      }
      bool bad = false;
      for (std::uint32_t x = tid; x < 4u * D; x += T) {
        const std::uint32_t quad = unit_quad(x);
        u32x2 w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const u32x2 t = *reinterpret_cast<const u32x2*>(kv.vt + place(4u * quad + e) + 4u * unit_dims(x));
          w[e] = (seen >> (4u * quad + e) & 1u) != 0u ? t : u32x2{0u, 0u};
          bad |= drop(w[e]);
        }
        uint2 v[4];
        turn_halves(w, v);
        put_values(buf, x, v);
      }
      ks1 = vs1 = 1.0f;
      put_scales(buf);
      if (bad) odd = 1u;
    }
  };

  // ---- one tile's scores, terms and products, 32 positions at a time ----
  // Of the 16-byte slots that a lane reads only the low bits depend on more than a constant offset.
  constexpr int kKeyAts = D == 64 ? 2 : 4;
  std::uint32_t kat[kKeyAts], vat[4];
#pragma unroll
  for (int j = 0; j < kKeyAts; ++j) kat[j] = col * (D * 2u) + 16u * key_slot<D>(col, 4u * j + qq);
#pragma unroll
  for (int y = 0; y < 4; ++y) vat[y] = col * 128u + 16u * (value_slot(col, qq) ^ (y & 1) ^ (4u * (y >> 1)));  // odd b, x 1
  auto compute = [&](int buf, std::uint32_t j0, unsigned long long sees_any, bool tail) {
    // every column of the wave sees every position
    const bool plain = sees_any == ~0ull && j0 + kTile - 1u <= pa && (pb - j0 < a.window || j0 + kTile <= a.sinks);
    if (CODES && tail) {  // values of scale 1, whatever their size, and last: their terms alone say where they are held
#pragma unroll
      for (int n = 0; n < NB; ++n) lead[n] = -INFINITY;
    }
    const std::uint8_t* const kt = keys[buf];
    const std::uint8_t* const vt = vals[buf];
    // AHEAD: a half tile's values are read ahead of its softmax. (Its keys as well, ahead of the products before: spills,
    // 904 us where this was 842. Heads of 64 over codes: spills too, 670 instead of 644.)
    half8 kf[2][J];
    auto load_keys = [&](int x) {
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int j = 0; j < J; ++j)
          kf[t][j] = *reinterpret_cast<const half8*>(kt + kat[j % kKeyAts] + ((2 * x + t) * 32 * D + (j / kKeyAts) * 64 * kKeyAts));
    };
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      f32x4 s[NB][2];
      load_keys(x);
#pragma unroll
      for (int t = 0; t < 2; ++t) {
#pragma unroll
        for (int n = 0; n < NB; ++n) s[n][t] = f32x4{};
#pragma unroll
        for (int j = 0; j < J; ++j) {
#pragma unroll
          for (int n = 0; n < NB; ++n) {
            s[n][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[t][j], qh[n][j], s[n][t], 0, 0, 0);
            if constexpr (F32) s[n][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[t][j], ql[n][j], s[n][t], 0, 0, 0);
          }
        }
      }
      half8 vf[B];
      auto load_values = [&]() {
#pragma unroll
        for (int b = 0; b < B; ++b) vf[b] = *reinterpret_cast<const half8*>(vt + vat[(b & 1) + 2 * x] + b * 2048);
      };
      if (AHEAD) {
        load_values();
        __builtin_amdgcn_sched_barrier(0);
      }
      f32x4 sc[2];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        sc[t] = f32x4{1.0f, 1.0f, 0.0f, 0.0f};
        if constexpr (CODES) sc[t] = *reinterpret_cast<const f32x4*>(scales[buf][32 * x + 16 * t + 4u * qq]);
      }
      float c[NB][2], top[NB], most[NB];
      bool moves = false;
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        c[n][0] = sc[0][0] * qscale[n], c[n][1] = sc[1][0] * qscale[n];
        if (!plain) {
          // of the lane's positions j0 + 32 x + 4 qq + (16 t + i): up to `last`, behind `past` or before `first`
          std::uint32_t quad = qq;
          asm volatile("" : "+v"(quad));  // (nothing of this is kept over the loop)
          const auto base = static_cast<int>(j0 + 32u * x + 4u * quad);
          const int last = static_cast<int>(pc[n]) - base, past = last - static_cast<int>(a.window), first = static_cast<int>(a.sinks) - base;
          const std::uint32_t bits = static_cast<std::uint32_t>(sees_any >> (32 * x)) >> (4u * quad);
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int at = 16 * t + i;
              const bool yes = (at <= last) & ((at > past) | (at < first)) & ((bits >> at & 1u) != 0u);
              s[n][t][i] = yes ? s[n][t][i] * c[n][t] : -INFINITY;
            }
          c[n][0] = c[n][1] = 1.0f;
        }
        top[n] = most[n] = -INFINITY;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const float quad = fmaxf(fmaxf(s[n][t][0], s[n][t][1]), fmaxf(s[n][t][2], s[n][t][3])) * c[n][t];
          top[n] = fmaxf(top[n], quad);
          if constexpr (CODES) most[n] = fmaxf(most[n], quad + sc[t][2]);
        }
        constexpr float kLag = F32 ? 0.0f : kSlack;
        moves |= top[n] > m[n] + kLag;  // (from no maximum: anything)
        if constexpr (CODES) moves |= most[n] > lead[n] + kLag;
      }
      // F16: the maxima counted from move once they are 2^4 behind
      if (__ballot(moves) != 0ull) {
#pragma unroll
        for (int n = 0; n < NB; ++n) {
          float t = fmaxf(top[n], lane_xor<16>(top[n]));
          t = fmaxf(t, lane_xor<32>(t));
          const float mn = fmaxf(m[n], t), base = mn == -INFINITY ? 0.0f : mn;
          float alpha = __builtin_amdgcn_exp2f(m[n] - base);
          l[n] *= alpha;
          if constexpr (CODES) {
            t = fmaxf(most[n], lane_xor<16>(most[n]));
            lead[n] = fmaxf(lead[n], fmaxf(t, lane_xor<32>(t)));
            int e = lead[n] - base > -126.0f ? static_cast<int>(ceilf(lead[n] - base)) : E[n];
            if (tail && e < E[n] - 60) e = E[n] - 60;  // (o has room for that)
            alpha = __builtin_amdgcn_exp2f((m[n] - base) + static_cast<float>(E[n] - e));
            E[n] = e;
          }
          m[n] = mn;
#pragma unroll
          for (int b = 0; b < B; ++b) o[n][b] *= alpha;
        }
      }
      half8 ph[NB], pl[NB];
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        const float base = (m[n] == -INFINITY ? 0.0f : m[n]) - static_cast<float>(F32 ? kPairLift : kLift);
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          float scale = 1.0f;
          if constexpr (CODES) scale = fminf(ldexpf(sc[t][1], -E[n]), 3e38f);  // (finite also where the row does not see)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float p = __builtin_amdgcn_exp2f(fmaf(s[n][t][i], c[n][t], -base));
            l[n] += p;
            if constexpr (CODES) p *= scale;
            asm("" : "+v"(p));  // one rounded value for hi and lo
            ph[n][4 * t + i] = static_cast<_Float16>(p);
            pl[n][4 * t + i] = static_cast<_Float16>(p - static_cast<float>(ph[n][4 * t + i]));
          }
        }
      }
      if (AHEAD)
        __builtin_amdgcn_sched_barrier(0);
      else
        load_values();
#pragma unroll
      for (int b = 0; b < B; ++b)
#pragma unroll
        for (int n = 0; n < NB; ++n) {
          o[n][b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf[b], ph[n], o[n][b], 0, 0, 0);
          o[n][b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf[b], pl[n], o[n][b], 0, 0, 0);
        }
    }
  };

  if (tid == 0u) odd = 0u;
  __syncthreads();
  page = load_page(u0);
  if (u0 < code1) {
    load_tile(u0);
    page = load_page(u0 + 1u);
    store_tile(0, first_of(u0));
  } else {
    tail_tile(0, first_of(u0));
  }
  unsigned long long now = seen;
  __syncthreads();
  int buf = 0;
  for (std::uint32_t u = u0; u < u1; ++u) {
    const std::uint32_t j0 = first_of(u);
    if (u + 1u < code1) {
      load_tile(u + 1u);
      page = load_page(u + 2u);
    }
    // (a wave whose rows see none of the tile: before it, or with their windows past it)
    if (!idle && j0 <= pb && (j0 + kTile - 1u + a.window > pa || j0 < a.sinks))
      compute(buf, j0, now, u >= sp.ncode);
    if (u + 1u < u1) {
      if (u + 1u < code1)
        store_tile(buf ^ 1, first_of(u + 1u));
      else
        tail_tile(buf ^ 1, first_of(u + 1u));
    }
    now = seen;
    lds_barrier();
    buf ^= 1;
  }

#pragma unroll
  for (int n = 0; n < NB; ++n) {
    float sum = l[n];
    sum += lane_xor<16>(sum);
    sum += lane_xor<32>(sum);
    const std::uint32_t c = (wave * NB + n) * 16u + col, ci = c / a.group;
    if (ci >= sp.nq) continue;
    if (per >= sp.total) {
      const float inv = sum == 0.0f ? 0.0f : ldexpf(1.0f / sum, E[n]);
      const std::size_t at = (static_cast<std::size_t>(sp.row + ci) * n_heads + g * a.group + (c - ci * a.group)) * D + 4u * qq;
#pragma unroll
      for (int b = 0; b < B; ++b) store_row4(a, at + 16 * b, o[n][b] * inv);
    } else {
      const std::size_t at = ((static_cast<std::size_t>(unit) * kv.p.n_kv + g) * (a.tq * a.group) + c) * a.splits + split;
#pragma unroll
      for (int b = 0; b < B; ++b)
        *reinterpret_cast<f32x4*>(a.part + at * D + 16 * b + 4u * qq) =
            f32x4{ldexpf(o[n][b][0], E[n]), ldexpf(o[n][b][1], E[n]), ldexpf(o[n][b][2], E[n]), ldexpf(o[n][b][3], E[n])};
      if (qq == 0u) a.ml[at] = make_float2(sum != sum ? INFINITY : m[n], sum);
    }
  }
  if (odd != 0u) not_finite_rows<D, CODES, true>(a, rows, kv, unit, g, split, kTile, 1u);
}

template <int D, Cached F, bool F32>
hipError_t launch(const AttnRows& a, const CallRows& rows, const RowsCache& kv, hipStream_t stream) {
  constexpr int NB = prompt_blocks(D, F32), NW = kPromptWaves;
  hipLaunchKernelGGL((attn_prompt_kernel<D, F, F32, NB, NW>), dim3(a.units * a.splits * kv.p.n_kv), dim3(64 * NW), 0, stream, a, rows, kv);
  return hipGetLastError();
}

template <int D>
hipError_t launch_dim(Cached kind, const AttnRows& a, const CallRows& rows, const RowsCache& kv, hipStream_t stream) {
  if (a.f16 != 0u)
    return kind == Cached::kF16    ? launch<D, Cached::kF16, false>(a, rows, kv, stream)
           : kind == Cached::kInt8 ? launch<D, Cached::kInt8, false>(a, rows, kv, stream)
                                   : launch<D, Cached::kE4m3, false>(a, rows, kv, stream);
  return kind == Cached::kF16    ? launch<D, Cached::kF16, true>(a, rows, kv, stream)
         : kind == Cached::kInt8 ? launch<D, Cached::kInt8, true>(a, rows, kv, stream)
                                 : launch<D, Cached::kE4m3, true>(a, rows, kv, stream);
}

}  // namespace

hipError_t attn_prompt(Cached kind, std::uint32_t head_dim, const AttnRows& a, const CallRows& rows, const RowsCache& kv,
                       hipStream_t stream) {
  return head_dim == 64u    ? launch_dim<64>(kind, a, rows, kv, stream)
         : head_dim == 128u ? launch_dim<128>(kind, a, rows, kv, stream)
                            : launch_dim<256>(kind, a, rows, kv, stream);
}

}  // namespace rtxllm
