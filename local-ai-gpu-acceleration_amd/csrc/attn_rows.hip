// Attention of new rows over a paged cache of fp16 values or 8-bit codes, with a
// sliding window and sinks: the form for few rows a sequence.
#include "attn_rows.cuh"

namespace rtxllm {
namespace {

constexpr std::uint32_t kThreads = 256, kWaves = kThreads / 64u, kCols = 16, kTile = kRowTile;
constexpr std::uint32_t kUnitsY = 32768;  // units of a launch's second dimension, at most
constexpr int kLift = 15;  // queries and softmax terms are brought to 2^15, as in paged_attn.hip

// A tile's keys and values in a lane's registers. Keys: position col of each half tile, the lane's
// quarter of the dimensions in D / 32 steps of 8. Values: VPL dimensions from VPL * col on of the 8 positions
// 16 (e / 4) + 4 qq + e % 4, which are those of the lane's scores.
template <int D, Cached F>
struct Frag {
  static constexpr Cached kind = F;
  static constexpr int VPL = D / 16, BYTES = F == Cached::kF16 ? 2 : 1;
  static constexpr int KN = D * BYTES / 64, VW = VPL * BYTES / 4;
  u32x4 k[2][KN];
  std::uint32_t v[8][VW];
  float ks[2], vs[2];  // 8-bit codes: scales of positions 16 t + 4 qq + 0..3

  __device__ __forceinline__ half8 key(int t, int j) const {
    if constexpr (F == Cached::kF16) {
      return __builtin_bit_cast(half8, k[t][j]);
    } else {
      const uint2 a = codes_to_half<F>(k[t][j / 2][2 * (j & 1)]), b = codes_to_half<F>(k[t][j / 2][2 * (j & 1) + 1]);
      return __builtin_bit_cast(half8, make_uint4(a.x, a.y, b.x, b.y));
    }
  }
  // dimensions VPL col + 4 w + i, i = 0..3, of the lane's 8 positions
  __device__ __forceinline__ void values(int w, half8* out) const {
    if constexpr (F == Cached::kF16) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const std::uint32_t sel = (i & 1) != 0 ? 0x07060302u : 0x05040100u;
        uint4 u;
        u.x = __builtin_amdgcn_perm(v[1][2 * w + i / 2], v[0][2 * w + i / 2], sel);
        u.y = __builtin_amdgcn_perm(v[3][2 * w + i / 2], v[2][2 * w + i / 2], sel);
        u.z = __builtin_amdgcn_perm(v[5][2 * w + i / 2], v[4][2 * w + i / 2], sel);
        u.w = __builtin_amdgcn_perm(v[7][2 * w + i / 2], v[6][2 * w + i / 2], sel);
        out[i] = __builtin_bit_cast(half8, u);
      }
    } else if constexpr (F == Cached::kInt8) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const std::uint32_t sel = 0x0C040C00u + 0x00010001u * i;  // byte i of two positions, each below a zero
        std::uint32_t u[4];
#pragma unroll
        for (int e = 0; e < 4; ++e)
          u[e] = less_1152(__builtin_amdgcn_perm(v[2 * e + 1][w], v[2 * e][w], sel) ^ 0x64806480u);
        out[i] = __builtin_bit_cast(half8, make_uint4(u[0], u[1], u[2], u[3]));
      }
    } else {
      uint2 u[2][4];
#pragma unroll
      for (int h = 0; h < 2; ++h) {  // the 4 x 4 bytes turned, then four positions of a dimension at a time
        const std::uint32_t a = v[4 * h][w], b = v[4 * h + 1][w], c = v[4 * h + 2][w], d = v[4 * h + 3][w];
        const std::uint32_t ab = __builtin_amdgcn_perm(b, a, 0x05010400u), AB = __builtin_amdgcn_perm(b, a, 0x07030602u);
        const std::uint32_t cd = __builtin_amdgcn_perm(d, c, 0x05010400u), CD = __builtin_amdgcn_perm(d, c, 0x07030602u);
        u[h][0] = codes_to_half<F>(__builtin_amdgcn_perm(cd, ab, 0x05040100u));
        u[h][1] = codes_to_half<F>(__builtin_amdgcn_perm(cd, ab, 0x07060302u));
        u[h][2] = codes_to_half<F>(__builtin_amdgcn_perm(CD, AB, 0x05040100u));
        u[h][3] = codes_to_half<F>(__builtin_amdgcn_perm(CD, AB, 0x07060302u));
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) out[i] = __builtin_bit_cast(half8, make_uint4(u[0][i].x, u[0][i].y, u[1][i].x, u[1][i].y));
    }
  }
};

// First dimension of score step j in the lane's quarter: the order in which the cache's 16-byte loads
// bring them.
template <bool CODES>
__device__ __forceinline__ std::uint32_t key_dim(int j, std::uint32_t qq) {
  return CODES ? 64u * (j / 2) + 16u * qq + 8u * (j & 1) : 32u * j + 8u * qq;
}

// One workgroup of four waves per (unit, kv head, split); 16 columns are the unit's query rows
// times the kv head's query heads. A wave takes tiles of 32 positions of its split in turn, with a running
// maximum and sum for every column:
//  * scores: S = K q^T by v_mfma_f32_16x16x32_f16, q as an fp16 pair lifted by a power of two
//    (F16 queries: hi alone); int8 and e4m3 codes are fp16 numbers, so a product is exact and the key's
//    scale multiplies the score;
//  * p = 2^(s - m + 15) enters the sum; times the value's scale over 2^E it is split into an fp16 pair. 2^E is the column's
//    own: the largest 2^(s - m) times scale that it has seen, so that what it does not see, or what hardly weighs, takes
//    no bits from the rest, whatever the scales' size;
//  * o += V^T p by the same instruction. The scores' layout (4 positions of each half tile a lane) is
//    taken as the order of the products' 32 positions, so p needs no exchange, and a lane loads its
//    values for those positions: rows of the cache in whole lines, bytes turned in registers.
// Bound by the reads of the cache where there are many: eight contexts to 65500 of 8 heads of 128 in e4m3 (604 MB)
// 102 us, 5.9 TB/s (a 1 GiB copy: 5.1); heads of 256 195 of 207 with keys past the caches, fp16 windows of 8000 41.6 of
// 46.7, values through the caches as well 208 and 45.8. Few positions are the chain of a wave: position, table, row and
// scales, some 1.6 us a tile (its 400 vector instructions, most of them codes becoming fp16), the merge: 16 positions
// 5.7 us, of which 2 are the launch.
template <int D, Cached F, bool QUAD>
__global__ __launch_bounds__(kThreads, (D == 256 ? 1 : 2)) void attn_rows_kernel(AttnRows a, CallRows rows, RowsCache kv) {
  constexpr bool CODES = F != Cached::kF16;
  constexpr int J = D / 32, B = D / 16, VPL = D / 16;
  constexpr std::uint32_t kPad = D + 4u;
  __shared__ __align__(16) float rec[kWaves][kCols][kPad];
  __shared__ float2 rml[kWaves][kCols];
  __shared__ std::uint32_t odd[kWaves];  // whether a wave left out values that are not finite: not_finite_rows
  // kv heads first: workgroups next to each other read what lies next to each other in a page
  const std::uint32_t split = blockIdx.x / kv.p.n_kv, g = blockIdx.x - split * kv.p.n_kv, unit = blockIdx.z * kUnitsY + blockIdx.y;
  if (unit >= a.units) return;
  const std::uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const std::uint32_t col = lane & 15u, qq = lane >> 4;
  const std::uint32_t n_heads = a.group * kv.p.n_kv;
  const bool f16 = a.f16 != 0u;
  const std::uint32_t qi = rows.start == nullptr ? (col < a.group ? 0u : 1u) : col / a.group;  // the column's query row
  const std::uint32_t h = col - qi * a.group;                                               // and head
  // The column's q, as it lies there: read before anything is known of the sequence where row and unit are one.
  // (16 bytes at a time; fp16: the second 16 are the first again and not used)
  u32x4 raw[J][2];
  auto load_q = [&](std::uint32_t row, bool there) {
    const std::size_t at = (static_cast<std::size_t>(row) * n_heads + g * a.group + (there ? h : 0u)) * D;
    const std::uint8_t* const base = static_cast<const std::uint8_t*>(a.q) + (f16 ? 2u : 4u) * at;
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const std::uint8_t* const x = base + (f16 ? 2u : 4u) * key_dim<CODES>(j, qq);
      raw[j][0] = u32x4(*reinterpret_cast<const u32x4_any*>(x));
      raw[j][1] = u32x4(*reinterpret_cast<const u32x4_any*>(x + (f16 ? 0u : 16u)));
    }
  };
  if (rows.start == nullptr) load_q(unit, qi == 0u);
  const RowSpan sp = row_span(rows, kv, unit, a.tq, a.window, a.sinks, kTile);
  if (sp.nq == 0u) return;
  const std::uint32_t per = span_per(sp.total, a.splits, kWaves), u0 = split * per;
  if (u0 >= sp.total) return;  // (merge_rows_kernel counts the records alike)
  const std::uint32_t u1 = u0 + per < sp.total ? u0 + per : sp.total;
  const bool mine = qi < sp.nq;
  if (rows.start != nullptr) load_q(sp.row + (mine ? qi : 0u), mine);
  const std::uint32_t pc = row_pos(sp.pos, mine ? qi : 0u, kv.p.capacity);
  const std::int32_t* const table = kv.p.table + static_cast<std::size_t>(sp.s) * kv.p.table_stride;

  // B operands of the scores and the column's power of two
  half8 qh[J], ql[J];
  float qscale;
  {
    float x[J][8], top = 0.0f;
    if (f16) {
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const half8 t = __builtin_bit_cast(half8, raw[j][0]);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[j][i] = static_cast<float>(t[i]);
      }
    } else {
#pragma unroll
      for (int j = 0; j < J; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const std::uint32_t w = raw[j][i / 4][i & 3];
          x[j][i] = __uint_as_float(w);
        }
    }
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(x[j][i]));
    top = fmaxf(top, lane_xor<16>(top));
    top = fmaxf(top, lane_xor<32>(top));
    int e = 0;
    if (top > 0.0f && top < INFINITY) frexpf(top, &e);
    qscale = ldexpf(score_scale<D>(), e - kLift);
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float v = mine ? ldexpf(x[j][i], kLift - e) : 0.0f;
        asm("" : "+v"(v));  // one rounded value for hi and lo
        qh[j][i] = static_cast<_Float16>(v);
        ql[j][i] = static_cast<_Float16>(v - static_cast<float>(qh[j][i]));
      }
  }

  float m = -INFINITY, l = 0.0f;
  float lead = -INFINITY;  // codes: the largest log2 of a position's term times its value's scale,
  int E = 0;               // lead - m in whole powers of two, over which o is held
  std::uint32_t left_out = 0u;  // the wave's own mark, in LDS only behind all tiles: nothing clears another wave's
  f32x4 o[B];
#pragma unroll
  for (int b = 0; b < B; ++b) o[b] = f32x4{};

  // One tile: `seen` has a bit for each of its positions that a column may see, of first position j0;
  // `next` runs once the keys are used.
  auto step = [&](auto& f, std::uint32_t j0, std::uint32_t seen, auto next) {
    using Fr = std::remove_reference_t<decltype(f)>;
    constexpr bool SCALED = Fr::kind != Cached::kF16, TAIL = CODES && !SCALED;
    f32x4 sc[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      sc[t] = f32x4{};
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const half8 kj = f.key(t, j);
        sc[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kj, qh[j], sc[t], 0, 0, 0);
        sc[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kj, ql[j], sc[t], 0, 0, 0);
      }
    }
    float ks[2] = {qscale, qscale}, vs[2] = {1.0f, 1.0f};
    if constexpr (SCALED) ks[0] *= f.ks[0], ks[1] *= f.ks[1], vs[0] = f.vs[0], vs[1] = f.vs[1];
    next();
    // every column sees every position
    const bool plain = seen == 0xFFFFFFFFu && (sp.nq == 1u || (j0 + kTile - 1u <= sp.p0 &&
                                                              (sp.plast - j0 < a.window || j0 + kTile <= a.sinks)));
    std::uint32_t sees = seen >> (4u * qq);  // bits 16 t + i: the lane's positions
    if (!plain && sp.nq > 1u) {
      // of the lane's positions j0 + 4 qq + (16 t + i): up to `last`, behind `past` or before `first`
      const auto base = static_cast<int>(j0 + 4u * qq);
      const int last = static_cast<int>(pc) - base, past = last - static_cast<int>(a.window), first = static_cast<int>(a.sinks) - base;
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int x = 16 * t + i;
          const bool yes = (x <= last) & ((x > past) | (x < first));
          sees &= yes ? ~0u : ~(1u << x);
        }
    }
    float s[2][4], top = -INFINITY, most = -INFINITY;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      float quad = -INFINITY;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float x = sc[t][i] * ks[t];
        s[t][i] = (sees >> (16 * t + i) & 1u) != 0u ? x : -INFINITY;
        quad = fmaxf(quad, s[t][i]);
      }
      top = fmaxf(top, quad);
      if constexpr (CODES)  // (a scale that is 0 or no number has no size)
        most = fmaxf(most, vs[t] > 0.0f && vs[t] < INFINITY ? quad + static_cast<float>(__builtin_amdgcn_frexp_expf(vs[t])) : -INFINITY);
    }
    top = fmaxf(top, lane_xor<16>(top));
    top = fmaxf(top, lane_xor<32>(top));
    const float mn = fmaxf(m, top), base = mn == -INFINITY ? 0.0f : mn;
    float alpha = __builtin_amdgcn_exp2f(m - base);
    l *= alpha;
    bool moved = mn != m;
    if constexpr (CODES) {
      most = fmaxf(most, lane_xor<16>(most));
      most = fmaxf(most, lane_xor<32>(most));
      // The tail's values are as they are, of scale 1 whatever their size, and come last: their terms alone say where
      // they are held (2^60 and o has room).
      lead = TAIL ? most : fmaxf(lead, most);
      int e = lead - base > -126.0f ? static_cast<int>(ceilf(lead - base)) : E;
      if (TAIL && e < E - 60) e = E - 60;
      alpha = __builtin_amdgcn_exp2f((m - base) + static_cast<float>(E - e));
      moved |= e != E;
      E = e;
#pragma unroll
      for (int t = 0; t < 2; ++t) {  // (a finite scale stays finite)
        const int room = 127 - __builtin_amdgcn_frexp_expf(vs[t]);
        vs[t] = ldexpf(vs[t], -E < room ? -E : room);
      }
    }
    m = mn;
    half8 ph, pl;
    float sum = 0.0f;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float p = __builtin_amdgcn_exp2f(s[t][i] - base + kLift);
        sum += p;
        if constexpr (CODES) p = (sees >> (16 * t + i) & 1u) != 0u ? p * vs[t] : 0.0f;
        asm("" : "+v"(p));
        ph[4 * t + i] = static_cast<_Float16>(p);
        pl[4 * t + i] = static_cast<_Float16>(p - static_cast<float>(ph[4 * t + i]));
      }
    l += sum;
    if (__ballot(moved) != 0ull) {
#pragma unroll
      for (int b = 0; b < B; ++b) o[b] *= alpha;
    }
    if (Fr::kind != Cached::kInt8 && seen != 0xFFFFFFFFu) {  // 0 times what no column sees must stay 0
#pragma unroll
      for (int e = 0; e < 8; ++e)
#pragma unroll
        for (int w = 0; w < Fr::VW; ++w) f.v[e][w] = (seen >> (16u * (e / 4) + 4u * qq + (e & 3)) & 1u) != 0u ? f.v[e][w] : 0u;
    }
    if constexpr (!SCALED) {
      if (!plain && sp.nq > 1u) {  // values that are not finite and that only some of the rows see: at the end
        u16x2 most = {0, 0};
#pragma unroll
        for (int e = 0; e < 8; ++e)
#pragma unroll
          for (int w = 0; w < Fr::VW; ++w) {
            const std::uint32_t m = f.v[e][w] & 0x7FFF7FFFu;
            most = __builtin_elementwise_max(most, __builtin_bit_cast(u16x2, m));
          }
        if (__ballot(most[0] >= 0x7C00u || most[1] >= 0x7C00u) != 0ull) {
          left_out = 1u;
#pragma unroll
          for (int e = 0; e < 8; ++e)
#pragma unroll
            for (int w = 0; w < Fr::VW; ++w) finite_only(f.v[e][w]);
        }
      }
    }
#pragma unroll
    for (int w = 0; w < VPL / 4; ++w) {
      half8 va[4];
      f.values(w, va);
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        o[4 * w + b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va[b], ph, o[4 * w + b], 0, 0, 0);
        o[4 * w + b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va[b], pl, o[4 * w + b], 0, 0, 0);
      }
    }
  };
  // Whether some row of the unit sees position j of the cache.
  auto some_row = [&](std::uint32_t j) { return j <= sp.plast && (j + a.window > sp.p0 || j < a.sinks); };

  const std::uint32_t code1 = u1 < sp.ncode ? u1 : sp.ncode, mine_at = lane & 31u;
  if (u0 + wave < code1) {
    // Tiles in the pages. A position that is not read takes row 0; its score and term are dropped.
    Frag<D, F> f;
    std::uint32_t seen = 0u, row = 0u, at = 0u;
    std::int32_t page = 0;
    auto position = [&](std::uint32_t u) {
      const std::uint32_t j = span_position(sp, u < code1 ? u : code1 - 1u, kTile) + mine_at;
      return j < kv.p.capacity ? j : kv.p.capacity - 1u;
    };
    auto load_page = [&](std::uint32_t u) { return table[page_of(kv.p, position(u))]; };
    auto settle = [&](std::uint32_t u) {  // from `page`, that of the lane's position of tile u
      const std::uint32_t j = position(u), j0 = span_position(sp, u < code1 ? u : code1 - 1u, kTile);
      const std::uint32_t r = paged_row(kv.p, page, g, j - page_of(kv.p, j) * kv.p.page_size);
      const bool there = j0 + mine_at < sp.code_end && r != kNoRow;
      row = there ? r : 0u;
      seen = static_cast<std::uint32_t>(__ballot(u < code1 && there && some_row(j)));
      at = j0;
    };
    auto load_k = [&]() {  // (through the caches: a line is two to four reads; values, whole lines at once, past them)
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const std::uint32_t r = from_lane(row, 16u * t + col);
        const u32x4* src = reinterpret_cast<const u32x4*>(kv.k + static_cast<std::size_t>(r) * (D * Frag<D, F>::BYTES)) + qq;
#pragma unroll
        for (int j = 0; j < Frag<D, F>::KN; ++j) f.k[t][j] = src[4 * j];
        if constexpr (CODES) f.ks[t] = kv.ks[from_lane(row, 16u * t + 4u * qq) >> kv.block_shift];
      }
    };
    auto load_v = [&]() {
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const std::uint32_t r0 = from_lane(row, 16u * t + 4u * qq);
        if constexpr (CODES) f.vs[t] = kv.vs[r0 >> kv.block_shift];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const std::uint32_t r = QUAD ? r0 + e : from_lane(row, 16u * t + 4u * qq + e);
          const std::uint32_t* src =
              reinterpret_cast<const std::uint32_t*>(kv.v + static_cast<std::size_t>(r) * (D * Frag<D, F>::BYTES)) + col * Frag<D, F>::VW;
          typedef std::uint32_t words __attribute__((ext_vector_type(Frag<D, F>::VW > 4 ? 4 : Frag<D, F>::VW)));
          constexpr int kParts = Frag<D, F>::VW > 4 ? Frag<D, F>::VW / 4 : 1;
#pragma unroll
          for (int x = 0; x < kParts; ++x) {
            const words w = __builtin_nontemporal_load(reinterpret_cast<const words*>(src) + x);
            if constexpr (Frag<D, F>::VW == 1) {
              f.v[4 * t + e][0] = w[0];
            } else {
#pragma unroll
              for (int i = 0; i < Frag<D, F>::VW / kParts; ++i) f.v[4 * t + e][4 * x + i] = w[i];
            }
          }
        }
      }
    };
    // Loads run ahead of use in the registers of one tile: the next tile's keys are read once this tile's scores
    // have used theirs, its values after this tile's products.
    page = load_page(u0 + wave);
    settle(u0 + wave);
    load_k();
    load_v();
    page = load_page(u0 + wave + kWaves);
    for (std::uint32_t u = u0 + wave; u < code1; u += kWaves) {
      const std::uint32_t now = seen, j0 = at;
      step(f, j0, now, [&]() {
        settle(u + kWaves);
        load_k();
        page = load_page(u + 2u * kWaves);
      });
      load_v();
    }
  }
  if constexpr (CODES) {
    // The newest block's positions, fp16, from the tail.
    const std::uint32_t block = 1u << kv.block_shift;
    const std::size_t base = (static_cast<std::size_t>(sp.s) * kv.p.n_kv + g) * block * D;
    std::uint32_t u = u0 + wave;
    if (u < sp.ncode) u += (sp.ncode - u + kWaves - 1u) / kWaves * kWaves;
    for (; u < u1; u += kWaves) {
      Frag<D, Cached::kF16> f;
      const std::uint32_t j0 = sp.tail + (u - sp.ncode) * kTile;
      const std::uint32_t seen = static_cast<std::uint32_t>(__ballot(some_row(j0 + mine_at)));
      auto place = [&](std::uint32_t i) {  // (the unit's last position lies in the tail)
        const std::uint32_t j = j0 + i < sp.plast ? j0 + i : sp.plast;
        return base + static_cast<std::size_t>(j & (block - 1u)) * D;
      };
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const std::uint16_t* kr = kv.kt + place(16u * t + col);
#pragma unroll
        for (int j = 0; j < J; ++j) f.k[t][j] = *reinterpret_cast<const u32x4*>(kr + key_dim<true>(j, qq));
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const std::uint32_t* vr = reinterpret_cast<const std::uint32_t*>(kv.vt + place(16u * t + 4u * qq + e)) + col * (VPL / 2);
#pragma unroll
          for (int i = 0; i < VPL / 2; ++i) f.v[4 * t + e][i] = vr[i];
        }
      }
      step(f, j0, seen, []() {});
    }
  }

  // the waves' records, merged: o = sum 2^(m_w - M + E_w) o_w, the sums without E_w
  l += lane_xor<16>(l);
  l += lane_xor<32>(l);
  // a NaN among the scores makes the row NaN, also where no number gave a maximum
  if (qq == 0u) rml[wave][col] = make_float2(l != l ? INFINITY : m, l);
  if (lane == 0u) odd[wave] = left_out;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int b = 0; b < B; b += 4)
      *reinterpret_cast<f32x4*>(&rec[wave][col][VPL * (4u * qq + i) + b]) =
          CODES ? f32x4{ldexpf(o[b][i], E), ldexpf(o[b + 1][i], E), ldexpf(o[b + 2][i], E), ldexpf(o[b + 3][i], E)}
                : f32x4{o[b][i], o[b + 1][i], o[b + 2][i], o[b + 3][i]};
  __syncthreads();
  const bool whole = per >= sp.total;
  const std::uint32_t ncol = a.tq * a.group;
  for (std::uint32_t it = threadIdx.x; it < sp.nq * a.group * (D / 4u); it += kThreads) {
    const std::uint32_t c = it / (D / 4u), d = 4u * (it % (D / 4u));
    float M = -INFINITY;
#pragma unroll
    for (std::uint32_t w = 0; w < kWaves; ++w) M = fmaxf(M, rml[w][c].x);
    const float base = M == -INFINITY ? 0.0f : M;
    float L = 0.0f;
    f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (std::uint32_t w = 0; w < kWaves; ++w) {
      const float x = __builtin_amdgcn_exp2f(rml[w][c].x - base);
      L += x * rml[w][c].y;
      v += x * *reinterpret_cast<const f32x4*>(&rec[w][c][d]);
    }
    if (whole) {
      const float inv = L == 0.0f ? 0.0f : 1.0f / L;
      const std::uint32_t i = c / a.group;
      const std::size_t dst = (static_cast<std::size_t>(sp.row + i) * n_heads + g * a.group + (c - i * a.group)) * D + d;
      store_row4(a, dst, v * inv);
    } else {
      const std::size_t dst = ((static_cast<std::size_t>(unit) * kv.p.n_kv + g) * ncol + c) * a.splits + split;
      *reinterpret_cast<f32x4*>(a.part + dst * D + d) = v;
      if (d == 0u) a.ml[dst] = make_float2(M, L);
    }
  }
  if ((odd[0] | odd[1] | odd[2] | odd[3]) != 0u) not_finite_rows<D, CODES, false>(a, rows, kv, unit, g, split, kTile, kWaves);
}

// One workgroup a (unit, kv head, column): the splits' records merged, D / 4 lanes a record, eight records of a lane in
// flight; the first eight are read before it is known how many there are.
template <int D>
__global__ __launch_bounds__(kThreads) void merge_rows_kernel(AttnRows a, CallRows rows, RowsCache kv, std::uint32_t tile,
                                                              std::uint32_t round) {
  constexpr std::uint32_t kLanes = D / 4u, kSub = kThreads / kLanes;
  __shared__ __align__(16) float sums[kSub][D];
  __shared__ float2 tops[kSub];
  const std::uint32_t ncol = a.tq * a.group, ug = blockIdx.x / ncol, c = blockIdx.x - ug * ncol, g = ug % kv.p.n_kv;
  const std::uint32_t d = 4u * (threadIdx.x % kLanes), sub = threadIdx.x / kLanes;
  const std::size_t at = static_cast<std::size_t>(blockIdx.x) * a.splits;
  f32x4 o[8];
  float2 t[8];
  auto load = [&](std::uint32_t x0, std::uint32_t end) {
#pragma unroll
    for (std::uint32_t k = 0; k < 8u; ++k) {
      const std::uint32_t x = x0 + kSub * k < end ? x0 + kSub * k : 0u;  // past the last: not counted
      o[k] = *reinterpret_cast<const f32x4*>(a.part + (at + x) * D + d);
      t[k] = a.ml[at + x];
    }
  };
  load(sub, a.splits);
  const RowSpan sp = row_span(rows, kv, ug / kv.p.n_kv, a.tq, a.window, a.sinks, tile);
  if (c >= sp.nq * a.group) return;
  const std::uint32_t per = span_per(sp.total, a.splits, round), used = (sp.total + per - 1u) / per;
  if (used <= 1u) return;
  f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
  float M = -INFINITY, L = 0.0f;
  for (std::uint32_t x0 = sub; x0 < used; x0 += 8u * kSub) {
    if (x0 != sub) load(x0, used);
    float mn = M;
#pragma unroll
    for (std::uint32_t k = 0; k < 8u; ++k) mn = x0 + kSub * k < used ? fmaxf(mn, t[k].x) : mn;
    const float base = mn == -INFINITY ? 0.0f : mn, f0 = __builtin_amdgcn_exp2f(M - base);
    v *= f0;
    L *= f0;
#pragma unroll
    for (std::uint32_t k = 0; k < 8u; ++k) {
      if (x0 + kSub * k < used) {
        const float f1 = __builtin_amdgcn_exp2f(t[k].x - base);
        v += o[k] * f1, L += t[k].y * f1;
      }
    }
    M = mn;
  }
  *reinterpret_cast<f32x4*>(&sums[sub][d]) = v;
  if (d == 0u) tops[sub] = make_float2(M, L);
  __syncthreads();
  if (sub != 0u) return;
  float top = -INFINITY;
  for (std::uint32_t k = 0; k < kSub; ++k) top = fmaxf(top, tops[k].x);
  const float base = top == -INFINITY ? 0.0f : top;
  v = f32x4{0.0f, 0.0f, 0.0f, 0.0f}, L = 0.0f;
  for (std::uint32_t k = 0; k < kSub; ++k) {
    const float f = __builtin_amdgcn_exp2f(tops[k].x - base);
    L += f * tops[k].y;
    v += f * *reinterpret_cast<const f32x4*>(&sums[k][d]);
  }
  v *= L == 0.0f ? 0.0f : 1.0f / L;
  const std::uint32_t i = c / a.group;
  const std::size_t dst = (static_cast<std::size_t>(sp.row + i) * a.group * kv.p.n_kv + g * a.group + (c - i * a.group)) * D + d;
  store_row4(a, dst, v);
}

// The same for many columns of few splits: D / 4 lanes a column, its records one after the other.
template <int D>
__global__ __launch_bounds__(kThreads) void merge_few_kernel(AttnRows a, CallRows rows, RowsCache kv, std::uint32_t tile,
                                                             std::uint32_t round) {
  constexpr std::uint32_t kLanes = D / 4u, kPer = kThreads / kLanes;
  const std::uint32_t ncol = a.tq * a.group, blocks = (ncol + kPer - 1u) / kPer, ug = blockIdx.x / blocks, g = ug % kv.p.n_kv;
  const std::uint32_t c = (blockIdx.x % blocks) * kPer + threadIdx.x / kLanes, d = 4u * (threadIdx.x % kLanes);
  const RowSpan sp = row_span(rows, kv, ug / kv.p.n_kv, a.tq, a.window, a.sinks, tile);
  if (c >= sp.nq * a.group) return;
  const std::uint32_t per = span_per(sp.total, a.splits, round), used = (sp.total + per - 1u) / per;
  if (used <= 1u) return;
  const std::size_t at = (static_cast<std::size_t>(ug) * ncol + c) * a.splits;
  f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
  float M = -INFINITY, L = 0.0f;
#pragma unroll 4
  for (std::uint32_t x = 0; x < used; ++x) {
    const float2 t = a.ml[at + x];
    const f32x4 o = *reinterpret_cast<const f32x4*>(a.part + (at + x) * D + d);
    const float mn = fmaxf(M, t.x), base = mn == -INFINITY ? 0.0f : mn;
    const float f0 = __builtin_amdgcn_exp2f(M - base), f1 = __builtin_amdgcn_exp2f(t.x - base);
    v = v * f0 + o * f1;
    L = L * f0 + t.y * f1;
    M = mn;
  }
  const std::uint32_t i = c / a.group;
  store_row4(a, (static_cast<std::size_t>(sp.row + i) * a.group * kv.p.n_kv + g * a.group + (c - i * a.group)) * D + d,
             v * (L == 0.0f ? 0.0f : 1.0f / L));
}

struct RowsPlan {
  bool prompt = false;
  std::uint32_t tq = 0, units = 0, splits = 0;
  std::size_t ml = 0, bytes = 0;  // bytes 0: refused
};

RowsPlan rows_plan(Cached kind, const rtxllm_paged_kv* c, std::uint32_t n_heads, bool f16, bool one_each, std::uint32_t sequences,
                   std::uint32_t rows, std::uint32_t window, std::uint32_t sinks) {
  RowsPlan p;
  const std::uint32_t group = paged_group(c, n_heads);
  if (group == 0u || window == 0u) return p;
  const std::uint64_t sees = static_cast<std::uint64_t>(window) + sinks;  // positions that a row can see
  p.prompt = !one_each && rows_prompt(sequences, rows, group, c->head_dim, c->page_size, !f16, sees < c->capacity ? sees : c->capacity);
  p.tq = one_each ? 1u : (p.prompt ? prompt_columns(c->head_dim, !f16) : kCols) / group;
  p.units = one_each ? sequences : units_of(sequences, rows, p.tq, 1u);
  const std::uint64_t items = static_cast<std::uint64_t>(p.units) * c->n_kv_heads;
  const std::uint64_t near = sees + p.tq;
  const std::uint64_t tiles = (near < c->capacity ? near : c->capacity) / (p.prompt ? kPromptTile : kTile) + 3u;
  std::uint64_t splits = rows_splits(items, tiles, kind != Cached::kF16, c->head_dim);
  if (p.prompt) {
    const std::uint64_t most = (tiles + 3u) / 4u;
    splits = items >= 192u ? 1u : (256u + items - 1u) / items;
    if (splits > most) splits = most;
  }
  p.splits = static_cast<std::uint32_t>(splits);
  // the launches' thread counts
  if ((p.prompt ? items * splits * 64u * kPromptWaves : splits * c->n_kv_heads * kThreads) > 0xFFFFFFFFull ||
      (splits > 1u && items * p.tq * group > (1u << 24)))
    return p;
  const std::uint64_t records = splits > 1u ? items * p.tq * group * splits : 0u;
  p.ml = round_256(8u * records);
  p.bytes = p.ml + round_256(4u * records * c->head_dim) + 256u;
  return p;
}

template <int D>
hipError_t launch_rows(Cached kind, bool prompt, const AttnRows& a, const CallRows& rows, const RowsCache& kv, hipStream_t stream) {
  const std::uint32_t y = a.units < kUnitsY ? a.units : kUnitsY;
  const dim3 grid(a.splits * kv.p.n_kv, y, (a.units + y - 1u) / y), block(kThreads);
  hipError_t rc = hipSuccess;
  if (prompt)
    rc = attn_prompt(kind, D, a, rows, kv, stream);
  else if (kind == Cached::kInt8)
    hipLaunchKernelGGL((attn_rows_kernel<D, Cached::kInt8, true>), grid, block, 0, stream, a, rows, kv);
  else if (kind == Cached::kE4m3)
    hipLaunchKernelGGL((attn_rows_kernel<D, Cached::kE4m3, true>), grid, block, 0, stream, a, rows, kv);
  else if (kv.p.page_size % 4u == 0u)
    hipLaunchKernelGGL((attn_rows_kernel<D, Cached::kF16, true>), grid, block, 0, stream, a, rows, kv);
  else
    hipLaunchKernelGGL((attn_rows_kernel<D, Cached::kF16, false>), grid, block, 0, stream, a, rows, kv);
  if (rc == hipSuccess) rc = hipGetLastError();
  if (rc != hipSuccess || a.splits == 1u) return rc;
  const std::uint32_t cols = a.tq * a.group, per = kThreads / (D / 4u);
  if (prompt)
    hipLaunchKernelGGL(merge_few_kernel<D>, dim3(a.units * kv.p.n_kv * ((cols + per - 1u) / per)), block, 0, stream, a, rows, kv,
                       kPromptTile, 1u);
  else
    hipLaunchKernelGGL(merge_rows_kernel<D>, dim3(a.units * kv.p.n_kv * cols), block, 0, stream, a, rows, kv, kTile, kWaves);
  return hipGetLastError();
}

hipError_t attn_rows(Cached kind, const rtxllm_paged_kv* pages, const RowsCache& kv, const void* q, int type, std::uint32_t n_heads,
                     const CallRows& rows, std::uint32_t window, std::uint32_t sinks, void* out, void* workspace,
                     std::size_t workspace_bytes, hipStream_t stream) {
  if (q == nullptr || out == nullptr || workspace == nullptr || !type_ok(type) || !aligned_to(q, type_bytes(type)) ||
      !aligned_to(out, type_bytes(type)) || !aligned_to(workspace, 256u))
    return hipErrorInvalidValue;
  const RowsPlan p = rows_plan(kind, pages, n_heads, type == RTXLLM_F16, rows.start == nullptr, rows.sequences, rows.rows, window, sinks);
  if (p.bytes == 0u || workspace_bytes < p.bytes) return hipErrorInvalidValue;
  const std::uint64_t n = type_bytes(type) * static_cast<std::uint64_t>(rows.rows) * n_heads * pages->head_dim;
  const std::uint64_t table = 4ull * ((rows.sequences - 1ull) * pages->table_stride + pages->capacity / pages->page_size);
  // a unit has its result while others read theirs
  for (const auto& [at, bytes] : {std::pair<void*, std::uint64_t>{out, n}, {workspace, p.bytes}}) {
    if ((at != out || out != q) && overlap(at, bytes, q, n)) return hipErrorInvalidValue;
    if (overlap(at, bytes, rows.pos, 4ull * rows.sequences) || overlap(at, bytes, pages->block_table, table) ||
        (rows.start != nullptr && overlap(at, bytes, rows.start, 4ull * rows.sequences + 4u)))
      return hipErrorInvalidValue;
  }
  if (overlap(out, n, workspace, p.bytes)) return hipErrorInvalidValue;
  AttnRows a{};
  a.q = q;
  a.out = out;
  a.ml = static_cast<float2*>(workspace);
  a.part = reinterpret_cast<float*>(static_cast<std::uint8_t*>(workspace) + p.ml);
  a.f16 = type == RTXLLM_F16 ? 1u : 0u;
  a.group = paged_group(pages, n_heads);
  a.tq = p.tq;
  a.window = window < pages->capacity ? window : pages->capacity;  // (no sum with a position passes 32 bits)
  a.sinks = sinks < pages->capacity ? sinks : pages->capacity;
  a.splits = p.splits;
  a.units = p.units;
  return pages->head_dim == 64u    ? launch_rows<64>(kind, p.prompt, a, rows, kv, stream)
         : pages->head_dim == 128u ? launch_rows<128>(kind, p.prompt, a, rows, kv, stream)
                                   : launch_rows<256>(kind, p.prompt, a, rows, kv, stream);
}

// A workspace serves every call of its numbers: of either type, with starts or one row each.
std::size_t attn_rows_bytes(Cached kind, const rtxllm_paged_kv* c, std::uint32_t n_heads, std::uint32_t sequences, std::uint32_t rows,
                            std::uint32_t window, std::uint32_t sinks) {
  if (sequences == 0u || sequences > 65535u || rows == 0u || rows > (1u << 20)) return 0u;
  std::size_t most = 0u;
  for (const bool f16 : {false, true})
    for (const bool one_each : {false, true}) {
      if (one_each && rows != sequences) continue;
      const std::size_t n = rows_plan(kind, c, n_heads, f16, one_each, sequences, rows, window, sinks).bytes;
      if (n == 0u) return 0u;
      most = n > most ? n : most;
    }
  return most;
}

}  // namespace
}  // namespace rtxllm

using namespace rtxllm;

extern "C" size_t rtxllm_attn_window_workspace(const rtxllm_paged_kv* cache, uint32_t n_heads, uint32_t sequences,
                                               uint32_t rows, uint32_t window, uint32_t sinks) {
  return paged_cache_ok(cache, sequences) ? attn_rows_bytes(Cached::kF16, cache, n_heads, sequences, rows, window, sinks) : 0u;
}

extern "C" hipError_t rtxllm_attn_window_f16(const rtxllm_paged_kv* cache, const void* q, int type, uint32_t n_heads,
                                             const uint32_t* start, const uint32_t* pos, uint32_t sequences,
                                             uint32_t rows, uint32_t window, uint32_t sinks, void* out, void* workspace,
                                             size_t workspace_bytes, hipStream_t stream) {
  if (!rows_ok(start, pos, sequences, rows) || !paged_cache_ok(cache, sequences)) return hipErrorInvalidValue;
  const std::uint64_t n = 2ull * cache->n_pages * cache->n_kv_heads * cache->page_size * cache->head_dim;
  const std::uint64_t o = type_bytes(type) * static_cast<std::uint64_t>(rows) * n_heads * cache->head_dim;
  for (const void* c : {cache->k, cache->v})
    if (overlap(c, n, out, o) || overlap(c, n, workspace, workspace_bytes)) return hipErrorInvalidValue;
  return attn_rows(Cached::kF16, cache, f16_view(cache), q, type, n_heads, CallRows{start, pos, sequences, rows}, window, sinks, out,
                   workspace, workspace_bytes, stream);
}

extern "C" size_t rtxllm_attn_kv8_workspace(const rtxllm_paged_kv8* cache, uint32_t n_heads, uint32_t sequences,
                                            uint32_t rows, uint32_t window, uint32_t sinks) {
  if (!kv8_cache_ok(cache, sequences)) return 0u;
  const rtxllm_paged_kv pages = kv8_pages(cache);
  return attn_rows_bytes(kv8_kind(cache), &pages, n_heads, sequences, rows, window, sinks);
}

extern "C" hipError_t rtxllm_attn_kv8(const rtxllm_paged_kv8* cache, const void* q, int type, uint32_t n_heads,
                                      const uint32_t* start, const uint32_t* pos, uint32_t sequences, uint32_t rows,
                                      uint32_t window, uint32_t sinks, void* out, void* workspace, size_t workspace_bytes,
                                      hipStream_t stream) {
  if (!rows_ok(start, pos, sequences, rows) || !kv8_cache_ok(cache, sequences)) return hipErrorInvalidValue;
  const std::uint64_t o = type_bytes(type) * static_cast<std::uint64_t>(rows) * n_heads * cache->head_dim;
  const Kv8Ranges r = kv8_ranges(cache, sequences);
  if (!apart(r, out, o) || !apart(r, workspace, workspace_bytes)) return hipErrorInvalidValue;
  const rtxllm_paged_kv pages = kv8_pages(cache);
  return attn_rows(kv8_kind(cache), &pages, kv8_view(cache), q, type, n_heads,
                   CallRows{start, pos, sequences, rows}, window, sinks, out, workspace, workspace_bytes, stream);
}
