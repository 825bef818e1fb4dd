// GQA decode attention over a paged cache: over listed pages, and over every
// slot with its softmax weight gathered.
#include "common.h"
#include "layer_common.cuh"
#include "paged.h"

namespace rtxllm {
namespace {

typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef std::uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef std::uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr std::uint32_t kThreads = 256, kWaves = kThreads / 64u, kTile = 16;
constexpr std::uint32_t kMaxPer = 64;  // tiles of a split, at most: what its scores take in the LDS
constexpr int kLift = 15;  // queries and softmax terms are brought to 2^15 (see the kernel)

struct AttnArgs {
  const float* q;
  const std::uint32_t* pos;
  const std::int32_t* pages;
  float* out;
  float2* ml;      // [row][kv head][query head][split]: maximum (in log2), sum
  float* part;     // [row][kv head][query head][split][head_dim]
  float* scores;   // [row][kv head][query head][score_stride], in log2 (weights only)
  std::uint32_t group, n_select, per, splits, score_stride;  // per: tiles of a split
};

__device__ __forceinline__ std::uint32_t from_lane(std::uint32_t v, std::uint32_t lane) {
  return static_cast<std::uint32_t>(__builtin_amdgcn_ds_bpermute(static_cast<int>(4u * lane), static_cast<int>(v)));
}

// Tiles of a split (one workgroup), of at most `tiles`. Of one size for all rows but much
// shorter ones (row_per), so that a longer context is more workgroups; the largest of 4 to 64 that leaves a
// workgroup for each CU, as a wave's prologue and the merge cost what two or three
// tiles do; over whole contexts, whose lengths differ, more than 16 only where the row
// still makes 12 of them (eight rows of 12000, us with at least 16 / 12 / 8: 87 / 82 / 81, of 8000 63 / 64 / 69,
// up to 16384 62 / 62 / 67). us at 4 / 8 / 16 / 32 / 64 tiles, 32 heads over 8 kv heads of 128
// - whole: 1024 slots of one sequence 7.9 / 8.8 / 10.7 / 14.5 / 22.1, 4001 of one 10.9 / 10.0 /
//   11.8 / 15.9 / 23.9, 65536 of one 88 / 68 / 58 / 53 / 51, up to 4096 of eight 31.1 / 25.9 / 23.3 /
//   26.0 / 27.2, up to 16384 of eight 100 / 78 / 71 / 70 / 66;
// - listed: 4096 positions of eight 39.6 / 32.0 / 29.1 / 27.9 / 24.7.
// 8 tiles already where 4 would make more workgroups than CUs, 16 where they make 160 (workgroups
// at 8, us at 4 / 8: 128 8.3 / 9.0, 160 12.4 / 11.3, 192 10.1 / 9.4, 132 of 16 heads of 256 30.7 / 21.3;
// at 16, us at 8 / 16: 156 9.9 / 11.4, 160 11.8 / 11.2, 208 12.5 / 12.0, 208 of 8 heads a kv head of 256
// 21.8 / 19.2; at 32, us at 16 / 32: 192 of 64 15.1 / 17.0).
// A short list is one workgroup's, which saves the merge's launch: 128 positions 7.2 us at 4 tiles,
// 5.4 at 8 (8 heads a kv head of 256 10.3 / 9.1), 256 positions 7.5 at 4, 7.2 at 16 (64 heads of 64 7.5 /
// 7.1; but 5 heads a kv head of 256 10.6 / 13.4, 12 of 128 8.9 / 9.2), 512 7.9 at 4, 10.9 at 32.
RTXLLM_HD std::uint32_t attn_per(std::uint64_t items, std::uint64_t tiles, bool whole, bool light) {
  if (!whole && tiles <= (light ? 16u : 8u)) return tiles <= 8u ? 8u : 16u;
  std::uint32_t per = kMaxPer;
  for (; per > kWaves; per /= 2u) {
    const std::uint64_t splits = (tiles + per - 1u) / per, enough = per == 8u ? 129u : per == 16u ? 160u : 256u;
    if (items * splits >= enough && (!whole || per <= 16u || splits >= 12u)) break;
  }
  return per;
}

// The tiles of a split of a row that has `tiles`: a.per, but a row much shorter than what
// there is room for (a list that ends early, a cache that is not full) is split anew, into at
// most as many parts (us without / with: 9997 positions of four, lists of 120 pages of 256
// 37.9 / 22.1; one of 600, lists of 1024 pages of 16 15.8 / 10.3; 2000 slots of 32768 21.9 / 9.7, of
// eight 51.3 / 26.8, contexts up to 16384 of eight in 16384 68 / 62). A list's end is looked for
// by every workgroup from the list's start, 64 entries at a time: full lists of 128 pages of 16
// of 8 kv heads take 8.9 us and 0.2 less with the end known, 1024 19.7 and 2.2, 8192 122 and
// 34, 65536, the most, 2230 and 1530.
template <bool WEIGHTS>
__device__ __forceinline__ std::uint32_t row_per(const AttnArgs& a, std::uint32_t items, std::uint32_t tiles, bool light) {
  if (a.splits == 1u || 2u * tiles > a.per * a.splits) return a.per;
  std::uint32_t per = attn_per(items, tiles, WEIGHTS, light);
  while (per * a.splits < tiles) per *= 2u;
  return WEIGHTS && per > a.per ? a.per : per;
}

// One workgroup of four waves per (split, kv head, row); a wave takes tiles of 16
// positions of its split in turn, with a running maximum and sum for every head:
//  * scores: S = K q^T by v_mfma_f32_16x16x32_f16. A = the K rows as stored (lane:
//    position l % 16, 8 dims of each 32); B = q of head n / 2 as an fp16 hi (n even) / lo
//    (n odd) pair, brought by a power of two to 2^14..2^15 in its largest element, so that
//    the subnormals come late: products are exact, an element is off by 2^-22 of itself or,
//    where lo is subnormal, by 2^-25 of 2^14, 2^-39 of the largest;
//  * p = 2^(s - m + 15) split into an fp16 hi / lo pair alike (the largest p is 2^15, the
//    sum l is lifted as well): terms down to 2^-18 of the largest keep 22 bits, smaller
//    ones are off by 2^-40 of the largest at most, which 2^16 positions add up to one
//    rounding of fp32;
//  * o += V^T p by v_mfma_f32_4x4x4_16b_f16: a lane holds its own dimensions of
//    four positions, as the V rows' coalesced loads leave them, and one column of p,
//    fetched from the score layout by ds_bpermute. A lane's 4 results are one head's,
//    so its rescaling is one factor;
//  * WIDE (9 to 16 heads): a column a head, hi and lo in two MFMAs of the scores, and o by
//    v_mfma_f32_16x16x4_4b_f16, whose A has the same layout: a quarter of the
//    instructions and exchanges of four 4x4 columns (12 heads of 128 83 -> 63 us).
// T: heads in fours (1, 2, 4). WEIGHTS: every slot, the scores kept for merge_weights_kernel.
// Bound by the reads of K and V: 4096 listed positions of eight sequences (134 MB)
// 25.2 us, 5.3 TB/s (a 1 GiB copy: 5.2); without loads running ahead 33.9, with two sets of
// registers in flight, at half the waves, 31.4; with loads that stay in the caches, which a
// step's other reads need more, 26.8. Workgroups next to each other take the
// kv heads of one place, which lie next to each other in a page.
// Waves a SIMD that the registers are held down for, where that pays: 9 to 16 heads (with
// weights, 12 heads a kv head, 8 kv heads, six contexts to 16000: of 64 35.9 -> 33.1 us, though
// two registers spill, of 128 62.9 -> 58.9; 52 listed pages of 64 of seven to 4377, of 256: 51.0 ->
// 45.7; of 256 with weights it spills more, six to 8000 67 -> 109, and up to 8 heads of 128 with
// weights lose, eight to 16384 of 4 heads 68 -> 80). 12 heads over 64 listed pages of 64 of eight
// take the time of their reads: of 128 (134 MB) 25.1 us, of 256 (268 MB) 49.1, 5.4 TB/s.
template <int D, int T, bool WEIGHTS>
constexpr int attn_waves() { return T < 4 || (D == 256 && WEIGHTS) ? 1 : D == 64 ? 3 : 2; }
template <int D, int T, bool WEIGHTS>
__global__ __launch_bounds__(kThreads, (attn_waves<D, T, WEIGHTS>())) void paged_attn_kernel(AttnArgs a, PagedView kv) {
  constexpr bool WIDE = T == 4;
  constexpr std::uint32_t kHeads = 4u * T;   // heads a workgroup has room for
  constexpr int J = D / 32;                  // score MFMAs of a tile
  constexpr int VD = D == 256 ? 4 : 2;       // dims a lane holds of a V row
  constexpr int RPL = D == 64 ? 2 : 1;       // V rows a load covers
  constexpr int STEPS = 4 / RPL;             // 4-position steps of a tile
  __shared__ __align__(16) float rec[kWaves][kHeads][D];
  __shared__ float2 rml[kWaves][kHeads];
  extern __shared__ __align__(16) float held[];
  const std::uint32_t split = blockIdx.x / kv.n_kv, g = blockIdx.x % kv.n_kv, r = blockIdx.y;
  const std::uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const std::uint32_t col = lane & 15u, qq = lane >> 4;
  const std::size_t gr = static_cast<std::size_t>(r) * kv.n_kv + g;
  const std::size_t head0 = gr * a.group;  // first query head of the kv head, over all rows
  const std::int32_t* const table = kv.table + static_cast<std::size_t>(r) * kv.table_stride;
  // (WEIGHTS: every slot; else the listed pages)
  const std::int32_t* const list = WEIGHTS ? nullptr : a.pages + gr * a.n_select;
  const std::uint32_t room = WEIGHTS ? kv.capacity : a.n_select * kv.page_size;

  // From a tile to the cache row of the lane's position (place col of it) in two
  // dependent reads, each with a register of its own, so that they run ahead: the
  // list's entry three tiles, the table's two. Indices past the end read the last entry.
  auto place_of = [&](std::uint32_t tile) {
    const std::uint32_t x = tile * kTile + col;
    return x < room ? x : room - 1u;
  };
  std::int32_t entry = 0, entry_next = 0, page = 0;
  auto load_entry = [&](std::uint32_t tile) {
    const std::uint32_t e = page_of(kv, place_of(tile));
    return WEIGHTS ? static_cast<std::int32_t>(e) : list[e];
  };
  auto load_page = [&](std::int32_t e) {
    const auto lp = static_cast<std::uint32_t>(e);
    return table[lp < kv.entries ? lp : kv.entries - 1u];
  };
  std::uint32_t per = a.per, tile0 = split * per + wave;
  // the list's first 64 entries, a lane each, for its length below
  const std::int32_t listed = WEIGHTS ? 0 : list[lane < a.n_select ? lane : 0u];
  entry = load_entry(tile0);
  entry_next = load_entry(tile0 + kWaves);

  // B operands of the scores and the column's power of two
  const std::uint32_t h = WIDE ? col : col / 2u;  // the lane's head
  const bool my_head = h < a.group;
  uint4 qb[WIDE ? 2 : 1][J];
  float qscale;
  {
    const float* qr = a.q + (head0 + (my_head ? h : 0u)) * D + 8u * qq;
    f32x4_any x[J][2];
    float m = 0.0f;
#pragma unroll
    for (int j = 0; j < J; ++j) {
      x[j][0] = *reinterpret_cast<const f32x4_any*>(qr + 32 * j);
      x[j][1] = *reinterpret_cast<const f32x4_any*>(qr + 32 * j + 4);
    }
    page = load_page(entry);  // with the query in flight
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) m = fmaxf(m, fmaxf(fabsf(x[j][0][i]), fabsf(x[j][1][i])));
    m = fmaxf(m, lane_xor<16>(m));
    m = fmaxf(m, lane_xor<32>(m));
    int e = 0;
    if (m > 0.0f && m < INFINITY) frexpf(m, &e);
    qscale = ldexpf(1.4426950408889634f / (D == 64 ? 8.0f : D == 128 ? 11.313708498984761f : 16.0f), e - kLift);
#pragma unroll
    for (int j = 0; j < J; ++j) {
      half8 hi, lo;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float v = my_head ? ldexpf(x[j][i / 4][i & 3], kLift - e) : 0.0f;
        asm("" : "+v"(v));  // one rounded value for hi and lo
        hi[i] = static_cast<_Float16>(v);
        lo[i] = static_cast<_Float16>(v - static_cast<float>(hi[i]));
      }
      if constexpr (WIDE) {
        qb[0][j] = __builtin_bit_cast(uint4, hi);
        qb[1][j] = __builtin_bit_cast(uint4, lo);
      } else {
        const uint4 uh = __builtin_bit_cast(uint4, hi), ul = __builtin_bit_cast(uint4, lo);
        qb[0][j] = (col & 1u) == 0u ? uh : ul;
      }
    }
  }

  const std::uint32_t n = paged_filled(kv, a.pos[r]);
  if (n == 0u) return;  // a padded row
  std::uint32_t total = n;
  if constexpr (!WEIGHTS) {  // up to the list's last entry that names a page of the table
    total = 0u;
    for (std::uint32_t i = 0; i < a.n_select; i += 64u) {
      const std::uint32_t e = i + lane;
      const std::int32_t lp = i == 0u ? listed : list[e < a.n_select ? e : 0u];
      const unsigned long long b = __ballot(e < a.n_select && static_cast<std::uint32_t>(lp) < kv.entries);
      if (b != 0ull) total = (i + 64u - static_cast<std::uint32_t>(__builtin_clzll(b))) * kv.page_size;
    }
  }
  const std::uint32_t tiles = (total + kTile - 1u) / kTile;
  per = row_per<WEIGHTS>(a, gridDim.y * kv.n_kv, tiles, D < 256 && !WIDE);
  if (per != a.per) {
    tile0 = split * per + wave;
    entry = load_entry(tile0);
    entry_next = load_entry(tile0 + kWaves);
    page = load_page(entry);
  }
  if (split * per >= tiles) {  // nothing of the row is here
    if constexpr (!WEIGHTS) {
      for (std::uint32_t i = threadIdx.x; i < a.group * D; i += kThreads) {
        if (a.splits == 1u)
          a.out[head0 * D + i] = 0.0f;
        else
          a.part[((head0 + i / D) * a.splits + split) * D + i % D] = 0.0f;
      }
      if (a.splits > 1u && threadIdx.x < a.group)
        a.ml[(head0 + threadIdx.x) * a.splits + split] = make_float2(-INFINITY, 0.0f);
    }
    return;
  }
  const std::uint32_t tile1 = split * per + per < tiles ? split * per + per : tiles;

  float m = -INFINITY, l = 0.0f;
  f32x4 o[WIDE ? 1 : T][VD];
  f32x16 ow[WIDE ? VD : 1];
  if constexpr (WIDE) {
#pragma unroll
    for (int s = 0; s < VD; ++s) ow[s] = f32x16{};
  } else {
#pragma unroll
    for (int t = 0; t < T; ++t)
#pragma unroll
      for (int s = 0; s < VD; ++s) o[t][s] = f32x4{};
  }

  // A tile's keys and values and which of its positions count. One that does not reads
  // row 0 of the cache; its score and value are dropped.
  u32x4 ka[J];
  std::uint32_t vw[16 / RPL][VD / 2], valid = 0u, row = 0u;
  auto settle = [&](std::uint32_t tile) {  // from `entry` and `page`, those of the tile
    const std::uint32_t x = place_of(tile), off = x - page_of(kv, x) * kv.page_size;
    const auto lp = static_cast<std::uint32_t>(entry);
    const std::uint32_t at = paged_row(kv, page, g, off);
    const bool there = tile < tile1 && tile * kTile + col < room && lp < kv.entries && at != kNoRow &&
                       lp * kv.page_size + off < n;
    valid = static_cast<std::uint32_t>(__ballot(there)) & 0xFFFFu;
    row = there ? at : 0u;
  };
  auto load_k = [&]() {
    const u32x4* kr = reinterpret_cast<const u32x4*>(kv.k + static_cast<std::size_t>(row) * D) + qq;
#pragma unroll
    for (int j = 0; j < J; ++j) ka[j] = __builtin_nontemporal_load(kr + 4 * j);
  };
  auto load_v = [&]() {
#pragma unroll
    for (int j = 0; j < 16 / RPL; ++j) {
      if constexpr (D == 64) {
        const std::uint32_t r0 = __builtin_amdgcn_readlane(row, 8 * (j / 4) + (j & 3)),
                            r1 = __builtin_amdgcn_readlane(row, 8 * (j / 4) + 4 + (j & 3));
        const std::uint32_t rr = lane < 32u ? r0 : r1;
        vw[j][0] = __builtin_nontemporal_load(reinterpret_cast<const std::uint32_t*>(kv.v + static_cast<std::size_t>(rr) * D) + (lane & 31u));
      } else {
        const std::uint32_t rr = __builtin_amdgcn_readlane(row, j);
        const std::uint16_t* vr = kv.v + static_cast<std::size_t>(rr) * D;
        if constexpr (D == 128) {
          vw[j][0] = __builtin_nontemporal_load(reinterpret_cast<const std::uint32_t*>(vr) + lane);
        } else {
          const u32x2 t = __builtin_nontemporal_load(reinterpret_cast<const u32x2*>(vr) + lane);
          vw[j][0] = t.x, vw[j][1] = t.y;
        }
      }
    }
  };
  // Loads run ahead of use without a second set of registers: the next tile's keys are
  // read once this tile's scores have used theirs, its values after this tile's sums.
  // No branch skips a load, so each wait is for the loads it needs alone (behind the
  // last tile row 0 is read, from the L2).
  settle(tile0);
  load_k();
  entry = entry_next;
  page = load_page(entry);
  entry_next = load_entry(tile0 + 2u * kWaves);
  load_v();
  for (std::uint32_t tile = tile0; tile < tile1; tile += kWaves) {
    const std::uint32_t now = valid;
    f32x4 sc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int k = 0; k < (WIDE ? 2 : 1); ++k)
#pragma unroll
      for (int j = 0; j < J; ++j)
        sc = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, ka[j]), __builtin_bit_cast(half8, qb[k][j]),
                                                    sc, 0, 0, 0);
    settle(tile + kWaves);
    load_k();
    entry = entry_next;
    page = load_page(entry);
    entry_next = load_entry(tile + 3u * kWaves);
    // positions 4 qq + i of the lane's head
    float s4[4], top = -INFINITY;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float t = (WIDE ? sc[i] : sc[i] + lane_xor<1>(sc[i])) * qscale;
      s4[i] = (now >> (4u * qq + i) & 1u) != 0u ? t : -INFINITY;
      top = fmaxf(top, s4[i]);
    }
    if constexpr (WEIGHTS) {
      if ((WIDE || (col & 1u) == 0u) && my_head)
        *reinterpret_cast<f32x4*>(&held[(h * a.per + (tile - split * per)) * kTile + 4u * qq]) = f32x4{s4[0], s4[1], s4[2], s4[3]};
    }
    top = fmaxf(top, lane_xor<16>(top));
    top = fmaxf(top, lane_xor<32>(top));
    const float mn = fmaxf(m, top), base = mn == -INFINITY ? 0.0f : mn;
    const float alpha = __builtin_amdgcn_exp2f(m - base);
    const bool moved = mn != m;
    m = mn;
    float sum = 0.0f;
    half4 p_hi, p_lo;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float p = __builtin_amdgcn_exp2f(s4[i] - base + kLift);
      asm("" : "+v"(p));
      sum += p;
      p_hi[i] = static_cast<_Float16>(p);
      p_lo[i] = static_cast<_Float16>(p - static_cast<float>(p_hi[i]));
    }
    l = l * alpha + sum;
    if (__ballot(moved) != 0ull) {
      if constexpr (WIDE) {
#pragma unroll
        for (int s = 0; s < VD; ++s) ow[s] *= alpha;  // a lane's results are its own head's
      } else {
#pragma unroll
        for (int t = 0; t < T; ++t) {
          const float f = __uint_as_float(from_lane(__float_as_uint(alpha), 8u * t + 2u * (lane & 3u)));
#pragma unroll
          for (int s = 0; s < VD; ++s) o[t][s] *= f;
        }
      }
    }
    if (now != 0xFFFFu) {  // 0 times what lies behind the context must stay 0
#pragma unroll
      for (int j = 0; j < 16 / RPL; ++j) {
        const std::uint32_t at = D == 64 ? 8u * (j / 4) + (lane < 32u ? 0u : 4u) + (j & 3) : j;
#pragma unroll
        for (int s = 0; s < VD / 2; ++s) vw[j][s] = (now >> at & 1u) != 0u ? vw[j][s] : 0u;
      }
    }
#pragma unroll
    for (int st = 0; st < STEPS; ++st) {
      half4 va[VD];
#pragma unroll
      for (int s = 0; s < VD; ++s) {
        const std::uint32_t sel = (s & 1) != 0 ? 0x07060302u : 0x05040100u;  // the high / low halves of two words
        uint2 w;
        w.x = __builtin_amdgcn_perm(vw[4 * st + 1][s / 2], vw[4 * st][s / 2], sel);
        w.y = __builtin_amdgcn_perm(vw[4 * st + 3][s / 2], vw[4 * st + 2][s / 2], sel);
        va[s] = __builtin_bit_cast(half4, w);
      }
      const std::uint32_t row16 = 16u * (RPL == 2 ? 2u * st + (lane >> 5) : st);  // where the step's p lies
      if constexpr (WIDE) {
        const uint2 hi = __builtin_bit_cast(uint2, p_hi), lo = __builtin_bit_cast(uint2, p_lo);
        const half4 bh = __builtin_bit_cast(half4, make_uint2(from_lane(hi.x, row16 + col), from_lane(hi.y, row16 + col)));
        const half4 bl = __builtin_bit_cast(half4, make_uint2(from_lane(lo.x, row16 + col), from_lane(lo.y, row16 + col)));
#pragma unroll
        for (int s = 0; s < VD; ++s) ow[s] = __builtin_amdgcn_mfma_f32_16x16x4f16(va[s], bh, ow[s], 0, 0, 0);
#pragma unroll
        for (int s = 0; s < VD; ++s) ow[s] = __builtin_amdgcn_mfma_f32_16x16x4f16(va[s], bl, ow[s], 0, 0, 0);
      } else {
        const uint2 pk = __builtin_bit_cast(uint2, (col & 1u) == 0u ? p_hi : p_lo);
#pragma unroll
        for (int t = 0; t < T; ++t) {
#pragma unroll
          for (int part = 0; part < 2; ++part) {
            const std::uint32_t src = row16 + 8u * t + 2u * (lane & 3u) + part;
            const half4 pb = __builtin_bit_cast(half4, make_uint2(from_lane(pk.x, src), from_lane(pk.y, src)));
#pragma unroll
            for (int s = 0; s < VD; ++s) o[t][s] = __builtin_amdgcn_mfma_f32_4x4x4f16(va[s], pb, o[t][s], 0, 0, 0);
          }
        }
      }
    }
    load_v();
  }

  // the waves' records, merged: o = sum e^(m_w - M) o_w, L alike
  l += lane_xor<16>(l);
  l += lane_xor<32>(l);
  // a NaN among the scores makes the row NaN, also where no number gave a maximum
  if (qq == 0u && (WIDE || (col & 1u) == 0u) && h < kHeads) rml[wave][h] = make_float2(l != l ? INFINITY : m, l);
  if constexpr (WIDE) {
    // register 4 b + i: lane 16 b + 4 qq + i of the values' loads
#pragma unroll
    for (int b = 0; b < (D == 64 ? 2 : 4); ++b) {
      float v[4 * VD];
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int s = 0; s < VD; ++s)
          v[VD * i + s] = D == 64 ? ow[s][4 * b + i] + ow[s][(4 * b + i + 8) % 16] : ow[s][4 * b + i];
      float* dst = &rec[wave][col][VD * (16 * b + 4u * qq)];
#pragma unroll
      for (int i = 0; i < VD; ++i)
        *reinterpret_cast<f32x4*>(dst + 4 * i) = f32x4{v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]};
    }
  } else {
#pragma unroll
    for (int t = 0; t < T; ++t) {
      if constexpr (D == 64) {
#pragma unroll
        for (int s = 0; s < VD; ++s)
#pragma unroll
          for (int i = 0; i < 4; ++i) o[t][s][i] += lane_xor<32>(o[t][s][i]);
      }
      if (D != 64 || lane < 32u) {
        float* dst = &rec[wave][4 * t + (lane & 3u)][VD * (lane & ~3u)];
#pragma unroll
        for (int i = 0; i < 4; i += 4 / VD) {
          if constexpr (VD == 2)
            *reinterpret_cast<f32x4*>(dst + 2 * i) = f32x4{o[t][0][i], o[t][1][i], o[t][0][i + 1], o[t][1][i + 1]};
          else
            *reinterpret_cast<f32x4*>(dst + 4 * i) = f32x4{o[t][0][i], o[t][1][i], o[t][VD - 2][i], o[t][VD - 1][i]};
        }
      }
    }
  }
  __syncthreads();
  if constexpr (WEIGHTS) {  // at once and in whole lines: tile by tile from the loop 68 us instead of 61
    const std::uint32_t own = (tile1 - split * per) * (kTile / 4u);
    for (std::uint32_t h = 0; h < a.group; ++h)
      for (std::uint32_t i = threadIdx.x; i < own; i += kThreads)
        *reinterpret_cast<f32x4*>(a.scores + (head0 + h) * a.score_stride + split * per * kTile + 4u * i) =
            *reinterpret_cast<const f32x4*>(&held[h * a.per * kTile + 4u * i]);
  }
  const std::uint32_t items = a.group * (D / 4u);
  for (std::uint32_t it = threadIdx.x; it < items; it += kThreads) {
    const std::uint32_t h = it / (D / 4u), d = 4u * (it % (D / 4u));
    float M = -INFINITY;
#pragma unroll
    for (std::uint32_t w = 0; w < kWaves; ++w) M = fmaxf(M, rml[w][h].x);
    const float base = M == -INFINITY ? 0.0f : M;
    float L = 0.0f;
    f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (std::uint32_t w = 0; w < kWaves; ++w) {
      const float f = __builtin_amdgcn_exp2f(rml[w][h].x - base);
      L += f * rml[w][h].y;
      v += f * *reinterpret_cast<const f32x4*>(&rec[w][h][d]);
    }
    if (!WEIGHTS && a.splits == 1u) {
      const float inv = L == 0.0f ? 0.0f : 1.0f / L;
      *reinterpret_cast<f32x4_any*>(a.out + (head0 + h) * D + d) = f32x4_any(v * inv);
    } else {
      const std::size_t at = (head0 + h) * a.splits + split;
      *reinterpret_cast<f32x4*>(a.part + at * D + d) = v;
      if (d == 0u) a.ml[at] = make_float2(M, L);
    }
  }
}

// Maximum and sum of one head over its splits' records, by one wave.
__device__ __forceinline__ float2 head_ml(const float2* __restrict__ ml, std::uint32_t splits, std::uint32_t lane) {
  float M = -INFINITY, l = 0.0f;
  for (std::uint32_t c0 = 0; c0 < splits; c0 += 256u) {  // (one round up to 32768 positions; 131072 of one pair: two)
    float2 x[4];
    float m = M;
#pragma unroll
    for (std::uint32_t i = 0; i < 4u; ++i) {
      const std::uint32_t c = c0 + lane + 64u * i;
      x[i] = c < splits ? ml[c] : make_float2(-INFINITY, 0.0f);
    }
#pragma unroll
    for (std::uint32_t i = 0; i < 4u; ++i) m = fmaxf(m, x[i].x);
    m = wave_max(m);
    const float base = m == -INFINITY ? 0.0f : m;
    l *= __builtin_amdgcn_exp2f(M - base);
#pragma unroll
    for (std::uint32_t i = 0; i < 4u; ++i) l += x[i].y * __builtin_amdgcn_exp2f(x[i].x - base);
    M = m;
  }
  return make_float2(M, wave_sum(l));
}

// One workgroup a query head (of all rows): its splits' records merged, D / 4
// lanes a record, eight records of a lane in flight.
template <int D>
__device__ __forceinline__ void merge_head(const AttnArgs& a, std::size_t head, std::uint32_t splits) {
  constexpr std::uint32_t kLanes = D / 4u, kSub = kThreads / kLanes;
  __shared__ __align__(16) float sums[kSub][D];
  const std::uint32_t d = 4u * (threadIdx.x % kLanes), sub = threadIdx.x / kLanes;
  const float2* const ml = a.ml + head * a.splits;
  const float* const part = a.part + head * a.splits * D + d;
  f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
  float M = -INFINITY;
  for (std::uint32_t c0 = sub; c0 < splits; c0 += 8u * kSub) {
    f32x4 x[8];
    float m[8], top = M;
#pragma unroll
    for (std::uint32_t j = 0; j < 8u; ++j) {
      const std::uint32_t c = c0 + kSub * j < splits ? c0 + kSub * j : c0;  // past the last: read again, weighted 0
      x[j] = *reinterpret_cast<const f32x4*>(part + static_cast<std::size_t>(c) * D);
      m[j] = ml[c].x;
    }
#pragma unroll
    for (std::uint32_t j = 0; j < 8u; ++j) top = fmaxf(top, m[j]);
    const float base = top == -INFINITY ? 0.0f : top;
    v *= __builtin_amdgcn_exp2f(M - base);
#pragma unroll
    for (std::uint32_t j = 0; j < 8u; ++j) v += (c0 + kSub * j < splits ? __builtin_amdgcn_exp2f(m[j] - base) : 0.0f) * x[j];
    M = top;
  }
  const float2 t = head_ml(ml, splits, threadIdx.x & 63u);
  v *= __builtin_amdgcn_exp2f(M - (t.x == -INFINITY ? 0.0f : t.x));
  *reinterpret_cast<f32x4*>(&sums[sub][d]) = v;
  __syncthreads();
  if (sub != 0u) return;
#pragma unroll
  for (std::uint32_t k = 1; k < kSub; ++k) v += *reinterpret_cast<const f32x4*>(&sums[k][d]);
  const float inv = t.y == 0.0f ? 0.0f : 1.0f / t.y;
  *reinterpret_cast<f32x4_any*>(a.out + head * D + d) = f32x4_any(v * inv);
}

template <int D>
__global__ __launch_bounds__(kThreads) void merge_kernel(AttnArgs a, PagedView kv) {
  const std::uint32_t r = blockIdx.y;
  if (paged_filled(kv, a.pos[r]) == 0u) return;
  merge_head<D>(a, static_cast<std::size_t>(r) * gridDim.x + blockIdx.x, a.splits);
}

// The first `group` workgroups of (kv head, row) merge a head each; the others
// add the softmax weights of 1024 slots each.
template <int D>
__global__ __launch_bounds__(kThreads) void merge_weights_kernel(AttnArgs a, PagedView kv, const float* weight,
                                                                 float* weight_out) {
  __shared__ float base_s[kMaxQueryGroup], inv_s[kMaxQueryGroup];
  const std::uint32_t g = blockIdx.y, r = blockIdx.z, n = paged_filled(kv, a.pos[r]);
  if (n == 0u) return;
  const std::size_t gr = static_cast<std::size_t>(r) * kv.n_kv + g, head0 = gr * a.group;
  const std::uint32_t tiles = (n + kTile - 1u) / kTile;
  const std::uint32_t per = row_per<true>(a, gridDim.y * gridDim.z, tiles, false);
  const std::uint32_t splits = (tiles + per - 1u) / per;  // those with a record
  if (blockIdx.x < a.group) {
    merge_head<D>(a, head0 + blockIdx.x, splits);
    return;
  }
  const std::uint32_t i0 = (blockIdx.x - a.group) * 4u * kThreads + 4u * threadIdx.x;
  if (i0 - 4u * threadIdx.x >= n) return;
  const std::uint32_t lane = threadIdx.x & 63u;
  for (std::uint32_t h = threadIdx.x >> 6; h < a.group; h += kWaves) {
    const float2 t = head_ml(a.ml + (head0 + h) * a.splits, splits, lane);
    if (lane == 0u) {
      base_s[h] = t.x == -INFINITY ? 0.0f : t.x;
      inv_s[h] = t.y == 0.0f ? 0.0f : static_cast<float>(1 << kLift) / t.y;  // (a large base would swallow the lift)
    }
  }
  __syncthreads();
  if (i0 >= n) return;
  f32x4 w = {0.0f, 0.0f, 0.0f, 0.0f};
  for (std::uint32_t h = 0; h < a.group; ++h) {
    const f32x4 s = *reinterpret_cast<const f32x4*>(a.scores + (head0 + h) * a.score_stride + i0);
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] += __builtin_amdgcn_exp2f(s[i] - base_s[h]) * inv_s[h];
  }
  const std::size_t at = gr * kv.capacity + i0;
  if (i0 + 4u <= n) {
    *reinterpret_cast<f32x4_any*>(weight_out + at) =
        *reinterpret_cast<const f32x4_any*>(weight + at) + f32x4_any(w);
  } else {
    for (std::uint32_t i = 0; i < n - i0; ++i) weight_out[at + i] = weight[at + i] + w[i];
  }
}

struct AttnSpace {
  std::uint32_t per = 0, splits = 0, score_stride = 0;
  std::size_t ml = 0, part = 0, scores = 0;  // byte offsets past the start
  std::size_t bytes = 0;                     // 0: refused
};

AttnSpace attn_space(const rtxllm_paged_kv* c, std::uint32_t n_heads, std::uint64_t positions, std::uint32_t count,
                     bool weights) {
  AttnSpace s;
  if (!paged_cache_ok(c, count) || count == 0u || count > 65535u || c->n_kv_heads > 65535u ||
      paged_group(c, n_heads) == 0u || positions == 0u || positions > (1ull << 30))
    return s;
  s.per = attn_per(static_cast<std::uint64_t>(count) * c->n_kv_heads, (positions + kTile - 1u) / kTile, weights,
                   c->head_dim < 256u && paged_group(c, n_heads) <= 8u);
  s.splits = static_cast<std::uint32_t>((positions + kTile * s.per - 1u) / (kTile * s.per));
  if (static_cast<std::uint64_t>(s.splits) * c->n_kv_heads > (1u << 23)) return s;  // the launch's thread count
  const std::size_t records = static_cast<std::size_t>(count) * n_heads * s.splits;
  s.part = round_256(8u * records);
  s.scores = s.part + round_256(4u * records * c->head_dim);
  s.bytes = s.scores;
  if (weights) {
    s.score_stride = (c->capacity + kTile - 1u) / kTile * kTile;
    s.bytes += round_256(4u * static_cast<std::size_t>(count) * n_heads * s.score_stride);
  }
  return s;
}

template <int D, bool WEIGHTS>
void launch_partial(const AttnArgs& a, const PagedView& view, std::uint32_t count, hipStream_t stream) {
  const dim3 grid(a.splits * view.n_kv, count);
  // a split's scores: 64 KB at most (16 heads of 64 tiles), beside at most 66 KB of records
  static_assert(4u * kMaxQueryGroup * kMaxPer * kTile <= 65536u, "fits the LDS");
  const std::size_t lds = WEIGHTS ? 4u * a.group * a.per * kTile : 0u;
  if (a.group <= 4u)
    hipLaunchKernelGGL((paged_attn_kernel<D, 1, WEIGHTS>), grid, dim3(kThreads), lds, stream, a, view);
  else if (a.group <= 8u)
    hipLaunchKernelGGL((paged_attn_kernel<D, 2, WEIGHTS>), grid, dim3(kThreads), lds, stream, a, view);
  else
    hipLaunchKernelGGL((paged_attn_kernel<D, 4, WEIGHTS>), grid, dim3(kThreads), lds, stream, a, view);
}

template <int D>
hipError_t launch_pages(const AttnArgs& a, const PagedView& view, std::uint32_t count, hipStream_t stream) {
  launch_partial<D, false>(a, view, count, stream);
  const hipError_t rc = hipGetLastError();
  if (rc != hipSuccess || a.splits == 1u) return rc;
  hipLaunchKernelGGL(merge_kernel<D>, dim3(a.group * view.n_kv, count), dim3(kThreads), 0, stream, a, view);
  return hipGetLastError();
}

template <int D>
hipError_t launch_weights(const AttnArgs& a, const PagedView& view, std::uint32_t count, const float* weight,
                          float* weight_out, hipStream_t stream) {
  launch_partial<D, true>(a, view, count, stream);
  const hipError_t rc = hipGetLastError();
  if (rc != hipSuccess) return rc;
  const std::uint32_t chunks = (view.capacity + 4u * kThreads - 1u) / (4u * kThreads);
  hipLaunchKernelGGL(merge_weights_kernel<D>, dim3(a.group + chunks, view.n_kv, count), dim3(kThreads), 0, stream, a,
                     view, weight, weight_out);
  return hipGetLastError();
}

AttnArgs attn_args(const float* q, const std::uint32_t* pos, float* out, void* workspace, const AttnSpace& s,
                   std::uint32_t group) {
  auto* base = static_cast<std::uint8_t*>(workspace);
  AttnArgs a{};
  a.q = q;
  a.pos = pos;
  a.out = out;
  a.ml = reinterpret_cast<float2*>(base);
  a.part = reinterpret_cast<float*>(base + s.part);
  a.scores = reinterpret_cast<float*>(base + s.scores);
  a.group = group;
  a.per = s.per;
  a.splits = s.splits;
  a.score_stride = s.score_stride;
  return a;
}

// out is q itself (a workgroup has read its heads before it writes them) or shares no memory with it.
bool attn_pointers_ok(const float* q, const std::uint32_t* pos, const float* out, const void* workspace,
                      std::uint64_t rows_bytes) {
  return q != nullptr && pos != nullptr && out != nullptr && workspace != nullptr && aligned_to(q, 4u) &&
         aligned_to(pos, 4u) && aligned_to(out, 4u) && aligned_to(workspace, 256u) &&
         (out == q || !overlap(out, rows_bytes, q, rows_bytes));
}

std::uint64_t rows_bytes(const rtxllm_paged_kv* cache, std::uint32_t n_heads, std::uint32_t count) {
  return 4ull * count * n_heads * cache->head_dim;
}

}  // namespace
}  // namespace rtxllm

using namespace rtxllm;

extern "C" size_t rtxllm_attn_pages_workspace(const rtxllm_paged_kv* cache, uint32_t n_heads, uint32_t n_select,
                                              uint32_t count) {
  if (cache == nullptr || n_select == 0u || n_select > 65536u) return 0u;
  return attn_space(cache, n_heads, static_cast<std::uint64_t>(n_select) * cache->page_size, count, false).bytes;
}

extern "C" hipError_t rtxllm_attn_decode_pages_gqa_f16(const rtxllm_paged_kv* cache, const float* q, uint32_t n_heads,
                                                       const int32_t* pages, uint32_t n_select, const uint32_t* pos,
                                                       uint32_t count, float* out, void* workspace,
                                                       size_t workspace_bytes, hipStream_t stream) {
  if (cache == nullptr || pages == nullptr || !aligned_to(pages, 4u) || n_select == 0u || n_select > 65536u ||
      !attn_pointers_ok(q, pos, out, workspace, rows_bytes(cache, n_heads, count)))
    return hipErrorInvalidValue;
  const AttnSpace s = attn_space(cache, n_heads, static_cast<std::uint64_t>(n_select) * cache->page_size, count, false);
  if (s.bytes == 0u || workspace_bytes < s.bytes) return hipErrorInvalidValue;
  // a row of one split has its result while others read their lists and positions
  const std::uint64_t rows = rows_bytes(cache, n_heads, count);
  if (overlap(out, rows, pages, 4ull * count * cache->n_kv_heads * n_select) || overlap(out, rows, pos, 4u * count))
    return hipErrorInvalidValue;
  AttnArgs a = attn_args(q, pos, out, workspace, s, paged_group(cache, n_heads));
  a.pages = pages;
  a.n_select = n_select;
  const PagedView view = paged_view(cache);
  return cache->head_dim == 64u    ? launch_pages<64>(a, view, count, stream)
         : cache->head_dim == 128u ? launch_pages<128>(a, view, count, stream)
                                   : launch_pages<256>(a, view, count, stream);
}

extern "C" size_t rtxllm_attn_weights_workspace(const rtxllm_paged_kv* cache, uint32_t n_heads, uint32_t count) {
  if (cache == nullptr) return 0u;
  return attn_space(cache, n_heads, cache->capacity, count, true).bytes;
}

extern "C" hipError_t rtxllm_attn_decode_weights_gqa_f16(const rtxllm_paged_kv* cache, const float* q,
                                                         uint32_t n_heads, const uint32_t* last, uint32_t count,
                                                         float* out, const float* weight, float* weight_out,
                                                         void* workspace, size_t workspace_bytes, hipStream_t stream) {
  if (cache == nullptr || weight == nullptr || weight_out == nullptr || !aligned_to(weight, 4u) ||
      !aligned_to(weight_out, 4u) || !attn_pointers_ok(q, last, out, workspace, rows_bytes(cache, n_heads, count)) ||
      (cache->table_stride == 0u && count > 1u))
    return hipErrorInvalidValue;
  const AttnSpace s = attn_space(cache, n_heads, cache->capacity, count, true);
  if (s.bytes == 0u || workspace_bytes < s.bytes) return hipErrorInvalidValue;
  const std::size_t n = 4u * static_cast<std::size_t>(count) * cache->n_kv_heads * cache->capacity;
  const std::uint64_t rows = rows_bytes(cache, n_heads, count);
  // some workgroups of the merge write results while others read weights
  if ((weight_out != weight && overlap(weight_out, n, weight, n)) || overlap(out, rows, weight, n) ||
      overlap(out, rows, weight_out, n) || overlap(weight_out, n, last, 4u * count) || overlap(out, rows, last, 4u * count))
    return hipErrorInvalidValue;
  const AttnArgs a = attn_args(q, last, out, workspace, s, paged_group(cache, n_heads));
  const PagedView view = paged_view(cache);
  return cache->head_dim == 64u    ? launch_weights<64>(a, view, count, weight, weight_out, stream)
         : cache->head_dim == 128u ? launch_weights<128>(a, view, count, weight, weight_out, stream)
                                   : launch_weights<256>(a, view, count, weight, weight_out, stream);
}
