/* C-ABI of the operators that keep long contexts affordable over the paged fp16
 * KV cache: the append of new keys and values with the norm of every head and
 * its rotation in the same pass; decode attention over pages that a cheap score
 * selects; decode attention that gathers each position's softmax weight, and the
 * eviction of the positions that gathered least. No counterpart in the reference
 * (its KV is a flat fp32 arena of side-writes, decode_kernels.cu:1600-1606).
 *
 * All functions but the workspace sizes are asynchronous on `stream`, allocate
 * nothing, synchronise nothing and are capture-safe; pointers are device
 * pointers of the stream's device except for the cache description, which is
 * read during the call. They return hipSuccess, hipErrorInvalidValue for refused
 * arguments (before any launch), or the launch's error. A workspace belongs to
 * one call until that call's work is done: calls that may overlap (two streams,
 * two graphs replayed at once) need one each. Results do not depend on it or on
 * timing: no call adds with atomics. What a call writes (the workspace among it) shares
 * memory with no other array of the call but where its description allows it. */
#ifndef RTXLLM_PAGED_KV_H
#define RTXLLM_PAGED_KV_H

#include <hip/hip_runtime_api.h>
#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* The position of a padded row: its inputs do not count, whatever they hold (they
 * must be allocated), and no output of it is written. */
#define RTXLLM_NO_POSITION 0xFFFFFFFFu

/* A layer's cache as a call's rows see it. Row r of a call reads the block table
 * row r, table_stride entries after row 0's start; with table_stride 0 every row
 * of the call is of one sequence (a prompt's tokens). capacity / page_size
 * entries of a table row are used. An entry outside [0, n_pages) names no page:
 * its positions are neither read nor written. */
typedef struct {
  uint16_t* k;                /* fp16 [n_pages][n_kv_heads][page_size][head_dim], */
  uint16_t* v;                /* 16-byte aligned both */
  const int32_t* block_table; /* logical page -> physical page */
  uint32_t table_stride;      /* 0, or >= capacity / page_size */
  uint32_t n_pages;
  uint32_t n_kv_heads;
  uint32_t head_dim;  /* 64, 128 or 256 */
  uint32_t page_size; /* positions of a page, any >= 1 */
  uint32_t capacity;  /* positions of a sequence, % page_size == 0, <= 2^24 */
} rtxllm_paged_kv;

/* New tokens of count rows. Per row r and head, with x the head's head_dim fp32
 * values of q or k: x' = x / sqrt(sum(x^2) / head_dim + eps) * weight (q_weight or
 * k_weight, fp32 [head_dim], null: ones), then the first rotary_dim values are
 * rotated in pairs by the angle pos[r] * theta^(-2 i / rotary_dim): (a, b) ->
 * (a cos - b sin, a sin + b cos), pair i being (i, i + rotary_dim / 2) with
 * RTXLLM_PAIR_HALVES and (2 i, 2 i + 1) with RTXLLM_PAIR_ADJACENT. The angle is
 * taken in 64 bits (rtxllm_rope_theta rounds it to fp32: up to pos 2^-24 of a
 * radian apart). q' goes to q_out [count][n_heads][head_dim] (fp32, in place
 * allowed when q_stride is n_heads * head_dim), k' and v, each rounded to fp16
 * once (beyond its range to an infinity), into slot slot[r] of the row's sequence (slot null: pos[r]).
 * q, k and v rows lie q_stride, k_stride and v_stride floats apart (one stacked
 * projection's output: the same stride three times); any 4-byte alignment.
 * rotary_dim % 8 == 0, 8..head_dim. pos[r] RTXLLM_NO_POSITION: a padded row. A slot >=
 * capacity stores nothing, one in no page its position and weight alone; q_out is written all the
 * same.
 * slot_pos, slot_weight (each may be null): uint32 and fp32 [rows][n_kv_heads]
 * [capacity], one row per sequence (one in all with table_stride 0); the new slot
 * gets pos[r] and 0 for every head. Rows of one call must not share a slot.
 * heads = n_heads + 2 n_kv_heads <= 4096, count <= 2^20. */
enum { RTXLLM_PAIR_ADJACENT = 0, RTXLLM_PAIR_HALVES = 1 };
hipError_t rtxllm_qk_norm_rope_append_f16(const rtxllm_paged_kv* cache, const float* q, size_t q_stride,
                                          const float* k, size_t k_stride, const float* v, size_t v_stride,
                                          const float* q_weight, const float* k_weight, uint32_t n_heads,
                                          uint32_t rotary_dim, int pairing, float theta, float eps,
                                          const uint32_t* pos, const uint32_t* slot, uint32_t count, float* q_out,
                                          uint32_t* slot_pos, float* slot_weight, hipStream_t stream);

/* Page bounds: fp16 [n_pages][n_kv_heads][2][head_dim], per physical page and
 * kv head the largest (index 0) and the smallest (1) value of each dimension over
 * the page's filled positions. A NaN does not count, and both are clamped to
 * +-65504 (so a page of NaN alone has -65504 and 65504 in reverse order). The
 * pages that hold positions first[r]..last[r] of sequence r are computed anew
 * (first null: the newest page, last[r]'s), at most `span` of them (1..2^20) from the
 * first on; last[r] >= capacity counts as capacity - 1; last[r] RTXLLM_NO_POSITION
 * or first[r] > last[r]: none. Rows that share pages compute the same values
 * where they fill them alike. bounds 16-byte aligned; count <= 65535; span *
 * n_kv_heads <= 2^24 (a larger span than a sequence has pages counts as that; the
 * launch is sized by it). */
hipError_t rtxllm_kv_page_bounds_f16(const rtxllm_paged_kv* cache, const uint32_t* first, const uint32_t* last,
                                     uint32_t count, uint32_t span, uint16_t* bounds, hipStream_t stream);

/* Per query r (fp32 q [count][n_heads][head_dim], any 4-byte alignment) and kv head
 * the logical pages worth attending, of those that hold positions 0..pos[r]:
 * the first n_first and the last n_last pages, and those with the largest scores,
 * n_select in all (or all there are); pages[r][kv head][n_select], ascending, -1
 * behind the last. score = max over the kv head's query heads h of sum_d
 * max(q_hd largest_d, q_hd smallest_d): no key of the page has a larger product
 * with any of them. The larger product is that with the extreme on q's side (the larger
 * one where q_hd >= 0), the other extreme has no effect. Products are exact and
 * summed in 64 bits, in one order for all pages: scores of like terms are equal, and others
 * come out in order unless they lie within some 2^-45 of their terms' sizes. The lower page wins
 * between equal scores; a head whose
 * sum is NaN does not count (an infinite q gives one where it meets an extreme of 0), and
 * a page where none does ranks last. A page with
 * no entry in the table is never listed.
 * n_heads / n_kv_heads 1..16, n_first + n_last <= n_select <= 65536, count <= 65535.
 * workspace: rtxllm_attn_select_workspace() bytes, 256-byte aligned. */
size_t rtxllm_attn_select_workspace(const rtxllm_paged_kv* cache, uint32_t count);
hipError_t rtxllm_attn_select_pages(const rtxllm_paged_kv* cache, const uint16_t* bounds, const float* q,
                                    uint32_t n_heads, const uint32_t* pos, uint32_t count, uint32_t n_first,
                                    uint32_t n_last, uint32_t n_select, int32_t* pages, void* workspace,
                                    size_t workspace_bytes, hipStream_t stream);

/* GQA decode attention over listed pages: query r attends, for each kv head, the
 * positions <= pos[r] of the logical pages in pages[r][kv head][n_select], in any
 * order; an entry outside the table (-1) is passed over, a page listed twice
 * counts twice. Scores q k / sqrt(head_dim), softmax with the maximum subtracted,
 * sums in fp32; out fp32 [count][n_heads][head_dim]; a row that attends nothing
 * is 0. What a position that is not attended holds, NaN and infinities included, has
 * no effect; a NaN or an infinity among the attended keys or values makes NaN of what
 * it enters, a score beyond fp32 of its head's result. q and the softmax terms enter the products as pairs of fp16: a query off by
 * 2^-22 of itself or 2^-39 of its head's largest at most, a term by 2^-22 of itself or 2^-40
 * of the largest term. out may be q, and shares no memory with it otherwise. n_heads /
 * n_kv_heads 1..16; count <= 65535; n_select 1..65536, n_select * page_size <= 2^30.
 * workspace: rtxllm_attn_pages_workspace() bytes, 256-byte aligned. */
size_t rtxllm_attn_pages_workspace(const rtxllm_paged_kv* cache, uint32_t n_heads, uint32_t n_select,
                                   uint32_t count);
hipError_t rtxllm_attn_decode_pages_gqa_f16(const rtxllm_paged_kv* cache, const float* q, uint32_t n_heads,
                                            const int32_t* pages, uint32_t n_select, const uint32_t* pos,
                                            uint32_t count, float* out, void* workspace, size_t workspace_bytes,
                                            hipStream_t stream);

/* GQA decode attention over slots 0..last[r], which also gathers what each of them
 * weighed: weight_out[r][kv head][s] = weight[r][kv head][s] + the sum over the kv
 * head's query heads of slot s's softmax weight, s <= last[r]; the rest of
 * weight_out is left as it was. weight, weight_out fp32 [count][n_kv_heads]
 * [capacity] (the same array: adds in place). Otherwise as
 * rtxllm_attn_decode_pages_gqa_f16; table_stride 0 only with count 1. */
size_t rtxllm_attn_weights_workspace(const rtxllm_paged_kv* cache, uint32_t n_heads, uint32_t count);
hipError_t rtxllm_attn_decode_weights_gqa_f16(const rtxllm_paged_kv* cache, const float* q, uint32_t n_heads,
                                              const uint32_t* last, uint32_t count, float* out, const float* weight,
                                              float* weight_out, void* workspace, size_t workspace_bytes,
                                              hipStream_t stream);

/* Eviction: sequence r's first length[r] slots are filled (more than capacity
 * counts as capacity); if they are more than `keep`, keep of them stay, for each
 * kv head its own: first those whose position is protected (slot_pos < n_first,
 * or slot_pos + n_recent > pos[r], pos[r] being the newest position; they are all
 * alike), then those with the largest weight; the lower slot between equals; a NaN
 * weight ranks below every number. The i-th kept slot at or behind `keep` moves into the i-th freed slot
 * below it (its key, value, weight and position), so that slots 0..keep - 1 are
 * filled and few rows move; order among slots means nothing to attention, the
 * keys being rotated already. K and V move in the cache; weight_out and
 * slot_pos_out get slots 0..min(length, keep) - 1 and are left as they were
 * behind (each may be its input); length_out[r] = min(length[r], keep) (may be
 * length). A row with pos[r] RTXLLM_NO_POSITION is a padded row. A slot in no
 * page has nothing to move and no room: whatever its weight and position it stays where
 * it lies below keep and leaves where it lies behind, and the others fill what is left of keep.
 * Page bounds do not follow: those of the kept slots' pages are to be computed anew (first 0, last
 * keep - 1). Sequences of one call must not share pages. n_first + n_recent <= keep <=
 * capacity, keep >= 1, count <= 65535; table_stride 0 only with count 1. */
size_t rtxllm_kv_evict_workspace(const rtxllm_paged_kv* cache, uint32_t keep, uint32_t count);
hipError_t rtxllm_kv_evict_f16(const rtxllm_paged_kv* cache, const uint32_t* length, const uint32_t* pos,
                               uint32_t count, uint32_t keep, uint32_t n_first, uint32_t n_recent,
                               const float* weight, const uint32_t* slot_pos, float* weight_out,
                               uint32_t* slot_pos_out, uint32_t* length_out, void* workspace,
                               size_t workspace_bytes, hipStream_t stream);

#ifdef __cplusplus
}
#endif

#endif
