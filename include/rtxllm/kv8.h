/* C-ABI of a paged KV cache held in 8 bits: new keys and values are quantised as they
 * are written, with one scale for each block of positions and head; positions are read
 * back as rows; new tokens (one a sequence, a few, a prompt) attend over it, with or
 * without a sliding window. No counterpart in the reference (its KV is a flat fp32
 * arena of side-writes, decode_kernels.cu:1600-1606). The rules of rtxllm/paged_kv.h
 * for streams, captures, workspaces and errors hold here too.
 *
 * Positions b block .. b block + block - 1 of a sequence are block b. A block of which all
 * positions are held is whole: it lies in the pages as codes. The newest block, while
 * it is not whole, lies in the tail as fp16 values. So what a cache holds does not
 * depend on how its tokens came, one at a time or as a prompt.
 *
 * A value enters as fp16 (to nearest, beyond its range to an infinity). With top the
 * largest |value| of a whole block of one head, over positions and dimensions:
 * RTXLLM_KV8_INT8: scale = top times the fp32 number 1 / 127, rounded to fp32, code = the nearest integer to
 * value / scale, the even one of two, decided exactly (so |code| <= 127); RTXLLM_KV8_E4M3: scale = the least power of two
 * with top / scale <= 448, code = the nearest e4m3 number (OCP: 4 exponent bits,
 * largest 448, subnormals of 2^-9) to value / scale, the even one of two. top 0: scale 0 and
 * codes 0. A block with a value that is not finite: scale NaN and codes 0, so that all
 * of it reads as NaN. What a code stands for is code * scale. */
#ifndef RTXLLM_KV8_H
#define RTXLLM_KV8_H

#include <hip/hip_runtime_api.h>
#include <stddef.h>
#include <stdint.h>

#include "rtxllm/paged_kv.h"

#ifdef __cplusplus
extern "C" {
#endif

enum { RTXLLM_KV8_INT8 = 0, RTXLLM_KV8_E4M3 = 1 };

/* A layer's cache. Sequence s reads the block table's row s, table_stride entries
 * after row 0's start (0: a call is of one sequence), and row s of the tails. An entry
 * outside [0, n_pages) names no page: its positions are neither read nor written. */
typedef struct {
  uint8_t* k;      /* codes [n_pages][n_kv_heads][page_size][head_dim], */
  uint8_t* v;      /* 16-byte aligned both */
  float* k_scale;  /* [n_pages][n_kv_heads][page_size / block] */
  float* v_scale;
  uint16_t* k_tail; /* fp16 [sequences][n_kv_heads][block][head_dim], 16-byte aligned: */
  uint16_t* v_tail; /* position p of the newest block, while it is not whole, at p % block */
  const int32_t* block_table;
  uint32_t table_stride; /* 0, or >= capacity / page_size */
  uint32_t n_pages;
  uint32_t n_kv_heads;
  uint32_t head_dim;  /* 64, 128 or 256 */
  uint32_t page_size; /* positions of a page, % block == 0 */
  uint32_t capacity;  /* positions of a sequence, % page_size == 0, <= 2^24 */
  uint32_t block;     /* 8, 16, 32 or 64 */
  int format;         /* RTXLLM_KV8_* */
} rtxllm_paged_kv8;

/* The rows of a call are as rtxllm_attn_window_f16 (rtxllm/paged_kv.h) describes them: sequence s
 * has rows start[s] .. start[s + 1] - 1 (start null: row s alone), which are its
 * positions pos[s], pos[s] + 1, ...
 *
 * New tokens: k and v of `type` (RTXLLM_F32, RTXLLM_F16), heads of head_dim values one
 * behind the other, rows k_stride and v_stride elements apart, any alignment to an
 * element. The cache has to hold the positions before pos[s]; of those the newest block's
 * are read from the tail where the new tokens make it whole. To write a sequence anew from an earlier
 * position, go back to a block's start or within the newest block. Rows that make a block whole leave codes alone, and
 * the rows behind them go over its tail, so a program that may drop rows it has appended (drafts) has to keep the
 * keys and values of the newest block itself, up to block - 1 positions before the first such row: if the dropped rows
 * had made that block whole, append again from its start. Nothing marks a sequence that was cut shorter without that;
 * its next calls read what the dropped rows left. Rows at or behind the capacity store
 * nothing; those of a whole block in no page are dropped. Sequences of one call must not share pages that they
 * write. rows <= 2^20, sequences <= 65535. */
hipError_t rtxllm_kv8_append(const rtxllm_paged_kv8* cache, const void* k, size_t k_stride, const void* v,
                             size_t v_stride, int type, const uint32_t* start, const uint32_t* pos,
                             uint32_t sequences, uint32_t rows, hipStream_t stream);

/* Positions back as rows, k_out and v_out [rows][n_kv_heads][head_dim] of `type` (either null: not wanted; fp16:
 * rounded to nearest), of a cache that holds held[s] positions of sequence s (more than capacity
 * counts as capacity). A row whose position is not held, or lies in no page, is left as it was. */
hipError_t rtxllm_kv8_read(const rtxllm_paged_kv8* cache, const uint32_t* held, const uint32_t* start,
                           const uint32_t* pos, uint32_t sequences, uint32_t rows, int type, void* k_out, void* v_out,
                           hipStream_t stream);

/* rtxllm_attn_window_f16 (rtxllm/paged_kv.h) over this cache, which holds the call's
 * rows already: sequence s holds pos[s] + its rows positions. A query sees the positions as the cache holds them, those
 * of its own call too. Codes enter the products as they are, a key's scale multiplies its scores and a value's its
 * softmax term, which enters as a pair then: off by 2^-22 of itself or 2^-34 of the largest term times scale that
 * the query attends, whatever lies where it does not. Scales that are not finite and tails behind what is held have no effect where they are not
 * attended. (e4m3 codes of NaN, which the append never writes, make NaN of the queries whose call reads
 * them, attended or not.) */
size_t rtxllm_attn_kv8_workspace(const rtxllm_paged_kv8* cache, uint32_t n_heads, uint32_t sequences, uint32_t rows,
                                 uint32_t window, uint32_t sinks);
hipError_t rtxllm_attn_kv8(const rtxllm_paged_kv8* cache, const void* q, int type, uint32_t n_heads,
                           const uint32_t* start, const uint32_t* pos, uint32_t sequences, uint32_t rows,
                           uint32_t window, uint32_t sinks, void* out, void* workspace, size_t workspace_bytes,
                           hipStream_t stream);

#ifdef __cplusplus
}
#endif

#endif
