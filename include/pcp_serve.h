/*
 * C ABI of the serving operators around the paged KV cache: norm and rotation
 * of query and key heads, scaled quantised append and read-back, and causal
 * attention of each sequence's new tokens over its paged cache.  No
 * counterpart in the reference, which attends one striped history at unit
 * scale and leaves "current-token attention" and serving for later
 * (README.md:17-18,52-54); the cache blocks keep its payload format
 * (pcp_attention/kernel.py:17-29).
 *
 * Conventions are those of pcp_attn.h (status codes, pcp_last_error, streams,
 * caller-owned buffers, device pointers of the current device).  Calls are
 * asynchronous on `stream`, allocate nothing, read no device value on the
 * host and may be captured into a CUDA graph.
 *
 * A batch of sequences: rows offsets[b] .. offsets[b + 1] of a packed
 * [heads][rows][head_dim] tensor are sequence b's tokens of this call, and
 * they are the LAST tokens of the kv_len[b] tokens it then has: row r sits at
 * position kv_len[b] - (offsets[b + 1] - r).  Rows outside every sequence are
 * never written.  Position p lives in row p % block_size of pool block
 * block_tables[b][p / block_size].
 *
 * Device status word (DEVICE int32; a call stores its code only over 0, so the
 * first failure since the caller last cleared the word stands):
 *   109  a table entry outside the pool, or a position past the table's width
 *        (append skips the token, read-back writes zeros; attention reads
 *        block 0 in the entry's place and stops at the table's end: rows of
 *        that sequence are then meaningless);
 *   112  a sequence the call does not take.  Append and read-back: a position
 *        below 0 (the token is skipped).  Attention: a negative kv_len (taken
 *        as 0), more rows than max_chunk (the sequence's rows are not
 *        written), offsets that decrease or leave the rows (nothing is
 *        written);
 *   1xx  a wait in the attention kernel that ran out (see pcp_attn.h): rows that
 *        the failed part of the work shares with others are not written.
 */
#ifndef PCP_SERVE_H
#define PCP_SERVE_H

#include <stddef.h>
#include <stdint.h>

#include "pcp_attn.h"

#ifdef __cplusplus
extern "C" {
#endif

/* A packed tensor [heads][rows][head_dim]: head_dim contiguous, the other two
 * axes at any stride (in elements).  Base and strides keep every row 16-byte
 * aligned. */
typedef struct pcp_heads {
  void* data;
  int64_t head_stride;
  int64_t row_stride;
  int32_t heads;
  int32_t reserved;
} pcp_heads_t;

enum pcp_float_dtype { PCP_F32 = 0, PCP_F16 = 1, PCP_BF16 = 2 };

/* Position rotation of the first rotary_dim elements of a head. */
enum pcp_rotary_layout {
  PCP_ROTARY_HALF = 0,       /* pairs (i, i + rotary_dim / 2) */
  PCP_ROTARY_INTERLEAVED = 1 /* pairs (2 i, 2 i + 1) */
};

/* q and k heads, each normed over its head_dim (when its weight is given) and
 * rotated by its row's position, in one pass, rounded once:
 *   y = x * rsqrt(mean(x^2) + eps) * weight
 *   (a, b) -> magnitude * (a cos t - b sin t, b cos t + a sin t)
 * with t = 2 pi * frac(position * turns[i] / 2^64) for pair i: `turns` (DEVICE
 * uint64[rotary_dim / 2]) is a pair's turns per position as a 64-bit fraction,
 * so the product's whole turns fall away exactly and far positions lose
 * nothing.
 *   - dtype: enum pcp_float_dtype of inputs, outputs and weights.
 *   - k.heads may be 0 (queries only).  Outputs may be the inputs themselves
 *     (same base and strides); any other overlap is undefined.
 *   - positions: DEVICE int32 or int64 (positions_64) [rows].
 *   - head_dim a multiple of 16 up to 512, rotary_dim a multiple of 16 up to
 *     head_dim (0: no rotation). */
int pcp_qk_norm_rope(int32_t dtype, int32_t rows, int32_t head_dim, int32_t rotary_dim, int32_t layout,
                     const pcp_heads_t* q, const pcp_heads_t* k, const pcp_heads_t* q_out, const pcp_heads_t* k_out,
                     const void* positions, int32_t positions_64, const uint64_t* turns, float magnitude,
                     const void* q_weight, const void* k_weight, float eps, void* stream);

/* A paged cache: blocks of [2][num_kv_heads][block_size][head_dim] e4m3fn or
 * bf16, K then V.  scales (e4m3 only; NULL: unit scale): one byte b per token,
 * head and K/V, [blocks][2][num_kv_heads][block_size]; the row's values are
 * code * 2^(b - 127), b from 27 to 247, as pcp_cache_append writes them (what other
 * bytes of tokens that are read give is not specified). */
typedef struct pcp_pool {
  void* data;
  uint8_t* scales;
  int64_t blocks;
  int32_t num_kv_heads;
  int32_t head_dim; /* 128 or 256 */
  int32_t block_size; /* a multiple of 16 */
  int32_t kv_dtype; /* enum pcp_kv_dtype */
} pcp_pool_t;

typedef struct pcp_batch {
  const int32_t* offsets;      /* DEVICE [num_seqs + 1] */
  const int32_t* kv_len;       /* DEVICE [num_seqs] */
  const int32_t* block_tables; /* DEVICE [num_seqs][table_width], rows table_stride apart */
  int64_t table_stride;
  int32_t table_width;
  int32_t num_seqs;
  int32_t rows; /* rows of the packed tensors */
  int32_t reserved;
} pcp_batch_t;

/* Writes every sequence's rows of k and v (bf16) into the cache.  With scales,
 * a row of a head is stored as e4m3 codes of x * 2^-e, e the least whole
 * number with max|x| <= 448 * 2^e (0 for a row of zeros, held to -100 .. 120)
 * over the row's finite elements, and b = e + 127: products by powers of two
 * lose nothing, and what is read back is exact in bf16 (but for values that
 * round up to 2^128, which read as infinity; attention takes them as 2^128).
 * Non-finite elements become NaN codes.  Without scales, as pcp_cache_write.  Two rows that map to
 * one slot race. */
int pcp_cache_append(const pcp_pool_t* pool, const pcp_batch_t* batch, const pcp_heads_t* k, const pcp_heads_t* v,
                     int32_t* device_status, void* stream);

/* Reads the last offsets[b + 1] - offsets[b] tokens of every sequence back as
 * bf16 rows of k_out and v_out. */
int pcp_cache_read(const pcp_pool_t* pool, const pcp_batch_t* batch, const pcp_heads_t* k_out,
                   const pcp_heads_t* v_out, int32_t* device_status, void* stream);

/* Causal attention of every sequence's rows of q over its paged cache (the new
 * tokens' K and V already appended): the row at position p sees positions 0 ..
 * p of its own sequence,
 *   out = sum_j softmax_j(softmax_scale * q . k_j) v_j,
 * KV head h serving query heads h * G .. h * G + G - 1.  Single tokens, chunks
 * of a prompt and whole prompts may be mixed in a batch.  Rows that see nothing
 * (positions below 0) are zeros; rows of no sequence are left as they were.
 * What a row does not see (later tokens, pages past the length) costs it
 * nothing, whatever it holds: infinities and NaN there too.  An element of V that is
 * not finite makes its column of the rows that see it not finite (NaN for those of
 * the new tokens themselves).
 * Scores, sums and accumulators are fp32.  Weights are rounded before they meet V: to
 * bf16 over bf16 caches, and over e4m3 caches that chunks read through a bf16 copy
 * (max_chunk * G >= 1024, where the workspace has room for it); to f16 over other e4m3
 * caches, a key's scale included, where contributions of keys below 2^-24 of the
 * row's largest are lost.  Weights up to 2^8 times V are summed before the division:
 * V of a bf16 cache beyond some 2^100 may overflow there.
 *   - max_chunk bounds every sequence's rows (HOST value; it picks which
 *     kernels are launched).  Lengths and tables are read on the device.
 *   - q, out: bf16 [num_q_heads][rows][head_dim] at any 16-byte aligned stride.
 *   - workspace: device memory of pcp_chunk_attention_workspace_size bytes,
 *     aligned to 256, needed until the call's work has run; calls that may
 *     overlap need one each. */
int pcp_chunk_attention_workspace_size(const pcp_pool_t* pool, int32_t num_q_heads, int32_t num_seqs, int32_t rows,
                                       int32_t table_width, int32_t max_chunk, size_t* bytes);
int pcp_chunk_attention(const pcp_pool_t* pool, const pcp_batch_t* batch, const pcp_heads_t* q, const pcp_heads_t* out,
                        int32_t max_chunk, float softmax_scale, void* workspace, size_t workspace_bytes,
                        int32_t* device_status, void* stream);

/* Host-side view of the merge of a unit that work ranges share (the same code
 * the kernel runs), for tests and tools: the parts of the unit that range
 * `range` of `ranges` leaves unfinished.  states (HOST [ranges]): a range's first
 * part is 0 none (of a unit begun before it), 1 one that goes on behind it, 2 the
 * unit's last; failed (HOST [ranges]): not 0 where a wait ran out.  *parts is 0 when
 * the unit is not merged: a part of it is missing or may be unwritten. */
int pcp_chunk_cut_parts(const int32_t* states, const int32_t* failed, int32_t ranges, int32_t range, int32_t* parts);

#ifdef __cplusplus
}
#endif

#endif /* PCP_SERVE_H */
