/*
 * Decode attention that reads the paged cache in place: the consumer of the gather, fused with
 * it.  One query token per sequence attends over that sequence's cached tokens, found through
 * the block table exactly as kvx_launch_gather_kv finds them, so the contiguous K/V copy the
 * gather would write (and attention would read back) never exists.
 *
 * No reference counterpart: the reference stops at the gather (kernels/kvx_paged_kv.h:19-21)
 * and names this fusion as future work.  The cache side keeps the reference's descriptors
 * (kvx_abi.h:73-128: cache tensors with their layout and strides, PACKED block table, sequence
 * lengths) and the gather's conventions for bad data.
 *
 *   out[s][q][:] = sum_t softmax_t(scale * <query[s][q][:], K[s][t][kv(q)][:]>) * V[s][t][kv(q)][:]
 *
 * over the cached tokens t < min(seq_lens[s], max_seq_len) of sequence s that the table
 * resolves (a token whose logical block is >= max_blocks_per_seq, or whose page id is negative
 * or >= num_blocks, takes no part, as in the gather), with kv(q) = q / (num_q_heads /
 * num_kv_heads) (grouped-query attention; num_q_heads a multiple of num_kv_heads).  A sequence
 * with no token that takes part gets out = 0.  Scores, softmax and the weighted sum are
 * accumulated in f32; the result is rounded once to the query's type.
 */
#ifndef KVX_ATTENTION_H
#define KVX_ATTENTION_H

#include "kvx_abi.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef struct kvx_attention_desc {
  uint32_t size;
  uint32_t num_q_heads;   /* a multiple of cache->num_kv_heads */
  uint32_t max_seq_len;   /* tokens beyond it are ignored; bounds the work split */
  float scale;            /* multiplies the scores before the softmax, e.g. 1/sqrt(head_dim) */
  kvx_tensor_desc_t query; /* [seq_count, num_q_heads, head_dim], F16 / BF16 / F32, dense */
  kvx_tensor_desc_t out;   /* same shape and type as query, dense */
  kvx_block_table_t block_table; /* PACKED */
  kvx_seq_lens_t seq_lens;       /* same index type as the table */
} kvx_attention_desc_t;

#if defined(__cplusplus)
static_assert(sizeof(kvx_attention_desc_t) == 328, "kvx_attention_desc_t layout");
#elif defined(__STDC_VERSION__) && __STDC_VERSION__ >= 201112L
_Static_assert(sizeof(kvx_attention_desc_t) == 328, "kvx_attention_desc_t layout");
#endif

/* Bytes of caller-owned DEVICE scratch kvx_launch_paged_attention_decode needs for this
 * problem size: a work counter and, when contexts are split in chunks, the chunks' partial
 * results.  The library allocates nothing itself; the scratch needs no initialisation and may
 * be reused by the next call on the same stream. */
KVX_API size_t kvx_paged_attention_workspace_bytes(uint32_t seq_count, uint32_t num_q_heads,
                                                   uint32_t num_kv_heads, uint32_t head_dim,
                                                   uint32_t max_seq_len);

/* Enqueues the attention on `stream` (1 to 3 kernels) and returns without synchronising.
 *
 * Cache: F16 / BF16 / F32 (query and out of the same type), or F8_E4M3 with 16/32-bit query
 * and F32 scales in k_scale / v_scale (PER_TENSOR or PER_HEAD, as for the fp8 gather; NULL
 * otherwise): K and V are dequantised on the fly as value * scale.
 *
 * Status: INVALID_ARGUMENT for NULL / undersized descriptors, shapes that disagree, a query
 * head count that is not a multiple of the KV heads, scratch smaller than
 * kvx_paged_attention_workspace_bytes() or misaligned (16 bytes); UNSUPPORTED for a table that
 * is not PACKED, mismatched types and non-dense query / out; OK without a launch when there is
 * no sequence.  Bad DATA is skipped as described above. */
KVX_API kvx_status_t kvx_launch_paged_attention_decode(const kvx_cache_desc_t *cache,
                                                       const kvx_attention_desc_t *attn,
                                                       const kvx_scale_desc_t *k_scale,
                                                       const kvx_scale_desc_t *v_scale,
                                                       void *workspace, size_t workspace_bytes,
                                                       void *stream);

/* ------------------------------------------------------------------ a chunk of new tokens ----
 * Several query tokens per sequence over the same pages: a prompt, the next piece of a long one
 * after a cached prefix, drafted tokens that are verified together.  The new tokens' K and V are
 * in the cache already (written by kvx_launch_write_kv or kvx_launch_rotary_write_kv); they are
 * the last ones of the sequence.  With n = query_indptr[s + 1] - query_indptr[s] new tokens,
 * row query_indptr[s] + i of query / out is token i at position seq_lens[s] - n + i, and
 *
 *   out[row][q][:] = sum_t softmax_t(scale * <query[row][q][:], K[s][t][kv(q)][:]>) * V[s][t][kv(q)][:]
 *
 * over the cached tokens t < min(seq_lens[s], max_seq_len) that the table resolves (as above), for
 * causal = 1 only those with t <= the row's position.  A row that sees no token, or whose scores
 * are all -inf, gets out = 0.  A token that is not seen has no influence beyond the rounding of the
 * weights, whatever its page holds.  n may differ from sequence to sequence and may be 0 or exceed
 * seq_lens[s] (rows at negative positions see nothing).  Rows at or beyond `rows`, rows of a
 * sequence with a negative query_indptr, and rows that belong to no sequence stay untouched.  The
 * row ranges of the sequences must not overlap, and out must not overlap query (query rows are
 * read after others were written).  Scores, softmax and sums are f32; on the tensor-core path the
 * softmax weights are rounded once to the query's type before they multiply V: a relative error of
 * half a unit in the last place of that type, of the order of the output's own rounding, and in f16
 * for weights below 2^-21 of the row's largest an absolute one of at most 2^-32 of it (an infinity in
 * the V of a token whose weight becomes zero gives NaN).  The result is rounded once to the query's
 * type. */
typedef struct kvx_chunk_attention_desc {
  uint32_t size;
  uint32_t num_q_heads;    /* a multiple of cache->num_kv_heads */
  uint32_t max_seq_len;    /* cached tokens beyond it are ignored */
  float scale;
  uint32_t causal;         /* 1 or 0 */
  kvx_dtype_t query_indptr_dtype; /* S32 or S64 */
  kvx_tensor_desc_t query; /* [rows, num_q_heads, head_dim], F16 / BF16 / F32; heads and dims dense, */
  kvx_tensor_desc_t out;   /* token rows may be further apart; out: same shape and type */
  kvx_block_table_t block_table; /* PACKED */
  kvx_seq_lens_t seq_lens;       /* same index type as the table */
  const void *query_indptr;      /* DEVICE array of seq_count + 1 row numbers */
} kvx_chunk_attention_desc_t;

#if defined(__cplusplus)
static_assert(sizeof(kvx_chunk_attention_desc_t) == 344, "kvx_chunk_attention_desc_t layout");
#elif defined(__STDC_VERSION__) && __STDC_VERSION__ >= 201112L
_Static_assert(sizeof(kvx_chunk_attention_desc_t) == 344, "kvx_chunk_attention_desc_t layout");
#endif

/* Bytes of caller-owned DEVICE scratch for a batch of `num_rows` new tokens (all sequences): the
 * work plan and the partial results of the tiles that are cut.  At most about 40 MB, whatever the
 * context length; no initialisation needed; may be reused by the next call on the same stream. */
KVX_API size_t kvx_paged_attention_chunk_workspace_bytes(uint32_t seq_count, uint32_t num_rows,
                                                         uint32_t num_q_heads, uint32_t num_kv_heads,
                                                         uint32_t head_dim, uint32_t max_seq_len);

/* Enqueues the attention on `stream` (1 to 3 kernels) and returns without synchronising.  Cache
 * types, layouts and scales as for kvx_launch_paged_attention_decode; head_dim up to 1024 (up to
 * 256 with a 16-bit query on the tensor cores).  Calls that may overlap on the GPU need scratch of
 * their own.
 *
 * Status: INVALID_ARGUMENT for NULL / undersized descriptors, shapes that disagree, a query head
 * count that is not a multiple of the KV heads, causal above 1, out at the query's address,
 * max_seq_len above 2^31 - 1025, scratch smaller than kvx_paged_attention_chunk_workspace_bytes()
 * or misaligned (16 bytes); UNSUPPORTED for a table that is not PACKED, mismatched types, token
 * rows with gaps between or inside heads, rows that overlap, more than 2^31 - 1024 rows x
 * (num_q_heads / num_kv_heads), head_dim above 1024; OK without a launch when there is no sequence
 * or no row. */
KVX_API kvx_status_t kvx_launch_paged_attention_chunk(const kvx_cache_desc_t *cache,
                                                      const kvx_chunk_attention_desc_t *attn,
                                                      const kvx_scale_desc_t *k_scale,
                                                      const kvx_scale_desc_t *v_scale,
                                                      void *workspace, size_t workspace_bytes,
                                                      void *stream);

/* The give-up word of the chunk kernel on the current device, as kvx_b200_device_error: its waits on
 * its own copies and products are abandoned after two seconds, the kernel then returns and leaves
 * rows unwritten.  0 = never happened, 1 = it did, -1 = unreadable; `reset` clears it.  Copies from
 * the device synchronously. */
KVX_API int kvx_attention_device_error(int reset);

#ifdef __cplusplus
}
#endif
#endif /* KVX_ATTENTION_H */
