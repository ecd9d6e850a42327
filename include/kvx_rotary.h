/*
 * Rotary positions on queries and keys, alone or fused with the cache write: the step ahead of
 * kvx_launch_write_kv and of the attention entry points (kvx_attention.h).  No reference
 * counterpart; the fused form keeps the reference's write descriptor (kvx_abi.h:172-180).
 *
 * Of every head's `head_dim` elements the first `rotary_dim` are turned in pairs, pair i by the
 * angle a = position * inv_freq[i]:
 *
 *   y1 = factor * (x1 cos a - x2 sin a)        half layout:         x1 = x[i], x2 = x[i + rotary_dim / 2]
 *   y2 = factor * (x2 cos a + x1 sin a)        interleaved layout:  x1 = x[2 i], x2 = x[2 i + 1]
 *
 * and the others are copied.  inv_freq carries whatever scaling for long contexts the model uses
 * (kvx_b200.ops.rotary_inv_freq computes the common ones); `factor` is its factor on the values,
 * 1 where it has none.  KVX_ROTARY_INVERSE turns by -a: the transposed map, i.e. the gradient of the
 * forward call, and (with 1 / factor) its undoing.  Angles are reduced in f64, so far positions
 * keep their accuracy; cosines and products are f32, and a result is rounded once to its type.
 */
#ifndef KVX_ROTARY_H
#define KVX_ROTARY_H

#include "kvx_abi.h"

#ifdef __cplusplus
extern "C" {
#endif

enum { KVX_ROTARY_INTERLEAVED = 1, KVX_ROTARY_INVERSE = 2 };

typedef struct kvx_rotary_desc {
  uint32_t size;
  uint32_t rotary_dim;        /* even, at most head_dim */
  uint32_t flags;             /* KVX_ROTARY_* bits */
  kvx_dtype_t position_dtype; /* S32 or S64 */
  const void *positions;      /* DEVICE [num_tokens]; any sign */
  const double *inv_freq;     /* DEVICE [rotary_dim / 2], radians per position */
  double factor;
  kvx_tensor_desc_t query;     /* [num_tokens, q_heads, head_dim], F16 / BF16 / F32; heads and dims */
  kvx_tensor_desc_t query_out; /* dense, token rows may be further apart; out may be the same memory */
  kvx_tensor_desc_t key;       /* [num_tokens, kv_heads, head_dim] of the query's type, or data = NULL */
  kvx_tensor_desc_t key_out;
} kvx_rotary_desc_t;

#if defined(__cplusplus)
static_assert(sizeof(kvx_rotary_desc_t) == 488, "kvx_rotary_desc_t layout");
#elif defined(__STDC_VERSION__) && __STDC_VERSION__ >= 201112L
_Static_assert(sizeof(kvx_rotary_desc_t) == 488, "kvx_rotary_desc_t layout");
#endif

/* Turns query into query_out and, where given, key into key_out (one kernel).  The two may be the
 * same memory (with the same strides); other overlaps are not supported.
 *
 * Status: INVALID_ARGUMENT for NULL / undersized descriptors, unknown flags, an odd rotary_dim or
 * one above head_dim, shapes that disagree; UNSUPPORTED for mismatched types, heads or dims that
 * are not dense, rows that overlap; OK without a launch when there is no token. */
KVX_API kvx_status_t kvx_launch_rotary(const kvx_rotary_desc_t *rotary, void *stream);

/* Turns query as above (query.data may be NULL: none) and writes the turned keys of write->io.key
 * and the values of write->io.value to their pages: the cache holds what kvx_launch_rotary followed
 * by kvx_launch_write_kv would put there, bit for bit, and io.key itself is only read.  Slots,
 * scales of an e4m3 cache and bad slots as for kvx_launch_write_kv; a token whose slot is skipped
 * still has its query turned.  rotary->key / key_out must have data = NULL (INVALID_ARGUMENT).
 * Status otherwise as kvx_launch_rotary and kvx_launch_write_kv. */
KVX_API kvx_status_t kvx_launch_rotary_write_kv(const kvx_cache_desc_t *cache, const kvx_write_desc_t *write,
                                                const kvx_rotary_desc_t *rotary, void *stream);

#ifdef __cplusplus
}
#endif
#endif /* KVX_ROTARY_H */
