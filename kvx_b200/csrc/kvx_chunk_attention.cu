/*
 * Attention of a chunk of new tokens over the paged KV cache (include/kvx_attention.h): several
 * query tokens per sequence -- a prompt, the next piece of one, drafted tokens to verify -- attend
 * over the sequence's pages in place.  No reference counterpart; pages are found as the gather
 * finds them (reference: kernels/kvx_paged_kv.cu:232-266, :54-75).
 *
 *   rows      The query heads of one KV head and the new tokens form the rows of one product: row
 *             r = token * group + head of the group, so K and V are read once per KV head.
 *   schedule  Tiles of rows, each with its causal number of K/V steps, are laid end to end and cut
 *             into equal shares, one per CTA (a share may begin and end inside a tile).  Only the
 *             tiles a cut goes through have partial results; the merge kernel joins them.
 *   product   scores = Q K^T and out += P V on tcgen05.mma, accumulators in tensor memory, one pass
 *             over K and V with the running maximum and sum of the softmax in f32.
 *
 * Nothing here allocates; plan and partial results live in caller-provided scratch.
 */
#include "kvx_attention.h"
#include "kvx_paged_kv.h"

#include "kvx_pages.h"

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>
#include <atomic>

namespace {

using kvx_detail::dtype_bytes;
using kvx_detail::make_page_view;
using kvx_detail::PageView;
using kvx_detail::ScaleView;

// ------------------------------------------------------------------ parameters ---------

struct ChunkParams {
  PageView k, v;
  ScaleView ks, vs;
  const void *table, *lens, *indptr;
  const char *query;
  char *out;
  int64_t q_pitch, o_pitch;  // bytes between token rows
  int64_t *prefix;           // [seq_count + 1] steps ahead of each sequence (all KV heads)
  float *part_o;             // [2 * grid][slot_rows][dim] unnormalised sums of cut tiles
  float *part_ml;            // [2 * grid][slot_rows][2] their maxima (unscaled scores) and denominators
  float scale_log2;          // scale * log2(e)
  int32_t seq_count, rows, max_blocks, max_seq_len, num_blocks, block_size;
  int32_t heads_kv, group, dim;
  int32_t causal, table64, indptr64;
  int32_t cache_code, io_code;
  int32_t grid, slot_rows, min_share;
  int32_t tile_rows, kv_tile;  // rows and tokens of one step of this kernel
  int32_t pair;                // 1: a tile of at most half the rows walks two K/V tiles per step
  int32_t bs_shift;            // log2(block_size) or -1
  int32_t box;                 // tokens one TMA box loads
  int32_t tile_cost;           // what a tile costs beyond its steps, in steps
  // how K and V tiles lie in shared memory: bytes between groups of 8 tokens and between panels of 64 dims
  int32_t group_stride, panel_stride;
  int32_t whole_boxes;         // 1: a box carries all panels of its tokens, [8 tokens][panel]; 0: one panel
  int32_t head_panels, head_groups;  // whole boxes: what a head adds to the panel and the group coordinate
  int32_t head_inner;          // else: heads are closer together than tokens
  int32_t plan_inside;         // 1: few sequences, planned by the attention kernel itself
  int32_t q_tma;               // 1: query tiles are loaded by TMA
  int32_t q_vec;               // 1: query rows can be read, out rows written in 16-byte pieces
  int32_t kv_vec;              // 1: page rows can be read in 16-byte pieces
  int32_t test_stall;          // 1: the first CTA's schedule waits for something that never comes, see the kernel
};

__device__ int g_chunk_error;  // set to 1 when a bounded wait gave up

__device__ __forceinline__ int64_t read_index(const void *p, int64_t i, int wide) {
  return wide ? static_cast<const int64_t *>(p)[i] : static_cast<const int32_t *>(p)[i];
}

__device__ __forceinline__ void pdl_prologue() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
}

// ------------------------------------------------------------------ schedule -----------

// One sequence of the batch.  Row r of its group rows belongs to token r / group, whose position is
// pos0 + token; it sees the cached tokens below limit(r).
struct Seq {
  int32_t first;  // first row of query / out
  int32_t rows;   // new tokens * group
  int32_t len;    // cached tokens that can take part
  int32_t pos0;
};

__device__ __forceinline__ Seq load_seq(const ChunkParams &p, int s) {
  const int64_t a = read_index(p.indptr, s, p.indptr64);
  const int64_t b = read_index(p.indptr, s + 1, p.indptr64);
  int64_t len = read_index(p.lens, s, p.table64);
  if (len < 0) len = 0;
  const bool none = a < 0 || b <= a || a >= p.rows;
  // (rows behind the last are left out, the others keep their positions)
  const int64_t n = none ? 0 : min(b, static_cast<int64_t>(p.rows)) - a;
  const int64_t pos0 = none ? 0 : max(len - (b - a), static_cast<int64_t>(INT32_MIN));
  len = min(len, static_cast<int64_t>(p.max_seq_len));
  len = min(len, static_cast<int64_t>(p.max_blocks) * p.block_size);
  Seq q;
  q.first = n > 0 ? static_cast<int32_t>(a) : 0;
  q.rows = static_cast<int32_t>(n * p.group);
  q.len = static_cast<int32_t>(len);
  q.pos0 = static_cast<int32_t>(min(pos0, len));  // at or beyond len every token sees all of it
  return q;
}

__device__ __forceinline__ int32_t row_limit(const ChunkParams &p, const Seq &q, int32_t r) {
  if (!p.causal) return q.len;
  const int64_t end = static_cast<int64_t>(q.pos0) + r / p.group + 1;
  return static_cast<int32_t>(max(static_cast<int64_t>(0), min(static_cast<int64_t>(q.len), end)));
}
__device__ __forceinline__ int32_t tiles_of(const ChunkParams &p, const Seq &q) {
  return (q.rows + p.tile_rows - 1) / p.tile_rows;
}
__device__ __forceinline__ bool is_narrow(const ChunkParams &p, const Seq &q) {
  return p.pair != 0 && q.rows <= p.tile_rows / 2;
}
// K/V tiles and steps of row tile `t`.  A tile without any is still one step: its rows are written;
// loading its queries and writing its result count as `tile_cost` steps ahead of the first.
__device__ __forceinline__ int32_t kv_tiles_of(const ChunkParams &p, const Seq &q, int32_t t) {
  const int32_t last = min(q.rows, (t + 1) * p.tile_rows) - 1;
  return (row_limit(p, q, last) + p.kv_tile - 1) / p.kv_tile;
}
__device__ __forceinline__ int32_t steps_of(const ChunkParams &p, const Seq &q, int32_t t) {
  int32_t n = kv_tiles_of(p, q, t);
  if (is_narrow(p, q)) n = (n + 1) / 2;
  return max(1, n) + p.tile_cost;
}

// Steps of one sequence over all KV heads, for every lane's own; the lanes of a warp help each other
// with sequences of many tiles.
__device__ __forceinline__ int64_t sequence_steps(const ChunkParams &p, int s) {
  const int lane = threadIdx.x & 31;
  Seq q{0, 0, 0, 0};
  int32_t tiles = 0;
  if (s < p.seq_count) {
    q = load_seq(p, s);
    tiles = tiles_of(p, q);
  }
  int64_t mine = 0;
  if (tiles <= 8)
    for (int t = 0; t < tiles; ++t) mine += steps_of(p, q, t);
  unsigned big = __ballot_sync(0xFFFFFFFFu, tiles > 8);
  while (big != 0) {
    const int from = __ffs(big) - 1;
    big &= big - 1;
    Seq x;
    x.first = 0;
    x.rows = __shfl_sync(0xFFFFFFFFu, q.rows, from);
    x.len = __shfl_sync(0xFFFFFFFFu, q.len, from);
    x.pos0 = __shfl_sync(0xFFFFFFFFu, q.pos0, from);
    const int32_t nt = tiles_of(p, x);
    int64_t sum = 0;
    for (int t = lane; t < nt; t += 32) sum += steps_of(p, x, t);
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, d);
    if (lane == from) mine = sum;
  }
  return mine * p.heads_kv;
}

constexpr int kPlanThreads = 1024;
constexpr int kPlanInside = 32;  // up to that many sequences every CTA makes the plan itself

// prefix[s] = steps of the sequences ahead of s, for at most kPlanInside sequences; one warp.
__device__ void plan_few(const ChunkParams &p, int64_t *prefix) {
  const int lane = threadIdx.x & 31;
  int64_t incl = sequence_steps(p, lane);
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int64_t y = __shfl_up_sync(0xFFFFFFFFu, incl, d);
    if (lane >= d) incl += y;
  }
  if (lane == 0) prefix[0] = 0;
  if (lane < p.seq_count) prefix[lane + 1] = incl;
}

// The same for any number.
__global__ void __launch_bounds__(kPlanThreads) kvx_chunk_plan_kernel(const ChunkParams p) {
  pdl_prologue();
  __shared__ int64_t s_sum[32];
  __shared__ int64_t s_base;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (threadIdx.x == 0) s_base = 0;
  __syncthreads();
  for (int s0 = 0; s0 < p.seq_count; s0 += kPlanThreads) {
    const int s = s0 + threadIdx.x;
    const int64_t mine = sequence_steps(p, s);
    int64_t incl = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int64_t y = __shfl_up_sync(0xFFFFFFFFu, incl, d);
      if (lane >= d) incl += y;
    }
    if (lane == 31) s_sum[warp] = incl;
    __syncthreads();
    int64_t before = s_base;
    for (int w = 0; w < warp; ++w) before += s_sum[w];
    if (s < p.seq_count) p.prefix[s] = before + incl - mine;
    __syncthreads();
    if (threadIdx.x == kPlanThreads - 1) s_base = before + incl;
    __syncthreads();
  }
  if (threadIdx.x == 0) p.prefix[p.seq_count] = s_base;
}

// A place in the laid-out work: step `off` of tile `tile` of KV head `head` of sequence `seq`.
struct Place {
  int32_t seq, head, tile, off;
  int32_t steps;  // of the tile
  Seq q;
};

__device__ __forceinline__ int shares(const ChunkParams &p, int64_t total) {
  const int64_t want = (total + p.min_share - 1) / p.min_share;
  return static_cast<int>(min(want, static_cast<int64_t>(p.grid)));
}
__device__ __forceinline__ int64_t share_begin(int64_t total, int n, int c) {
  return total * c / n;  // total < 2^48, n < 2^15
}
// A cut at `at` inside the tile [begin, end) goes to the tile's edge where it would leave next to
// nothing on one side.
__device__ __forceinline__ int64_t snap(const ChunkParams &p, int64_t at, int64_t begin, int64_t end) {
  if (at - begin <= p.tile_cost + 1) return begin;
  return end - at <= 1 ? end : at;
}

// All lanes of a warp call it together and get the same answer.  `at` < prefix[seq_count].
__device__ Place find_place(const ChunkParams &p, const int64_t *prefix, int64_t at) {
  const int lane = threadIdx.x & 31;
  int lo = 0, hi = p.seq_count;  // the last s with prefix[s] <= at lies in [lo, hi)
  while (hi - lo > 1) {
    const int step = max(1, (hi - lo + 31) / 32);
    const int s = lo + lane * step;
    const unsigned in = __ballot_sync(0xFFFFFFFFu, s < hi && prefix[s] <= at);
    lo = lo + (31 - __clz(in)) * step;
    hi = min(hi, lo + step);
  }
  Place w;
  w.seq = lo;
  w.q = load_seq(p, lo);
  const int64_t in_seq = at - prefix[lo];
  const int64_t per_head = (prefix[lo + 1] - prefix[lo]) / p.heads_kv;
  w.head = static_cast<int32_t>(in_seq / per_head);
  int64_t left = in_seq - w.head * per_head;
  const int32_t nt = tiles_of(p, w.q);
  for (int t0 = 0;; t0 += 32) {
    const int32_t n = t0 + lane < nt ? steps_of(p, w.q, t0 + lane) : 0;
    int64_t incl = n;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int64_t y = __shfl_up_sync(0xFFFFFFFFu, incl, d);
      if (lane >= d) incl += y;
    }
    const unsigned beyond = __ballot_sync(0xFFFFFFFFu, incl > left);
    if (beyond != 0) {
      const int l = __ffs(beyond) - 1;
      w.tile = t0 + l;
      w.steps = __shfl_sync(0xFFFFFFFFu, n, l);
      w.off = static_cast<int32_t>(left - (__shfl_sync(0xFFFFFFFFu, incl, l) - w.steps));
      return w;
    }
    left -= __shfl_sync(0xFFFFFFFFu, incl, 31);
    if (t0 + 32 >= nt) {  // not reached: `at` lies inside the sequence
      w.tile = 0, w.off = 0, w.steps = 1;
      return w;
    }
  }
}

// Share `share` of the schedule: from `w` on, `left` steps.
__device__ __forceinline__ int64_t find_share(const ChunkParams &p, const int64_t *prefix, int share, Place *w) {
  const int64_t total = prefix[p.seq_count];
  const int n = shares(p, total);
  if (share >= n) return 0;
  int64_t at[2];
  Place e[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    at[i] = share_begin(total, n, share + i);
    if (at[i] >= total) continue;
    e[i] = find_place(p, prefix, at[i]);
    const int64_t begin = at[i] - e[i].off, to = snap(p, at[i], begin, begin + e[i].steps);
    e[i].off = static_cast<int32_t>(to - begin);
    at[i] = to;
  }
  *w = e[0];
  return at[1] - at[0];
}

// The next tile after w's, in the order of the schedule; w.seq = seq_count when there is none.
__device__ __forceinline__ void next_tile(const ChunkParams &p, Place &w) {
  w.off = 0;
  if (++w.tile >= tiles_of(p, w.q)) {
    w.tile = 0;
    if (++w.head >= p.heads_kv) {
      w.head = 0;
      do {
        if (++w.seq >= p.seq_count) return;
        w.q = load_seq(p, w.seq);
      } while (w.q.rows == 0);
    }
  }
  w.steps = steps_of(p, w.q, w.tile);
}

// One CTA's part of one tile: steps [begin, end) of it.
struct Piece {
  Seq q;
  int32_t seq, head, row0, rows;  // rows [row0, row0 + rows) of the sequence's group rows
  int32_t kv0, kv1;               // K/V tiles of the piece
  int32_t kv_masked;              // the first K/V tile of which some of the tile's rows may not see every token
  int32_t narrow;
  int32_t slot;                   // partial-result slot, -1 = the piece is the whole tile
};

__device__ __forceinline__ Piece piece_of(const ChunkParams &p, const Place &w, int32_t end, int share) {
  Piece x;
  x.q = w.q;
  x.seq = w.seq;
  x.head = w.head;
  x.row0 = w.tile * p.tile_rows;
  x.rows = min(p.tile_rows, w.q.rows - x.row0);
  x.narrow = is_narrow(p, w.q) ? 1 : 0;
  const int32_t n = kv_tiles_of(p, w.q, w.tile);
  const int32_t mul = x.narrow ? 2 : 1;
  x.kv0 = min(n, max(0, w.off - p.tile_cost) * mul);
  x.kv1 = min(n, max(0, end - p.tile_cost) * mul);
  x.kv_masked = p.causal ? row_limit(p, w.q, x.row0) / p.kv_tile : n;
  // a share holds at most one piece that continues a tile begun earlier and one that begins a
  // tile ended later
  x.slot = (w.off == 0 && end == w.steps) ? -1 : (w.off > 0 ? 2 * share : 2 * share + 1);
  return x;
}

// ------------------------------------------------------------------ element access -----

__device__ __forceinline__ float load_f32(const char *at, int code) {
  switch (code) {
    case KVX_DTYPE_BF16:
      return __uint_as_float(static_cast<uint32_t>(*reinterpret_cast<const uint16_t *>(at)) << 16);
    case KVX_DTYPE_F16:
      return __half2float(__ushort_as_half(*reinterpret_cast<const uint16_t *>(at)));
    case KVX_DTYPE_F8_E4M3: {
      uint32_t h2;
      asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h2) : "h"(static_cast<uint16_t>(*reinterpret_cast<const uint8_t *>(at))));
      return __half2float(__ushort_as_half(static_cast<uint16_t>(h2 & 0xFFFFu)));
    }
    default:
      return *reinterpret_cast<const float *>(at);
  }
}
__device__ __forceinline__ void store_f32(char *base, int64_t i, float x, int code) {
  if (code == KVX_DTYPE_BF16)
    reinterpret_cast<uint16_t *>(base)[i] = __bfloat16_as_ushort(__float2bfloat16_rn(x));
  else if (code == KVX_DTYPE_F16)
    reinterpret_cast<uint16_t *>(base)[i] = __half_as_ushort(__float2half_rn(x));
  else
    reinterpret_cast<float *>(base)[i] = x;
}
__device__ __forceinline__ int elem_bytes(int code) {
  return code == KVX_DTYPE_F32 ? 4 : code == KVX_DTYPE_F8_E4M3 ? 1 : 2;
}
__device__ __forceinline__ int64_t head_offset(const PageView &v, int64_t o, int64_t h, int32_t d) {
  const int32_t hi = d / v.pack;
  return o * v.tok + h * v.head + hi * v.dhi + (d - hi * v.pack) * v.dlo;
}

// Page of token `tok` of sequence `seq`, -1 when it takes no part.
__device__ __forceinline__ int32_t page_of(const ChunkParams &p, int32_t seq, int32_t tok) {
  const int32_t lb = p.bs_shift >= 0 ? tok >> p.bs_shift : tok / p.block_size;
  if (lb >= p.max_blocks) return -1;
  const int64_t b = read_index(p.table, static_cast<int64_t>(seq) * p.max_blocks + lb, p.table64);
  return b < 0 || b >= p.num_blocks ? -1 : static_cast<int32_t>(b);
}

// exp2 of a difference of scaled maxima, 0 when nothing was accumulated under `a`.
__device__ __forceinline__ float weight_of(float a, float m, float mul) { return a == -INFINITY ? 0.f : exp2f((a - m) * mul); }

// Score multiplier of a KV head in the exp2 domain (the K scale of an e4m3 cache folded in).
__device__ __forceinline__ float score_mul(const ChunkParams &p, int head) {
  return p.ks.base != nullptr ? p.scale_log2 * p.ks.base[head * p.ks.stride] : p.scale_log2;
}

// Running maxima are kept of scores times the sign of the multiplier, and weighted with its size.  A
// multiplier of zero (zero times the -inf of a masked score would be a NaN) is taken as 2^-126, which
// makes every score's exponent zero all the same.
__device__ __forceinline__ float nonzero(float mul) { return mul == 0.f ? 1.17549435e-38f : mul; }

// ------------------------------------------------------------------ merge of pieces ----

constexpr int kMergeThreads = 128;

// One warp per (cut, row of the tile the cut goes through); the first cut through a tile does the
// work.
__global__ void __launch_bounds__(kMergeThreads) kvx_chunk_merge_kernel(const ChunkParams p) {
  pdl_prologue();
  const int64_t total = p.prefix[p.seq_count];
  const int n = shares(p, total);
  const int cut = blockIdx.x + 1;
  if (cut >= n) return;
  const int64_t raw = share_begin(total, n, cut);
  const Place w = find_place(p, p.prefix, raw);
  const int64_t tile_at = raw - w.off, tile_end = tile_at + w.steps;
  const int64_t at = snap(p, raw, tile_at, tile_end);
  if (at == tile_at || at == tile_end) return;
  const int64_t ahead = share_begin(total, n, cut - 1);
  if (ahead > tile_at && snap(p, ahead, tile_at, tile_end) > tile_at) return;  // an earlier cut goes through this tile
  // shares cut .. last continue the tile, share cut - 1 began it
  int last = cut;
  while (last + 1 < n) {
    const int64_t next = share_begin(total, n, last + 1);
    if (next >= tile_end || snap(p, next, tile_at, tile_end) == tile_end) break;
    ++last;
  }
  const int32_t row0 = w.tile * p.tile_rows, rows = min(p.tile_rows, w.q.rows - row0);
  const int lane = threadIdx.x & 31;
  const float mul = fabsf(nonzero(score_mul(p, w.head)));
  for (int r = blockIdx.y * (kMergeThreads / 32) + (threadIdx.x >> 5); r < rows; r += gridDim.y * (kMergeThreads / 32)) {
    float m = -INFINITY;
    for (int c = cut - 1 + lane; c <= last; c += 32) {
      const int64_t slot = c == cut - 1 ? 2 * c + 1 : 2 * c;
      m = fmaxf(m, p.part_ml[(slot * p.slot_rows + r) * 2]);
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, d));
    float l = 0.f;
    for (int c = cut - 1; c <= last; ++c) {
      const int64_t slot = c == cut - 1 ? 2 * c + 1 : 2 * c;
      const float2 ml = reinterpret_cast<const float2 *>(p.part_ml)[slot * p.slot_rows + r];
      l += ml.y * weight_of(ml.x, m, mul);
    }
    const int32_t token = (row0 + r) / p.group, head = w.head * p.group + (row0 + r) % p.group;
    char *out = p.out + (w.q.first + token) * p.o_pitch + static_cast<int64_t>(head) * p.dim * elem_bytes(p.io_code);
    for (int d = lane; d < p.dim; d += 32) {
      float acc = 0.f;
      for (int c = cut - 1; c <= last; ++c) {
        const int64_t slot = c == cut - 1 ? 2 * c + 1 : 2 * c;
        const float f = weight_of(p.part_ml[(slot * p.slot_rows + r) * 2], m, mul);
        acc += f * p.part_o[(slot * p.slot_rows + r) * p.dim + d];
      }
      store_f32(out, d, l == 0.f ? 0.f : acc / l, p.io_code);
    }
  }
}

// ------------------------------------------------------------------ mbarriers, TMA, tensor memory --

__device__ __forceinline__ uint32_t elect_lane() {
  uint32_t e;
  asm volatile("{ .reg .pred p;\n\telect.sync _|p, 0xFFFFFFFF;\n\tselp.u32 %0, 1, 0, p; }" : "=r"(e));
  return e;
}
__device__ __forceinline__ uint32_t smem_addr(const void *p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void mbar_expect_tx(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool mbar_try(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{ .reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p; }"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
// Waits for the phase, two seconds at most; a wait that gives up sets the device's word and answers false,
// upon which its role returns.  Few instructions on purpose, see the note at the kernel: tries are
// counted, not time.  A try that fails takes 4.0 us on B200 (measured over 1 to 100 000 of them, with one warp of
// the CTA waiting and with twelve), whatever the suspension asked for.
constexpr uint32_t kTries = 500000;
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{ .reg .pred p;\n\t"
      ".reg .u32 n;\n\t"
      "mov.u32 n, %3;\n\t"
      "AGAIN:\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %4;\n\t"
      "@p bra DONE;\n\t"
      "sub.u32 n, n, 1;\n\t"
      "setp.ne.u32 p, n, 0;\n\t"
      "@p bra AGAIN;\n\t"
      "DONE:\n\t"
      "selp.u32 %0, 1, 0, p; }"
      : "=r"(ok)
      : "r"(bar), "r"(parity), "n"(kTries), "r"(1000u)
      : "memory");
  if (ok == 0) g_chunk_error = 1;
  return ok != 0;
}
// The same for a whole warp: all lanes get one answer, and the compiler knows that they do.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity) {
  return __all_sync(0xFFFFFFFFu, mbar_wait(bar, parity)) != 0;
}

// Issued by the elected lane of a warp whose lanes agree on all operands.
__device__ __forceinline__ void tma_load4(uint32_t elected, uint32_t dst, const CUtensorMap *map, int x, int c1, int c2, int c3, uint32_t bar) {
  asm volatile(
      "{ .reg .pred q;\n\t"
      "setp.ne.b32 q, %7, 0;\n\t"
      "@q cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6]; }" ::"r"(dst),
      "l"(map), "r"(x), "r"(c1), "r"(c2), "r"(c3), "r"(bar), "r"(elected)
      : "memory");
}
__device__ __forceinline__ void tma_load5(uint32_t elected, uint32_t dst, const CUtensorMap *map, int panel, int group, int page, uint32_t bar) {
  asm volatile(
      "{ .reg .pred q;\n\t"
      "setp.ne.b32 q, %6, 0;\n\t"
      "@q cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%7, %7, %2, %3, %4}], [%5]; }" ::"r"(dst),
      "l"(map), "r"(panel), "r"(group), "r"(page), "r"(bar), "r"(elected), "r"(0)
      : "memory");
}
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_commit(uint32_t elected, uint32_t bar) {
  asm volatile(
      "{ .reg .pred q;\n\t"
      "setp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0]; }" ::"r"(bar), "r"(elected)
      : "memory");
}
// d[128 x N] (+)= a[128 x 16] b[N x 16]^T; a and b in shared memory.  Called by a whole warp, issued by
// the elected lane: in code that the compiler can see to be uniform, descriptors live in uniform
// registers, which is where the instruction wants them.
__device__ __forceinline__ void mma_ss(uint32_t elected, uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{ .reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p; }" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(elected)
      : "memory");
}
// the same with a in tensor memory
__device__ __forceinline__ void mma_ts(uint32_t elected, uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{ .reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p; }" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(elected)
      : "memory");
}
__device__ __forceinline__ void tc_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// 32 columns of this warp's 32 lanes
__device__ __forceinline__ void tc_ld32(float *x, uint32_t at) {
  uint32_t *r = reinterpret_cast<uint32_t *>(x);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,"
      "%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
        "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
        "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(at));
}
__device__ __forceinline__ void tc_st32(uint32_t at, const float *x) {
  const uint32_t *r = reinterpret_cast<const uint32_t *>(x);
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,"
      "%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(at),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]),
      "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]),
      "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tc_ld16(float *x, uint32_t at) {
  uint32_t *r = reinterpret_cast<uint32_t *>(x);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(at));
}
__device__ __forceinline__ void tc_st16(uint32_t at, const uint32_t *r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(at),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
// Shared-memory operand descriptor, 128-byte swizzle: rows of 128 bytes, 8 of them to an atom of
// 1 024 bytes.  `stride` bytes between groups of 8 rows; `lead` bytes between blocks of 64
// elements along the rows (used when the rows run along the reduction, i.e. for V).
__device__ __forceinline__ uint64_t operand_desc(uint32_t addr, uint32_t lead, uint32_t stride) {
  return static_cast<uint64_t>((addr & 0x3FFFF) >> 4) | (static_cast<uint64_t>(lead >> 4) << 16) |
         (static_cast<uint64_t>(stride >> 4) << 32) | (1ull << 46) | (2ull << 61);
}

__device__ __forceinline__ float fast_exp2(float x) {  // ex2.approx: 2 ulp, -inf -> 0
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

struct Bf16 {
  static constexpr uint32_t kFormat = 1;  // operand format of the instruction descriptor
  static constexpr float kShift = 0.f;    // of the softmax weights, see kLazy; bf16 has the exponents of f32
  static __device__ __forceinline__ float get(uint16_t b) { return __uint_as_float(static_cast<uint32_t>(b) << 16); }
  static __device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    const __nv_bfloat162 r = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&r);
  }
  static __device__ __forceinline__ uint32_t from_f16x2(uint32_t x) {  // e4m3 values: exact
    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&x));
    return pack2(f.x, f.y);
  }
};
struct Fp16 {
  static constexpr uint32_t kFormat = 0;
  static constexpr float kShift = 7.f;
  static __device__ __forceinline__ float get(uint16_t b) { return __half2float(__ushort_as_half(b)); }
  static __device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    const __half2 r = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&r);
  }
  static __device__ __forceinline__ uint32_t from_f16x2(uint32_t x) { return x; }
};

// ------------------------------------------------------------------ tensor-core kernel --
//
// Roles of a CTA (one per SM, 384 threads, 512 where loading takes more than TMA):
//   warps 0-3, 4-7   softmax of stream 0 and of stream 1: a thread owns one of the 128 rows
//   warp 8           issues every tcgen05.mma
//   warp 9           walks the schedule, publishes pieces, loads Q and K tiles (TMA)
//   warp 10          loads V tiles
//   (e4m3: warp 9 loads K and V bytes, warps 10 to 15 convert them; pages that TMA cannot read:
//   warps 9 to 15 copy them)
// Two streams of 128 rows keep the tensor pipe and the exponentials busy in turn: while one
// stream's scores are turned into weights the other stream's products run.  A tile with at most
// 128 rows gives both streams the same rows and every K/V tile to one of them; the two halves are
// joined in shared memory.  head_dim above 128 leaves tensor memory for one stream, which then has
// two score buffers instead.
//
// Tensor memory (512 columns): scores of 128 x 128 f32 at 0 and 128, weights written over the
// first 64 columns of their scores, output sums at 256 (and 256 + kDp).  The MMAs of a CTA run in
// the order of their issue, which is what lets the scores of the next tile overwrite the weights
// the previous product read.

constexpr int kMmaWarp = 8;
// How K and V get into shared memory.
enum Loads { kTmaLoads, kRawLoads, kCopyLoads };  // TMA; e4m3 bytes by TMA, converted; copied by warps
constexpr int kCopyWarps = 7, kConvertWarps = 6;
constexpr int threads_of(Loads loads) { return loads == kTmaLoads ? 384 : 512; }
constexpr int kTile = 128;          // rows of a stream, tokens of a K/V tile
constexpr int kPanelBytes = 16384;  // 128 rows x 128 bytes
constexpr int kItems = 2;           // pieces published ahead

template <int kDp>
struct Shape {
  static constexpr int kStreams = kDp > 128 ? 1 : 2;
  static constexpr int kScoreBufs = kDp > 128 ? 2 : 1;     // per stream
  static constexpr int kPanels = kDp / 64;                 // 64 dims (128 bytes) each
  static constexpr int kUnitPanels = kPanels > 2 ? 2 : kPanels;
  static constexpr int kUnits = kPanels / kUnitPanels;     // ring entries per tile
  static constexpr int kUnitBytes = kUnitPanels * kPanelBytes;
  static constexpr int kRing = kDp == 64 ? 4 : 2;          // entries of the K ring and of the V ring (powers of two)
  static constexpr int kQBytes = kPanels * kPanelBytes;    // per stream
  static constexpr int kRingAt = kStreams * kQBytes;
  static constexpr int kRawBytes = kTile * kUnitPanels * 64;  // an entry's e4m3 bytes
  static constexpr int kRawAt = kRingAt + 2 * kRing * kUnitBytes;
  static constexpr int kMiscAt = kRawAt + 2 * kRawBytes;
};

struct Misc {
  uint64_t item_full[kItems], item_empty[kItems];
  uint64_t kv_full[8], kv_empty[8];
  uint64_t q_full[2], q_empty[2], s_full[2], p_part[2], p_full[2], pv_done[2];
  uint64_t join_full, join_empty;
  uint64_t raw_full[2], raw_empty[2];
  uint64_t tail, drain;
  Piece items[kItems];
  int64_t prefix[kPlanInside + 1];
  float join_m[kTile], join_l[kTile];
  uint32_t tmem;
};

template <int kDp>
constexpr size_t chunk_smem_bytes() {
  return 1024 + Shape<kDp>::kMiscAt + sizeof(Misc);
}

// K/V tiles [b, e) stream `s` walks in this piece.
template <int kStreams>
__device__ __forceinline__ void stream_range(const ChunkParams &p, const Piece &x, int s, int *b, int *e) {
  if (kStreams == 2 && x.narrow) {
    const int h = x.kv0 + (x.kv1 - x.kv0 + 1) / 2;
    *b = s == 0 ? x.kv0 : h;
    *e = s == 0 ? h : x.kv1;
    return;
  }
  const int rows = min(kTile, x.rows - s * kTile);
  *b = *e = x.kv0;
  if (rows <= 0) return;
  const int32_t limit = row_limit(p, x.q, x.row0 + s * kTile + rows - 1);
  *e = max(x.kv0, min(x.kv1, (limit + kTile - 1) / kTile));
}

// K/V tiles are taken from the last to the first.  A masked token has weight zero in the products, but
// zero times an infinity or a NaN that its V holds is a NaN; and tokens that are masked for some of a tile's
// rows lie in its last tiles only (three at most: the rows of one tile lie within 256 tokens).  So those
// come first, and behind them, before anything else is added, rows whose sums are not finite get that
// part again without the masked tokens (repair_rows).  What is not finite later comes from tokens that
// the row sees, and stays.
//
// Of two streams that share their tiles, stream 0 may begin `late` tiles behind stream 1: none of its
// rows sees those.
struct Walk {
  int32_t b, e, late;
  __device__ __forceinline__ int32_t count() const { return e - b; }
};
template <int kStreams>
__device__ __forceinline__ Walk stream_walk(const ChunkParams &p, const Piece &x, int s) {
  Walk w;
  stream_range<kStreams>(p, x, s, &w.b, &w.e);
  w.late = 0;
  if (kStreams == 2 && !x.narrow && s == 0) {
    int b, e;
    stream_range<kStreams>(p, x, 1, &b, &e);
    w.late = max(0, e - w.e);
  }
  return w;
}

// The K tiles (and the V tiles) of a piece in the order in which they are consumed: one after the
// other, or for a narrow piece from the two streams in turn.
struct TileOrder {
  int32_t e0, e1, count, narrow;
  __device__ __forceinline__ int32_t tile(int q) const { return narrow ? ((q & 1) ? e1 : e0) - 1 - (q >> 1) : e0 - 1 - q; }
};
template <int kStreams>
__device__ __forceinline__ TileOrder tile_order(const ChunkParams &p, const Piece &x) {
  int b0, e0, b1 = 0, e1 = 0;
  stream_range<kStreams>(p, x, 0, &b0, &e0);
  if (kStreams == 2) stream_range<kStreams>(p, x, 1, &b1, &e1);
  const bool narrow = kStreams == 2 && x.narrow;
  return TileOrder{narrow ? e0 : max(e0, e1), e1, narrow ? (e0 - b0) + (e1 - b1) : max(e0, e1) - x.kv0, narrow ? 1 : 0};
}

// Whether stream 1 hands its half of a narrow tile to stream 0 (it has K/V tiles of its own).
__device__ __forceinline__ bool joins_streams(const Piece &x) { return x.narrow && x.kv1 - x.kv0 > 1; }

__device__ __forceinline__ void tma_load3(uint32_t dst, const CUtensorMap *map, int x, int c1, int c2, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
      "l"(map), "r"(x), "r"(c1), "r"(c2), "r"(bar)
      : "memory");
}

// Query tiles of a piece by TMA, one lane: `group` is a power of two, so the 128 rows of a stream are
// the group's heads of 128 / group whole tokens.  Rows behind the sequence are other sequences'
// or zeros; nothing is written for them.
template <int kDp>
__device__ bool load_queries(const ChunkParams &p, const CUtensorMap *qmap, const Piece &x, uint32_t base, Misc *m, uint32_t *count) {
  using S = Shape<kDp>;
  for (int s = 0; s < S::kStreams; ++s) {
    int b, e;
    stream_range<S::kStreams>(p, x, s, &b, &e);
    if (e == b) continue;
    const uint32_t bar = smem_addr(&m->q_full[s]);
    if (count[s] > 0 && !mbar_wait(smem_addr(&m->q_empty[s]), (count[s] - 1) & 1)) return false;
    ++count[s];
    mbar_expect_tx(bar, S::kQBytes);
    const int32_t token = x.q.first + (x.row0 + (x.narrow ? 0 : s * kTile)) / p.group;
    for (int k = 0; k < S::kPanels; ++k)
      tma_load3(base + s * S::kQBytes + k * kPanelBytes, qmap, k * 64, x.head * p.group, token, bar);
  }
  return true;
}

// Place in the K ring (0) or the V ring (1): entries are used in turn.
template <int kDp>
struct Ring {
  using S = Shape<kDp>;
  uint32_t at;     // the ring's first entry in shared memory
  uint32_t first;  // its first barrier's number
  uint32_t entry = 0;
  __device__ __forceinline__ Ring(uint32_t base, int which) : at(base + S::kRingAt + which * S::kRing * S::kUnitBytes), first(which * S::kRing) {}
  __device__ __forceinline__ uint32_t slot() const { return first + (entry & (S::kRing - 1)); }
  __device__ __forceinline__ uint32_t addr() const { return at + (entry & (S::kRing - 1)) * S::kUnitBytes; }
  __device__ __forceinline__ uint32_t phase() const { return entry / S::kRing & 1; }
};

// ---- loads ------------------------------------------------------------------------------

// The pieces of this CTA's share, one after the other; behind the last a piece without rows.  All lanes
// of a warp call it together.
struct Schedule {
  Place w;
  int64_t left;
  __device__ __forceinline__ Schedule(const ChunkParams &p, const int64_t *prefix) {
    left = find_share(p, prefix, blockIdx.x, &w);
    if (left > 0 && w.off >= w.steps) next_tile(p, w);
  }
  __device__ __forceinline__ Piece next(const ChunkParams &p) {
    Piece x;
    x.rows = 0;
    if (left > 0) {
      const int32_t stop = static_cast<int32_t>(min(static_cast<int64_t>(w.steps), w.off + left));
      x = piece_of(p, w, stop, blockIdx.x);
      left -= stop - w.off;
      if (left > 0) next_tile(p, w);
    }
    return x;
  }
};

// Hands piece `item` to the other warps, and its queries to TMA.
template <int kDp>
__device__ __forceinline__ bool publish(const ChunkParams &p, const CUtensorMap *qmap, const Piece &x, uint32_t item, uint32_t base, Misc *m,
                                        uint32_t elected, uint32_t *queries) {
  const uint32_t slot = item % kItems;
  if (item >= kItems && !warp_wait(smem_addr(&m->item_empty[slot]), (item / kItems - 1) & 1)) return false;
  bool ok = true;
  if (elected) {
    m->items[slot] = x;
    mbar_arrive(smem_addr(&m->item_full[slot]));
    if (p.q_tma && x.rows > 0) ok = load_queries<kDp>(p, qmap, x, base, m, queries);
  }
  return __all_sync(0xFFFFFFFFu, ok) != 0;
}
// Takes piece `item`.
__device__ __forceinline__ bool receive(Misc *m, uint32_t item, uint32_t elected, Piece *x) {
  const uint32_t slot = item % kItems;
  if (!warp_wait(smem_addr(&m->item_full[slot]), (item / kItems) & 1)) return false;
  *x = m->items[slot];
  __syncwarp();
  if (elected) mbar_arrive(smem_addr(&m->item_empty[slot]));
  __syncwarp();
  return true;
}

// Two warps load by TMA: the first walks the schedule, publishes the pieces, loads the queries and the
// K tiles, the second loads the V tiles.  What a single warp does per box and per tile is on the
// kernel's critical path (one instruction every ten clocks or so), so a box carries all panels of
// its tokens where the layout allows, its coordinates are looked up a tile ahead, one box per lane,
// and the boxes are issued by one lane of converged code.
template <int kDp>
__device__ __forceinline__ void load_role_tma(const ChunkParams &p, const CUtensorMap *kmap, const CUtensorMap *vmap, const CUtensorMap *qmap, uint32_t base,
                              Misc *m, bool mine_v) {
  using S = Shape<kDp>;
  const int lane = threadIdx.x & 31;
  const uint32_t elected = elect_lane();
  Ring<kDp> ring(base, mine_v ? 1 : 0);
  uint32_t queries[2] = {0, 0};
  uint32_t tail_phase = 0;
  const int boxes = kTile / p.box;
  const CUtensorMap *map = mine_v ? vmap : kmap;
  const uint32_t box_bytes = p.box / 8 * p.group_stride;
  // Page of this lane's box of a tile (beyond the sequence, or where there is no such page, a number
  // behind the pool, which TMA answers with zeros), and its first token's place in the page.
  auto look_up = [&](const Piece &x, int tile, int32_t *in_page) {
    const int32_t tok = tile * kTile + lane * p.box;
    *in_page = 0;
    if (lane >= boxes || tok >= x.q.len) return p.num_blocks;
    const int32_t page = page_of(p, x.seq, tok);
    *in_page = p.bs_shift >= 0 ? tok & (p.block_size - 1) : tok % p.block_size;
    return page >= 0 ? page : p.num_blocks;
  };
  auto load_piece = [&](const Piece &x) {
    const TileOrder order = tile_order<S::kStreams>(p, x);
    if (order.count == 0) return true;  // no tile, and so none whose pages could be looked up ahead
    const int32_t c_panel = x.head * p.head_panels, c_group = x.head * p.head_groups;
    int32_t in_page = 0, page = p.num_blocks;
#pragma unroll 1
    for (int q = -1; q < order.count; ++q) {
      const int32_t now_page = page, now_in = in_page;
      page = look_up(x, order.tile(min(q + 1, order.count - 1)), &in_page);
      if (q < 0) continue;
      const int tile = order.tile(q);
      const int valid = x.q.len - tile * kTile;  // tokens of the tile that exist
      const bool tail = __any_sync(0xFFFFFFFFu, mine_v && valid < kTile && valid % p.box != 0) != 0;
#pragma unroll 1
      for (int u = 0; u < S::kUnits; ++u, ++ring.entry) {
        const uint32_t st = ring.slot();
        if (ring.entry >= S::kRing && !warp_wait(smem_addr(&m->kv_empty[st]), ring.phase() ^ 1)) return false;
        uint32_t dst = ring.addr();
        const uint32_t bar = smem_addr(tail ? &m->tail : &m->kv_full[st]);
        if (elected) mbar_expect_tx(bar, S::kUnitBytes);
        __syncwarp();
        if (p.whole_boxes) {
#pragma unroll 2
          for (int k = 0; k < boxes; ++k, dst += box_bytes)
            tma_load5(elected, dst, map, c_panel + u * S::kUnitPanels, c_group + (__shfl_sync(0xFFFFFFFFu, now_in, k) >> 3),
                      __shfl_sync(0xFFFFFFFFu, now_page, k), bar);
        } else {
          const bool head_inner = p.head_inner != 0;
#pragma unroll 1
          for (int k = 0; k < boxes; ++k, dst += box_bytes) {
            const int32_t pg = __shfl_sync(0xFFFFFFFFu, now_page, k), in = __shfl_sync(0xFFFFFFFFu, now_in, k);
#pragma unroll
            for (int pp = 0; pp < S::kUnitPanels; ++pp)
              tma_load4(elected, dst + pp * kPanelBytes, map, (u * S::kUnitPanels + pp) * 64, head_inner ? x.head : in,
                        head_inner ? in : x.head, pg, bar);
          }
        }
        if (tail) {
          // Rows of the last page behind the sequence hold whatever the page holds; their weight
          // is zero, but zero times a NaN is not: overwrite them.
          if (!warp_wait(bar, tail_phase)) return false;
          tail_phase ^= 1;
          const int rows = min(kTile, (valid + p.box - 1) / p.box * p.box) - valid;
#pragma unroll 1
          for (int i = lane; i < rows * 8 * S::kUnitPanels; i += 32) {
            const int row = valid + i / (8 * S::kUnitPanels), c = i % (8 * S::kUnitPanels);
            const uint32_t to = ring.addr() + (row >> 3) * p.group_stride + (row & 7) * 128 + (c >> 3) * p.panel_stride + (c & 7) * 16;
            asm volatile("st.shared.v4.u32 [%0], {%1,%1,%1,%1};" ::"r"(to), "r"(0u) : "memory");
          }
          fence_async_smem();
          __syncwarp();
          if (elected) mbar_arrive(smem_addr(&m->kv_full[st]));
        }
      }
    }
    return true;
  };
  bool ok = true;
  Schedule schedule(p, p.plan_inside ? m->prefix : p.prefix);
#pragma unroll 1
  for (uint32_t item = 0; ok; ++item) {
    Piece x;
    if (mine_v) {
      ok = receive(m, item, elected, &x);
    } else {
      x = schedule.next(p);
      ok = publish<kDp>(p, qmap, x, item, base, m, elected, queries);
    }
    if (!ok || __all_sync(0xFFFFFFFFu, x.rows == 0)) break;
    ok = load_piece(x);
  }
  // Nothing may be in flight towards this CTA's shared memory when it ends.  Normally: every
  // entry's release has arrived.  After giving up: the loads themselves, as far as they come.
  const uint32_t held = min(ring.entry, static_cast<uint32_t>(S::kRing)), end = ring.entry;
#pragma unroll 1
  for (ring.entry = end - held; ring.entry != end; ++ring.entry) {
    if (ok) ok = warp_wait(smem_addr(&m->kv_empty[ring.slot()]), ring.phase());
    if (!ok) {
      int ignore = 0;
      for (int i = 0; i < 4096 && ignore == 0; ++i) ignore = mbar_try(smem_addr(&m->kv_full[ring.slot()]), ring.phase()) ? 1 : 0;
    }
  }
}

// 16 bytes, or zeros; no branch, so that several loads of a lane are in flight together.
__device__ __forceinline__ uint4 load16_if(bool there, const char *from) {
  uint4 r = make_uint4(0, 0, 0, 0);
  asm volatile(
      "{ .reg .pred q;\n\t"
      "setp.ne.u32 q, %5, 0;\n\t"
      "@q ld.global.v4.u32 {%0,%1,%2,%3}, [%4]; }"
      : "+r"(r.x), "+r"(r.y), "+r"(r.z), "+r"(r.w)
      : "l"(from), "r"(static_cast<uint32_t>(there)));
  return r;
}

// Eight elements of one token's head from `d` on, element by element; behind head_dim zeros.  e4m3 in
// the first two words, 16-bit elements in all four.
__device__ __noinline__ uint4 gather_elements(const PageView &view, const char *page, int32_t o, int32_t head, int32_t d, int32_t dim, int elem) {
  uint32_t w[4] = {0, 0, 0, 0};
  for (int c = 0; c < 8 && d + c < dim; ++c) {
    const char *src = page + head_offset(view, o, head, d + c);
    if (elem == 2)
      w[c >> 1] |= static_cast<uint32_t>(*reinterpret_cast<const uint16_t *>(src)) << ((c & 1) * 16);
    else
      w[c >> 2] |= static_cast<uint32_t>(*reinterpret_cast<const uint8_t *>(src)) << ((c & 3) * 8);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Pages that TMA cannot read (HND_PACKED, pages of less than 8 tokens, odd strides): seven warps
// copy rows into the same swizzled tiles, converting on the way.  A warp's load instruction covers
// whole rows in 16-byte pieces; pages are looked up a tile ahead, and the loads of an entry are in
// flight while the one before it is converted.  Each warp walks the schedule for itself, the first
// one publishes the pieces.
template <typename T, int kDp>
__device__ __forceinline__ void load_role_copy(const ChunkParams &p, const CUtensorMap *qmap, uint32_t base, Misc *m) {
  using S = Shape<kDp>;
  constexpr int kPieces = S::kUnitPanels * 4;  // 16-byte pieces of a row of e4m3 (twice as many of 16-bit elements)
  constexpr int kSteps = (4 * kPieces + kCopyWarps - 1) / kCopyWarps;  // loads of a lane and entry (twice as many ..)
  const int lane = threadIdx.x & 31, warp = (threadIdx.x >> 5) - (kMmaWarp + 1);
  Ring<kDp> rings[2] = {Ring<kDp>(base, 0), Ring<kDp>(base, 1)};
  uint32_t queries[2] = {0, 0};
  const uint32_t elected = elect_lane();
  Schedule schedule(p, p.plan_inside ? m->prefix : p.prefix);
  const bool wide = p.cache_code != KVX_DTYPE_F8_E4M3;  // 16-bit elements
  const int elem = wide ? 2 : 1, pieces = wide ? 2 * kPieces : kPieces;
  const int in_group = lane / pieces, piece = lane % pieces;
  auto row_of = [&](int k) { return (warp + kCopyWarps * k) * (32 / pieces) + in_group; };  // of load k; 128 and more: none

  int32_t page[kSteps], next_page[kSteps];  // e4m3: of the rows in the tile being fetched, and in the one after it
  auto look_up = [&](const Piece &x, int tile, int row) {
    const int32_t tok = tile * kTile + row;
    return row < kTile && tok < x.q.len ? page_of(p, x.seq, tok) : -1;
  };
  // Entry n of a piece is (tile, K or V, unit): K and V of a tile, then the next tile's.
  auto fetch = [&](const Piece &x, const TileOrder &order, int n, int first, uint4 *r) {
    const int u = n % S::kUnits, kv = n / S::kUnits & 1, q = n / (2 * S::kUnits), tile = order.tile(q);
    if (!wide && u == 0 && kv == 0) {
#pragma unroll
      for (int k = 0; k < kSteps; ++k) {
        page[k] = q == 0 ? look_up(x, tile, row_of(k)) : next_page[k];
        next_page[k] = q + 1 < order.count ? look_up(x, order.tile(q + 1), row_of(k)) : -1;
      }
    }
    const PageView &view = kv ? p.v : p.k;
    const int d = u * S::kUnitPanels * 64 + piece * (16 / elem);
    const char *const in_head = view.base + x.head * view.head + d * elem;
    if (p.kv_vec) {
#pragma unroll
      for (int k = 0; k < kSteps; ++k) {
        const int32_t pg = wide ? look_up(x, tile, row_of(first + k)) : page[k];
        const int32_t tok = tile * kTile + row_of(first + k);
        const int32_t o = p.bs_shift >= 0 ? tok & (p.block_size - 1) : tok % p.block_size;
        r[k] = load16_if(pg >= 0 && d < p.dim, in_head + pg * view.blk + o * view.tok);
      }
      return;
    }
#pragma unroll 1
    for (int k = 0; k < kSteps; ++k) {
      const int row = row_of(first + k);
      const int32_t pg = look_up(x, tile, row);
      uint4 y = make_uint4(0, 0, 0, 0);
      if (pg >= 0 && d < p.dim) {
        const int32_t o = (tile * kTile + row) % p.block_size;
        const char *from = view.base + pg * view.blk;
        y = gather_elements(view, from, o, x.head, d, p.dim, elem);
        if (!wide) {
          const uint4 hi = gather_elements(view, from, o, x.head, d + 8, p.dim, elem);
          y.z = hi.x, y.w = hi.y;
        }
      }
#pragma unroll
      for (int i = 0; i < kSteps; ++i)  // (registers have no index)
        if (i == k) r[i] = y;
    }
  };
  auto place = [&](uint32_t dst, int first, const uint4 *r) {
#pragma unroll
    for (int k = 0; k < kSteps; ++k) {
      const int row = row_of(first + k);
      if (row >= kTile) continue;
      const uint32_t at = dst + (row >> 3) * p.group_stride + (row & 7) * 128;
      auto put = [&](int c, uint32_t a, uint32_t b, uint32_t e, uint32_t f) {
        asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(at + (c >> 3) * p.panel_stride + (((c & 7) ^ (row & 7)) << 4)), "r"(a),
                     "r"(b), "r"(e), "r"(f)
                     : "memory");
      };
      if (wide) {
        put(piece, r[k].x, r[k].y, r[k].z, r[k].w);
      } else {
        const uint32_t from[4] = {r[k].x, r[k].y, r[k].z, r[k].w};
        uint32_t y[8];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          uint32_t lo, hi;
          asm("{ .reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b; }"
              : "=r"(lo), "=r"(hi)
              : "r"(from[q]));
          y[2 * q] = T::from_f16x2(lo), y[2 * q + 1] = T::from_f16x2(hi);
        }
        put(2 * piece, y[0], y[1], y[2], y[3]);
        put(2 * piece + 1, y[4], y[5], y[6], y[7]);
      }
    }
  };

#pragma unroll 1
  for (uint32_t item = 0;; ++item) {
    const Piece x = schedule.next(p);
    if (warp == 0 && !publish<kDp>(p, qmap, x, item, base, m, elected, queries)) return;
    if (x.rows == 0) break;
    const TileOrder order = tile_order<S::kStreams>(p, x);
    const int entries = 2 * S::kUnits * order.count;
    uint4 ahead[kSteps];
    if (entries > 0) fetch(x, order, 0, 0, ahead);
#pragma unroll 1
    for (int n = 0; n < entries; ++n) {
      Ring<kDp> &ring = rings[n / S::kUnits & 1];
      const uint32_t st = ring.slot();
      uint4 now[kSteps];
#pragma unroll
      for (int k = 0; k < kSteps; ++k) now[k] = ahead[k];
      if (n + 1 < entries) fetch(x, order, n + 1, 0, ahead);
      if (ring.entry >= S::kRing && !warp_wait(smem_addr(&m->kv_empty[st]), ring.phase() ^ 1)) return;
      const uint32_t dst = ring.addr();
      place(dst, 0, now);
      if (wide) {  // twice as many loads: the others without looking ahead
        fetch(x, order, n, kSteps, now);
        place(dst, kSteps, now);
      }
      fence_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_addr(&m->kv_full[st]));
      ++ring.entry;
    }
  }
#pragma unroll 1
  for (int k = 0; k < 2; ++k) {  // releases that are still to arrive
    Ring<kDp> &ring = rings[k];
    const uint32_t held = min(ring.entry, static_cast<uint32_t>(S::kRing)), last = ring.entry;
    for (ring.entry = last - held; ring.entry != last; ++ring.entry)
      if (!warp_wait(smem_addr(&m->kv_empty[ring.slot()]), ring.phase())) return;
  }
}

// e4m3 pages by TMA: one warp loads the bytes of an entry's rows as they are into a small ring, six
// warps turn them into operand rows of the query's type (exact).  K and V of a tile, then the next
// tile's.  Against warps that fetch the bytes themselves this takes look-ups, addresses and the
// memory's latency off the converting warps: 16 x 128 new tokens over 1000 to 4000 cached ones in
// 444 us that way.
template <int kDp>
__device__ __forceinline__ void load_role_raw(const ChunkParams &p, const CUtensorMap *kmap, const CUtensorMap *vmap, const CUtensorMap *qmap, uint32_t base,
                              Misc *m) {
  using S = Shape<kDp>;
  const int lane = threadIdx.x & 31;
  const uint32_t elected = elect_lane();
  uint32_t queries[2] = {0, 0};
  uint32_t entry = 0;
  const int boxes = kTile / p.box;
  const bool head_inner = p.head_inner != 0;
  Schedule schedule(p, p.plan_inside ? m->prefix : p.prefix);
#pragma unroll 1
  for (uint32_t item = 0;; ++item) {
    const Piece x = schedule.next(p);
    if (!publish<kDp>(p, qmap, x, item, base, m, elected, queries)) break;
    if (__all_sync(0xFFFFFFFFu, x.rows == 0)) break;
    const TileOrder order = tile_order<S::kStreams>(p, x);
    if (order.count == 0) continue;  // no tile, and so none whose pages could be looked up ahead
    bool ok = true;
    int32_t page = p.num_blocks, in_page = 0;
#pragma unroll 1
    for (int q = -1; q < order.count && ok; ++q) {
      const int32_t now_page = page, now_in = in_page;
      const int32_t tok = order.tile(min(q + 1, order.count - 1)) * kTile + lane * p.box;
      page = p.num_blocks, in_page = 0;
      if (lane < boxes && tok < x.q.len) {
        const int32_t b = page_of(p, x.seq, tok);
        if (b >= 0) page = b;
        in_page = p.bs_shift >= 0 ? tok & (p.block_size - 1) : tok % p.block_size;
      }
      if (q < 0) continue;
#pragma unroll 1
      for (int n = 0; n < 2 * S::kUnits && ok; ++n, ++entry) {
        const uint32_t st = entry & 1;
        if (entry >= 2 && !warp_wait(smem_addr(&m->raw_empty[st]), (entry >> 1 & 1) ^ 1)) {
          ok = false;
          break;
        }
        const int u = n % S::kUnits;
        const uint32_t bar = smem_addr(&m->raw_full[st]);
        uint32_t dst = base + S::kRawAt + st * S::kRawBytes;
        if (elected) mbar_expect_tx(bar, S::kRawBytes);
        __syncwarp();
#pragma unroll 1
        for (int k = 0; k < boxes; ++k, dst += p.box * S::kUnitPanels * 64) {
          const int32_t pg = __shfl_sync(0xFFFFFFFFu, now_page, k), in = __shfl_sync(0xFFFFFFFFu, now_in, k);
          tma_load4(elected, dst, n >= S::kUnits ? vmap : kmap, u * S::kUnitPanels * 64, head_inner ? x.head : in, head_inner ? in : x.head, pg,
                    bar);
        }
      }
    }
    if (!ok) break;
  }
  // what is in flight arrives before the CTA ends
#pragma unroll 1
  for (uint32_t n = entry - min(entry, 2u); n != entry; ++n) warp_wait(smem_addr(&m->raw_full[n & 1]), n >> 1 & 1);
}

template <typename T, int kDp>
__device__ __forceinline__ void convert_role(const ChunkParams &p, char *smem, uint32_t base, Misc *m) {
  using S = Shape<kDp>;
  constexpr int kPieces = S::kUnitPanels * 4;                                 // 16-byte pieces of a row
  constexpr int kSteps = (4 * kPieces + kConvertWarps - 1) / kConvertWarps;  // of a lane and entry
  const int lane = threadIdx.x & 31, warp = (threadIdx.x >> 5) - (kMmaWarp + 2);
  const uint32_t elected = elect_lane();
  const int piece = lane % kPieces, in_group = lane / kPieces;
  Ring<kDp> rings[2] = {Ring<kDp>(base, 0), Ring<kDp>(base, 1)};
  uint32_t entry = 0;
#pragma unroll 1
  for (uint32_t item = 0;; ++item) {
    Piece x;
    if (!receive(m, item, elected, &x)) return;
    if (__all_sync(0xFFFFFFFFu, x.rows == 0)) break;
    const TileOrder order = tile_order<S::kStreams>(p, x);
#pragma unroll 1
    for (int n = 0; n < order.count * 2 * S::kUnits; ++n, ++entry) {
      const int valid = x.q.len - order.tile(n / (2 * S::kUnits)) * kTile;  // rows behind the sequence become zeros
      Ring<kDp> &ring = rings[n / S::kUnits & 1];
      const uint32_t st = entry & 1;
      if (!warp_wait(smem_addr(&m->raw_full[st]), entry >> 1 & 1)) return;
      const char *raw = smem + S::kRawAt + st * S::kRawBytes;
      uint4 r[kSteps];
#pragma unroll
      for (int k = 0; k < kSteps; ++k) {
        const int row = (warp + kConvertWarps * k) * (32 / kPieces) + in_group;
        r[k] = make_uint4(0, 0, 0, 0);
        if (row < min(valid, kTile)) r[k] = *reinterpret_cast<const uint4 *>(raw + row * (kPieces * 16) + piece * 16);
      }
      __syncwarp();
      if (elected) mbar_arrive(smem_addr(&m->raw_empty[st]));
      if (ring.entry >= S::kRing && !warp_wait(smem_addr(&m->kv_empty[ring.slot()]), ring.phase() ^ 1)) return;
      const uint32_t dst = ring.addr();
#pragma unroll
      for (int k = 0; k < kSteps; ++k) {
        const int row = (warp + kConvertWarps * k) * (32 / kPieces) + in_group;
        const uint32_t from[4] = {r[k].x, r[k].y, r[k].z, r[k].w};
        uint32_t y[8];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          uint32_t lo, hi;
          asm("{ .reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b; }"
              : "=r"(lo), "=r"(hi)
              : "r"(from[q]));
          y[2 * q] = T::from_f16x2(lo), y[2 * q + 1] = T::from_f16x2(hi);
        }
        if (row >= kTile) continue;
        const uint32_t at = dst + (row >> 3) * p.group_stride + (row & 7) * 128 + (2 * piece >> 3) * p.panel_stride;
#pragma unroll
        for (int c = 0; c < 2; ++c)
          asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(at + ((((2 * piece + c) & 7) ^ (row & 7)) << 4)), "r"(y[4 * c]),
                       "r"(y[4 * c + 1]), "r"(y[4 * c + 2]), "r"(y[4 * c + 3])
                       : "memory");
      }
      fence_async_smem();
      __syncwarp();
      if (elected) mbar_arrive(smem_addr(&m->kv_full[ring.slot()]));
      ++ring.entry;
    }
  }
#pragma unroll 1
  for (int k = 0; k < 2; ++k) {  // releases that are still to arrive
    Ring<kDp> &ring = rings[k];
    const uint32_t held = min(ring.entry, static_cast<uint32_t>(S::kRing)), last = ring.entry;
    for (ring.entry = last - held; ring.entry != last; ++ring.entry)
      if (!warp_wait(smem_addr(&m->kv_empty[ring.slot()]), ring.phase())) return;
  }
}

// ---- products -----------------------------------------------------------------------------
//
// A tcgen05.commit that follows another one waits in the issuing warp until the products ahead of the
// first have ended (about 800 clocks here), so there is one commit per group of products: scores
// announce themselves and with them every product issued earlier.  What else waits for the products
// -- the rings, the query tile -- is told by the softmax warps.

template <typename T, int kDp>
struct Products {
  using S = Shape<kDp>;
  // instruction descriptors: f32 accumulator, M = 128, B K-major (scores) or N-major (output)
  static constexpr uint32_t kTypes = (1u << 4) | (T::kFormat << 7) | (T::kFormat << 10) | ((kTile >> 4) << 24);
  static constexpr uint32_t kScores = kTypes | ((kTile >> 3) << 17);
  static constexpr uint32_t kOutput = kTypes | (1u << 16) | ((S::kUnitPanels * 64 / 8) << 17);

  const ChunkParams &p;
  uint32_t elected;
  uint32_t base, tmem;
  Misc *m;
  Ring<kDp> k_ring, v_ring;
  uint32_t q_phase = 0, p_phase = 0;  // bit s: parity of the next wait for stream s's queries / weights
  uint32_t tiles = 0, weights = 0;    // one stream: score tiles and output products issued
  __device__ __forceinline__ Products(const ChunkParams &params, uint32_t smem_base, uint32_t tmem_base, Misc *misc)
      : p(params), elected(elect_lane()), base(smem_base), tmem(tmem_base), m(misc), k_ring(smem_base, 0), v_ring(smem_base, 1) {}

  __device__ __forceinline__ bool acquire(Ring<kDp> ring) {  // one tile
#pragma unroll
    for (int u = 0; u < S::kUnits; ++u, ++ring.entry)
      if (!warp_wait(smem_addr(&m->kv_full[ring.slot()]), ring.phase())) return false;
    return true;
  }
  __device__ __forceinline__ void scores(uint32_t s) {
    tc_fence_after();
    const uint32_t buf = S::kScoreBufs == 2 ? (tiles++ & 1) : s;
    const uint32_t d = tmem + buf * kTile;
    Ring<kDp> k = k_ring;
    uint32_t q = base + s * S::kQBytes;
#pragma unroll
    for (int u = 0; u < S::kUnits; ++u, ++k.entry) {
#pragma unroll
      for (int pp = 0; pp < S::kUnitPanels; ++pp, q += kPanelBytes) {
        const uint64_t qd = operand_desc(q, 16, 1024);
        const uint64_t kd = operand_desc(k.addr() + pp * p.panel_stride, 16, p.group_stride);
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) mma_ss(elected, d, qd + kk * 2, kd + kk * 2, kScores, u > 0 || pp > 0 || kk > 0);
      }
    }
    tc_commit(elected, smem_addr(&m->s_full[0]) + 8 * buf);
  }
  // The product over the first three quarters of the tokens runs while the last weights are still
  // being made.
  __device__ __forceinline__ bool output(uint32_t s, bool first, bool last) {
    const uint32_t buf = S::kScoreBufs == 2 ? (weights & 1) : s;
    const uint32_t ph = S::kScoreBufs == 2 ? (weights >> 1 & 1) : (p_phase >> s & 1);
    const uint32_t a = tmem + buf * kTile, d = tmem + 256 + s * kDp;
    const uint32_t step = p.group_stride >> 3;  // 16 tokens, in descriptor units
    if (!warp_wait(smem_addr(&m->p_part[0]) + 8 * buf, ph)) return false;
    tc_fence_after();
    Ring<kDp> v = v_ring;
#pragma unroll
    for (int u = 0; u < S::kUnits; ++u, ++v.entry) {
      const uint64_t vd = operand_desc(v.addr(), p.panel_stride, p.group_stride);
#pragma unroll
      for (int kk = 0; kk < 6; ++kk) mma_ts(elected, d + u * 128, a + kk * 8, vd + kk * step, kOutput, !first || kk > 0);
    }
    if (!warp_wait(smem_addr(&m->p_full[0]) + 8 * buf, ph)) return false;
    tc_fence_after();
    v = v_ring;
#pragma unroll
    for (int u = 0; u < S::kUnits; ++u, ++v.entry) {
      const uint64_t vd = operand_desc(v.addr(), p.panel_stride, p.group_stride);
#pragma unroll
      for (int kk = 6; kk < 8; ++kk) mma_ts(elected, d + u * 128, a + kk * 8, vd + kk * step, kOutput, 1);
    }
    // two streams: until the last tile, the stream's next scores tell that this product has ended
    if (S::kScoreBufs == 2 || last) tc_commit(elected, smem_addr(&m->pv_done[0]) + 8 * s);
    p_phase ^= 1u << s;
    ++weights;
    return true;
  }

  __device__ __forceinline__ bool piece(const Piece &x) {
    int late = 0, end[2] = {0, 0};  // places of the streams' tiles: [late, end) and [0, end)
#pragma unroll
    for (int s = 0; s < S::kStreams; ++s) {
      const Walk w = stream_walk<S::kStreams>(p, x, s);
      const int n = __reduce_max_sync(0xFFFFFFFFu, w.count());  // (uniform, and known to be)
      if (n == 0) continue;
      if (s == 0) late = __reduce_max_sync(0xFFFFFFFFu, w.late);
      end[s] = s == 0 ? late + n : n;
      if (!warp_wait(smem_addr(&m->q_full[s]), q_phase >> s & 1)) return false;
      q_phase ^= 1u << s;
    }
    const bool narrow = S::kStreams == 2 && __any_sync(0xFFFFFFFFu, x.narrow) != 0;
    const int most = max(end[0], end[1]);
    if (most == 0) return true;
#pragma unroll 1
    for (int i = 0; i <= most; ++i) {
      if (S::kStreams == 1) {  // scores of the next tile ahead of the output product of this one
        if (i < most) {
          if (!acquire(k_ring)) return false;
          scores(0);
          k_ring.entry += S::kUnits;
        }
        if (i > 0) {
          if (!acquire(v_ring) || !output(0, i == 1, i == most)) return false;
          v_ring.entry += S::kUnits;
        }
        continue;
      }
      bool has_k = false, has_v = false;
#pragma unroll
      for (uint32_t s = 0; s < 2; ++s) {
        const int from = s == 0 ? late : 0;
        if (i > from && i <= end[s]) {
          if (!has_v && !acquire(v_ring)) return false;
          has_v = true;
          if (!output(s, i - 1 == from, i == end[s])) return false;
        }
        if (i >= from && i < end[s]) {
          if (!has_k && !acquire(k_ring)) return false;
          has_k = true;
          scores(s);
        }
        if (narrow || s == 1) {  // the tiles' last reader
          v_ring.entry += has_v;
          k_ring.entry += has_k;
          has_k = has_v = false;
        }
      }
    }
    return true;
  }
};

// ---- softmax ------------------------------------------------------------------------------

// Raises the weights' reference maximum only when it has moved by more than this (in the exp2
// domain): weights then stay below 2^8, and the sums in tensor memory are rescaled on a few tiles instead
// of on every one.  Weights, and with them their sums, are carried as 2^kShift times themselves: below
// 2^15 in f16 (whose largest value is 65504), where the rounding of a weight is relative down to 2^-21 and at most
// 2^-32 below that, so that a long context of little weight beside one dominant token is not lost.
constexpr float kLazy = 8.f;

// Weights of 32 scores of one row: exponentials, their sum, and the rounded pairs to tensor memory.
// (Making a quarter of the exponentials by a polynomial on the f32 pipes was slower: the softmax warps
// are bound by the latency of their own instructions, not by the exponential unit.)
template <typename T>
__device__ __forceinline__ void weigh(const float *sc, float2 mul2, float2 sub2, float2 &sum2, uint32_t to) {
  uint32_t w[16];
#pragma unroll
  for (int k = 0; k < 16; ++k) {
    const float2 z = __ffma2_rn(make_float2(sc[2 * k], sc[2 * k + 1]), mul2, sub2);
    const float2 y = make_float2(fast_exp2(z.x), fast_exp2(z.y));
    sum2 = __fadd2_rn(sum2, y);
    w[k] = T::pack2(y.x, y.y);
  }
  tc_st16(to, w);
}

// Whether the page of this lane's four tokens of the tile at `first` exists; page sizes that are not a
// multiple of four are looked up token by token where it matters.
__device__ __forceinline__ bool pages_exist(const ChunkParams &p, const Piece &x, int32_t first) {
  const int32_t tok = first + (threadIdx.x & 31) * 4;
  return tok >= x.q.len || ((p.block_size & 3) == 0 && page_of(p, x.seq, tok) >= 0);
}

// Whether one of this row's sums is not finite.
template <int kDp>
__device__ __forceinline__ bool sums_not_finite(uint32_t o_at) {
  const float2 zero = make_float2(0.f, 0.f);
  float2 f0 = zero, f1 = zero;  // become NaN with the first value that is not finite
#pragma unroll 1
  for (int k = 0; k < kDp; k += 64) {
    float a[32], b[32];
    tc_ld32(a, o_at + k);
    tc_ld32(b, o_at + k + 32);
    tc_wait_ld();
#pragma unroll
    for (int i = 0; i < 32; i += 2) {
      f0 = __ffma2_rn(make_float2(a[i], a[i + 1]), zero, f0);
      f1 = __ffma2_rn(make_float2(b[i], b[i + 1]), zero, f1);
    }
  }
  return (f0.x + f0.y) + (f1.x + f1.y) != 0.f;
}

// The sums of the rows of a warp that are `bad` once more, over the tokens [first, limit) that the row sees,
// with the weights they were made with (exp2(mul * score + sub)).  A few tokens at a time, every lane its own
// row: all lanes read the same elements of K and V.  At most three tiles of tokens, about 4 ms at head_dim 128, far
// below what the other roles' waits allow: a prompt of 8 000 tokens x 8 heads with no finite value in V takes
// 8.8 ms (9.9 from packed pages, 22 at head_dim 256).  Looking for such rows costs the 16 prompts of the note
// at the kernel 1 %, the order of the tiles 2 % (4 x 512 tokens over 32k gain 3 % by it).
template <typename T, int kDp, bool kFp8>
__device__ __noinline__ void repair_rows(const ChunkParams &p, const Piece &x, bool bad, int32_t r, int32_t first, int32_t limit, float mul,
                                         float sub, uint32_t o_at) {
  constexpr int kTok = 8;
  auto q_at = [](const char *at) { return T::get(*reinterpret_cast<const uint16_t *>(at)); };
  auto kv_at = [&](const char *at) { return kFp8 ? load_f32(at, KVX_DTYPE_F8_E4M3) : q_at(at); };
  if (!bad) r = x.row0, limit = 0;
  const int32_t token = r / p.group, qh = x.head * p.group + r % p.group;
  const char *q = p.query + (x.q.first + token) * p.q_pitch + static_cast<int64_t>(qh) * p.dim * 2;
  const int32_t end = __reduce_max_sync(0xFFFFFFFFu, limit);
#pragma unroll 1
  for (int k = 0; k < kDp; k += 16) {
    float o[16];
    tc_ld16(o, o_at + k);
    tc_wait_ld();
#pragma unroll
    for (int i = 0; i < 16; ++i) o[i] = bad ? 0.f : o[i];
    tc_st16(o_at + k, reinterpret_cast<const uint32_t *>(o));
  }
  tc_wait_st();
  if (p.num_blocks == 0) return;
#pragma unroll 1
  for (int32_t t0 = first; t0 < end; t0 += kTok) {
    const char *at[kTok];  // K, then V; of page 0 for tokens that are left out
    float w[kTok];
    uint32_t in = 0;
    auto rows = [&](const PageView &v) {
#pragma unroll
      for (int i = 0; i < kTok; ++i) {
        const int32_t t = t0 + i, page = t < end ? page_of(p, x.seq, t) : -1;
        at[i] = v.base + max(page, 0) * v.blk + static_cast<int64_t>(t % p.block_size) * v.tok + x.head * v.head;
        if (page >= 0 && t < limit) in |= 1u << i;
      }
    };
    // from one element to the next
    int32_t left;
    auto step = [&](const PageView &v) {
      int64_t by = v.dlo;
      if (--left == 0) by = v.dhi - (v.pack - 1) * v.dlo, left = v.pack;
#pragma unroll
      for (int i = 0; i < kTok; ++i) at[i] += by;
    };
    rows(p.k);
    left = p.k.pack;
#pragma unroll
    for (int i = 0; i < kTok; ++i) w[i] = 0.f;
#pragma unroll 1
    for (int d = 0; d < p.dim; ++d) {
      const float y = q_at(q + d * 2);
#pragma unroll
      for (int i = 0; i < kTok; ++i) w[i] = fmaf(y, kv_at(at[i]), w[i]);
      step(p.k);
    }
#pragma unroll
    for (int i = 0; i < kTok; ++i) w[i] = exp2f(fmaf(w[i], mul, sub));
    rows(p.v);
    left = p.v.pack;
#pragma unroll 1
    for (int k = 0; k < p.dim; k += 16) {
      float o[16];
      tc_ld16(o, o_at + k);
      tc_wait_ld();
#pragma unroll
      for (int c = 0; c < 16; ++c) {
        if (k + c >= p.dim) continue;
#pragma unroll
        for (int i = 0; i < kTok; ++i) {
          const float v = kv_at(at[i]);
          o[c] = (in >> i) & 1 ? fmaf(w[i], v, o[c]) : o[c];
        }
        step(p.v);
      }
      tc_st16(o_at + k, reinterpret_cast<const uint32_t *>(o));
    }
    tc_wait_st();
  }
}

// Sets scores that must not count (tokens the row may not see, tokens without a page) to -inf, and
// gives the others the sign of the multiplier.
__device__ __forceinline__ void correct_scores(const ChunkParams &p, const Piece &x, uint32_t s_at, int32_t first, int32_t valid, bool gaps,
                                               float sign) {
#pragma unroll 1
  for (int k = 0; k < kTile; k += 32) {
    float c[32];
    tc_ld32(c, s_at + k);
    unsigned has = 0xFFFFFFFFu;
    if (gaps) {
      const int32_t tok = first + k + (threadIdx.x & 31);
      has = __ballot_sync(0xFFFFFFFFu, tok >= x.q.len || page_of(p, x.seq, tok) >= 0);
    }
    if (valid - k < 32) has &= valid <= k ? 0u : (1u << (valid - k)) - 1;
    tc_wait_ld();
#pragma unroll
    for (int i = 0; i < 32; ++i) c[i] = (has >> i) & 1 ? c[i] * sign : -INFINITY;
    tc_st32(s_at + k, c);
  }
  tc_wait_st();
}

template <typename T, int kDp>
__device__ __forceinline__ void softmax_role(const ChunkParams &p, uint32_t base, char *smem, uint32_t tmem0, Misc *m) {
  using S = Shape<kDp>;
  const int s = threadIdx.x >> 7;                 // stream
  const int tid = threadIdx.x & 127, lane = threadIdx.x & 31;
  const uint32_t lanes = static_cast<uint32_t>((tid >> 5) * 32) << 16;  // this warp's lanes of tensor memory
  uint32_t tiles = 0;   // score tiles of this stream so far
  uint32_t pieces = 0;  // pieces of this stream that had any
  uint32_t joins = 0;
  uint32_t entries = 0;  // tiles of both rings before this piece
  // The ring entries of a K or V tile (the `q`-th of the piece) may be filled again.
  auto release = [&](int which, int q) {
    if (tid != 0) return;
#pragma unroll
    for (int u = 0; u < S::kUnits; ++u)
      mbar_arrive(smem_addr(&m->kv_empty[0]) + 8 * (which * S::kRing + (((entries + q) * S::kUnits + u) & (S::kRing - 1))));
  };
#pragma unroll 1
  for (uint32_t item = 0;; ++item) {
    const uint32_t slot = item % kItems;
    if (!warp_wait(smem_addr(&m->item_full[slot]), (item / kItems) & 1)) return;
    const Piece x = m->items[slot];
    __syncwarp();
    if (lane == 0) mbar_arrive(smem_addr(&m->item_empty[slot]));
    if (x.rows == 0) return;
    int b, e, other = 0;  // tiles of this stream, number of the other stream's
    stream_range<S::kStreams>(p, x, s, &b, &e);
    if (S::kStreams == 2) {
      int ob, oe;
      stream_range<S::kStreams>(p, x, s ^ 1, &ob, &oe);
      other = oe - ob;
    }
    const bool narrow = S::kStreams == 2 && x.narrow;
    const int count = narrow ? e - b + other : max(e - b, other);  // tiles of the piece, each of K and of V
    // this stream is the last reader of its tiles (stream 1 comes after stream 0, and takes every tile)
    const bool last_reader = narrow || s == 1 || other == 0;
    auto place = [&](int i) { return narrow ? 2 * i + s : i; };  // of this stream's tile i, where it is the last reader
    const int32_t row_at = x.row0 + (narrow ? 0 : s * kTile);   // first group row of this stream
    const int32_t rows = min(kTile, x.rows - (narrow ? 0 : s * kTile));
    if (rows <= 0) {
      entries += count;
      continue;
    }
    const float mul = nonzero(score_mul(p, x.head));
    const float am = fabsf(mul), sign = mul > 0.f ? 1.f : -1.f;

    if (e > b && !p.q_tma) {
      // Query rows into the swizzled operand tile (its last reader, the scores of this stream's
      // previous tile, was waited for).
      constexpr int kChunks = kDp / 8, kBatch = 4;
#pragma unroll 1
      for (int i0 = tid; i0 < kTile * kChunks; i0 += 128 * kBatch) {
        uint4 y[kBatch];
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
          const int i = i0 + 128 * k, row = i / kChunks, d = i % kChunks * 8;
          y[k] = make_uint4(0, 0, 0, 0);
          if (row < rows && d < p.dim) {
            const int32_t r = row_at + row, token = r / p.group, hq = x.head * p.group + (r - token * p.group);
            const char *src = p.query + (x.q.first + token) * p.q_pitch + (static_cast<int64_t>(hq) * p.dim + d) * 2;
            if (p.q_vec) {
              y[k] = *reinterpret_cast<const uint4 *>(src);
            } else {
              uint32_t t[4] = {0, 0, 0, 0};
#pragma unroll
              for (int c = 0; c < 8; ++c)
                if (d + c < p.dim) t[c >> 1] |= static_cast<uint32_t>(reinterpret_cast<const uint16_t *>(src)[c]) << ((c & 1) * 16);
              y[k] = make_uint4(t[0], t[1], t[2], t[3]);
            }
          }
        }
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
          const int i = i0 + 128 * k, row = i / kChunks, c = i % kChunks;
          const uint32_t to = base + s * S::kQBytes + (c >> 3) * kPanelBytes + row * 128 + (((c & 7) ^ (row & 7)) << 4);
          asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(to), "r"(y[k].x), "r"(y[k].y), "r"(y[k].z), "r"(y[k].w) : "memory");
        }
      }
      fence_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_addr(&m->q_full[0]) + 8 * s);
    }

    // (rows behind the tile's last are never written: nothing is masked for them)
    const int32_t limit = tid < rows ? row_limit(p, x.q, row_at + tid) : INT32_MAX;
    float mx = -INFINITY, l = 0.f;
    const uint32_t o_at = tmem0 + lanes + 256 + s * kDp;
    int from = e;
    if ((tid & ~31) >= rows) {
      // All rows of this warp lie behind the tile's last: no weights to make.  What the products do
      // with its lanes stays in its lanes.
#pragma unroll 1
      for (; from > b; --from, ++tiles) {
        const uint32_t buf = S::kScoreBufs == 2 ? (tiles & 1) : s;
        if (!warp_wait(smem_addr(&m->s_full[0]) + 8 * buf, (S::kScoreBufs == 2 ? tiles >> 1 : tiles) & 1)) return;
        if (S::kStreams == 1 && from < e && !warp_wait(smem_addr(&m->pv_done[0]), (tiles - 1) & 1)) return;
        if (lane == 0) {
          mbar_arrive(smem_addr(&m->p_part[0]) + 8 * buf);
          mbar_arrive(smem_addr(&m->p_full[0]) + 8 * buf);
        }
        __syncwarp();
      }
    }
    // Called when all products so far have ended, and only tiles with masked tokens are among them: [masked, e).
    const int masked = max(b, min(e, x.kv_masked));
    const bool any_masked = __any_sync(0xFFFFFFFFu, limit < min(x.q.len, e * kTile)) != 0 && masked < e;
    auto repair = [&]() {
      const bool bad = sums_not_finite<kDp>(o_at) && limit < min(x.q.len, e * kTile);
      if (!__any_sync(0xFFFFFFFFu, bad)) return;
      const Piece y = x;  // (a copy: the reference keeps it in memory)
      const float sub = mx == -INFINITY ? T::kShift : fmaf(-mx, am, T::kShift);
      if (p.cache_code == KVX_DTYPE_F8_E4M3)
        repair_rows<T, kDp, true>(p, y, bad, row_at + tid, masked * kTile, limit, mul, sub, o_at);
      else
        repair_rows<T, kDp, false>(p, y, bad, row_at + tid, masked * kTile, limit, mul, sub, o_at);
    };
    const int repair_at = any_masked ? masked - 1 : -1;  // the tile ahead of which that is
    bool page_ok = pages_exist(p, x, max(e - 1, 0) * kTile);
#pragma unroll 1
    for (int j = from - 1; j >= b; --j, ++tiles) {
      const uint32_t buf = S::kScoreBufs == 2 ? (tiles & 1) : s;
      const uint32_t ph = (S::kScoreBufs == 2 ? tiles >> 1 : tiles) & 1;
      const uint32_t s_at = tmem0 + lanes + buf * kTile;
      const int32_t valid = limit == INT32_MAX ? kTile : min(kTile, limit - j * kTile);  // visible tokens of this row (may be negative)
      const bool plain = __all_sync(0xFFFFFFFFu, valid == kTile && page_ok && mul > 0.f) != 0;
      const bool gaps = __all_sync(0xFFFFFFFFu, page_ok) == 0;
      if (!warp_wait(smem_addr(&m->s_full[0]) + 8 * buf, ph)) return;
      tc_fence_after();
      // these scores have read their K tile, and (two streams) the product ahead of them its V tile
      const int i = e - 1 - j;
      if (last_reader) release(0, place(i));
      if (S::kStreams == 2 && i > 0 && last_reader) release(1, place(i - 1));
      if (j == b && p.q_tma && tid == 0 && !(s == 1 && joins_streams(x))) mbar_arrive(smem_addr(&m->q_empty[0]) + 8 * s);
      if (j == repair_at) {
        if (S::kStreams == 1 && !warp_wait(smem_addr(&m->pv_done[0]), (tiles - 1) & 1)) return;
        tc_fence_after();
        repair();
      }
      if (!plain) correct_scores(p, x, s_at, j * kTile, valid, gaps, sign);
      float top = -INFINITY;
#pragma unroll 1
      for (int k = 0; k < kTile; k += 64) {
        float c0[32], c1[32];
        tc_ld32(c0, s_at + k);
        tc_ld32(c1, s_at + k + 32);
        tc_wait_ld();
        float t0 = top, t1 = -INFINITY, t2 = -INFINITY, t3 = -INFINITY;
#pragma unroll
        for (int i = 0; i < 32; i += 4) {
          t0 = fmaxf(fmaxf(t0, c0[i]), c0[i + 1]);
          t1 = fmaxf(fmaxf(t1, c1[i]), c1[i + 1]);
          t2 = fmaxf(fmaxf(t2, c0[i + 2]), c0[i + 3]);
          t3 = fmaxf(fmaxf(t3, c1[i + 2]), c1[i + 3]);
        }
        top = fmaxf(fmaxf(t0, t1), fmaxf(t2, t3));
      }
      page_ok = pages_exist(p, x, max(j - 1, 0) * kTile);  // of the next tile: on its way meanwhile
      const bool raise = top > mx && (mx == -INFINITY || (top - mx) * am > kLazy);
      if (__any_sync(0xFFFFFFFFu, raise)) {
        const float c = raise ? weight_of(mx, top, am) : 1.f;
        if (raise) mx = top;
        if (j < e - 1) {
          l *= c;
          // the sums of the tiles so far must be complete before they are rescaled (two streams: they
          // are, these scores were announced behind them)
          if (S::kStreams == 1 && !warp_wait(smem_addr(&m->pv_done[0]), (tiles - 1) & 1)) return;
          tc_fence_after();
#pragma unroll 1
          for (int k = 0; k < kDp; k += 16) {
            float o[16];
            tc_ld16(o, o_at + k);
            tc_wait_ld();
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] *= c;
            tc_st16(o_at + k, reinterpret_cast<const uint32_t *>(o));
          }
        }
      }
      // weights exp2((score - mx) * am + kShift); a row that has seen no token yet subtracts 0
      const float sub = mx == -INFINITY ? T::kShift : fmaf(-mx, am, T::kShift);
      const float2 mul2 = make_float2(am, am), sub2 = make_float2(sub, sub);
      float2 sum2 = make_float2(0.f, 0.f);
      {
        // 32 columns at a time, the next 32 on their way; the weights of columns c, c + 1 go to column
        // c / 2, which has been read by then.
        float c0[32], c1[32];
        tc_ld32(c0, s_at);
#pragma unroll 1
        for (int k = 0; k < 2; ++k) {
          tc_wait_ld();
          tc_ld32(c1, s_at + 64 * k + 32);
          weigh<T>(c0, mul2, sub2, sum2, s_at + 32 * k);
          tc_wait_ld();
          if (k == 0) {
            tc_ld32(c0, s_at + 64);
          } else {
            // Three quarters are made.  One stream: the scores of this tile were issued ahead of the
            // previous output product, so they do not tell that it has ended.  Weights are handed over
            // only after it has -- its barrier is then never more than one phase away from the
            // parity that is waited for.
            if (S::kStreams == 1 && j < e - 1) {
              if (!warp_wait(smem_addr(&m->pv_done[0]), (tiles - 1) & 1)) return;
              release(1, i - 1);
            }
            tc_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_addr(&m->p_part[0]) + 8 * buf);
          }
          weigh<T>(c1, mul2, sub2, sum2, s_at + 32 * k + 16);
        }
      }
      l += sum2.x + sum2.y;
      tc_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_addr(&m->p_full[0]) + 8 * buf);
    }

    // ---- the piece's result ----
    if (e > b) {
      if (!warp_wait(smem_addr(&m->pv_done[0]) + 8 * s, (S::kStreams == 1 ? tiles - 1 : pieces) & 1)) return;
      tc_fence_after();
      ++pieces;
      if (last_reader) release(1, place(e - b - 1));
      if (masked == b && any_masked) repair();  // no other tiles came behind those with masked tokens
    }
    entries += count;
    const float vmul = p.vs.base != nullptr ? p.vs.base[x.head * p.vs.stride] : 1.f;
    const bool join = S::kStreams == 2 && joins_streams(x);
    // Stream 1 hands its sums to stream 0 through its query tile, [kDp / 2][128] at a time.
    float *joint = reinterpret_cast<float *>(smem + S::kQBytes) + tid;
    if (narrow && s == 1) {
      if (!join) continue;
      m->join_m[tid] = mx, m->join_l[tid] = l;
#pragma unroll 1
      for (int k = 0; k < kDp; k += 16) {
        if (k == kDp / 2) {
          if (!warp_wait(smem_addr(&m->join_empty), joins & 1)) return;
          ++joins;
        }
        float o[16];
        tc_ld16(o, o_at + k);
        tc_wait_ld();
#pragma unroll
        for (int i = 0; i < 16; ++i) joint[(k % (kDp / 2) + i) * kTile] = o[i];
        if (k % (kDp / 2) + 16 == kDp / 2) {
          fence_async_smem();  // TMA may fill the tile next
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_addr(&m->join_full));
        }
      }
      // the query tile is free again once stream 0 has read the second part
      if (!warp_wait(smem_addr(&m->join_empty), joins & 1)) return;
      ++joins;
      if (p.q_tma && tid == 0) mbar_arrive(smem_addr(&m->q_empty[1]));
      tc_fence_before();
      continue;
    }
    float f_own = 1.f, f_other = 0.f;
    if (join) {
      if (!warp_wait(smem_addr(&m->join_full), joins & 1)) return;
      const float m1 = m->join_m[tid], l1 = m->join_l[tid];
      const float top = fmaxf(mx, m1);
      f_own = weight_of(mx, top, am), f_other = weight_of(m1, top, am);
      l = l * f_own + l1 * f_other;
      mx = top;
    }
    const int32_t r = row_at + tid;
    const int32_t token = r / p.group, qh = x.head * p.group + r % p.group;
    char *out = p.out + (x.q.first + token) * p.o_pitch + static_cast<int64_t>(qh) * p.dim * 2;
    const int64_t part = x.slot < 0 ? 0 : static_cast<int64_t>(x.slot) * p.slot_rows + (r - x.row0);
    const float mul_out = l == 0.f ? 0.f : (x.slot < 0 ? vmul / l : vmul);
    const bool vec_out = p.q_vec != 0;
    char *quad_out[4];  // the rows of this thread and its three neighbours
#pragma unroll
    for (int c = 0; c < 4; ++c)
      quad_out[c] = reinterpret_cast<char *>(__shfl_sync(0xFFFFFFFFu, reinterpret_cast<unsigned long long>(out), (lane & ~3) + c));
#pragma unroll 1
    for (int k = 0; k < kDp; k += 32) {
      const int d0 = k;
      float o[32];
      if (e > b) {
        tc_ld32(o, o_at + k);
        tc_wait_ld();
      } else {
#pragma unroll
        for (int i = 0; i < 32; ++i) o[i] = 0.f;
      }
      if (join) {
        if (k == kDp / 2) {
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_addr(&m->join_empty));
          if (!warp_wait(smem_addr(&m->join_full), (joins + 1) & 1)) return;
        }
#pragma unroll
        for (int i = 0; i < 32; ++i) o[i] = o[i] * f_own + joint[(k % (kDp / 2) + i) * kTile] * f_other;
      }
#pragma unroll
      for (int i = 0; i < 32; ++i) o[i] = l == 0.f ? 0.f : o[i] * mul_out;
      if (x.slot < 0 && vec_out) {
        // A thread has 64 bytes of its row; four threads exchange 16-byte pieces so that each store
        // instruction writes 64 bytes of 8 rows instead of 16 bytes of 32.
        uint32_t w[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) w[i] = T::pack2(o[2 * i], o[2 * i + 1]);
#pragma unroll
        for (int bit = 1; bit <= 2; bit <<= 1) {
          const bool up = (lane & bit) != 0;
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            if (c & bit) continue;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint32_t got = __shfl_xor_sync(0xFFFFFFFFu, up ? w[4 * c + i] : w[4 * (c | bit) + i], bit);
              if (up)
                w[4 * c + i] = got;
              else
                w[4 * (c | bit) + i] = got;
            }
          }
        }
        const int d = d0 + (lane & 3) * 8;
#pragma unroll
        for (int c = 0; c < 4; ++c)
          if ((tid & ~3) + c < rows && d < p.dim)
            *reinterpret_cast<uint4 *>(quad_out[c] + d * 2) = make_uint4(w[4 * c], w[4 * c + 1], w[4 * c + 2], w[4 * c + 3]);
      } else if (tid < rows) {
        if (x.slot >= 0) {
          float *to = p.part_o + part * p.dim + d0;
          if ((p.dim & 3) == 0) {
#pragma unroll
            for (int i = 0; i < 32; i += 4)
              if (d0 + i < p.dim) *reinterpret_cast<float4 *>(to + i) = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (d0 + i < p.dim) to[i] = o[i];
          }
        } else {
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const uint32_t w = T::pack2(o[2 * i], o[2 * i + 1]);
            uint16_t *to = reinterpret_cast<uint16_t *>(out) + d0 + 2 * i;
            if (d0 + 2 * i < p.dim) to[0] = static_cast<uint16_t>(w);
            if (d0 + 2 * i + 1 < p.dim) to[1] = static_cast<uint16_t>(w >> 16);
          }
        }
      }
    }
    if (join) {
      joins += 2;
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_addr(&m->join_empty));
    }
    if (x.slot >= 0 && tid < rows) reinterpret_cast<float2 *>(p.part_ml)[part] = make_float2(mx, l);
    tc_fence_before();
  }
}

// Every role's instruction count is part of the kernel's speed: a single warp gets through about one
// instruction in eight clocks here, so loops over columns are kept as loops of 32 to 64 columns that
// fit the registers, and what is done per tile by the loading and the issuing warps is kept small.
// Measured on 16 prompts of 512 to 4096 tokens and on 4 x 512 tokens over 32k contexts (us), in runs too short to
// reach the power cap:
//   first version, one thread issuing everything, boxes issued by their lanes     2410   1310
//   queries by TMA, column loops, waits that do not read the timer first          1290   1110 - 1250
//   + whole boxes, two loading warps, converged issue, one commit per product     1180   1080 - 1220
// Back to back, at the cap, and with the tiles from the last to the first: 1390 and 1210 (700 and 850 TFLOP/s).
// 64 x 5 drafted tokens over up to 32k, bound by the loads: 245, 4.3 TB/s.  Two warps per 32 rows (half the
// columns each, 640 threads) ran at 1470 and 1340 against 1350 and 1250 then; keeping all 128 scores of a row in
// registers at 1490 and 1390, the column loops unrolled at 1440 and 1230; strict turns between the
// streams changed nothing.
template <typename T, int kDp, Loads kLoads>
__global__ void __launch_bounds__(kLoads == kTmaLoads ? 384 : 512, 1)  // = threads_of(kLoads)
    kvx_chunk_attention_kernel(const __grid_constant__ ChunkParams p, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                               const __grid_constant__ CUtensorMap qmap) {
  using S = Shape<kDp>;
  extern __shared__ char smem_raw[];
  char *smem = reinterpret_cast<char *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const uint32_t base = smem_addr(smem);
  Misc *m = reinterpret_cast<Misc *>(smem + S::kMiscAt);
  const int warp = threadIdx.x >> 5;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (threadIdx.x == 0) {
    for (int i = 0; i < kItems; ++i) {
      mbar_init(smem_addr(&m->item_full[i]), 1);
      mbar_init(smem_addr(&m->item_empty[i]), S::kStreams * 4 + (kLoads == kTmaLoads ? 2 : kLoads == kRawLoads ? 1 + kConvertWarps : 1));  // softmax, products, others
    }
    for (int i = 0; i < 2 * S::kRing; ++i) {
      mbar_init(smem_addr(&m->kv_full[i]), kLoads == kTmaLoads ? 1 : kLoads == kRawLoads ? kConvertWarps : kCopyWarps);
      mbar_init(smem_addr(&m->kv_empty[i]), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_addr(&m->raw_full[i]), 1);
      mbar_init(smem_addr(&m->raw_empty[i]), kConvertWarps);
      mbar_init(smem_addr(&m->q_full[i]), p.q_tma ? 1 : 4);
      mbar_init(smem_addr(&m->q_empty[i]), 1);
      mbar_init(smem_addr(&m->s_full[i]), 1);
      mbar_init(smem_addr(&m->p_part[i]), 4);
      mbar_init(smem_addr(&m->p_full[i]), 4);
      mbar_init(smem_addr(&m->pv_done[i]), 1);
    }
    mbar_init(smem_addr(&m->join_full), 4);
    mbar_init(smem_addr(&m->join_empty), 4);
    mbar_init(smem_addr(&m->tail), 1);
    mbar_init(smem_addr(&m->drain), 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_addr(&m->tmem)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (p.plan_inside && warp == 0) {
    plan_few(p, m->prefix);
    // (the merge kernel reads it, too)
    if (blockIdx.x == 0) plan_few(p, p.prefix);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = m->tmem;

  if (warp < kMmaWarp) {
    if (S::kStreams == 2 || warp < 4) softmax_role<T, kDp>(p, base, smem, tmem, m);
  } else if (p.test_stall != 0 && blockIdx.x == 0 && warp == kMmaWarp + 1 && !warp_wait(smem_addr(&m->tail), 0)) {
    // A test of the bounded waits: the warp that publishes the pieces gives up before it has published or loaded
    // anything, the others when no piece comes.
  } else {
    if (warp == kMmaWarp) {
      Products<T, kDp> pr(p, base, __reduce_max_sync(0xFFFFFFFFu, tmem), m);
#pragma unroll 1
      for (uint32_t item = 0;; ++item) {
        const uint32_t slot = item % kItems;
        if (!warp_wait(smem_addr(&m->item_full[slot]), (item / kItems) & 1)) break;
        const Piece x = m->items[slot];
        __syncwarp();
        if (pr.elected) mbar_arrive(smem_addr(&m->item_empty[slot]));
        __syncwarp();
        if (__all_sync(0xFFFFFFFFu, x.rows == 0) || !pr.piece(x)) break;
      }
      // every product has ended before tensor memory is given back
      tc_commit(pr.elected, smem_addr(&m->drain));
      mbar_wait(smem_addr(&m->drain), 0);
      __syncwarp();
    } else if (kLoads == kTmaLoads) {
      if (warp <= kMmaWarp + 2) load_role_tma<kDp>(p, &kmap, &vmap, &qmap, base, m, warp == kMmaWarp + 2);
    } else if (kLoads == kRawLoads) {
      if (warp == kMmaWarp + 1)
        load_role_raw<kDp>(p, &kmap, &vmap, &qmap, base, m);
      else
        convert_role<T, kDp>(p, smem, base, m);
    } else {
      load_role_copy<T, kDp>(p, &qmap, base, m);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == kMmaWarp) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
}

// ------------------------------------------------------------------ everything else, f32 --
//
// head_dim above 256, f32 with odd strides, HND_PACKED pages or an e4m3 cache: the same schedule and the
// same one-pass softmax on the f32 units, every element read through the layout's rule.  A step is 32 rows
// x kN tokens: scores from shared memory, a warp owns 4 rows of the softmax and of the output sums (a lane
// owns every 32nd dim), K and V share one buffer.
constexpr int kSimtThreads = 256;
constexpr int kSimtRows = 32;
constexpr int simt_tokens(int dim_bucket) { return dim_bucket > 512 ? 16 : 32; }

template <int kDb>  // head_dim rounded up to 64, 128, 256, 512 or 1024
__global__ void __launch_bounds__(kSimtThreads) kvx_chunk_attention_simt_kernel(const ChunkParams p) {
  constexpr int kN = kDb > 512 ? 16 : 32;  // = simt_tokens(kDb)
  constexpr int kPer = kDb / 32;
  extern __shared__ float sm[];
  const int dp = (p.dim + 3) & ~3, pitch = dp + 4;
  float *sm_q = sm;                          // [32][pitch]
  float *sm_kv = sm_q + kSimtRows * pitch;   // [kN][pitch]
  float *sm_p = sm_kv + kN * pitch;          // [32][kN + 4]
  int32_t *sm_page = reinterpret_cast<int32_t *>(sm_p + kSimtRows * (kN + 4));  // [kN]
  pdl_prologue();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int share = blockIdx.x;
  Place w;
  int64_t left = find_share(p, p.prefix, share, &w);
  if (left > 0 && w.off >= w.steps) next_tile(p, w);
  const int io = elem_bytes(p.io_code);
  while (left > 0) {
    const int32_t stop = static_cast<int32_t>(min(static_cast<int64_t>(w.steps), w.off + left));
    const Piece x = piece_of(p, w, stop, share);
    const float mul = nonzero(score_mul(p, x.head)), am = fabsf(mul);
    __syncthreads();  // the previous piece is done with shared memory
    for (int i = tid; i < kSimtRows * dp; i += kSimtThreads) {
      const int row = i / dp, d = i - row * dp;
      float y = 0.f;
      if (row < x.rows && d < p.dim) {
        const int32_t r = x.row0 + row, token = r / p.group, h = x.head * p.group + (r - token * p.group);
        y = load_f32(p.query + (x.q.first + token) * p.q_pitch + (static_cast<int64_t>(h) * p.dim + d) * io, p.io_code);
      }
      sm_q[row * pitch + d] = mul < 0.f ? -y : y;
    }
    float acc[4][kPer], m[4], l[4];
    int32_t limit[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      m[i] = -INFINITY, l[i] = 0.f;
      limit[i] = warp * 4 + i < x.rows ? row_limit(p, x.q, x.row0 + warp * 4 + i) : 0;
#pragma unroll
      for (int k = 0; k < kPer; ++k) acc[i][k] = 0.f;
    }
    for (int j = x.kv0; j < x.kv1; ++j) {
      const int32_t t0 = j * kN;
      if (tid < kN) sm_page[tid] = t0 + tid < x.q.len ? page_of(p, x.seq, t0 + tid) : -1;
      __syncthreads();  // pages known, query in place; the previous step is done with K/V and weights
      for (int i = tid; i < kN * dp; i += kSimtThreads) {
        const int c = i / dp, d = i - c * dp;
        const int32_t page = sm_page[c];
        float y = 0.f;
        if (page >= 0 && d < p.dim)
          y = load_f32(p.k.base + page * p.k.blk + head_offset(p.k, (t0 + c) % p.block_size, x.head, d), p.cache_code);
        sm_kv[c * pitch + d] = y;
      }
      __syncthreads();
      {
        constexpr int kC = kN / 16;
        const int ty = tid >> 4, tx = tid & 15;
        float s[2][kC];
#pragma unroll
        for (int a = 0; a < 2; ++a)
#pragma unroll
          for (int b = 0; b < kC; ++b) s[a][b] = 0.f;
        for (int d = 0; d < dp; d += 4) {
          float4 q[2], k[kC];
#pragma unroll
          for (int a = 0; a < 2; ++a) q[a] = *reinterpret_cast<const float4 *>(&sm_q[(ty + 16 * a) * pitch + d]);
#pragma unroll
          for (int b = 0; b < kC; ++b) k[b] = *reinterpret_cast<const float4 *>(&sm_kv[(tx + 16 * b) * pitch + d]);
#pragma unroll
          for (int a = 0; a < 2; ++a)
#pragma unroll
            for (int b = 0; b < kC; ++b)
              s[a][b] = fmaf(q[a].w, k[b].w, fmaf(q[a].z, k[b].z, fmaf(q[a].y, k[b].y, fmaf(q[a].x, k[b].x, s[a][b]))));
        }
#pragma unroll
        for (int a = 0; a < 2; ++a)
#pragma unroll
          for (int b = 0; b < kC; ++b) sm_p[(ty + 16 * a) * (kN + 4) + tx + 16 * b] = s[a][b];
      }
      __syncthreads();  // scores in place, K no longer needed
      for (int i = tid; i < kN * dp; i += kSimtThreads) {
        const int c = i / dp, d = i - c * dp;
        const int32_t page = sm_page[c];
        float y = 0.f;
        if (page >= 0 && d < p.dim)
          y = load_f32(p.v.base + page * p.v.blk + head_offset(p.v, (t0 + c) % p.block_size, x.head, d), p.cache_code);
        sm_kv[c * pitch + d] = y;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {  // a warp's own rows: no barrier between scores and weights
        const int row = warp * 4 + i;
        const bool in = lane < kN && t0 + lane < limit[i] && sm_page[lane < kN ? lane : 0] >= 0;
        const float s = in ? sm_p[row * (kN + 4) + lane] : -INFINITY;
        float top = s;
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, d));
        const float mn = fmaxf(m[i], top);
        const float c = weight_of(m[i], mn, am);
        float wgt = 0.f;
        if (in) wgt = mn == -INFINITY ? (s == s ? 0.f : s) : exp2f((s - mn) * am);
        float sum = wgt;
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, d);
        l[i] = l[i] * c + sum;
        m[i] = mn;
#pragma unroll
        for (int k = 0; k < kPer; ++k) acc[i][k] *= c;
        if (lane < kN) sm_p[row * (kN + 4) + lane] = wgt;
      }
      __syncthreads();  // V in place, weights in place
#pragma unroll 1
      for (int c0 = 0; c0 < kN; c0 += 4) {
        float4 wv[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) wv[i] = *reinterpret_cast<const float4 *>(&sm_p[(warp * 4 + i) * (kN + 4) + c0]);
#pragma unroll
        for (int k = 0; k < kPer; ++k) {
          const int d = lane + 32 * k;
          if (d >= p.dim) continue;
          float v[4];
#pragma unroll
          for (int c = 0; c < 4; ++c) v[c] = sm_kv[(c0 + c) * pitch + d];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if (t0 + c0 + 3 < limit[i]) {
              acc[i][k] = fmaf(wv[i].w, v[3], fmaf(wv[i].z, v[2], fmaf(wv[i].y, v[1], fmaf(wv[i].x, v[0], acc[i][k]))));
            } else {  // tokens this row may not see are left out, not weighted with zero
              if (t0 + c0 < limit[i]) acc[i][k] = fmaf(wv[i].x, v[0], acc[i][k]);
              if (t0 + c0 + 1 < limit[i]) acc[i][k] = fmaf(wv[i].y, v[1], acc[i][k]);
              if (t0 + c0 + 2 < limit[i]) acc[i][k] = fmaf(wv[i].z, v[2], acc[i][k]);
            }
          }
        }
      }
    }
    const float vmul = p.vs.base != nullptr ? p.vs.base[x.head * p.vs.stride] : 1.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = warp * 4 + i;
      if (row >= x.rows) continue;
      const int32_t r = x.row0 + row, token = r / p.group, qh = x.head * p.group + r % p.group;
      char *out = p.out + (x.q.first + token) * p.o_pitch + static_cast<int64_t>(qh) * p.dim * io;
      const int64_t part = x.slot < 0 ? 0 : static_cast<int64_t>(x.slot) * p.slot_rows + row;
#pragma unroll
      for (int k = 0; k < kPer; ++k) {
        const int d = lane + 32 * k;
        if (d >= p.dim) continue;
        if (x.slot >= 0)
          p.part_o[part * p.dim + d] = acc[i][k] * vmul;
        else
          store_f32(out, d, l[i] == 0.f ? 0.f : acc[i][k] / l[i] * vmul, p.io_code);
      }
      if (x.slot >= 0 && lane == 0) reinterpret_cast<float2 *>(p.part_ml)[part] = make_float2(m[i], l[i]);
    }
    left -= stop - w.off;
    if (left > 0) next_tile(p, w);
  }
}

// f32 caches whose rows 16-byte copies can read, head_dim up to 256: steps of 64 rows x 64 tokens, bound by
// the FMA units where the rows are many.  A thread has 4 rows x 4 tokens of the scores and 4 rows x kDb / 16
// dims of the output; the 16 lanes that share rows are half a warp, so weights pass through shared memory
// without a barrier of the CTA.  K and V have a buffer each, filled asynchronously: the next K while the
// softmax and the output product run, the next V while the next scores do.  Against the kernel above, us:
// 113 tokens x 16 heads over 5k-10k tokens of 4 heads x 64  2540 -> 586;  392 x 5 over 1.2k, 8 x 128  1231 -> 353;
// with few rows, where the copies count:  8 x (1 token x 8 heads) over up to 6.6k, 8 x 128  1012 -> 262.
constexpr int kWideRows = 64, kWideTokens = 64;
constexpr size_t wide_smem_bytes(int bucket) {
  return (static_cast<size_t>(kWideRows + 2 * kWideTokens) * (bucket + 4) + kWideRows * (kWideTokens + 4) + 2 * kWideTokens) * sizeof(float);
}

__device__ __forceinline__ void copy16_async(uint32_t to, const char *from, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kPending>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(kPending) : "memory");
}

template <int kDb>  // head_dim (a multiple of 4) rounded up to 64, 128 or 256
__global__ void __launch_bounds__(kSimtThreads, kDb > 64 ? 1 : 2) kvx_chunk_attention_f32_kernel(const ChunkParams p) {
  constexpr int kPitch = kDb + 4, kPitchP = kWideTokens + 4, kCols = kDb / 64;
  extern __shared__ float4 sm_wide[];
  float *sm_q = reinterpret_cast<float *>(sm_wide);  // [64][kPitch]
  float *sm_k = sm_q + kWideRows * kPitch;            // [64][kPitch]
  float *sm_v = sm_k + kWideTokens * kPitch;          // [64][kPitch]
  float *sm_p = sm_v + kWideTokens * kPitch;          // [64][kPitchP]
  int32_t *sm_page = reinterpret_cast<int32_t *>(sm_p + kWideRows * kPitchP);  // [2][64]: of this tile and the next
  pdl_prologue();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, ty = tid >> 4, tx = tid & 15;
  const int quads = p.dim / 4;
  __shared__ int64_t sm_prefix[kPlanInside + 1];
  if (p.plan_inside) {
    if (warp == 0) plan_few(p, sm_prefix);
    if (warp == 0 && blockIdx.x == 0) plan_few(p, p.prefix);  // (the merge kernel reads it, too)
    __syncthreads();
  }
  Place w;
  int64_t left = find_share(p, p.plan_inside ? sm_prefix : p.prefix, blockIdx.x, &w);
  if (left > 0 && w.off >= w.steps) next_tile(p, w);
#pragma unroll 1
  while (left > 0) {
    const int32_t stop = static_cast<int32_t>(min(static_cast<int64_t>(w.steps), w.off + left));
    const Piece x = piece_of(p, w, stop, blockIdx.x);
    const float mul = nonzero(score_mul(p, x.head)), am = fabsf(mul);
    auto look_up = [&](int j) { return j < x.kv1 && j * kWideTokens + tid < x.q.len ? page_of(p, x.seq, j * kWideTokens + tid) : -1; };
    auto fetch = [&](const PageView &view, float *to, int j) {  // tokens without a page become zeros
      const int32_t *pages = sm_page + (j & 1) * kWideTokens;
#pragma unroll 4
      for (int i = tid; i < kWideTokens * quads; i += kSimtThreads) {
        const int c = i / quads, d = (i - c * quads) * 4;
        const int32_t page = pages[c], tok = j * kWideTokens + c;
        const int32_t o = p.bs_shift >= 0 ? tok & (p.block_size - 1) : tok % p.block_size;
        const char *from = page < 0 ? view.base : view.base + page * view.blk + o * view.tok + x.head * view.head + d * 4;
        copy16_async(smem_addr(to + c * kPitch + d), from, page >= 0);
      }
    };
    __syncthreads();  // the previous piece is done with shared memory
    if (tid < kWideTokens) sm_page[(x.kv0 & 1) * kWideTokens + tid] = look_up(x.kv0);
    for (int row = warp; row < kWideRows; row += kSimtThreads / 32) {
      const int32_t r = x.row0 + row, token = r / p.group, h = x.head * p.group + (r - token * p.group);
      const float *from = reinterpret_cast<const float *>(p.query + (x.q.first + token) * p.q_pitch) + static_cast<int64_t>(h) * p.dim;
      for (int d = lane; d < p.dim; d += 32) {
        const float y = row < x.rows ? from[d] : 0.f;
        sm_q[row * kPitch + d] = mul < 0.f ? -y : y;
      }
    }
    __syncthreads();
    if (x.kv0 < x.kv1) fetch(p.k, sm_k, x.kv0);
    copies_commit();
    if (x.kv0 < x.kv1) fetch(p.v, sm_v, x.kv0);
    copies_commit();
    float acc[4][kCols][4], m[4], l[4];
    int32_t limit[4];  // (rows behind the tile's last are never written: nothing is masked for them)
#pragma unroll
    for (int a = 0; a < 4; ++a) {
      m[a] = -INFINITY, l[a] = 0.f;
      limit[a] = ty * 4 + a < x.rows ? row_limit(p, x.q, x.row0 + ty * 4 + a) : INT32_MAX;
#pragma unroll
      for (int c = 0; c < kCols; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[a][c][e] = 0.f;
    }
    const bool works = (warp * 8) < x.rows;  // warps without rows only load
    const int32_t least = min(min(limit[0], limit[1]), min(limit[2], limit[3]));
#pragma unroll 1
    for (int j = x.kv0; j < x.kv1; ++j) {
      const int32_t t0 = j * kWideTokens;
      const int32_t next_page = tid < kWideTokens ? look_up(j + 1) : -1;
      copies_wait<1>();
      __syncthreads();  // K of this tile is there
      float s[4][4];
#pragma unroll
      for (int a = 0; a < 4; ++a)
#pragma unroll
        for (int b = 0; b < 4; ++b) s[a][b] = 0.f;
      if (works) {
#pragma unroll 2
        for (int d = 0; d < p.dim; d += 4) {
          float4 q[4], k[4];
#pragma unroll
          for (int a = 0; a < 4; ++a) q[a] = *reinterpret_cast<const float4 *>(&sm_q[(ty * 4 + a) * kPitch + d]);
#pragma unroll
          for (int b = 0; b < 4; ++b) k[b] = *reinterpret_cast<const float4 *>(&sm_k[(tx + 16 * b) * kPitch + d]);
#pragma unroll
          for (int a = 0; a < 4; ++a)
#pragma unroll
            for (int b = 0; b < 4; ++b)
              s[a][b] = fmaf(q[a].w, k[b].w, fmaf(q[a].z, k[b].z, fmaf(q[a].y, k[b].y, fmaf(q[a].x, k[b].x, s[a][b]))));
        }
      }
      if (tid < kWideTokens) sm_page[((j + 1) & 1) * kWideTokens + tid] = next_page;
      __syncthreads();  // K is free, the next tile's pages are known
      if (j + 1 < x.kv1) fetch(p.k, sm_k, j + 1);
      copies_commit();
      if (works) {
        bool there[4];
#pragma unroll
        for (int b = 0; b < 4; ++b) there[b] = sm_page[(j & 1) * kWideTokens + tx + 16 * b] >= 0;
#pragma unroll
        for (int a = 0; a < 4; ++a) {
          float top = -INFINITY;
#pragma unroll
          for (int b = 0; b < 4; ++b)
            if (there[b] && t0 + tx + 16 * b < limit[a]) top = fmaxf(top, s[a][b]);
#pragma unroll
          for (int d = 8; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, d));
          const float mn = fmaxf(m[a], top), c = weight_of(m[a], mn, am);
          float sum = 0.f;
#pragma unroll
          for (int b = 0; b < 4; ++b) {
            float y = 0.f;
            if (there[b] && t0 + tx + 16 * b < limit[a])
              y = mn == -INFINITY ? (s[a][b] == s[a][b] ? 0.f : s[a][b]) : exp2f((s[a][b] - mn) * am);
            sum += y;
            sm_p[(ty * 4 + a) * kPitchP + tx + 16 * b] = y;
          }
          l[a] = l[a] * c + sum;  // of this lane's tokens
          m[a] = mn;
#pragma unroll
          for (int e = 0; e < kCols; ++e)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[a][e][i] *= c;
        }
      }
      copies_wait<1>();
      __syncthreads();  // V of this tile and the weights are there
      if (works) {
#pragma unroll 1
        for (int c0 = 0; c0 < kWideTokens; c0 += 4) {
          float wv[4][4];
#pragma unroll
          for (int a = 0; a < 4; ++a) {
            const float4 y = *reinterpret_cast<const float4 *>(&sm_p[(ty * 4 + a) * kPitchP + c0]);
            wv[a][0] = y.x, wv[a][1] = y.y, wv[a][2] = y.z, wv[a][3] = y.w;
          }
          const bool all = t0 + c0 + 3 < least;
#pragma unroll
          for (int t = 0; t < 4; ++t) {
#pragma unroll
            for (int c = 0; c < kCols; ++c) {
              const float4 v = *reinterpret_cast<const float4 *>(&sm_v[(c0 + t) * kPitch + c * 64 + tx * 4]);
#pragma unroll
              for (int a = 0; a < 4; ++a) {
                if (!all && t0 + c0 + t >= limit[a]) continue;  // left out, not weighted with zero
                acc[a][c][0] = fmaf(wv[a][t], v.x, acc[a][c][0]);
                acc[a][c][1] = fmaf(wv[a][t], v.y, acc[a][c][1]);
                acc[a][c][2] = fmaf(wv[a][t], v.z, acc[a][c][2]);
                acc[a][c][3] = fmaf(wv[a][t], v.w, acc[a][c][3]);
              }
            }
          }
        }
      }
      __syncthreads();  // V is free
      if (j + 1 < x.kv1) fetch(p.v, sm_v, j + 1);
      copies_commit();
    }
#pragma unroll
    for (int a = 0; a < 4; ++a) {
#pragma unroll
      for (int d = 8; d > 0; d >>= 1) l[a] += __shfl_xor_sync(0xFFFFFFFFu, l[a], d);
      const int row = ty * 4 + a;
      if (row >= x.rows) continue;
      const int32_t r = x.row0 + row, token = r / p.group, h = x.head * p.group + (r - token * p.group);
      float *out = reinterpret_cast<float *>(p.out + (x.q.first + token) * p.o_pitch) + static_cast<int64_t>(h) * p.dim;
      const int64_t part = x.slot < 0 ? 0 : static_cast<int64_t>(x.slot) * p.slot_rows + row;
#pragma unroll
      for (int c = 0; c < kCols; ++c) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int d = c * 64 + tx * 4 + i;
          if (d >= p.dim) continue;
          if (x.slot >= 0)
            p.part_o[part * p.dim + d] = acc[a][c][i];
          else
            out[d] = l[a] == 0.f ? 0.f : acc[a][c][i] / l[a];
        }
      }
      if (x.slot >= 0 && tx == 0) reinterpret_cast<float2 *>(p.part_ml)[part] = make_float2(m[a], l[a]);
    }
    left -= stop - w.off;
    if (left > 0) next_tile(p, w);
  }
}

// ------------------------------------------------------------------ host ---------------

constexpr int kMaxShares = 148;      // of the tensor-core kernel: one CTA per SM
constexpr int kMaxSimtShares = 296;  // of the kernels on the f32 units, where two CTAs share an SM
constexpr int kMinShare = 2;         // steps; a shorter share costs more in its partial result than it saves
constexpr int kMinSimtShare = 4;
constexpr int kTileCost = 2;  // steps that loading a tile's queries and writing its result are worth
constexpr int kSimtTileCost = 1;

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// The tensor-core kernel, the f32 kernel of large steps, the one for everything else.
enum Family { kTensor, kWide, kSimt };

struct Split {
  int32_t tile_rows, kv_tile, grid, slot_rows, min_share, tile_cost;
  bool cuts;  // whether tiles may be cut
  size_t prefix_bytes, ml_bytes, o_bytes;
  size_t total() const { return prefix_bytes + ml_bytes + o_bytes; }
};

// Scratch and shares of one kernel family.  Every share that begins or ends inside a tile has a
// slot for it; there are never more shares than steps / min_share.
Split split_of(Family family, int64_t seqs, int64_t rows, int64_t heads_q, int64_t heads_kv, int64_t dim, int64_t max_len) {
  Split s;
  const int64_t group = heads_q / heads_kv;
  const bool tensor = family == kTensor;
  s.tile_rows = tensor ? (dim > 128 ? kTile : 2 * kTile) : family == kWide ? kWideRows : kSimtRows;
  s.kv_tile = tensor ? kTile : family == kWide ? kWideTokens : simt_tokens(static_cast<int>(dim > 512 ? 1024 : 64));
  s.min_share = tensor ? kMinShare : kMinSimtShare;
  s.tile_cost = tensor ? kTileCost : kSimtTileCost;
  const int64_t most = tensor ? kMaxShares : family == kWide ? (dim > 64 ? kMaxShares : kMaxSimtShares) : (dim > 256 ? kMaxShares : kMaxSimtShares);
  const int64_t tiles = (seqs + rows * group / s.tile_rows) * heads_kv;
  const int64_t per_tile = std::max<int64_t>(1, (max_len + s.kv_tile - 1) / s.kv_tile) + s.tile_cost;
  int64_t steps;
  if (__builtin_mul_overflow(tiles, per_tile, &steps)) steps = INT64_MAX / 2;
  s.grid = static_cast<int32_t>(std::max<int64_t>(1, std::min<int64_t>(most, (steps + s.min_share - 1) / s.min_share)));
  s.slot_rows = static_cast<int32_t>(std::min<int64_t>(s.tile_rows, rows * group));
  s.prefix_bytes = (static_cast<size_t>(seqs + 1) * sizeof(int64_t) + 15) / 16 * 16;
  // (a cut that would leave a tile of at most two steps in two parts goes to its edge: see snap)
  s.cuts = s.grid > 1 && per_tile - s.tile_cost > 2;
  const size_t slots = s.cuts ? static_cast<size_t>(2) * s.grid * s.slot_rows : 0;
  s.ml_bytes = slots * 2 * sizeof(float);
  s.o_bytes = slots * dim * sizeof(float);
  return s;
}

// Token rows of heads x dim elements without gaps, further apart than that or not.
kvx_status_t check_rows(const kvx_tensor_desc_t *t, int64_t rows, int64_t heads, int64_t dim) {
  if (t->size < sizeof(kvx_tensor_desc_t)) return KVX_STATUS_INVALID_ARGUMENT;
  if (t->ndim != 3 || t->shape[0] != rows || t->shape[1] != heads || t->shape[2] != dim) return KVX_STATUS_INVALID_ARGUMENT;
  if ((dim > 1 && t->stride[2] != 1) || (heads > 1 && t->stride[1] != dim)) return KVX_STATUS_UNSUPPORTED;
  if (rows > 1 && t->stride[0] < heads * dim) return KVX_STATUS_UNSUPPORTED;
  return KVX_STATUS_OK;
}

// Launch with the programmatic-stream-serialization attribute (see pdl_prologue).
template <typename... Args>
void launch_pdl(void (*kernel)(Args...), dim3 grid, unsigned block, size_t smem, cudaStream_t st, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(block);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaLaunchKernelEx(&cfg, kernel, args...);
}

using EncodeTiled = decltype(&cuTensorMapEncodeTiled);
EncodeTiled encode_tiled() {
  static std::atomic<void *> cached{nullptr};
  void *f = cached.load(std::memory_order_acquire);
  if (f == nullptr) {
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &found) != cudaSuccess ||
        found != cudaDriverEntryPointSuccess) {
      cudaGetLastError();
      return nullptr;
    }
    cached.store(f, std::memory_order_release);
  }
  return reinterpret_cast<EncodeTiled>(f);
}

// Pages as a tensor that is loaded in boxes of `box` tokens of one head of one page, swizzled as the
// operands want them.  Whole boxes: (64 dims, 8 tokens, panels, groups of 8 tokens, pages), with the
// head folded into the panels (heads next to each other) or into the groups (heads behind each
// other's tokens), so that all panels come with one box.  Otherwise (dim, head and token in the
// order of their strides, page), one panel to a box; dims behind head_dim come as zeros.
bool make_map(CUtensorMap *map, const ChunkParams &p, const PageView &v, bool bf16, int unit_panels) {
  const EncodeTiled encode = encode_tiled();
  if (encode == nullptr) return false;
  const CUtensorMapDataType type = bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  const cuuint64_t heads = static_cast<cuuint64_t>(p.heads_kv), toks = static_cast<cuuint64_t>(p.block_size);
  const cuuint64_t pages = static_cast<cuuint64_t>(p.num_blocks);
  if (p.whole_boxes) {
    const cuuint64_t dims[5] = {64, 8, (heads - 1) * p.head_panels + p.dim / 64, (heads - 1) * p.head_groups + toks / 8, pages};
    const cuuint64_t strides[4] = {static_cast<cuuint64_t>(v.tok), 128, static_cast<cuuint64_t>(v.tok) * 8, static_cast<cuuint64_t>(v.blk)};
    const cuuint32_t box[5] = {64, 8, static_cast<cuuint32_t>(unit_panels), static_cast<cuuint32_t>(p.box / 8), 1};
    const cuuint32_t step[5] = {1, 1, 1, 1, 1};
    return encode(map, type, 5, v.base, dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
  }
  const cuuint64_t dims[4] = {static_cast<cuuint64_t>(p.dim), p.head_inner ? heads : toks, p.head_inner ? toks : heads, pages};
  const cuuint64_t strides[3] = {static_cast<cuuint64_t>(p.head_inner ? v.head : v.tok), static_cast<cuuint64_t>(p.head_inner ? v.tok : v.head),
                                 static_cast<cuuint64_t>(v.blk)};
  const cuuint32_t rows = static_cast<cuuint32_t>(p.box);
  const cuuint32_t box[4] = {64, p.head_inner ? 1 : rows, p.head_inner ? rows : 1, 1};
  const cuuint32_t step[4] = {1, 1, 1, 1};
  return encode(map, type, 4, v.base, dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// e4m3 pages: (dim, head and token in the order of their strides, page), rows of one entry's dims.
bool make_raw_map(CUtensorMap *map, const ChunkParams &p, const PageView &v, int unit_panels) {
  const EncodeTiled encode = encode_tiled();
  if (encode == nullptr) return false;
  const cuuint64_t heads = static_cast<cuuint64_t>(p.heads_kv), toks = static_cast<cuuint64_t>(p.block_size);
  const cuuint64_t dims[4] = {static_cast<cuuint64_t>(p.dim), p.head_inner ? heads : toks, p.head_inner ? toks : heads,
                              static_cast<cuuint64_t>(p.num_blocks)};
  const cuuint64_t strides[3] = {static_cast<cuuint64_t>(p.head_inner ? v.head : v.tok), static_cast<cuuint64_t>(p.head_inner ? v.tok : v.head),
                                 static_cast<cuuint64_t>(v.blk)};
  const cuuint32_t rows = static_cast<cuuint32_t>(p.box);
  const cuuint32_t box[4] = {static_cast<cuuint32_t>(unit_panels * 64), p.head_inner ? 1 : rows, p.head_inner ? rows : 1, 1};
  const cuuint32_t step[4] = {1, 1, 1, 1};
  return encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, v.base, dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// What a head adds to the coordinates of whole boxes; false when K or V does not fold that way.  A
// box must not reach behind its head (head_dim 192 in two boxes of 128): the next head's values are
// not zeros there, and zero queries times its infinities would be NaN.
bool fold_heads(ChunkParams *p, int unit_panels) {
  if (p->dim % (64 * unit_panels) != 0) return false;
  p->head_panels = p->head_groups = 0;
  if (p->heads_kv == 1) return true;
  const PageView &k = p->k, &v = p->v;
  if (p->head_inner) {  // heads are panels further on
    if (k.head != v.head || k.head % 128 != 0) return false;
    p->head_panels = static_cast<int32_t>(k.head / 128);
    return k.head / 128 * (p->heads_kv - 1) < INT32_MAX / 2;
  }
  if (k.head % (8 * k.tok) != 0 || v.head % (8 * v.tok) != 0 || k.head / k.tok != v.head / v.tok) return false;
  p->head_groups = static_cast<int32_t>(k.head / (8 * k.tok));
  return k.head / (8 * k.tok) * (p->heads_kv - 1) < INT32_MAX / 2;
}

// Query rows as a 3-d tensor (dim, head, token) loaded as the 128 rows of a stream.
bool make_query_map(CUtensorMap *map, const ChunkParams &p, bool bf16) {
  const EncodeTiled encode = encode_tiled();
  if (encode == nullptr) return false;
  const cuuint64_t dims[3] = {static_cast<cuuint64_t>(p.dim), static_cast<cuuint64_t>(p.heads_kv) * p.group, static_cast<cuuint64_t>(p.rows)};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(p.dim) * 2, static_cast<cuuint64_t>(p.q_pitch)};
  const cuuint32_t box[3] = {64, static_cast<cuuint32_t>(p.group), static_cast<cuuint32_t>(kTile / p.group)};
  const cuuint32_t step[3] = {1, 1, 1};
  return encode(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<char *>(p.query), dims, strides,
                box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

bool tma_strides(const PageView &v, int64_t elem) {
  const int64_t most = int64_t{1} << 40;
  return v.pack == 1 && v.dhi == elem && aligned16(v.base) && v.blk % 16 == 0 && v.tok % 16 == 0 && v.head % 16 == 0 && v.blk > 0 &&
         v.tok > 0 && v.head > 0 && v.blk < most && v.tok < most && v.head < most;
}

template <typename T, int kDp, Loads kLoads>
void launch_tensor(const ChunkParams &p, const CUtensorMap &k, const CUtensorMap &v, const CUtensorMap &q, cudaStream_t st) {
  const size_t smem = chunk_smem_bytes<kDp>();
  // (the attribute is per device and cheap to set, so it is set on every launch)
  cudaFuncSetAttribute(kvx_chunk_attention_kernel<T, kDp, kLoads>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
  launch_pdl(kvx_chunk_attention_kernel<T, kDp, kLoads>, dim3(static_cast<unsigned>(p.grid)), static_cast<unsigned>(threads_of(kLoads)), smem, st, p, k, v, q);
}
template <typename T, Loads kLoads>
void launch_tensor_dim(const ChunkParams &p, const CUtensorMap &k, const CUtensorMap &v, const CUtensorMap &q, cudaStream_t st) {
  if (p.dim <= 64)
    launch_tensor<T, 64, kLoads>(p, k, v, q, st);
  else if (p.dim <= 128)
    launch_tensor<T, 128, kLoads>(p, k, v, q, st);
  else
    launch_tensor<T, 256, kLoads>(p, k, v, q, st);
}
template <int kDb>
void launch_simt(const ChunkParams &p, cudaStream_t st) {
  const int pitch = ((p.dim + 3) & ~3) + 4, tokens = simt_tokens(kDb);
  const size_t smem = static_cast<size_t>((kSimtRows + tokens) * pitch + kSimtRows * (tokens + 4) + tokens) * sizeof(float);
  cudaFuncSetAttribute(kvx_chunk_attention_simt_kernel<kDb>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
  launch_pdl(kvx_chunk_attention_simt_kernel<kDb>, dim3(static_cast<unsigned>(p.grid)), kSimtThreads, smem, st, p);
}

template <int kDb>
void launch_wide(const ChunkParams &p, cudaStream_t st) {
  const size_t smem = wide_smem_bytes(kDb);
  cudaFuncSetAttribute(kvx_chunk_attention_f32_kernel<kDb>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
  launch_pdl(kvx_chunk_attention_f32_kernel<kDb>, dim3(static_cast<unsigned>(p.grid)), kSimtThreads, smem, st, p);
}

}  // namespace

extern "C" {

KVX_API size_t kvx_paged_attention_chunk_workspace_bytes(uint32_t seq_count, uint32_t num_rows, uint32_t num_q_heads,
                                                         uint32_t num_kv_heads, uint32_t head_dim, uint32_t max_seq_len) {
  if (seq_count == 0 || num_rows == 0 || num_q_heads == 0 || num_kv_heads == 0 || num_q_heads < num_kv_heads || head_dim == 0) return 0;
  size_t most = 0;
  for (const Family family : {kTensor, kWide, kSimt}) {
    if (family != kSimt && head_dim > 256) continue;
    most = std::max(most, split_of(family, seq_count, num_rows, num_q_heads, num_kv_heads, head_dim, max_seq_len).total());
  }
  return most;
}

KVX_API kvx_status_t kvx_launch_paged_attention_chunk(const kvx_cache_desc_t *cache, const kvx_chunk_attention_desc_t *attn,
                                                      const kvx_scale_desc_t *k_scale, const kvx_scale_desc_t *v_scale,
                                                      void *workspace, size_t workspace_bytes, void *stream) {
  if (cache == nullptr || attn == nullptr) return KVX_STATUS_INVALID_ARGUMENT;
  if (cache->size < sizeof(kvx_cache_desc_t) || attn->size < sizeof(kvx_chunk_attention_desc_t) ||
      attn->block_table.size < sizeof(kvx_block_table_t) || attn->seq_lens.size < sizeof(kvx_seq_lens_t))
    return KVX_STATUS_INVALID_ARGUMENT;
  const int64_t H = cache->num_kv_heads, D = cache->head_dim, Hq = attn->num_q_heads;
  if (H == 0 || D == 0 || Hq == 0 || Hq % H != 0 || cache->block_size == 0 || attn->max_seq_len == 0)
    return KVX_STATUS_INVALID_ARGUMENT;
  if (cache->k.dtype != cache->v.dtype || attn->causal > 1) return KVX_STATUS_INVALID_ARGUMENT;
  if (attn->block_table.format != KVX_BLOCK_TABLE_PACKED) return KVX_STATUS_UNSUPPORTED;
  const kvx_dtype_t io = attn->query.dtype, cd = cache->k.dtype;
  if ((io != KVX_DTYPE_F16 && io != KVX_DTYPE_BF16 && io != KVX_DTYPE_F32) || attn->out.dtype != io) return KVX_STATUS_UNSUPPORTED;
  ChunkParams p = {};
  if (cd == KVX_DTYPE_F8_E4M3) {
    if (!kvx_detail::resolve_scale(k_scale, nullptr, cache->num_kv_heads, &p.ks) ||
        !kvx_detail::resolve_scale(v_scale, nullptr, cache->num_kv_heads, &p.vs))
      return KVX_STATUS_UNSUPPORTED;
  } else if (cd != io) {
    return KVX_STATUS_UNSUPPORTED;
  }
  const int64_t S = attn->block_table.seq_count, R = attn->query.shape[0];
  if (attn->seq_lens.seq_count != S || R < 0) return KVX_STATUS_INVALID_ARGUMENT;
  kvx_status_t st = check_rows(&attn->query, R, Hq, D);
  if (st != KVX_STATUS_OK) return st;
  st = check_rows(&attn->out, R, Hq, D);
  if (st != KVX_STATUS_OK) return st;
  const bool s32 = attn->block_table.index_dtype == KVX_DTYPE_S32 && attn->seq_lens.dtype == KVX_DTYPE_S32;
  const bool s64 = attn->block_table.index_dtype == KVX_DTYPE_S64 && attn->seq_lens.dtype == KVX_DTYPE_S64;
  if (!s32 && !s64) return KVX_STATUS_INVALID_ARGUMENT;
  if (attn->query_indptr_dtype != KVX_DTYPE_S32 && attn->query_indptr_dtype != KVX_DTYPE_S64) return KVX_STATUS_INVALID_ARGUMENT;
  if (S == 0 || R == 0) return KVX_STATUS_OK;
  const int64_t elem = dtype_bytes(cd), io_elem = dtype_bytes(io);
  st = make_page_view(cache, &cache->k, elem, &p.k);
  if (st != KVX_STATUS_OK) return st;
  st = make_page_view(cache, &cache->v, elem, &p.v);
  if (st != KVX_STATUS_OK) return st;
  if (attn->query.data == nullptr || attn->out.data == nullptr || attn->query_indptr == nullptr ||
      attn->block_table.indices == nullptr || attn->seq_lens.lengths == nullptr || cache->k.data == nullptr ||
      cache->v.data == nullptr || attn->block_table.max_blocks_per_seq == 0 || attn->query.data == attn->out.data ||
      attn->block_table.max_blocks_per_seq > static_cast<uint32_t>(INT32_MAX) || cache->num_blocks > static_cast<uint32_t>(INT32_MAX) ||
      cache->block_size > static_cast<uint32_t>(INT32_MAX) || attn->max_seq_len > static_cast<uint32_t>(INT32_MAX) - 1024u ||
      S > INT32_MAX || D > INT32_MAX)
    return KVX_STATUS_INVALID_ARGUMENT;
  const int64_t group = Hq / H;
  if (R > (INT32_MAX - 1024) / group) return KVX_STATUS_UNSUPPORTED;  // group rows are counted in 32 bits

  const bool tensor = io != KVX_DTYPE_F32 && D <= 256;
  if (!tensor && D > 1024) return KVX_STATUS_UNSUPPORTED;
  auto f32_rows = [](const PageView &v) {  // rows that 16-byte copies can read
    return v.pack == 1 && v.dhi == 4 && aligned16(v.base) && v.blk % 16 == 0 && v.tok % 16 == 0 && v.head % 16 == 0;
  };
  const Family family = tensor                                                                        ? kTensor
                        : cd == KVX_DTYPE_F32 && D <= 256 && D % 4 == 0 && f32_rows(p.k) && f32_rows(p.v)
                            ? kWide
                            : kSimt;
  const Split sp = split_of(family, S, R, Hq, H, D, attn->max_seq_len);
  const size_t need = kvx_paged_attention_chunk_workspace_bytes(static_cast<uint32_t>(S), static_cast<uint32_t>(R), attn->num_q_heads,
                                                                cache->num_kv_heads, cache->head_dim, attn->max_seq_len);
  if (workspace == nullptr || workspace_bytes < need || !aligned16(workspace)) return KVX_STATUS_INVALID_ARGUMENT;

  p.table = attn->block_table.indices;
  p.lens = attn->seq_lens.lengths;
  p.indptr = attn->query_indptr;
  p.query = static_cast<const char *>(attn->query.data);
  p.out = static_cast<char *>(attn->out.data);
  p.q_pitch = (R > 1 ? attn->query.stride[0] : Hq * D) * io_elem;
  p.o_pitch = (R > 1 ? attn->out.stride[0] : Hq * D) * io_elem;
  p.prefix = static_cast<int64_t *>(workspace);
  p.part_ml = reinterpret_cast<float *>(static_cast<char *>(workspace) + sp.prefix_bytes);
  p.part_o = reinterpret_cast<float *>(static_cast<char *>(workspace) + sp.prefix_bytes + sp.ml_bytes);
  p.scale_log2 = attn->scale * 1.4426950408889634f;
  p.seq_count = static_cast<int32_t>(S);
  p.rows = static_cast<int32_t>(R);
  p.max_blocks = static_cast<int32_t>(attn->block_table.max_blocks_per_seq);
  p.max_seq_len = static_cast<int32_t>(attn->max_seq_len);
  p.num_blocks = static_cast<int32_t>(cache->num_blocks);
  p.block_size = static_cast<int32_t>(cache->block_size);
  p.bs_shift = (p.block_size & (p.block_size - 1)) == 0 ? __builtin_ctz(cache->block_size) : -1;
  p.heads_kv = static_cast<int32_t>(H);
  p.group = static_cast<int32_t>(group);
  p.dim = static_cast<int32_t>(D);
  p.causal = static_cast<int32_t>(attn->causal);
  p.table64 = s64 ? 1 : 0;
  p.indptr64 = attn->query_indptr_dtype == KVX_DTYPE_S64 ? 1 : 0;
  p.cache_code = static_cast<int32_t>(cd);
  p.io_code = static_cast<int32_t>(io);
  p.grid = sp.grid;
  p.slot_rows = sp.slot_rows;
  p.min_share = sp.min_share;
  p.tile_rows = sp.tile_rows;
  p.kv_tile = sp.kv_tile;
  p.tile_cost = sp.tile_cost;
  p.pair = tensor && D <= 128 ? 1 : 0;
  p.test_stall = kvx_b200_get_option("chunk_test_stall") != 0 ? 1 : 0;
  p.q_vec = D % 8 == 0 && p.q_pitch % 16 == 0 && p.o_pitch % 16 == 0 && aligned16(p.query) && aligned16(p.out) ? 1 : 0;
  const cudaStream_t cs = reinterpret_cast<cudaStream_t>(stream);

  p.plan_inside = family != kSimt && S <= kPlanInside ? 1 : 0;
  if (!p.plan_inside) launch_pdl(kvx_chunk_plan_kernel, dim3(1), static_cast<unsigned>(kPlanThreads), size_t{0}, cs, p);
  if (tensor) {
    p.box = 1;
    while (p.box < kTile && p.block_size % (2 * p.box) == 0) p.box *= 2;
    if (H == 1) {  // a stride nothing is multiplied by
      if (p.k.head <= 0 || p.k.head % 16 != 0) p.k.head = p.k.tok;
      if (p.v.head <= 0 || p.v.head % 16 != 0) p.v.head = p.v.tok;
    }
    CUtensorMap kmap = {}, vmap = {};
    const int unit_panels = D <= 64 ? 1 : 2;
    const bool bf16 = io == KVX_DTYPE_BF16;
    p.head_inner = p.k.head < p.k.tok ? 1 : 0;
    const bool strides = tma_strides(p.k, elem) && tma_strides(p.v, elem) && (p.k.head < p.k.tok) == (p.v.head < p.v.tok);
    bool tma = elem == 2 && p.box >= 8 && strides;
    p.whole_boxes = tma && fold_heads(&p, unit_panels) ? 1 : 0;
    if (p.whole_boxes && !(make_map(&kmap, p, p.k, bf16, unit_panels) && make_map(&vmap, p, p.v, bf16, unit_panels))) p.whole_boxes = 0;
    if (tma && !p.whole_boxes) tma = make_map(&kmap, p, p.k, bf16, unit_panels) && make_map(&vmap, p, p.v, bf16, unit_panels);
    const bool raw = elem == 1 && p.box >= 8 && strides && make_raw_map(&kmap, p, p.k, unit_panels) && make_raw_map(&vmap, p, p.v, unit_panels);
    p.group_stride = p.whole_boxes ? unit_panels * 1024 : 1024;
    p.panel_stride = p.whole_boxes ? 1024 : kPanelBytes;
    CUtensorMap qmap = {};
    p.q_tma = p.q_vec && (p.group & (p.group - 1)) == 0 && p.group <= kTile && p.q_pitch < (int64_t{1} << 40) &&
                      make_query_map(&qmap, p, io == KVX_DTYPE_BF16)
                  ? 1
                  : 0;
    auto rows_ok = [&](const PageView &v) {  // rows that 16-byte loads can read where TMA is not used
      return v.pack == 1 && v.dhi == elem && aligned16(v.base) && v.blk % 16 == 0 && v.tok % 16 == 0 && v.head % 16 == 0;
    };
    p.kv_vec = D * elem % 16 == 0 && rows_ok(p.k) && rows_ok(p.v) ? 1 : 0;
    auto launch = [&](auto type) {
      using T = decltype(type);
      if (tma)
        launch_tensor_dim<T, kTmaLoads>(p, kmap, vmap, qmap, cs);
      else if (raw)
        launch_tensor_dim<T, kRawLoads>(p, kmap, vmap, qmap, cs);
      else
        launch_tensor_dim<T, kCopyLoads>(p, kmap, vmap, qmap, cs);
    };
    if (bf16)
      launch(Bf16{});
    else
      launch(Fp16{});
  } else if (family == kWide) {
    if (D <= 64)
      launch_wide<64>(p, cs);
    else if (D <= 128)
      launch_wide<128>(p, cs);
    else
      launch_wide<256>(p, cs);
  } else if (D <= 64) {
    launch_simt<64>(p, cs);
  } else if (D <= 128) {
    launch_simt<128>(p, cs);
  } else if (D <= 256) {
    launch_simt<256>(p, cs);
  } else if (D <= 512) {
    launch_simt<512>(p, cs);
  } else {
    launch_simt<1024>(p, cs);
  }
  if (sp.cuts) {
    const unsigned y = static_cast<unsigned>(std::max(1, std::min(16, p.slot_rows / 16)));
    launch_pdl(kvx_chunk_merge_kernel, dim3(static_cast<unsigned>(p.grid - 1), y), static_cast<unsigned>(kMergeThreads), size_t{0}, cs, p);
  }
  return cudaGetLastError() == cudaSuccess ? KVX_STATUS_OK : KVX_STATUS_INTERNAL_ERROR;
}

KVX_API int kvx_attention_device_error(int reset) {
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, g_chunk_error, sizeof(v)) != cudaSuccess) {
    cudaGetLastError();
    return -1;
  }
  if (reset && v != 0) {
    const int zero = 0;
    if (cudaMemcpyToSymbol(g_chunk_error, &zero, sizeof(zero)) != cudaSuccess) cudaGetLastError();
  }
  return v != 0 ? 1 : 0;
}

}  // extern "C"
