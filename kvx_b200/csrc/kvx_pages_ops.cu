/*
 * Upkeep of the page pool (include/kvx_pages_ops.h): copy, fork, free, compact.  No reference
 * counterpart; page tensors are addressed by the reference's per-layout rule
 * (reference: kernels/kvx_paged_kv.cu:54-75).
 *
 * copy     HBM-bound byte mover.  A warp takes (a block of pairs, one K or V tensor of one layer, a
 *          span of the page) and streams the span with 16-byte loads, several in flight per lane.
 *          One launch moves up to kMaxTensors / 2 layers, so that a copy-on-write of a few pages
 *          is one launch and not one per layer.
 * plans    integer work on the tables; one CTA walks the reference counts (a prefix sum decides who
 *          gets which page, so the result does not depend on timing), a second kernel edits rows.
 */
#include "kvx_pages_ops.h"
#include "kvx_paged_kv.h"

#include "kvx_pages.h"

#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>

namespace {

using kvx_detail::dtype_bytes;
using kvx_detail::make_page_view;
using kvx_detail::PageView;

__device__ __forceinline__ int64_t read_index(const void *p, int64_t i, int wide) {
  return wide ? static_cast<const int64_t *>(p)[i] : static_cast<const int32_t *>(p)[i];
}
__device__ __forceinline__ void write_index(void *p, int64_t i, int64_t x, int wide) {
  if (wide)
    static_cast<int64_t *>(p)[i] = x;
  else
    static_cast<int32_t *>(p)[i] = static_cast<int32_t>(x);
}

__device__ __forceinline__ void pdl_prologue() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
}

template <typename... Args>
void launch_pdl(void (*kernel)(Args...), unsigned grid, unsigned block, cudaStream_t st, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(block);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaLaunchKernelEx(&cfg, kernel, args...);
}

kvx_status_t finished() { return cudaGetLastError() == cudaSuccess ? KVX_STATUS_OK : KVX_STATUS_INTERNAL_ERROR; }

// ------------------------------------------------------------------ copy ---------------

constexpr int kMaxTensors = 128;    // K and V of 64 layers per launch
constexpr int kCheckInline = 256;   // pairs up to which every warp checks its pairs itself
constexpr int kCopyThreads = 256;
constexpr int kUnroll = 8;
constexpr int kSpan = 32 * 16 * kUnroll;  // bytes a warp moves per iteration

struct CopyTensor {
  char *base;
  int64_t blk;  // bytes between pages
};
struct CopyParams {
  const void *src, *dst;
  const uint8_t *flags;  // one per pair, or NULL: check in place
  int32_t pairs, wide, num_blocks, tensors;
  int64_t page_bytes;        // of one page of one tensor (contiguous pages)
  int32_t spans;             // warps that share a page
  int32_t pair_block;        // pairs a warp looks at together
  // element walk of pages with gaps: extents and byte strides of the page's four inner axes
  int32_t elem, n[4];
  int64_t s[4];
  CopyTensor t[kMaxTensors];
};

__device__ __forceinline__ bool in_range(int64_t a, int64_t b, int32_t num_blocks) {
  return a >= 0 && a < num_blocks && b >= 0 && b < num_blocks && a != b;
}

// Whether pair i takes part; all lanes of a warp call it with the same i.
__device__ bool takes_part(const CopyParams &p, int64_t i) {
  const int64_t a = read_index(p.src, i, p.wide), b = read_index(p.dst, i, p.wide);
  if (!in_range(a, b, p.num_blocks)) return false;
  // four targets of a lane are in flight together
  constexpr int kAhead = 4;
  bool clash = false;
  for (int64_t j0 = threadIdx.x & 31; j0 < p.pairs && !clash; j0 += 32 * kAhead) {
    int64_t d[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int64_t j = j0 + 32 * k;
      d[k] = j < p.pairs ? read_index(p.dst, j, p.wide) : -1;
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int64_t j = j0 + 32 * k;
      if (d[k] == a || (d[k] == b && j > i)) clash = clash || in_range(read_index(p.src, j, p.wide), d[k], p.num_blocks);
    }
  }
  return __any_sync(0xFFFFFFFFu, clash) == 0;
}

__global__ void __launch_bounds__(kCopyThreads) kvx_copy_pages_check_kernel(const CopyParams p, uint8_t *flags) {
  pdl_prologue();
  const int64_t warps = static_cast<int64_t>(gridDim.x) * (kCopyThreads / 32);
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * (kCopyThreads / 32) + (threadIdx.x >> 5); i < p.pairs; i += warps) {
    const bool ok = takes_part(p, i);
    if ((threadIdx.x & 31) == 0) flags[i] = ok ? 1 : 0;
  }
}

// Contiguous pages in 16-byte pieces.
__global__ void __launch_bounds__(kCopyThreads) kvx_copy_pages_kernel(const CopyParams p) {
  pdl_prologue();
  const int lane = threadIdx.x & 31;
  const int64_t warps = static_cast<int64_t>(gridDim.x) * (kCopyThreads / 32);
  const int64_t blocks = (p.pairs + p.pair_block - 1) / p.pair_block;
  const int64_t units = blocks * p.tensors * p.spans;
  for (int64_t u = static_cast<int64_t>(blockIdx.x) * (kCopyThreads / 32) + (threadIdx.x >> 5); u < units; u += warps) {
    // spans of one page are neighbours, then the tensors, then the pairs
    const int span = static_cast<int>(u % p.spans);
    const int64_t r = u / p.spans;
    const int tensor = static_cast<int>(r % p.tensors);
    const int64_t i0 = r / p.tensors * p.pair_block;
    const int n = static_cast<int>(min(static_cast<int64_t>(p.pair_block), p.pairs - i0));
    unsigned todo;
    if (p.flags != nullptr) {
      todo = __ballot_sync(0xFFFFFFFFu, lane < n && p.flags[i0 + lane] != 0);
    } else {
      todo = 0;
      for (int k = 0; k < n; ++k)
        if (takes_part(p, i0 + k)) todo |= 1u << k;
    }
    char *const base = p.t[tensor].base;
    const int64_t blk = p.t[tensor].blk;
    while (todo != 0) {
      const int k = __ffs(todo) - 1;
      todo &= todo - 1;
      const char *from = base + read_index(p.src, i0 + k, p.wide) * blk;
      char *to = base + read_index(p.dst, i0 + k, p.wide) * blk;
      for (int64_t at = static_cast<int64_t>(span) * kSpan + lane * 16; at - lane * 16 < p.page_bytes;
           at += static_cast<int64_t>(p.spans) * kSpan) {
        uint4 x[kUnroll];
#pragma unroll
        for (int c = 0; c < kUnroll; ++c)
          if (at + c * 512 < p.page_bytes)
            asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                         : "=r"(x[c].x), "=r"(x[c].y), "=r"(x[c].z), "=r"(x[c].w)
                         : "l"(from + at + c * 512));
#pragma unroll
        for (int c = 0; c < kUnroll; ++c)
          if (at + c * 512 < p.page_bytes)
            asm volatile("st.global.cs.v4.u32 [%0], {%1,%2,%3,%4};" ::"l"(to + at + c * 512), "r"(x[c].x), "r"(x[c].y), "r"(x[c].z),
                         "r"(x[c].w)
                         : "memory");
      }
    }
  }
}

// Pages with gaps between their elements, misaligned ones: element by element.
__global__ void __launch_bounds__(kCopyThreads) kvx_copy_pages_element_kernel(const CopyParams p) {
  pdl_prologue();
  const int lane = threadIdx.x & 31;
  const int64_t warps = static_cast<int64_t>(gridDim.x) * (kCopyThreads / 32);
  const int64_t units = static_cast<int64_t>(p.pairs) * p.tensors;
  const int64_t count = static_cast<int64_t>(p.n[0]) * p.n[1] * p.n[2] * p.n[3];
  for (int64_t u = static_cast<int64_t>(blockIdx.x) * (kCopyThreads / 32) + (threadIdx.x >> 5); u < units; u += warps) {
    const int tensor = static_cast<int>(u % p.tensors);
    const int64_t i = u / p.tensors;
    if (p.flags != nullptr ? p.flags[i] == 0 : !takes_part(p, i)) continue;
    const char *from = p.t[tensor].base + read_index(p.src, i, p.wide) * p.t[tensor].blk;
    char *to = p.t[tensor].base + read_index(p.dst, i, p.wide) * p.t[tensor].blk;
    for (int64_t e = lane; e < count; e += 32) {
      int64_t r = e;
      const int64_t i3 = r % p.n[3];
      r /= p.n[3];
      const int64_t i2 = r % p.n[2];
      r /= p.n[2];
      const int64_t off = (r / p.n[1]) * p.s[0] + (r % p.n[1]) * p.s[1] + i2 * p.s[2] + i3 * p.s[3];
      if (p.elem == 1)
        to[off] = from[off];
      else if (p.elem == 2)
        *reinterpret_cast<uint16_t *>(to + off) = *reinterpret_cast<const uint16_t *>(from + off);
      else
        *reinterpret_cast<uint32_t *>(to + off) = *reinterpret_cast<const uint32_t *>(from + off);
    }
  }
}

// How a tensor's pages lie: inner extents and strides, and whether a page is one run of bytes.
struct PageShape {
  int64_t n[4], s[4];
  bool run;
  bool same(const PageShape &o) const {
    for (int i = 0; i < 4; ++i)
      if (n[i] != o.n[i] || s[i] != o.s[i]) return false;
    return run == o.run;
  }
};

kvx_status_t shape_of(const kvx_cache_desc_t *c, const kvx_tensor_desc_t *t, int64_t elem, PageView *v, PageShape *out) {
  const kvx_status_t st = make_page_view(c, t, elem, v);
  if (st != KVX_STATUS_OK) return st;
  out->n[0] = c->num_kv_heads, out->s[0] = v->head;
  out->n[1] = c->block_size, out->s[1] = v->tok;
  out->n[2] = c->head_dim / v->pack, out->s[2] = v->dhi;
  out->n[3] = v->pack, out->s[3] = v->pack > 1 ? v->dlo : elem;
  if (v->pack == 1) out->n[3] = 1;
  // one run: sorted by stride, every axis steps over exactly what lies inside it
  int order[4] = {0, 1, 2, 3};
  std::sort(order, order + 4, [&](int a, int b) { return out->s[a] != out->s[b] ? out->s[a] < out->s[b] : out->n[a] < out->n[b]; });
  int64_t run = elem;
  out->run = true;
  for (int k : order) {
    if (out->n[k] == 1) continue;
    if (out->s[k] != run) out->run = false;
    run *= out->n[k];
  }
  return KVX_STATUS_OK;
}

}  // namespace

extern "C" {

KVX_API size_t kvx_copy_pages_workspace_bytes(uint32_t pair_count) {
  return pair_count > static_cast<uint32_t>(kCheckInline) ? (static_cast<size_t>(pair_count) + 15) / 16 * 16 : 0;
}

KVX_API kvx_status_t kvx_launch_copy_pages(const kvx_cache_desc_t *caches, uint32_t cache_count, const void *src, const void *dst,
                                           kvx_dtype_t index_dtype, uint32_t pair_count, void *workspace, size_t workspace_bytes,
                                           void *stream) {
  if (caches == nullptr && cache_count > 0) return KVX_STATUS_INVALID_ARGUMENT;
  if (index_dtype != KVX_DTYPE_S32 && index_dtype != KVX_DTYPE_S64) return KVX_STATUS_INVALID_ARGUMENT;
  // all checks ahead of the first launch
  for (uint32_t i = 0; i < cache_count; ++i) {
    const kvx_cache_desc_t *c = &caches[i];
    if (c->size < sizeof(kvx_cache_desc_t) || c->k.dtype != c->v.dtype || c->num_blocks != caches[0].num_blocks ||
        c->num_blocks > static_cast<uint32_t>(INT32_MAX) || c->block_size == 0 || c->num_kv_heads == 0 || c->head_dim == 0 ||
        c->block_size > static_cast<uint32_t>(INT32_MAX) || c->num_kv_heads > static_cast<uint32_t>(INT32_MAX) ||
        c->head_dim > static_cast<uint32_t>(INT32_MAX))
      return KVX_STATUS_INVALID_ARGUMENT;
    const int64_t elem = c->k.dtype == KVX_DTYPE_F8_E5M2 || c->k.dtype == KVX_DTYPE_U8 ? 1 : dtype_bytes(c->k.dtype);
    if (elem == 0) return KVX_STATUS_UNSUPPORTED;
    PageView v;
    PageShape s;
    kvx_status_t st = shape_of(c, &c->k, elem, &v, &s);
    if (st != KVX_STATUS_OK) return st;
    st = shape_of(c, &c->v, elem, &v, &s);
    if (st != KVX_STATUS_OK) return st;
    if (pair_count > 0 && c->num_blocks > 0 && (c->k.data == nullptr || c->v.data == nullptr)) return KVX_STATUS_INVALID_ARGUMENT;
  }
  if (pair_count == 0 || cache_count == 0 || caches[0].num_blocks == 0) return KVX_STATUS_OK;
  if (src == nullptr || dst == nullptr || pair_count > static_cast<uint32_t>(INT32_MAX)) return KVX_STATUS_INVALID_ARGUMENT;
  const size_t need = kvx_copy_pages_workspace_bytes(pair_count);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need)) return KVX_STATUS_INVALID_ARGUMENT;

  const cudaStream_t cs = reinterpret_cast<cudaStream_t>(stream);
  CopyParams p = {};
  p.src = src, p.dst = dst;
  p.pairs = static_cast<int32_t>(pair_count);
  p.wide = index_dtype == KVX_DTYPE_S64 ? 1 : 0;
  p.num_blocks = static_cast<int32_t>(caches[0].num_blocks);
  if (need > 0) {
    uint8_t *flags = static_cast<uint8_t *>(workspace);
    const unsigned grid = static_cast<unsigned>(std::min<int64_t>(148 * 8, (pair_count + 7) / 8));
    launch_pdl(kvx_copy_pages_check_kernel, grid, static_cast<unsigned>(kCopyThreads), cs, p, flags);
    p.flags = flags;
  }
  // tensors whose pages lie alike go into one launch; K and V of a layer usually do
  PageShape shape = {};
  int64_t elem = 0;
  bool vec = false;
  auto flush = [&]() {
    if (p.tensors == 0) return;
    p.elem = static_cast<int32_t>(elem);
    for (int i = 0; i < 4; ++i) p.n[i] = static_cast<int32_t>(shape.n[i]), p.s[i] = shape.s[i];
    p.page_bytes = shape.n[0] * shape.n[1] * shape.n[2] * shape.n[3] * elem;
    if (vec) {
      // as many warps per page as it has spans; long lists (a compaction's list is mostly its unused
      // tail) are looked at up to 32 pairs at a time, as long as there are four units for every
      // warp (460 moves of 32 KB in 16 tensors: 128 us with 32 pairs, where a quarter of the warps
      // had work)
      const int64_t warps = 148 * 64;
      const int64_t most = (p.page_bytes + kSpan - 1) / kSpan;
      p.spans = static_cast<int32_t>(std::min<int64_t>(most, 1024));
      p.pair_block = 1;
      while (p.flags != nullptr && p.pair_block < 32 &&
             static_cast<int64_t>(p.pairs) / (2 * p.pair_block) * p.tensors * p.spans >= 4 * warps)
        p.pair_block *= 2;
      const int64_t units = (static_cast<int64_t>(p.pairs) + p.pair_block - 1) / p.pair_block * p.tensors * p.spans;
      const unsigned grid = static_cast<unsigned>(std::min<int64_t>((units + 7) / 8, warps / 8));
      launch_pdl(kvx_copy_pages_kernel, grid, static_cast<unsigned>(kCopyThreads), cs, p);
    } else {
      const int64_t units = static_cast<int64_t>(p.pairs) * p.tensors;
      const unsigned grid = static_cast<unsigned>(std::min<int64_t>((units + 7) / 8, 148 * 8));
      launch_pdl(kvx_copy_pages_element_kernel, grid, static_cast<unsigned>(kCopyThreads), cs, p);
    }
    p.tensors = 0;
  };
  for (uint32_t i = 0; i < cache_count; ++i) {
    for (int kv = 0; kv < 2; ++kv) {
      const kvx_cache_desc_t *c = &caches[i];
      const kvx_tensor_desc_t *t = kv == 0 ? &c->k : &c->v;
      const int64_t e = t->dtype == KVX_DTYPE_F8_E5M2 || t->dtype == KVX_DTYPE_U8 ? 1 : dtype_bytes(t->dtype);
      PageView v;
      PageShape s;
      shape_of(c, t, e, &v, &s);
      const bool sv = s.run && reinterpret_cast<uintptr_t>(v.base) % 16 == 0 && v.blk % 16 == 0 &&
                      s.n[0] * s.n[1] * s.n[2] * s.n[3] * e % 16 == 0;
      if (p.tensors > 0 && (p.tensors == kMaxTensors || sv != vec || e != elem || !s.same(shape))) flush();
      shape = s, elem = e, vec = sv;
      p.t[p.tensors++] = CopyTensor{v.base, v.blk};
    }
  }
  flush();
  return finished();
}

}  // extern "C"

// ------------------------------------------------------------------ free, fork, compact --

namespace {

struct TableParams {
  void *table, *lens;
  int32_t *refs;
  int32_t rows, max_blocks, num_blocks, block_size, wide;
};

constexpr int kRowThreads = 128;

// One CTA per named row.
__global__ void __launch_bounds__(kRowThreads) kvx_free_rows_kernel(const TableParams p, const void *rows) {
  pdl_prologue();
  const int64_t i = blockIdx.x;
  const int64_t row = read_index(rows, i, p.wide);
  if (row < 0 || row >= p.rows) return;
  bool seen = false;  // a row that is named twice is freed once
  for (int64_t j = threadIdx.x; j < i; j += kRowThreads) seen |= read_index(rows, j, p.wide) == row;
  if (__syncthreads_or(seen)) return;
  for (int64_t b = threadIdx.x; b < p.max_blocks; b += kRowThreads) {
    const int64_t at = row * p.max_blocks + b;
    const int64_t page = read_index(p.table, at, p.wide);
    if (page >= 0 && page < p.num_blocks) {
      // one reference back, never below zero: what was not there is put back
      if (atomicSub(&p.refs[page], 1) <= 0) atomicAdd(&p.refs[page], 1);
    }
    write_index(p.table, at, -1, p.wide);
  }
  if (threadIdx.x == 0) write_index(p.lens, row, 0, p.wide);
}

constexpr int kPlanThreads = 1024;

// Exclusive prefix sum over the CTA; *total = the sum.
__device__ int32_t cta_scan(int32_t x, int32_t *total) {
  __shared__ int32_t s[kPlanThreads / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int32_t incl = x;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int32_t y = __shfl_up_sync(0xFFFFFFFFu, incl, d);
    if (lane >= d) incl += y;
  }
  __syncthreads();  // the previous scan's sums were read
  if (lane == 31) s[warp] = incl;
  __syncthreads();
  int32_t w = s[lane];  // kPlanThreads / 32 = 32 sums: every warp adds them up by shuffles
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int32_t y = __shfl_up_sync(0xFFFFFFFFu, w, d);
    if (lane >= d) w += y;
  }
  *total = __shfl_sync(0xFFFFFFFFu, w, 31);
  const int32_t before = __shfl_sync(0xFFFFFFFFu, w, warp == 0 ? 0 : warp - 1);
  return incl - x + (warp == 0 ? 0 : before);
}

// Which pairs can be forked, and the new page of each that needs one.  copy_dst holds -3 - rank for
// those in between the two passes.
__global__ void __launch_bounds__(kPlanThreads)
    kvx_fork_plan_kernel(const TableParams p, const void *parents, const void *children, int32_t n, void *copy_src, void *copy_dst,
                         int32_t *spare) {
  pdl_prologue();
  int32_t needed = 0;
  for (int32_t i0 = 0; i0 < n; i0 += kPlanThreads) {
    const int32_t i = i0 + threadIdx.x;
    int64_t src = -2, dst = -2;
    bool need = false;
    if (i < n) {
      const int64_t a = read_index(parents, i, p.wide), c = read_index(children, i, p.wide);
      bool ok = a >= 0 && a < p.rows && c >= 0 && c < p.rows && a != c;
      for (int32_t j = 0; j < n && ok; ++j) {
        const int64_t other = read_index(children, j, p.wide);
        if ((other == c && j < i) || other == a) ok = false;
      }
      if (ok) {
        src = dst = -1;
        const int64_t len = max(static_cast<int64_t>(0), read_index(p.lens, a, p.wide));
        const int64_t full = len / p.block_size;
        if (len % p.block_size != 0 && full < p.max_blocks) {
          const int64_t page = read_index(p.table, a * p.max_blocks + full, p.wide);
          if (page >= 0 && page < p.num_blocks) src = page, need = true;
        }
      }
    }
    int32_t total;
    const int32_t rank = needed + cta_scan(need ? 1 : 0, &total);
    needed += total;
    if (i < n) {
      write_index(copy_src, i, src, p.wide);
      write_index(copy_dst, i, need ? -3 - rank : dst, p.wide);
    }
  }
  // the lowest free pages, as many as are needed
  int32_t found = 0;
  for (int32_t b0 = 0; b0 < p.num_blocks && found < needed; b0 += kPlanThreads) {
    const int32_t b = b0 + threadIdx.x;
    const bool free_page = b < p.num_blocks && p.refs[b] == 0;
    int32_t total;
    const int32_t rank = found + cta_scan(free_page ? 1 : 0, &total);
    if (free_page && rank < needed) spare[rank] = b;
    found += total;
  }
  __syncthreads();
  for (int32_t i = threadIdx.x; i < n; i += kPlanThreads) {
    const int64_t code = read_index(copy_dst, i, p.wide);
    if (code > -3) continue;
    const int64_t rank = -3 - code;
    if (rank < found) {
      write_index(copy_dst, i, spare[rank], p.wide);
    } else {
      write_index(copy_src, i, -2, p.wide);
      write_index(copy_dst, i, -2, p.wide);
    }
  }
}

// One CTA per pair writes the child's row.
__global__ void __launch_bounds__(kRowThreads)
    kvx_fork_rows_kernel(const TableParams p, const void *parents, const void *children, const void *copy_dst) {
  pdl_prologue();
  const int64_t i = blockIdx.x;
  const int64_t fresh = read_index(copy_dst, i, p.wide);
  if (fresh == -2) return;
  const int64_t a = read_index(parents, i, p.wide), c = read_index(children, i, p.wide);
  const int64_t len = max(static_cast<int64_t>(0), read_index(p.lens, a, p.wide));
  const int64_t full = len / p.block_size;
  for (int64_t b = threadIdx.x; b < p.max_blocks; b += kRowThreads) {
    int64_t page = -1;
    if (b < full) {
      page = read_index(p.table, a * p.max_blocks + b, p.wide);
      if (page >= 0 && page < p.num_blocks) atomicAdd(&p.refs[page], 1);
    } else if (b == full && fresh >= 0) {
      page = fresh;
      atomicAdd(&p.refs[page], 1);
    }
    write_index(p.table, c * p.max_blocks + b, page, p.wide);
  }
  if (threadIdx.x == 0) write_index(p.lens, c, len, p.wide);
}

// Moves and their lists; references follow.
__global__ void __launch_bounds__(kPlanThreads)
    kvx_compact_plan_kernel(const TableParams p, void *copy_src, void *copy_dst, int32_t capacity) {
  pdl_prologue();
  constexpr int kPer = 4;
  int32_t mine = 0;
  for (int32_t b = threadIdx.x; b < p.num_blocks; b += kPlanThreads) mine += p.refs[b] > 0;
  int32_t live;
  cta_scan(mine, &live);
  int32_t movers = 0, holes = 0;
  for (int32_t b0 = 0; b0 < p.num_blocks; b0 += kPlanThreads * kPer) {
    // a thread looks at neighbouring pages; live ones behind the line move, free ones before it fill
    int32_t take[kPer], m = 0, h = 0;
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      const int32_t b = b0 + threadIdx.x * kPer + k;
      take[k] = 0;
      if (b < p.num_blocks) {
        const bool used = p.refs[b] > 0;
        if (used && b >= live) take[k] = 1, ++m;
        if (!used && b < live) take[k] = 2, ++h;
      }
    }
    int32_t total;
    const int32_t both = cta_scan(m | h << 16, &total);  // at most 4 096 of either per round
    int32_t mr = movers + (both & 0xFFFF), hr = holes + (both >> 16);
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      const int32_t b = b0 + threadIdx.x * kPer + k;
      if (take[k] == 1) write_index(copy_src, mr++, b, p.wide);
      if (take[k] == 2) write_index(copy_dst, hr++, b, p.wide);
    }
    movers += total & 0xFFFF, holes += total >> 16;
  }
  for (int32_t i = movers + threadIdx.x; i < capacity; i += kPlanThreads) {
    write_index(copy_src, i, -1, p.wide);
    write_index(copy_dst, i, -1, p.wide);
  }
  __syncthreads();
  for (int32_t i = threadIdx.x; i < movers; i += kPlanThreads) {
    const int64_t from = read_index(copy_src, i, p.wide), to = read_index(copy_dst, i, p.wide);
    p.refs[to] = p.refs[from];
    p.refs[from] = 0;
  }
}

// Table entries that name a moved page: found by bisection in the ascending list of moved pages.
__global__ void __launch_bounds__(256) kvx_compact_rows_kernel(const TableParams p, const void *copy_src, const void *copy_dst, int32_t capacity) {
  pdl_prologue();
  const int64_t all = static_cast<int64_t>(p.rows) * p.max_blocks;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < all; i += static_cast<int64_t>(gridDim.x) * 256) {
    const int64_t page = read_index(p.table, i, p.wide);
    if (page < 0 || page >= p.num_blocks) continue;
    int32_t lo = 0, hi = capacity;  // the first entry that is not below `page` (-1 stands for the end)
    while (lo < hi) {
      const int32_t mid = (lo + hi) >> 1;
      const int64_t x = read_index(copy_src, mid, p.wide);
      if (x >= 0 && x < page)
        lo = mid + 1;
      else
        hi = mid;
    }
    if (lo < capacity && read_index(copy_src, lo, p.wide) == page) write_index(p.table, i, read_index(copy_dst, lo, p.wide), p.wide);
  }
}

kvx_status_t check_table(const kvx_block_table_t *t, const kvx_seq_lens_t *l, const int32_t *refs, uint32_t num_blocks, TableParams *p) {
  if (t == nullptr || t->size < sizeof(kvx_block_table_t)) return KVX_STATUS_INVALID_ARGUMENT;
  if (t->format != KVX_BLOCK_TABLE_PACKED) return KVX_STATUS_UNSUPPORTED;
  if (t->index_dtype != KVX_DTYPE_S32 && t->index_dtype != KVX_DTYPE_S64) return KVX_STATUS_INVALID_ARGUMENT;
  if (l != nullptr && (l->size < sizeof(kvx_seq_lens_t) || l->dtype != t->index_dtype || l->seq_count != t->seq_count))
    return KVX_STATUS_INVALID_ARGUMENT;
  if (num_blocks > static_cast<uint32_t>(INT32_MAX) || t->seq_count > static_cast<uint32_t>(INT32_MAX) ||
      t->max_blocks_per_seq > static_cast<uint32_t>(INT32_MAX))
    return KVX_STATUS_INVALID_ARGUMENT;
  const int64_t entries = static_cast<int64_t>(t->seq_count) * t->max_blocks_per_seq;
  if ((entries > 0 && t->indices == nullptr) || (num_blocks > 0 && refs == nullptr)) return KVX_STATUS_INVALID_ARGUMENT;
  if (l != nullptr && t->seq_count > 0 && l->lengths == nullptr) return KVX_STATUS_INVALID_ARGUMENT;
  p->table = const_cast<void *>(t->indices);
  p->lens = l != nullptr ? const_cast<void *>(l->lengths) : nullptr;
  p->refs = const_cast<int32_t *>(refs);
  p->rows = static_cast<int32_t>(t->seq_count);
  p->max_blocks = static_cast<int32_t>(t->max_blocks_per_seq);
  p->num_blocks = static_cast<int32_t>(num_blocks);
  p->wide = t->index_dtype == KVX_DTYPE_S64 ? 1 : 0;
  return KVX_STATUS_OK;
}

}  // namespace

extern "C" {

KVX_API kvx_status_t kvx_launch_free_sequences(const kvx_block_table_t *table, const kvx_seq_lens_t *seq_lens, int32_t *page_refs,
                                               uint32_t num_blocks, const void *rows, uint32_t row_count, void *stream) {
  if (seq_lens == nullptr) return KVX_STATUS_INVALID_ARGUMENT;
  TableParams p = {};
  const kvx_status_t st = check_table(table, seq_lens, page_refs, num_blocks, &p);
  if (st != KVX_STATUS_OK) return st;
  if (row_count == 0 || p.rows == 0) return KVX_STATUS_OK;
  if (rows == nullptr || row_count > static_cast<uint32_t>(INT32_MAX)) return KVX_STATUS_INVALID_ARGUMENT;
  launch_pdl(kvx_free_rows_kernel, row_count, static_cast<unsigned>(kRowThreads), reinterpret_cast<cudaStream_t>(stream), p, rows);
  return finished();
}

KVX_API size_t kvx_fork_workspace_bytes(uint32_t pair_count) { return (static_cast<size_t>(pair_count) * 4 + 15) / 16 * 16; }

KVX_API kvx_status_t kvx_launch_fork_sequences(const kvx_block_table_t *table, const kvx_seq_lens_t *seq_lens, int32_t *page_refs,
                                               uint32_t num_blocks, uint32_t block_size, const void *parents, const void *children,
                                               uint32_t pair_count, void *copy_src, void *copy_dst, void *workspace,
                                               size_t workspace_bytes, void *stream) {
  if (seq_lens == nullptr || block_size == 0 || block_size > static_cast<uint32_t>(INT32_MAX)) return KVX_STATUS_INVALID_ARGUMENT;
  TableParams p = {};
  const kvx_status_t st = check_table(table, seq_lens, page_refs, num_blocks, &p);
  if (st != KVX_STATUS_OK) return st;
  p.block_size = static_cast<int32_t>(block_size);
  if (pair_count == 0) return KVX_STATUS_OK;
  if (parents == nullptr || children == nullptr || copy_src == nullptr || copy_dst == nullptr || workspace == nullptr ||
      workspace_bytes < kvx_fork_workspace_bytes(pair_count) || reinterpret_cast<uintptr_t>(workspace) % 4 != 0 ||
      pair_count > static_cast<uint32_t>(INT32_MAX) - 4u)
    return KVX_STATUS_INVALID_ARGUMENT;
  const cudaStream_t cs = reinterpret_cast<cudaStream_t>(stream);
  launch_pdl(kvx_fork_plan_kernel, 1u, static_cast<unsigned>(kPlanThreads), cs, p, parents, children, static_cast<int32_t>(pair_count),
             copy_src, copy_dst, static_cast<int32_t *>(workspace));
  launch_pdl(kvx_fork_rows_kernel, pair_count, static_cast<unsigned>(kRowThreads), cs, p, parents, children,
             static_cast<const void *>(copy_dst));
  return finished();
}

KVX_API kvx_status_t kvx_launch_compact_pages(const kvx_block_table_t *table, int32_t *page_refs, uint32_t num_blocks, void *copy_src,
                                              void *copy_dst, void *stream) {
  TableParams p = {};
  const kvx_status_t st = check_table(table, nullptr, page_refs, num_blocks, &p);
  if (st != KVX_STATUS_OK) return st;
  if (copy_src == nullptr || copy_dst == nullptr) return KVX_STATUS_INVALID_ARGUMENT;
  const int32_t capacity = std::max(1, p.num_blocks / 2);
  const cudaStream_t cs = reinterpret_cast<cudaStream_t>(stream);
  launch_pdl(kvx_compact_plan_kernel, 1u, static_cast<unsigned>(kPlanThreads), cs, p, copy_src, copy_dst, capacity);
  const int64_t entries = static_cast<int64_t>(p.rows) * p.max_blocks;
  if (entries > 0) {
    const unsigned grid = static_cast<unsigned>(std::min<int64_t>((entries + 255) / 256, 148 * 8));
    launch_pdl(kvx_compact_rows_kernel, grid, 256u, cs, p, static_cast<const void *>(copy_src), static_cast<const void *>(copy_dst),
               capacity);
  }
  return finished();
}

}  // extern "C"
