/*
 * Rotary positions (include/kvx_rotary.h), alone and fused with the cache write.  No reference
 * counterpart; slots and pages are addressed as the reference's write does it
 * (reference: kernels/kvx_paged_kv.cu:93-160, :54-75).
 *
 * HBM-bound: every element is read and written once, about 3 flop each.  The angles are not read
 * from a table: a CTA takes a few tokens, computes their cosines and sines once (f64 reduction,
 * f32 functions) into shared memory, and all heads of Q and K use them.
 *
 *   vector tier   16-byte vectors; a thread turns a whole vector (interleaved) or the two vectors
 *                 that pair up (half layout), V vectors pass through to the cache.
 *   element tier  odd rotary_dim / head_dim, misaligned rows, HND_PACKED pages: one pair per thread.
 */
#include "kvx_rotary.h"
#include "kvx_paged_kv.h"

#include "kvx_pages.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>

namespace {

using kvx_detail::dtype_bytes;
using kvx_detail::make_page_view;
using kvx_detail::PageView;
using kvx_detail::ScaleView;

struct RotaryParams {
  const char *q, *k, *v;  // sources; NULL = absent
  char *q_out, *k_out;    // k_out NULL = keys and values go to pages
  int64_t q_pitch, k_pitch, v_pitch, qo_pitch, ko_pitch;  // bytes between token rows
  const void *positions, *slots;
  const double *inv_freq;
  PageView kc, vc;
  ScaleView ks, vs;
  float factor;
  int32_t tokens, q_heads, k_heads, dim, half;  // half = rotary_dim / 2
  int32_t pos64, slot64, inverse, interleaved;
  int32_t num_blocks, block_size, fp8;
  int32_t q_in_place, k_in_place;  // what is not turned need not be copied
  int32_t tile;                    // tokens per CTA
  // vector tier: units of a head and V vectors of one, with their shifts (-1: no power of two)
  int32_t units, units_shift, v_units, v_shift;
};

__device__ __forceinline__ int64_t read_index(const void *p, int64_t i, int wide) {
  return wide ? static_cast<const int64_t *>(p)[i] : static_cast<const int32_t *>(p)[i];
}

struct Bf16 {
  using Bits = uint16_t;
  static constexpr int kPerVec = 8;
  static __device__ __forceinline__ float get(uint16_t b) { return __uint_as_float(static_cast<uint32_t>(b) << 16); }
  static __device__ __forceinline__ uint16_t put(float x) { return __bfloat16_as_ushort(__float2bfloat16_rn(x)); }
  static __device__ __forceinline__ void unpack(const uint4 &x, float *f) {
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) f[2 * i] = __uint_as_float(w[i] << 16), f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
  }
  static __device__ __forceinline__ uint4 pack(const float *f) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 r = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t *>(&r);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};
struct Fp16 {
  using Bits = uint16_t;
  static constexpr int kPerVec = 8;
  static __device__ __forceinline__ float get(uint16_t b) { return __half2float(__ushort_as_half(b)); }
  static __device__ __forceinline__ uint16_t put(float x) { return __half_as_ushort(__float2half_rn(x)); }
  static __device__ __forceinline__ void unpack(const uint4 &x, float *f) {
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 t = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
      f[2 * i] = t.x, f[2 * i + 1] = t.y;
    }
  }
  static __device__ __forceinline__ uint4 pack(const float *f) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __half2 r = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t *>(&r);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};
struct Fp32 {
  using Bits = uint32_t;
  static constexpr int kPerVec = 4;
  static __device__ __forceinline__ float get(uint32_t b) { return __uint_as_float(b); }
  static __device__ __forceinline__ uint32_t put(float x) { return __float_as_uint(x); }
  static __device__ __forceinline__ void unpack(const uint4 &x, float *f) {
    f[0] = __uint_as_float(x.x), f[1] = __uint_as_float(x.y), f[2] = __uint_as_float(x.z), f[3] = __uint_as_float(x.w);
  }
  static __device__ __forceinline__ uint4 pack(const float *f) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  }
};

// Quantisation of the cache write: one IEEE division, one rounding to E4M3 (NaN -> 0x7F).
__device__ __forceinline__ uint32_t quant2(float lo, float hi, float scale) {
  lo = __fdiv_rn(lo, scale), hi = __fdiv_rn(hi, scale);
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  uint32_t q = r;
  if (lo != lo) q = (q & 0xFF00u) | 0x7Fu;
  if (hi != hi) q = (q & 0x00FFu) | 0x7F00u;
  return q;
}

__device__ __forceinline__ uint4 load_stream(const void *p) {
  uint4 r;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(p));
  return r;
}
__device__ __forceinline__ void store_stream(void *p, const uint4 &r) {
  asm volatile("st.global.cs.v4.u32 [%0], {%1,%2,%3,%4};" ::"l"(p), "r"(r.x), "r"(r.y), "r"(r.z), "r"(r.w) : "memory");
}

// Cosine and sine (times factor) of pos * inv_freq.  The turns are reduced in f64: what is left,
// at most half a turn, loses 2^-25 of a turn when it becomes an f32.
__device__ __forceinline__ float2 turn(const RotaryParams &p, int64_t pos, int i) {
  const double turns = static_cast<double>(pos) * (p.inv_freq[i] * 0.15915494309189535);  // 1 / (2 pi)
  const double part = turns - rint(turns);
  float s, c;
  sincospif(static_cast<float>(2.0 * part), &s, &c);
  return make_float2(c * p.factor, (p.inverse ? -s : s) * p.factor);
}

// The turned pair, with the roundings spelled out: both tiers give the same bits.
__device__ __forceinline__ void turn_pair(float &y, float &z, float c, float s) {
  const float a = __fmaf_rn(y, c, -__fmul_rn(z, s)), b = __fmaf_rn(z, c, __fmul_rn(y, s));
  y = a, z = b;
}

struct SlotAt {
  int64_t block, off;  // block < 0: skipped
};
__device__ __forceinline__ SlotAt slot_at(const RotaryParams &p, int64_t t) {
  const int64_t slot = read_index(p.slots, t, p.slot64);
  SlotAt a{-1, 0};
  if (slot < 0) return a;
  const int64_t b = slot / p.block_size;
  if (b >= p.num_blocks) return a;
  a.block = b, a.off = slot - b * p.block_size;
  return a;
}

__device__ __forceinline__ void pdl_prologue() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
}

// ------------------------------------------------------------------ vector tier --------

constexpr int kThreads = 128;
constexpr int kMaxTile = 16;

template <typename T, bool kInterleaved>
__global__ void __launch_bounds__(kThreads) kvx_rotary_kernel(const RotaryParams p) {
  constexpr int kVec = T::kPerVec;
  constexpr int kE = 16 / kVec;  // bytes per element
  extern __shared__ float sm_turn[];  // [tile][half] cosines, [tile][half] sines
  __shared__ SlotAt sm_slot[kMaxTile];
  pdl_prologue();
  const int t0 = blockIdx.x * p.tile, n = min(p.tile, p.tokens - t0);
  float *cosines = sm_turn, *sines = sm_turn + p.tile * p.half;
  for (int i = threadIdx.x; i < n * p.half; i += kThreads) {
    const int t = i / p.half;
    const float2 cs = turn(p, read_index(p.positions, t0 + t, p.pos64), i - t * p.half);
    cosines[i] = cs.x, sines[i] = cs.y;
  }
  const bool paged = p.k != nullptr && p.k_out == nullptr;
  if (paged && threadIdx.x < n) sm_slot[threadIdx.x] = slot_at(p, t0 + threadIdx.x);
  __syncthreads();

  // units of a head: the vectors (or pairs of vectors) that are turned, then those that are not
  const int turned = kInterleaved ? 2 * p.half / kVec : p.half / kVec;
  const int units = p.units;
  const int heads = p.q_heads + p.k_heads;             // turned heads of a token
  const int v_units = paged ? p.k_heads * p.v_units : 0;
  const int per_token = heads * units + v_units;
  for (int i = threadIdx.x; i < n * per_token; i += kThreads) {
    const int t = i / per_token;
    int rest = i - t * per_token;
    const int64_t tok = t0 + t;
    if (rest >= heads * units) {  // a vector of V, on its way to the cache
      const SlotAt at = sm_slot[t];
      if (at.block < 0) continue;
      rest -= heads * units;
      const int h = p.v_shift >= 0 ? rest >> p.v_shift : rest / p.v_units, d = (rest - h * p.v_units) * kVec;
      const uint4 x = load_stream(p.v + tok * p.v_pitch + (static_cast<int64_t>(h) * p.dim + d) * kE);
      char *to = p.vc.base + at.block * p.vc.blk + at.off * p.vc.tok + h * p.vc.head;
      if (!p.fp8) {
        store_stream(to + d * kE, x);
      } else {
        float f[kVec];
        T::unpack(x, f);
        const float s = p.vs.base[h * p.vs.stride];
#pragma unroll
        for (int c = 0; c < kVec; c += 4)
          *reinterpret_cast<uint32_t *>(to + d + c) = quant2(f[c], f[c + 1], s) | quant2(f[c + 2], f[c + 3], s) << 16;
      }
      continue;
    }
    const int h = p.units_shift >= 0 ? rest >> p.units_shift : rest / units, u = rest - h * units;
    const bool is_k = h >= p.q_heads;
    const int kh = h - p.q_heads;
    const bool pass = u >= turned;
    const int d0 = pass ? 2 * p.half + (u - turned) * kVec : u * kVec;
    const int d1 = d0 + p.half;  // the vector that pairs up (half layout)
    const char *from;
    char *to;
    bool skip, quant = false;
    if (!is_k) {
      from = p.q + tok * p.q_pitch + static_cast<int64_t>(h) * p.dim * kE;
      to = p.q_out + tok * p.qo_pitch + static_cast<int64_t>(h) * p.dim * kE;
      skip = pass && p.q_in_place;
    } else {
      from = p.k + tok * p.k_pitch + static_cast<int64_t>(kh) * p.dim * kE;
      if (paged) {
        const SlotAt at = sm_slot[t];
        skip = at.block < 0;
        to = p.kc.base + at.block * p.kc.blk + at.off * p.kc.tok + kh * p.kc.head;
        quant = p.fp8 != 0;
      } else {
        to = p.k_out + tok * p.ko_pitch + static_cast<int64_t>(kh) * p.dim * kE;
        skip = pass && p.k_in_place;
      }
    }
    if (skip) continue;
    uint4 x0 = load_stream(from + d0 * kE), x1 = make_uint4(0, 0, 0, 0);
    const bool two = !kInterleaved && !pass;
    if (two) x1 = load_stream(from + d1 * kE);
    if (!pass) {
      float a[kVec], b[kVec];
      T::unpack(x0, a);
      if (kInterleaved) {
        const float *c = cosines + t * p.half + u * (kVec / 2), *s = sines + t * p.half + u * (kVec / 2);
#pragma unroll
        for (int k = 0; k < kVec / 2; ++k) turn_pair(a[2 * k], a[2 * k + 1], c[k], s[k]);
      } else {
        T::unpack(x1, b);
        const float *c = cosines + t * p.half + d0, *s = sines + t * p.half + d0;
#pragma unroll
        for (int k = 0; k < kVec; ++k) turn_pair(a[k], b[k], c[k], s[k]);
        x1 = T::pack(b);
      }
      x0 = T::pack(a);
    }
    if (!quant) {
      store_stream(to + d0 * kE, x0);
      if (two) store_stream(to + d1 * kE, x1);
    } else {
      // the values the IO type holds are what is quantised, as by a write of the turned keys
      const float s = p.ks.base[kh * p.ks.stride];
      float f[kVec];
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        if (half == 1 && !two) break;
        T::unpack(half == 0 ? x0 : x1, f);
#pragma unroll
        for (int c = 0; c < kVec; c += 4)
          *reinterpret_cast<uint32_t *>(to + (half == 0 ? d0 : d1) + c) =
              quant2(f[c], f[c + 1], s) | quant2(f[c + 2], f[c + 3], s) << 16;
      }
    }
  }
}

// ------------------------------------------------------------------ element tier -------

__device__ __forceinline__ int64_t elem_offset(const PageView &v, const SlotAt &a, int64_t h, int32_t d) {
  const int32_t hi = d / v.pack;
  return a.block * v.blk + a.off * v.tok + h * v.head + hi * v.dhi + (d - hi * v.pack) * v.dlo;
}

// One thread per pair of a head (then per element that is not turned, then per element of V).
template <typename T>
__global__ void __launch_bounds__(kThreads) kvx_rotary_element_kernel(const RotaryParams p) {
  using Bits = typename T::Bits;
  pdl_prologue();
  const bool paged = p.k != nullptr && p.k_out == nullptr;
  const int units = p.dim - p.half;  // pairs, then single elements
  const int heads = p.q_heads + p.k_heads;
  const int64_t per_token = static_cast<int64_t>(heads) * units + (paged ? static_cast<int64_t>(p.k_heads) * p.dim : 0);
  const int64_t all = per_token * p.tokens;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; i < all; i += static_cast<int64_t>(gridDim.x) * kThreads) {
    const int64_t t = i / per_token;
    int64_t rest = i - t * per_token;
    auto put_page = [&](const PageView &view, const ScaleView &sc, const SlotAt &at, int h, int d, float x) {
      char *to = view.base + elem_offset(view, at, h, d);
      if (p.fp8)
        *reinterpret_cast<uint8_t *>(to) = static_cast<uint8_t>(quant2(x, 0.f, sc.base[h * sc.stride]));
      else
        *reinterpret_cast<Bits *>(to) = T::put(x);
    };
    if (rest >= static_cast<int64_t>(heads) * units) {
      rest -= static_cast<int64_t>(heads) * units;
      const SlotAt at = slot_at(p, t);
      if (at.block < 0) continue;
      const int h = static_cast<int>(rest / p.dim), d = static_cast<int>(rest - static_cast<int64_t>(h) * p.dim);
      const Bits x = reinterpret_cast<const Bits *>(p.v + t * p.v_pitch)[static_cast<int64_t>(h) * p.dim + d];
      if (p.fp8)
        put_page(p.vc, p.vs, at, h, d, T::get(x));
      else
        *reinterpret_cast<Bits *>(p.vc.base + elem_offset(p.vc, at, h, d)) = x;
      continue;
    }
    const int h = static_cast<int>(rest / units), u = static_cast<int>(rest - static_cast<int64_t>(h) * units);
    const bool is_k = h >= p.q_heads;
    const int hh = is_k ? h - p.q_heads : h;
    const Bits *from = reinterpret_cast<const Bits *>((is_k ? p.k + t * p.k_pitch : p.q + t * p.q_pitch)) + static_cast<int64_t>(hh) * p.dim;
    Bits *to = nullptr;
    SlotAt at{-1, 0};
    if (is_k && paged) {
      at = slot_at(p, t);
      if (at.block < 0) continue;
    } else {
      to = reinterpret_cast<Bits *>(is_k ? p.k_out + t * p.ko_pitch : p.q_out + t * p.qo_pitch) + static_cast<int64_t>(hh) * p.dim;
    }
    if (u >= p.half) {  // not turned: bits as they are
      const int d = u + p.half;
      const Bits x = from[d];
      if (to != nullptr)
        to[d] = x;
      else if (p.fp8)
        put_page(p.kc, p.ks, at, hh, d, T::get(x));
      else
        *reinterpret_cast<Bits *>(p.kc.base + elem_offset(p.kc, at, hh, d)) = x;
      continue;
    }
    const float2 cs = turn(p, read_index(p.positions, t, p.pos64), u);
    const int d0 = p.interleaved ? 2 * u : u, d1 = p.interleaved ? 2 * u + 1 : u + p.half;
    float y = T::get(from[d0]), z = T::get(from[d1]);
    turn_pair(y, z, cs.x, cs.y);
    const Bits a = T::put(y), b = T::put(z);
    if (to != nullptr) {
      to[d0] = a, to[d1] = b;
    } else {
      put_page(p.kc, p.ks, at, hh, d0, T::get(a));
      put_page(p.kc, p.ks, at, hh, d1, T::get(b));
    }
  }
}

// ------------------------------------------------------------------ host ---------------

bool aligned(const void *p, int64_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// Token rows of heads x dim elements, dense inside; `pitch` in bytes.
kvx_status_t check_rows(const kvx_tensor_desc_t *t, int64_t tokens, int64_t heads, int64_t dim, int64_t elem, int64_t *pitch) {
  if (t->size < sizeof(kvx_tensor_desc_t)) return KVX_STATUS_INVALID_ARGUMENT;
  if (t->ndim != 3 || t->shape[0] != tokens || t->shape[1] != heads || t->shape[2] != dim) return KVX_STATUS_INVALID_ARGUMENT;
  if ((dim > 1 && t->stride[2] != 1) || (heads > 1 && t->stride[1] != dim)) return KVX_STATUS_UNSUPPORTED;
  if (tokens > 1 && t->stride[0] < heads * dim) return KVX_STATUS_UNSUPPORTED;
  *pitch = (tokens > 1 ? t->stride[0] : heads * dim) * elem;
  return KVX_STATUS_OK;
}

bool io_type(kvx_dtype_t t) { return t == KVX_DTYPE_F16 || t == KVX_DTYPE_BF16 || t == KVX_DTYPE_F32; }

template <typename... Args>
void launch_pdl(void (*kernel)(Args...), unsigned grid, unsigned block, size_t smem, cudaStream_t st, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
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

template <typename T>
kvx_status_t launch(RotaryParams &p, cudaStream_t st) {
  constexpr int kVec = T::kPerVec;
  const int64_t e = 16 / kVec, ce = p.fp8 ? 1 : e;
  const bool paged = p.k != nullptr && p.k_out == nullptr;
  auto rows16 = [&](const void *base, int64_t pitch) { return base == nullptr || (aligned(base, 16) && pitch % 16 == 0); };
  auto pages16 = [&](const PageView &v) {
    const int64_t a = kVec * ce;  // bytes one vector becomes in the cache
    return v.pack == 1 && v.dhi == ce && aligned(v.base, a) && v.blk % a == 0 && v.tok % a == 0 && v.head % a == 0;
  };
  const bool shape = p.dim % kVec == 0 && (p.interleaved ? (2 * p.half) % kVec == 0 : p.half % kVec == 0);
  const bool vec = shape && rows16(p.q, p.q_pitch) && rows16(p.q_out, p.qo_pitch) && rows16(p.k, p.k_pitch) &&
                   rows16(p.k_out, p.ko_pitch) && (!paged || (rows16(p.v, p.v_pitch) && pages16(p.kc) && pages16(p.vc))) &&
                   static_cast<int64_t>(p.q_heads + 2 * p.k_heads) * p.dim <= (1 << 22) && p.half <= 1024;
  if (vec) {
    // Tokens per CTA: the angles' latency is hidden by the other CTAs of the SM, so small CTAs do
    // best.  16 384 tokens of 32 + 8 heads x 128 with the write of K and V (389 MB), us: 66.6 with 2
    // tokens and 128 threads (5.8 TB/s, 89 % of a copy), 67.7 / 4 / 256, 69.8 / 2 / 256, 72.1 / 8 / 256;
    // two or four units in flight per thread 75 and 101 (registers cost more CTAs than they bring loads).
    p.tile = 2;
    while (p.tile > 1 && (p.tokens + p.tile - 1) / p.tile < 148 * 4) p.tile >>= 1;
    auto shift_of = [](int32_t x) { return x > 0 && (x & (x - 1)) == 0 ? __builtin_ctz(static_cast<unsigned>(x)) : -1; };
    p.units = (p.interleaved ? 2 * p.half : p.half) / kVec + (p.dim - 2 * p.half) / kVec;
    p.v_units = p.dim / kVec;
    p.units_shift = shift_of(p.units), p.v_shift = shift_of(p.v_units);
    const unsigned grid = static_cast<unsigned>((p.tokens + p.tile - 1) / p.tile);
    const size_t smem = static_cast<size_t>(p.tile) * p.half * 2 * sizeof(float);
    if (p.interleaved)
      launch_pdl(kvx_rotary_kernel<T, true>, grid, kThreads, smem, st, p);
    else
      launch_pdl(kvx_rotary_kernel<T, false>, grid, kThreads, smem, st, p);
  } else {
    const int64_t all = (static_cast<int64_t>(p.q_heads + p.k_heads) * (p.dim - p.half) + (paged ? static_cast<int64_t>(p.k_heads) * p.dim : 0)) * p.tokens;
    const unsigned grid = static_cast<unsigned>(std::min<int64_t>((all + kThreads - 1) / kThreads, 148 * 32));
    launch_pdl(kvx_rotary_element_kernel<T>, grid, kThreads, size_t{0}, st, p);
  }
  return cudaGetLastError() == cudaSuccess ? KVX_STATUS_OK : KVX_STATUS_INTERNAL_ERROR;
}

// Everything of the descriptor that both entry points share.  `tokens` / `dim` are those of the keys
// (fused form) or -1: taken from the query.
kvx_status_t common(const kvx_rotary_desc_t *r, int64_t tokens, int64_t dim, kvx_dtype_t io, RotaryParams *p) {
  if ((r->flags & ~static_cast<uint32_t>(KVX_ROTARY_INTERLEAVED | KVX_ROTARY_INVERSE)) != 0) return KVX_STATUS_INVALID_ARGUMENT;
  if (r->rotary_dim % 2 != 0 || r->rotary_dim > static_cast<uint64_t>(dim)) return KVX_STATUS_INVALID_ARGUMENT;
  const int64_t elem = dtype_bytes(io);
  if (r->query.data != nullptr) {
    if (r->query.dtype != io || r->query_out.dtype != io) return KVX_STATUS_UNSUPPORTED;
    const int64_t hq = r->query.shape[1];
    if (hq < 0 || hq > INT32_MAX) return KVX_STATUS_INVALID_ARGUMENT;
    kvx_status_t st = check_rows(&r->query, tokens, hq, dim, elem, &p->q_pitch);
    if (st != KVX_STATUS_OK) return st;
    st = check_rows(&r->query_out, tokens, hq, dim, elem, &p->qo_pitch);
    if (st != KVX_STATUS_OK) return st;
    if (r->query_out.data == nullptr && tokens * hq * dim > 0) return KVX_STATUS_INVALID_ARGUMENT;
    p->q = static_cast<const char *>(r->query.data);
    p->q_out = static_cast<char *>(r->query_out.data);
    p->q_heads = static_cast<int32_t>(hq);
    p->q_in_place = p->q == p->q_out && p->q_pitch == p->qo_pitch ? 1 : 0;
  }
  if (tokens > INT32_MAX || dim > INT32_MAX) return KVX_STATUS_INVALID_ARGUMENT;
  if (tokens == 0) return KVX_STATUS_OK;
  if (r->position_dtype != KVX_DTYPE_S32 && r->position_dtype != KVX_DTYPE_S64) return KVX_STATUS_INVALID_ARGUMENT;
  if (r->positions == nullptr || (r->inv_freq == nullptr && r->rotary_dim > 0)) return KVX_STATUS_INVALID_ARGUMENT;
  p->positions = r->positions;
  p->pos64 = r->position_dtype == KVX_DTYPE_S64 ? 1 : 0;
  p->inv_freq = r->inv_freq;
  p->factor = static_cast<float>(r->factor);
  p->tokens = static_cast<int32_t>(tokens);
  p->dim = static_cast<int32_t>(dim);
  p->half = static_cast<int32_t>(r->rotary_dim / 2);
  p->interleaved = (r->flags & KVX_ROTARY_INTERLEAVED) != 0 ? 1 : 0;
  p->inverse = (r->flags & KVX_ROTARY_INVERSE) != 0 ? 1 : 0;
  return KVX_STATUS_OK;
}

kvx_status_t dispatch(RotaryParams &p, kvx_dtype_t io, cudaStream_t st) {
  if (static_cast<int64_t>(p.q_heads + p.k_heads) * p.dim == 0) return KVX_STATUS_OK;
  if (io == KVX_DTYPE_BF16) return launch<Bf16>(p, st);
  if (io == KVX_DTYPE_F16) return launch<Fp16>(p, st);
  return launch<Fp32>(p, st);
}

}  // namespace

extern "C" {

KVX_API kvx_status_t kvx_launch_rotary(const kvx_rotary_desc_t *r, void *stream) {
  if (r == nullptr || r->size < sizeof(kvx_rotary_desc_t)) return KVX_STATUS_INVALID_ARGUMENT;
  const bool has_q = r->query.data != nullptr, has_k = r->key.data != nullptr;
  if (!has_q && !has_k) {  // no data: nothing to turn, or a missing pointer
    const kvx_tensor_desc_t *t = &r->query;
    if (t->size < sizeof(kvx_tensor_desc_t) || t->ndim != 3) return KVX_STATUS_INVALID_ARGUMENT;
    return t->shape[0] == 0 ? KVX_STATUS_OK : KVX_STATUS_INVALID_ARGUMENT;
  }
  const kvx_tensor_desc_t *lead = has_q ? &r->query : &r->key;
  const kvx_dtype_t io = lead->dtype;
  if (!io_type(io)) return KVX_STATUS_UNSUPPORTED;
  if (lead->ndim != 3 || lead->shape[0] < 0 || lead->shape[2] < 0) return KVX_STATUS_INVALID_ARGUMENT;
  RotaryParams p = {};
  kvx_status_t st = common(r, lead->shape[0], lead->shape[2], io, &p);
  if (st != KVX_STATUS_OK) return st;
  if (has_k) {
    if (r->key.dtype != io || r->key_out.dtype != io) return KVX_STATUS_UNSUPPORTED;
    const int64_t hk = r->key.shape[1], elem = dtype_bytes(io);
    if (hk < 0 || hk > INT32_MAX / 2) return KVX_STATUS_INVALID_ARGUMENT;
    st = check_rows(&r->key, lead->shape[0], hk, lead->shape[2], elem, &p.k_pitch);
    if (st != KVX_STATUS_OK) return st;
    st = check_rows(&r->key_out, lead->shape[0], hk, lead->shape[2], elem, &p.ko_pitch);
    if (st != KVX_STATUS_OK) return st;
    if (r->key_out.data == nullptr) return KVX_STATUS_INVALID_ARGUMENT;
    p.k = static_cast<const char *>(r->key.data);
    p.k_out = static_cast<char *>(r->key_out.data);
    p.k_heads = static_cast<int32_t>(hk);
    p.k_in_place = p.k == p.k_out && p.k_pitch == p.ko_pitch ? 1 : 0;
  }
  if (lead->shape[0] == 0) return KVX_STATUS_OK;
  return dispatch(p, io, reinterpret_cast<cudaStream_t>(stream));
}

KVX_API kvx_status_t kvx_launch_rotary_write_kv(const kvx_cache_desc_t *cache, const kvx_write_desc_t *write, const kvx_rotary_desc_t *r,
                                                void *stream) {
  if (cache == nullptr || write == nullptr || r == nullptr) return KVX_STATUS_INVALID_ARGUMENT;
  if (cache->size < sizeof(kvx_cache_desc_t) || write->size < sizeof(kvx_write_desc_t) || write->io.size < sizeof(kvx_kv_io_desc_t) ||
      write->slots.size < sizeof(kvx_slot_mapping_t) || r->size < sizeof(kvx_rotary_desc_t))
    return KVX_STATUS_INVALID_ARGUMENT;
  if (r->key.data != nullptr || r->key_out.data != nullptr) return KVX_STATUS_INVALID_ARGUMENT;
  if (cache->k.dtype != cache->v.dtype) return KVX_STATUS_INVALID_ARGUMENT;
  const kvx_dtype_t io = write->io.key.dtype, cd = cache->k.dtype;
  if (!io_type(io) || write->io.value.dtype != io) return KVX_STATUS_UNSUPPORTED;
  RotaryParams p = {};
  if (cd == KVX_DTYPE_F8_E4M3) {
    if (!kvx_detail::resolve_scale(&write->k_scale_desc, write->k_scale, cache->num_kv_heads, &p.ks) ||
        !kvx_detail::resolve_scale(&write->v_scale_desc, write->v_scale, cache->num_kv_heads, &p.vs))
      return KVX_STATUS_UNSUPPORTED;
    p.fp8 = 1;
  } else if (cd != io) {
    return KVX_STATUS_UNSUPPORTED;
  }
  if (write->io.num_kv_heads != cache->num_kv_heads || write->io.head_dim != cache->head_dim) return KVX_STATUS_INVALID_ARGUMENT;
  const int64_t T = write->io.num_tokens, H = cache->num_kv_heads, D = cache->head_dim, elem = dtype_bytes(io);
  kvx_status_t st = check_rows(&write->io.key, T, H, D, elem, &p.k_pitch);
  if (st != KVX_STATUS_OK) return st;
  st = check_rows(&write->io.value, T, H, D, elem, &p.v_pitch);
  if (st != KVX_STATUS_OK) return st;
  if (write->slots.token_count != write->io.num_tokens) return KVX_STATUS_INVALID_ARGUMENT;
  st = common(r, T, D, io, &p);
  if (st != KVX_STATUS_OK) return st;
  st = make_page_view(cache, &cache->k, dtype_bytes(cd), &p.kc);
  if (st != KVX_STATUS_OK) return st;
  st = make_page_view(cache, &cache->v, dtype_bytes(cd), &p.vc);
  if (st != KVX_STATUS_OK) return st;
  if (T * D == 0 || (H == 0 && p.q == nullptr)) return KVX_STATUS_OK;
  if (write->slots.dtype != KVX_DTYPE_S32 && write->slots.dtype != KVX_DTYPE_S64) return KVX_STATUS_INVALID_ARGUMENT;
  if (write->io.key.data == nullptr || write->io.value.data == nullptr || write->slots.slots == nullptr || cache->k.data == nullptr ||
      cache->v.data == nullptr || cache->block_size == 0 || cache->block_size > static_cast<uint32_t>(INT32_MAX) ||
      cache->num_blocks > static_cast<uint32_t>(INT32_MAX) || H > INT32_MAX / 2)
    return KVX_STATUS_INVALID_ARGUMENT;
  p.k = static_cast<const char *>(write->io.key.data);
  p.v = static_cast<const char *>(write->io.value.data);
  p.k_heads = static_cast<int32_t>(H);
  p.slots = write->slots.slots;
  p.slot64 = write->slots.dtype == KVX_DTYPE_S64 ? 1 : 0;
  p.num_blocks = static_cast<int32_t>(cache->num_blocks);
  p.block_size = static_cast<int32_t>(cache->block_size);
  return dispatch(p, io, reinterpret_cast<cudaStream_t>(stream));
}

}  // extern "C"
