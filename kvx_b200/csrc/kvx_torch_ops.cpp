/*
 * torch operators over the C-ABI library, registered as torch.ops.kvx_b200.*:
 *
 *   reshape_and_cache_flash_kvx(key, value, key_cache!, value_cache!, slot_mapping,
 *                               kv_cache_dtype, k_scale, v_scale) -> ()
 *   gather_kv(key_cache, value_cache, block_table, seq_lens, key_out!, value_out!,
 *             kv_cache_dtype, k_scale, v_scale) -> ()
 *
 * The first has the schema, the checks and the descriptor filling of the operator the
 * reference's vLLM patch adds to vLLM's _C extension (reference: patches/vllm/kvx.patch:176-275,
 * schema :288-296): tensors are described as they are (sizes and strides, no copies), the cache
 * layout is inferred from sizes and strides (cache_form below), the batch is sized by
 * slot_mapping, the launch goes to the current CUDA stream, and a status other than OK
 * raises.  Going through the dispatcher instead of ctypes keeps the host cost of a decode-size
 * call at a few microseconds.  This file only marshals arguments; all data movement is in
 * kvx_paged_kv.cu.
 */
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/library.h>
#include <torch/types.h>

#include <algorithm>
#include <cstring>
#include <string>
#include <tuple>
#include <vector>

#include "kvx_attention.h"
#include "kvx_paged_kv.h"
#include "kvx_pages_ops.h"
#include "kvx_rotary.h"

namespace {

kvx_dtype_t float_code(at::ScalarType t) {
  switch (t) {
    case at::ScalarType::Float:
      return KVX_DTYPE_F32;
    case at::ScalarType::Half:
      return KVX_DTYPE_F16;
    case at::ScalarType::BFloat16:
      return KVX_DTYPE_BF16;
    default:
      return KVX_DTYPE_INVALID;
  }
}

kvx_dtype_t index_code(at::ScalarType t) {
  return t == at::ScalarType::Int ? KVX_DTYPE_S32 : t == at::ScalarType::Long ? KVX_DTYPE_S64 : KVX_DTYPE_INVALID;
}

void describe(kvx_tensor_desc_t *d, const torch::Tensor &t, kvx_dtype_t dtype, kvx_layout_t layout) {
  std::memset(d, 0, sizeof(*d));
  d->size = sizeof(*d);
  d->dtype = dtype;
  d->layout = layout;
  d->memory = KVX_MEMORY_DEVICE;
  d->ndim = static_cast<uint32_t>(t.dim());
  for (int64_t i = 0; i < t.dim() && i < KVX_MAX_TENSOR_DIMS; ++i) {
    d->shape[i] = t.size(i);
    d->stride[i] = t.stride(i);
  }
  d->data = t.data_ptr();
}

// Which page layout a 4-D cache tensor has.  The reference's operator decides by one stride
// (NHD when stride(2) == head_dim, reference: kvx.patch:132-135, :222-229), which misreads a
// contiguous [blocks, heads, block_size, dim] tensor; this rule agrees with it wherever it is
// right and also accepts that tensor and vLLM's permuted view of HND memory:
//   stride(1) < stride(2)          a [blocks, block_size, heads, dim] VIEW of HND memory
//   else size(2) == heads only     NHD   [blocks, block_size, heads, dim]
//   else size(1) == heads only     HND   [blocks, heads, block_size, dim]
//   else (block_size == heads)     the reference's stride rule
enum class CacheForm { kNhd, kHnd, kHndView };

CacheForm cache_form(const torch::Tensor &c, int64_t heads, int64_t head_dim) {
  if (c.stride(1) < c.stride(2)) return CacheForm::kHndView;
  const bool nhd = c.size(2) == heads, hnd = c.size(1) == heads;
  if (nhd != hnd) return nhd ? CacheForm::kNhd : CacheForm::kHnd;
  return c.stride(2) == head_dim ? CacheForm::kNhd : CacheForm::kHnd;
}

void describe_pages(kvx_tensor_desc_t *d, const torch::Tensor &t, kvx_dtype_t dtype, CacheForm form) {
  describe(d, t, dtype, form == CacheForm::kNhd ? KVX_LAYOUT_BLOCK_NHD : KVX_LAYOUT_BLOCK_HND);
  if (form == CacheForm::kHndView) {  // describe the memory: axes 1 and 2 swapped back
    d->shape[1] = t.size(2), d->shape[2] = t.size(1);
    d->stride[1] = t.stride(2), d->stride[2] = t.stride(1);
  }
}

// Cache descriptor from a pair of 4-D page tensors (reference: kvx.patch:222-245).
kvx_dtype_t describe_cache(kvx_cache_desc_t *c, const torch::Tensor &key_cache, const torch::Tensor &value_cache,
                           const std::string &kv_cache_dtype, int64_t heads, int64_t head_dim) {
  TORCH_CHECK(key_cache.is_cuda() && value_cache.is_cuda(), "cache tensors must be CUDA tensors");
  TORCH_CHECK(key_cache.dim() == 4 && key_cache.sizes() == value_cache.sizes(), "key/value cache shape mismatch");
  TORCH_CHECK(key_cache.scalar_type() == value_cache.scalar_type(), "cache dtype mismatch");
  kvx_dtype_t code;
  if (kv_cache_dtype == "auto") {
    code = float_code(key_cache.scalar_type());
    TORCH_CHECK(code != KVX_DTYPE_INVALID, "KVX cache: unsupported cache dtype");
  } else {
    TORCH_CHECK(kv_cache_dtype == "fp8" || kv_cache_dtype == "fp8_e4m3", "KVX cache: unsupported kv_cache_dtype ",
                kv_cache_dtype);
    TORCH_CHECK(key_cache.element_size() == 1, "an fp8 cache must have 1-byte elements");
    code = KVX_DTYPE_F8_E4M3;
  }
  const CacheForm form = cache_form(key_cache, heads, head_dim);
  TORCH_CHECK(cache_form(value_cache, heads, head_dim) == form, "key/value cache layout mismatch");
  std::memset(c, 0, sizeof(*c));
  c->size = sizeof(*c);
  c->num_blocks = static_cast<uint32_t>(key_cache.size(0));
  c->block_size = static_cast<uint32_t>(form == CacheForm::kHnd ? key_cache.size(2) : key_cache.size(1));
  c->num_kv_heads = static_cast<uint32_t>(form == CacheForm::kHnd ? key_cache.size(1) : key_cache.size(2));
  c->head_dim = static_cast<uint32_t>(key_cache.size(3));
  describe_pages(&c->k, key_cache, code, form);
  describe_pages(&c->v, value_cache, code, form);
  c->pool.size = sizeof(c->pool);
  return code;
}

void describe_scale(kvx_scale_desc_t *d, const torch::Tensor &scale, int64_t heads) {
  std::memset(d, 0, sizeof(*d));
  d->size = sizeof(*d);
  d->dtype = KVX_DTYPE_F32;
  if (!scale.defined() || scale.numel() == 0) return;
  TORCH_CHECK(scale.is_cuda() && scale.scalar_type() == at::ScalarType::Float, "scales must be float32 CUDA tensors");
  TORCH_CHECK(scale.numel() == 1 || (scale.dim() == 1 && scale.numel() == heads),
              "a scale must have 1 or num_kv_heads elements");
  d->granularity = scale.numel() == 1 ? KVX_SCALE_PER_TENSOR : KVX_SCALE_PER_HEAD;
  d->ndim = 1;
  d->shape[0] = scale.numel();
  d->stride[0] = scale.dim() == 1 ? scale.stride(0) : 1;
  d->data = scale.data_ptr();
}

void reshape_and_cache_flash_kvx(torch::Tensor &key, torch::Tensor &value, torch::Tensor &key_cache,
                                 torch::Tensor &value_cache, torch::Tensor &slot_mapping,
                                 const std::string &kv_cache_dtype, torch::Tensor &k_scale, torch::Tensor &v_scale) {
  TORCH_CHECK(key.is_cuda() && value.is_cuda(), "key/value must be CUDA tensors");
  TORCH_CHECK(key.dim() == 3 && value.dim() == 3, "key/value must be [num_tokens, num_heads, head_dim]");
  TORCH_CHECK(key.scalar_type() == value.scalar_type(), "key/value dtype mismatch");
  const kvx_dtype_t io = float_code(key.scalar_type());
  TORCH_CHECK(io != KVX_DTYPE_INVALID, "KVX cache write unsupported dtype");
  const kvx_dtype_t slot_dtype = index_code(slot_mapping.scalar_type());
  TORCH_CHECK(slot_dtype != KVX_DTYPE_INVALID && slot_mapping.dim() == 1, "slot_mapping must be 1-D int32 or int64");
  TORCH_CHECK(slot_mapping.is_cuda() && slot_mapping.is_contiguous(), "slot_mapping must be a contiguous CUDA tensor");
  const int64_t tokens = slot_mapping.size(0), heads = key.size(1), dim = key.size(2);
  // the batch is sized by slot_mapping (as in the operator this one stands in for), so key and
  // value must hold at least that many token rows
  TORCH_CHECK(key.size(0) >= tokens && value.size(0) >= tokens, "key/value hold fewer tokens than slot_mapping");
  TORCH_CHECK(key_cache.is_cuda() && value_cache.is_cuda(), "cache tensors must be CUDA tensors");
  const at::cuda::OptionalCUDAGuard guard(at::device_of(key_cache));  // launch on the tensors' device and its stream

  kvx_cache_desc_t cache;
  const kvx_dtype_t cache_code = describe_cache(&cache, key_cache, value_cache, kv_cache_dtype, heads, dim);
  TORCH_CHECK(cache_code == io || cache_code == KVX_DTYPE_F8_E4M3, "key/value dtype must match cache dtype");

  kvx_write_desc_t write;
  std::memset(&write, 0, sizeof(write));
  write.size = sizeof(write);
  write.io.size = sizeof(write.io);
  write.io.num_tokens = static_cast<uint32_t>(tokens);
  write.io.num_kv_heads = static_cast<uint32_t>(heads);
  write.io.head_dim = static_cast<uint32_t>(dim);
  describe(&write.io.key, key, io, KVX_LAYOUT_INVALID);
  describe(&write.io.value, value, io, KVX_LAYOUT_INVALID);
  write.io.key.shape[0] = write.io.value.shape[0] = tokens;  // the batch is sized by slot_mapping
  write.slots.size = sizeof(write.slots);
  write.slots.dtype = slot_dtype;
  write.slots.token_count = static_cast<uint32_t>(tokens);
  write.slots.invalid_slot = -1;
  write.slots.slots = slot_mapping.data_ptr();
  describe_scale(&write.k_scale_desc, k_scale, heads);
  describe_scale(&write.v_scale_desc, v_scale, heads);

  void *stream = reinterpret_cast<void *>(at::cuda::getCurrentCUDAStream().stream());
  const kvx_status_t status = kvx_launch_write_kv(&cache, &write, stream);
  TORCH_CHECK(status == KVX_STATUS_OK, "kvx cache write failed with status=", static_cast<int>(status));
}

void gather_kv(torch::Tensor &key_cache, torch::Tensor &value_cache, torch::Tensor &block_table,
               torch::Tensor &seq_lens, torch::Tensor &key_out, torch::Tensor &value_out,
               const std::string &kv_cache_dtype, torch::Tensor &k_scale, torch::Tensor &v_scale) {
  TORCH_CHECK(key_out.is_cuda() && value_out.is_cuda(), "outputs must be CUDA tensors");
  TORCH_CHECK(key_out.dim() == 4 && key_out.sizes() == value_out.sizes(),
              "outputs must be [seq_count, max_seq_len, heads, dim]");
  const kvx_dtype_t io = float_code(key_out.scalar_type());
  TORCH_CHECK(io != KVX_DTYPE_INVALID && value_out.scalar_type() == key_out.scalar_type(), "unsupported output dtype");
  TORCH_CHECK(block_table.dim() == 2 && block_table.is_contiguous(), "block_table must be contiguous and 2-D");
  const kvx_dtype_t idx = index_code(block_table.scalar_type());
  TORCH_CHECK(idx != KVX_DTYPE_INVALID && seq_lens.scalar_type() == block_table.scalar_type(),
              "block_table and seq_lens must share an int32 or int64 dtype");
  const int64_t seqs = key_out.size(0), max_len = key_out.size(1), heads = key_out.size(2), dim = key_out.size(3);
  TORCH_CHECK(block_table.is_cuda() && seq_lens.is_cuda() && seq_lens.is_contiguous(),
              "block_table and seq_lens must be contiguous CUDA tensors");
  TORCH_CHECK(seq_lens.dim() == 1 && seq_lens.numel() == block_table.size(0),
              "seq_lens must have one entry per row of block_table");
  TORCH_CHECK(key_cache.is_cuda() && value_cache.is_cuda(), "cache tensors must be CUDA tensors");
  const at::cuda::OptionalCUDAGuard guard(at::device_of(key_cache));

  kvx_cache_desc_t cache;
  const kvx_dtype_t cache_code = describe_cache(&cache, key_cache, value_cache, kv_cache_dtype, heads, dim);

  kvx_gather_desc_t g;
  std::memset(&g, 0, sizeof(g));
  g.size = sizeof(g);
  g.io.size = sizeof(g.io);
  g.io.num_tokens = static_cast<uint32_t>(seqs * max_len);
  g.io.num_kv_heads = static_cast<uint32_t>(heads);
  g.io.head_dim = static_cast<uint32_t>(dim);
  describe(&g.io.key, key_out, io, KVX_LAYOUT_INVALID);
  describe(&g.io.value, value_out, io, KVX_LAYOUT_INVALID);
  g.block_table.size = sizeof(g.block_table);
  g.block_table.format = KVX_BLOCK_TABLE_PACKED;
  g.block_table.index_dtype = idx;
  g.block_table.seq_count = static_cast<uint32_t>(block_table.size(0));
  g.block_table.beam_width = 1;
  g.block_table.max_blocks_per_seq = static_cast<uint32_t>(block_table.size(1));
  g.block_table.indices = block_table.data_ptr();
  g.block_table.indices_count = static_cast<uint32_t>(block_table.numel());
  g.seq_lens.size = sizeof(g.seq_lens);
  g.seq_lens.dtype = idx;
  g.seq_lens.seq_count = static_cast<uint32_t>(seq_lens.size(0));
  g.seq_lens.lengths = seq_lens.data_ptr();
  g.max_seq_len = static_cast<uint32_t>(max_len);

  void *stream = reinterpret_cast<void *>(at::cuda::getCurrentCUDAStream().stream());
  kvx_status_t status;
  if (cache_code == KVX_DTYPE_F8_E4M3) {
    kvx_scale_desc_t ks, vs;
    describe_scale(&ks, k_scale, heads);
    describe_scale(&vs, v_scale, heads);
    status = kvx_launch_gather_kv_f8e4m3(&cache, &g, &ks, &vs, stream);
  } else {
    status = kvx_launch_gather_kv(&cache, &g, stream);
  }
  TORCH_CHECK(status == KVX_STATUS_OK, "kvx cache gather failed with status=", static_cast<int>(status));
}

// Decode attention over the paged cache (include/kvx_attention.h).  `workspace` is a uint8 CUDA
// tensor of at least kvx_paged_attention_workspace_bytes() bytes (see attention_workspace_bytes).
void paged_attention_decode(torch::Tensor &out, torch::Tensor &query, torch::Tensor &key_cache,
                            torch::Tensor &value_cache, torch::Tensor &block_table, torch::Tensor &seq_lens,
                            double scale, int64_t max_seq_len, int64_t num_kv_heads, torch::Tensor &workspace,
                            const std::string &kv_cache_dtype, torch::Tensor &k_scale, torch::Tensor &v_scale) {
  TORCH_CHECK(query.is_cuda() && out.is_cuda(), "query/out must be CUDA tensors");
  TORCH_CHECK(query.dim() == 3 && query.sizes() == out.sizes() && query.scalar_type() == out.scalar_type(),
              "query/out must be matching [seq_count, q_heads, head_dim] tensors");
  const kvx_dtype_t io = float_code(query.scalar_type());
  TORCH_CHECK(io != KVX_DTYPE_INVALID, "unsupported query dtype");
  TORCH_CHECK(block_table.dim() == 2 && block_table.is_contiguous(), "block_table must be contiguous and 2-D");
  const kvx_dtype_t idx = index_code(block_table.scalar_type());
  TORCH_CHECK(idx != KVX_DTYPE_INVALID && seq_lens.scalar_type() == block_table.scalar_type(),
              "block_table and seq_lens must share an int32 or int64 dtype");
  const int64_t q_heads = query.size(1), dim = query.size(2);
  TORCH_CHECK(block_table.is_cuda() && seq_lens.is_cuda() && seq_lens.is_contiguous(),
              "block_table and seq_lens must be contiguous CUDA tensors");
  TORCH_CHECK(seq_lens.dim() == 1 && seq_lens.numel() == block_table.size(0),
              "seq_lens must have one entry per row of block_table");
  TORCH_CHECK(key_cache.is_cuda() && value_cache.is_cuda(), "cache tensors must be CUDA tensors");
  const at::cuda::OptionalCUDAGuard guard(at::device_of(key_cache));
  // KV heads: given, or read off the cache with the reference's stride rule (axis 2 when it is
  // contiguous over head_dim or the tensor is a permuted view, else axis 1)
  TORCH_CHECK(key_cache.dim() == 4, "cache tensors must be 4-D");
  const int64_t kv_heads = num_kv_heads > 0 ? num_kv_heads
                           : (key_cache.stride(1) < key_cache.stride(2) || key_cache.stride(2) == dim)
                               ? key_cache.size(2)
                               : key_cache.size(1);
  kvx_cache_desc_t cache;
  describe_cache(&cache, key_cache, value_cache, kv_cache_dtype, kv_heads, dim);

  kvx_attention_desc_t a;
  std::memset(&a, 0, sizeof(a));
  a.size = sizeof(a);
  a.num_q_heads = static_cast<uint32_t>(q_heads);
  a.max_seq_len = static_cast<uint32_t>(max_seq_len);
  a.scale = static_cast<float>(scale);
  describe(&a.query, query, io, KVX_LAYOUT_INVALID);
  describe(&a.out, out, io, KVX_LAYOUT_INVALID);
  a.block_table.size = sizeof(a.block_table);
  a.block_table.format = KVX_BLOCK_TABLE_PACKED;
  a.block_table.index_dtype = idx;
  a.block_table.seq_count = static_cast<uint32_t>(block_table.size(0));
  a.block_table.beam_width = 1;
  a.block_table.max_blocks_per_seq = static_cast<uint32_t>(block_table.size(1));
  a.block_table.indices = block_table.data_ptr();
  a.block_table.indices_count = static_cast<uint32_t>(block_table.numel());
  a.seq_lens.size = sizeof(a.seq_lens);
  a.seq_lens.dtype = idx;
  a.seq_lens.seq_count = static_cast<uint32_t>(seq_lens.size(0));
  a.seq_lens.lengths = seq_lens.data_ptr();
  kvx_scale_desc_t ks, vs;
  describe_scale(&ks, k_scale, cache.num_kv_heads);
  describe_scale(&vs, v_scale, cache.num_kv_heads);
  TORCH_CHECK(workspace.is_cuda() && workspace.is_contiguous(), "workspace must be a contiguous CUDA tensor");
  void *stream = reinterpret_cast<void *>(at::cuda::getCurrentCUDAStream().stream());
  const kvx_status_t status = kvx_launch_paged_attention_decode(
      &cache, &a, &ks, &vs, workspace.data_ptr(), static_cast<size_t>(workspace.numel() * workspace.element_size()), stream);
  TORCH_CHECK(status == KVX_STATUS_OK, "kvx paged attention failed with status=", static_cast<int>(status));
}

void *current_stream() { return reinterpret_cast<void *>(at::cuda::getCurrentCUDAStream().stream()); }

void describe_table(kvx_block_table_t *d, const torch::Tensor &t) {
  TORCH_CHECK(t.dim() == 2 && t.is_contiguous() && t.is_cuda(), "block_table must be a contiguous 2-D CUDA tensor");
  const kvx_dtype_t idx = index_code(t.scalar_type());
  TORCH_CHECK(idx != KVX_DTYPE_INVALID, "block_table must be int32 or int64");
  std::memset(d, 0, sizeof(*d));
  d->size = sizeof(*d);
  d->format = KVX_BLOCK_TABLE_PACKED;
  d->index_dtype = idx;
  d->seq_count = static_cast<uint32_t>(t.size(0));
  d->beam_width = 1;
  d->max_blocks_per_seq = static_cast<uint32_t>(t.size(1));
  d->indices = t.data_ptr();
  d->indices_count = static_cast<uint32_t>(t.numel());
}

void describe_lens(kvx_seq_lens_t *d, const torch::Tensor &t, const torch::Tensor &table) {
  TORCH_CHECK(t.is_cuda() && t.is_contiguous() && t.dim() == 1 && t.numel() == table.size(0),
              "seq_lens must be a contiguous CUDA tensor with one entry per row of block_table");
  TORCH_CHECK(t.scalar_type() == table.scalar_type(), "block_table and seq_lens must share an int32 or int64 dtype");
  TORCH_CHECK(t.device() == table.device(), "block_table and seq_lens must be on one device");
  d->size = sizeof(*d);
  d->dtype = index_code(t.scalar_type());
  d->seq_count = static_cast<uint32_t>(t.size(0));
  d->lengths = t.data_ptr();
}

// Attention of a chunk of new tokens (include/kvx_attention.h).  An empty or short `workspace` is
// replaced by scratch of torch's allocator; max_seq_len = 0 stands for what the table can address.
void paged_attention_chunk(torch::Tensor &out, const torch::Tensor &query, const torch::Tensor &key_cache,
                           const torch::Tensor &value_cache, const torch::Tensor &block_table, const torch::Tensor &seq_lens,
                           const torch::Tensor &query_indptr, double scale, bool causal, int64_t max_seq_len,
                           int64_t num_kv_heads, torch::Tensor &workspace, const std::string &kv_cache_dtype,
                           const torch::Tensor &k_scale, const torch::Tensor &v_scale) {
  TORCH_CHECK(query.is_cuda() && query.dim() == 3, "query must be a [rows, q_heads, head_dim] CUDA tensor");
  TORCH_CHECK(query.sizes() == out.sizes() && query.scalar_type() == out.scalar_type(),
              "out must have the shape and dtype of query");
  const kvx_dtype_t io = float_code(query.scalar_type());
  TORCH_CHECK(io != KVX_DTYPE_INVALID, "unsupported query dtype");
  const int64_t dim = query.size(2);
  kvx_chunk_attention_desc_t a;
  std::memset(&a, 0, sizeof(a));
  describe_table(&a.block_table, block_table);
  describe_lens(&a.seq_lens, seq_lens, block_table);
  a.query_indptr_dtype = index_code(query_indptr.scalar_type());
  TORCH_CHECK(a.query_indptr_dtype != KVX_DTYPE_INVALID && query_indptr.dim() == 1 && query_indptr.is_contiguous() &&
                  query_indptr.numel() == block_table.size(0) + 1,
              "query_indptr must hold seq_count + 1 int32 or int64 row numbers");
  TORCH_CHECK(key_cache.dim() == 4 && key_cache.is_cuda(), "cache tensors must be 4-D CUDA tensors");
  for (const torch::Tensor *t : {&key_cache, &value_cache, &block_table, &query_indptr, static_cast<const torch::Tensor *>(&out)})
    TORCH_CHECK(t->device() == query.device(), "all tensors must be on the query's device");
  const at::cuda::OptionalCUDAGuard guard(at::device_of(query));
  // KV heads: given, or read off the cache as paged_attention_decode does
  const int64_t kv_heads = num_kv_heads > 0 ? num_kv_heads
                           : (key_cache.stride(1) < key_cache.stride(2) || key_cache.stride(2) == dim)
                               ? key_cache.size(2)
                               : key_cache.size(1);
  kvx_cache_desc_t cache;
  describe_cache(&cache, key_cache, value_cache, kv_cache_dtype, kv_heads, dim);
  TORCH_CHECK(max_seq_len >= 0, "max_seq_len must not be negative");
  if (max_seq_len == 0)
    max_seq_len = std::min<int64_t>(block_table.size(1) * static_cast<int64_t>(cache.block_size), INT32_MAX - 2048);
  TORCH_CHECK(max_seq_len <= INT32_MAX - 1024, "max_seq_len is too large");
  a.size = sizeof(a);
  a.num_q_heads = static_cast<uint32_t>(query.size(1));
  a.max_seq_len = static_cast<uint32_t>(max_seq_len);
  a.scale = static_cast<float>(scale);
  a.causal = causal ? 1 : 0;
  describe(&a.query, query, io, KVX_LAYOUT_INVALID);
  describe(&a.out, out, io, KVX_LAYOUT_INVALID);
  a.query_indptr = query_indptr.data_ptr();
  kvx_scale_desc_t ks, vs;
  describe_scale(&ks, k_scale, cache.num_kv_heads);
  describe_scale(&vs, v_scale, cache.num_kv_heads);
  const size_t need = kvx_paged_attention_chunk_workspace_bytes(a.block_table.seq_count, static_cast<uint32_t>(query.size(0)),
                                                                a.num_q_heads, cache.num_kv_heads, cache.head_dim, a.max_seq_len);
  torch::Tensor scratch = workspace;
  if (static_cast<size_t>(scratch.numel() * scratch.element_size()) < need)
    scratch = torch::empty({static_cast<int64_t>(need)}, query.options().dtype(torch::kUInt8));
  TORCH_CHECK(scratch.device() == query.device() && scratch.is_contiguous(), "workspace must be contiguous, on the query's device");
  const kvx_status_t status = kvx_launch_paged_attention_chunk(
      &cache, &a, &ks, &vs, scratch.data_ptr(), static_cast<size_t>(scratch.numel() * scratch.element_size()), current_stream());
  TORCH_CHECK(status == KVX_STATUS_OK, "kvx chunk attention failed with status=", static_cast<int>(status));
}

// Fields of a rotary descriptor that both operators fill alike.
void describe_rotary(kvx_rotary_desc_t *r, const torch::Tensor &positions, const torch::Tensor &inv_freq, bool interleaved,
                     double factor, bool inverse, int64_t tokens, const torch::Device &device) {
  std::memset(r, 0, sizeof(*r));
  r->size = sizeof(*r);
  TORCH_CHECK(positions.device() == device && inv_freq.device() == device, "positions and inv_freq must be on the query's device");
  r->position_dtype = index_code(positions.scalar_type());
  TORCH_CHECK(r->position_dtype != KVX_DTYPE_INVALID && positions.dim() == 1 && positions.is_contiguous() &&
                  positions.numel() == tokens,
              "positions must hold one int32 or int64 per token");
  TORCH_CHECK(inv_freq.scalar_type() == at::ScalarType::Double && inv_freq.dim() == 1 && inv_freq.is_contiguous(),
              "inv_freq must be a contiguous float64 vector");
  r->rotary_dim = static_cast<uint32_t>(2 * inv_freq.numel());
  r->flags = (interleaved ? KVX_ROTARY_INTERLEAVED : 0) | (inverse ? KVX_ROTARY_INVERSE : 0);
  r->positions = positions.data_ptr();
  r->inv_freq = inv_freq.data_ptr<double>();
  r->factor = factor;
  for (kvx_tensor_desc_t *t : {&r->query, &r->query_out, &r->key, &r->key_out}) t->size = sizeof(*t);
}

void rotary_embedding(const torch::Tensor &query, const torch::Tensor &key, const torch::Tensor &positions,
                      const torch::Tensor &inv_freq, bool interleaved, double factor, bool inverse, torch::Tensor &query_out,
                      torch::Tensor &key_out) {
  TORCH_CHECK(query.is_cuda() && query.dim() == 3, "query must be a [tokens, heads, head_dim] CUDA tensor");
  const kvx_dtype_t io = float_code(query.scalar_type());
  TORCH_CHECK(io != KVX_DTYPE_INVALID, "unsupported query dtype");
  TORCH_CHECK(query_out.sizes() == query.sizes() && query_out.scalar_type() == query.scalar_type() &&
                  query_out.device() == query.device(),
              "query_out must match query");
  const at::cuda::OptionalCUDAGuard guard(at::device_of(query));
  kvx_rotary_desc_t r;
  describe_rotary(&r, positions, inv_freq, interleaved, factor, inverse, query.size(0), query.device());
  describe(&r.query, query, io, KVX_LAYOUT_INVALID);
  describe(&r.query_out, query_out, io, KVX_LAYOUT_INVALID);
  if (key.dim() == 3) {
    TORCH_CHECK(key.device() == query.device() && key.scalar_type() == query.scalar_type() && key.size(0) == query.size(0) &&
                    key.size(2) == query.size(2),
                "key must match query in device, dtype, tokens and head_dim");
    TORCH_CHECK(key_out.sizes() == key.sizes() && key_out.scalar_type() == key.scalar_type() && key_out.device() == key.device(),
                "key_out must match key");
    describe(&r.key, key, io, KVX_LAYOUT_INVALID);
    describe(&r.key_out, key_out, io, KVX_LAYOUT_INVALID);
  }
  const kvx_status_t status = kvx_launch_rotary(&r, current_stream());
  TORCH_CHECK(status == KVX_STATUS_OK, "kvx rotary failed with status=", static_cast<int>(status));
}

void rotary_and_cache(const torch::Tensor &query, const torch::Tensor &key, const torch::Tensor &value,
                      const torch::Tensor &positions, const torch::Tensor &inv_freq, torch::Tensor &key_cache,
                      torch::Tensor &value_cache, const torch::Tensor &slot_mapping, bool interleaved, double factor,
                      torch::Tensor &query_out, const std::string &kv_cache_dtype, const torch::Tensor &k_scale,
                      const torch::Tensor &v_scale) {
  TORCH_CHECK(key.is_cuda() && value.is_cuda() && query.is_cuda(), "query/key/value must be CUDA tensors");
  TORCH_CHECK(query.dim() == 3 && key.dim() == 3 && value.sizes() == key.sizes(), "query/key/value must be [tokens, heads, head_dim]");
  TORCH_CHECK(query.size(0) == key.size(0) && query.size(2) == key.size(2), "query and key must match in tokens and head_dim");
  const kvx_dtype_t io = float_code(key.scalar_type());
  TORCH_CHECK(io != KVX_DTYPE_INVALID && value.scalar_type() == key.scalar_type() && query.scalar_type() == key.scalar_type(),
              "query/key/value must share a float dtype");
  TORCH_CHECK(query_out.sizes() == query.sizes() && query_out.scalar_type() == query.scalar_type(), "query_out must match query");
  for (const torch::Tensor *t : {&key, &value, static_cast<const torch::Tensor *>(&key_cache), static_cast<const torch::Tensor *>(&value_cache),
                                 &slot_mapping, static_cast<const torch::Tensor *>(&query_out)})
    TORCH_CHECK(t->device() == query.device(), "all tensors must be on the query's device");
  const kvx_dtype_t slot_dtype = index_code(slot_mapping.scalar_type());
  TORCH_CHECK(slot_dtype != KVX_DTYPE_INVALID && slot_mapping.dim() == 1 && slot_mapping.is_contiguous(),
              "slot_mapping must be a contiguous int32 or int64 vector");
  // rows behind the last slot (a batch padded to a fixed size) are turned, but not cached
  const int64_t tokens = slot_mapping.numel(), rows = key.size(0), heads = key.size(1), dim = key.size(2);
  TORCH_CHECK(tokens <= rows, "key/value hold fewer tokens than slot_mapping");
  const at::cuda::OptionalCUDAGuard guard(at::device_of(query));
  kvx_cache_desc_t cache;
  describe_cache(&cache, key_cache, value_cache, kv_cache_dtype, heads, dim);
  kvx_write_desc_t write;
  std::memset(&write, 0, sizeof(write));
  write.size = sizeof(write);
  write.io.size = sizeof(write.io);
  write.io.num_tokens = static_cast<uint32_t>(tokens);
  write.io.num_kv_heads = static_cast<uint32_t>(heads);
  write.io.head_dim = static_cast<uint32_t>(dim);
  describe(&write.io.key, key, io, KVX_LAYOUT_INVALID);
  describe(&write.io.value, value, io, KVX_LAYOUT_INVALID);
  write.io.key.shape[0] = write.io.value.shape[0] = tokens;
  write.slots.size = sizeof(write.slots);
  write.slots.dtype = slot_dtype;
  write.slots.token_count = static_cast<uint32_t>(tokens);
  write.slots.invalid_slot = -1;
  write.slots.slots = slot_mapping.data_ptr();
  describe_scale(&write.k_scale_desc, k_scale, heads);
  describe_scale(&write.v_scale_desc, v_scale, heads);
  kvx_rotary_desc_t r;
  describe_rotary(&r, positions, inv_freq, interleaved, factor, false, rows, query.device());
  if (query.numel() > 0) {
    describe(&r.query, query, io, KVX_LAYOUT_INVALID);
    describe(&r.query_out, query_out, io, KVX_LAYOUT_INVALID);
    r.query.shape[0] = r.query_out.shape[0] = tokens;
  }
  kvx_status_t status = kvx_launch_rotary_write_kv(&cache, &write, &r, current_stream());
  TORCH_CHECK(status == KVX_STATUS_OK, "kvx rotary write failed with status=", static_cast<int>(status));
  if (tokens == rows || query.numel() == 0) return;
  const torch::Tensor rest = query.narrow(0, tokens, rows - tokens), rest_out = query_out.narrow(0, tokens, rows - tokens),
                      rest_at = positions.narrow(0, tokens, rows - tokens);
  describe_rotary(&r, rest_at, inv_freq, interleaved, factor, false, rows - tokens, query.device());
  describe(&r.query, rest, io, KVX_LAYOUT_INVALID);
  describe(&r.query_out, rest_out, io, KVX_LAYOUT_INVALID);
  status = kvx_launch_rotary(&r, current_stream());
  TORCH_CHECK(status == KVX_STATUS_OK, "kvx rotary failed with status=", static_cast<int>(status));
}

// Page upkeep (include/kvx_pages_ops.h).  Whole pages are moved, so a 4-D tensor is described with
// its axes as they are, whatever they mean; a 5-D one as packed pages.
void describe_any_pages(kvx_cache_desc_t *c, const torch::Tensor &k, const torch::Tensor &v) {
  TORCH_CHECK(k.is_cuda() && v.is_cuda() && (k.dim() == 4 || k.dim() == 5) && (v.dim() == 4 || v.dim() == 5),
              "cache tensors must be 4-D or 5-D CUDA tensors");
  TORCH_CHECK(k.scalar_type() == v.scalar_type() && k.size(0) == v.size(0), "key/value cache mismatch");
  kvx_dtype_t code = float_code(k.scalar_type());
  if (code == KVX_DTYPE_INVALID && k.element_size() == 1) code = KVX_DTYPE_F8_E4M3;  // bytes
  TORCH_CHECK(code != KVX_DTYPE_INVALID, "KVX cache: unsupported cache dtype");
  TORCH_CHECK(k.dim() == v.dim() && k.sizes() == v.sizes(), "key/value cache shape mismatch");
  std::memset(c, 0, sizeof(*c));
  c->size = sizeof(*c);
  c->num_blocks = static_cast<uint32_t>(k.size(0));
  const bool packed = k.dim() == 5;
  c->block_size = static_cast<uint32_t>(packed ? k.size(3) : k.size(1));
  c->num_kv_heads = static_cast<uint32_t>(packed ? k.size(1) : k.size(2));
  c->head_dim = static_cast<uint32_t>(packed ? k.size(2) * k.size(4) : k.size(3));
  const kvx_layout_t layout = packed ? KVX_LAYOUT_BLOCK_HND_PACKED : KVX_LAYOUT_BLOCK_NHD;
  describe(&c->k, k, code, layout);
  describe(&c->v, v, code, layout);
  c->pool.size = sizeof(c->pool);
}

void copy_pages(std::vector<torch::Tensor> key_caches, std::vector<torch::Tensor> value_caches, const torch::Tensor &src,
                const torch::Tensor &dst) {
  TORCH_CHECK(key_caches.size() == value_caches.size() && !key_caches.empty(), "one value cache per key cache");
  const kvx_dtype_t idx = index_code(src.scalar_type());
  TORCH_CHECK(idx != KVX_DTYPE_INVALID && src.dim() == 1 && src.is_contiguous() && dst.is_contiguous() && dst.sizes() == src.sizes() &&
                  dst.scalar_type() == src.scalar_type(),
              "src and dst must be matching contiguous int32 or int64 vectors");
  TORCH_CHECK(src.is_cuda() && dst.device() == src.device(), "src and dst must be on one CUDA device");
  std::vector<kvx_cache_desc_t> caches(key_caches.size());
  for (size_t i = 0; i < caches.size(); ++i) {
    TORCH_CHECK(key_caches[i].device() == src.device() && value_caches[i].device() == src.device(),
                "caches must be on the device of the page numbers");
    describe_any_pages(&caches[i], key_caches[i], value_caches[i]);
  }
  const at::cuda::OptionalCUDAGuard guard(at::device_of(src));
  const size_t need = kvx_copy_pages_workspace_bytes(static_cast<uint32_t>(src.numel()));
  torch::Tensor scratch;
  if (need > 0) scratch = torch::empty({static_cast<int64_t>(need)}, src.options().dtype(torch::kUInt8));
  const kvx_status_t status =
      kvx_launch_copy_pages(caches.data(), static_cast<uint32_t>(caches.size()), src.data_ptr(), dst.data_ptr(), idx,
                            static_cast<uint32_t>(src.numel()), need > 0 ? scratch.data_ptr() : nullptr, need, current_stream());
  TORCH_CHECK(status == KVX_STATUS_OK, "kvx page copy failed with status=", static_cast<int>(status));
}

void check_refs(const torch::Tensor &refs, const torch::Tensor &table) {
  TORCH_CHECK(refs.scalar_type() == at::ScalarType::Int && refs.dim() == 1 && refs.is_contiguous() && refs.device() == table.device(),
              "page_refs must be a contiguous int32 vector on the table's device");
}

void check_rows(const torch::Tensor &rows, const torch::Tensor &table, const char *name) {
  TORCH_CHECK(rows.scalar_type() == table.scalar_type() && rows.dim() == 1 && rows.is_contiguous() && rows.device() == table.device(),
              name, " must be a contiguous vector of the table's dtype on its device");
}

void free_sequences(torch::Tensor &block_table, torch::Tensor &seq_lens, torch::Tensor &page_refs, const torch::Tensor &rows) {
  kvx_block_table_t t;
  kvx_seq_lens_t l;
  describe_table(&t, block_table);
  describe_lens(&l, seq_lens, block_table);
  check_refs(page_refs, block_table);
  check_rows(rows, block_table, "rows");
  const at::cuda::OptionalCUDAGuard guard(at::device_of(block_table));
  const kvx_status_t status = kvx_launch_free_sequences(&t, &l, page_refs.data_ptr<int32_t>(), static_cast<uint32_t>(page_refs.numel()),
                                                        rows.data_ptr(), static_cast<uint32_t>(rows.numel()), current_stream());
  TORCH_CHECK(status == KVX_STATUS_OK, "kvx sequence free failed with status=", static_cast<int>(status));
}

std::tuple<torch::Tensor, torch::Tensor> fork_sequences(torch::Tensor &block_table, torch::Tensor &seq_lens, torch::Tensor &page_refs,
                                                        const torch::Tensor &parents, const torch::Tensor &children,
                                                        int64_t block_size) {
  kvx_block_table_t t;
  kvx_seq_lens_t l;
  describe_table(&t, block_table);
  describe_lens(&l, seq_lens, block_table);
  check_refs(page_refs, block_table);
  check_rows(parents, block_table, "parents");
  check_rows(children, block_table, "children");
  TORCH_CHECK(parents.numel() == children.numel(), "one child per parent");
  TORCH_CHECK(block_size > 0 && block_size <= INT32_MAX, "block_size must be positive");
  const at::cuda::OptionalCUDAGuard guard(at::device_of(block_table));
  const int64_t n = parents.numel();
  torch::Tensor src = torch::empty({n}, parents.options()), dst = torch::empty({n}, parents.options());
  const size_t need = kvx_fork_workspace_bytes(static_cast<uint32_t>(n));
  torch::Tensor scratch = torch::empty({static_cast<int64_t>(need)}, parents.options().dtype(torch::kUInt8));
  const kvx_status_t status = kvx_launch_fork_sequences(
      &t, &l, page_refs.data_ptr<int32_t>(), static_cast<uint32_t>(page_refs.numel()), static_cast<uint32_t>(block_size),
      parents.data_ptr(), children.data_ptr(), static_cast<uint32_t>(n), src.data_ptr(), dst.data_ptr(), scratch.data_ptr(), need,
      current_stream());
  TORCH_CHECK(status == KVX_STATUS_OK, "kvx sequence fork failed with status=", static_cast<int>(status));
  return {src, dst};
}

std::tuple<torch::Tensor, torch::Tensor> compact_pages(torch::Tensor &block_table, torch::Tensor &page_refs) {
  kvx_block_table_t t;
  describe_table(&t, block_table);
  check_refs(page_refs, block_table);
  const at::cuda::OptionalCUDAGuard guard(at::device_of(block_table));
  const int64_t n = page_refs.numel() / 2;
  torch::Tensor src = torch::empty({std::max<int64_t>(n, 1)}, block_table.options()),
                dst = torch::empty({std::max<int64_t>(n, 1)}, block_table.options());
  const kvx_status_t status = kvx_launch_compact_pages(&t, page_refs.data_ptr<int32_t>(), static_cast<uint32_t>(page_refs.numel()),
                                                       src.data_ptr(), dst.data_ptr(), current_stream());
  TORCH_CHECK(status == KVX_STATUS_OK, "kvx page compaction failed with status=", static_cast<int>(status));
  return {src, dst};
}

}  // namespace

TORCH_LIBRARY(kvx_b200, m) {
  m.def(
      "reshape_and_cache_flash_kvx(Tensor key, Tensor value, Tensor! key_cache, Tensor! value_cache,"
      " Tensor slot_mapping, str kv_cache_dtype, Tensor k_scale, Tensor v_scale) -> ()");
  m.def(
      "gather_kv(Tensor key_cache, Tensor value_cache, Tensor block_table, Tensor seq_lens, Tensor! key_out,"
      " Tensor! value_out, str kv_cache_dtype, Tensor k_scale, Tensor v_scale) -> ()");
  m.def(
      "paged_attention_decode(Tensor! out, Tensor query, Tensor key_cache, Tensor value_cache, Tensor block_table,"
      " Tensor seq_lens, float scale, int max_seq_len, int num_kv_heads, Tensor! workspace, str kv_cache_dtype,"
      " Tensor k_scale,"
      " Tensor v_scale) -> ()");
  m.def(
      "paged_attention_chunk(Tensor! out, Tensor query, Tensor key_cache, Tensor value_cache, Tensor block_table,"
      " Tensor seq_lens, Tensor query_indptr, float scale, bool causal, int max_seq_len, int num_kv_heads,"
      " Tensor! workspace, str kv_cache_dtype, Tensor k_scale, Tensor v_scale) -> ()");
  m.def(
      "rotary_embedding(Tensor query, Tensor key, Tensor positions, Tensor inv_freq, bool interleaved, float factor,"
      " bool inverse, Tensor! query_out, Tensor! key_out) -> ()");
  m.def(
      "rotary_and_cache(Tensor query, Tensor key, Tensor value, Tensor positions, Tensor inv_freq, Tensor! key_cache,"
      " Tensor! value_cache, Tensor slot_mapping, bool interleaved, float factor, Tensor! query_out, str kv_cache_dtype,"
      " Tensor k_scale, Tensor v_scale) -> ()");
  m.def("copy_pages(Tensor(a!)[] key_caches, Tensor(b!)[] value_caches, Tensor src, Tensor dst) -> ()");
  m.def("free_sequences(Tensor! block_table, Tensor! seq_lens, Tensor! page_refs, Tensor rows) -> ()");
  m.def(
      "fork_sequences(Tensor! block_table, Tensor! seq_lens, Tensor! page_refs, Tensor parents, Tensor children,"
      " int block_size) -> (Tensor, Tensor)");
  m.def("compact_pages(Tensor! block_table, Tensor! page_refs) -> (Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(kvx_b200, CUDA, m) {
  m.impl("reshape_and_cache_flash_kvx", &reshape_and_cache_flash_kvx);
  m.impl("gather_kv", &gather_kv);
  m.impl("paged_attention_decode", &paged_attention_decode);
  m.impl("paged_attention_chunk", &paged_attention_chunk);
  m.impl("rotary_embedding", &rotary_embedding);
  m.impl("rotary_and_cache", &rotary_and_cache);
  m.impl("copy_pages", &copy_pages);
  m.impl("free_sequences", &free_sequences);
  m.impl("fork_sequences", &fork_sequences);
  m.impl("compact_pages", &compact_pages);
}
