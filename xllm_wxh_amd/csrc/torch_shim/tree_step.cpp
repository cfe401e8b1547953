#include "tree_step.h"

#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <hip/hip_runtime_api.h>

#include <limits>

#include "../../../include/xllm_hip_paged_kv.h"
#include "stream_scratch.h"

namespace xllm::kernel::hip {
namespace {

using Maybe = std::optional<torch::Tensor>;

#define TREE_REQUIRE(cond, ...)                                                              \
  do {                                                                                       \
    if (!(cond)) throw StatusError(XLLM_HIP_INVALID_ARGUMENT, c10::str(__VA_ARGS__));        \
  } while (0)

void check(int status) {
  if (status != XLLM_HIP_OK) throw StatusError(status, xllm_hip_last_error());
}

bool has(const Maybe& t) { return t.has_value() && t->defined(); }

int32_t dtype_code(const torch::Tensor& t) {
  switch (t.scalar_type()) {
    case torch::kBFloat16:
      return XLLM_HIP_BF16;
    case torch::kHalf:
      return XLLM_HIP_FP16;
    case torch::kFloat:
      return XLLM_HIP_FP32;
    case torch::kFloat8_e4m3fn:
      return XLLM_HIP_FP8_E4M3;
    case torch::kChar:
      return XLLM_HIP_INT8;
    default:
      throw StatusError(XLLM_HIP_INVALID_ARGUMENT, c10::str("unsupported dtype ", t.scalar_type()));
  }
}

int32_t as_i32(int64_t v, const char* name) {
  TREE_REQUIRE(v >= std::numeric_limits<int32_t>::min() && v <= std::numeric_limits<int32_t>::max(), name, " ", v, " does not fit 32 bits");
  return (int32_t)v;
}

void vec32(const torch::Tensor& t, int64_t n, const char* name) {
  TREE_REQUIRE(t.scalar_type() == torch::kInt && t.dim() == 1 && t.size(0) == n && t.is_contiguous(), name,
               " must be a contiguous int32 vector of ", n, " entries");
}
void vec32(const Maybe& t, int64_t n, const char* name) {
  if (has(t)) vec32(*t, n, name);
}

// int32 [rows, width], rows contiguous
void matrix32(const torch::Tensor& t, const char* name) {
  TREE_REQUIRE(t.scalar_type() == torch::kInt && t.dim() == 2 && t.size(1) >= 1 && (t.stride(1) == 1 || t.size(1) == 1), name,
               " must be int32 [rows, width], rows contiguous");
}
// (the row stride of a one-row tensor is arbitrary in torch: such a tensor is its one row)
int64_t row_stride(const torch::Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }

const int32_t* i32(const Maybe& t) { return has(t) ? (const int32_t*)t->data_ptr() : nullptr; }
int32_t* i32_out(const Maybe& t) { return has(t) ? (int32_t*)t->data_ptr() : nullptr; }

void on(const c10::Device& dev, const torch::Tensor& t) {
  TREE_REQUIRE(t.device() == dev, "the tensors must live on one GPU");
}
void on(const c10::Device& dev, const Maybe& t) {
  if (has(t)) on(dev, *t);
}
// Every tensor lives on the GPU the first lives on, which is made current for the call.
template <class... T>
c10::Device one_gpu(const torch::Tensor& first, const T&... rest) {
  TREE_REQUIRE(first.is_cuda(), "the tensors must live on the GPU");
  const c10::Device dev = first.device();
  (on(dev, rest), ...);
  return dev;
}
xllm_hip_stream_t stream_of(const c10::Device& dev) {
  return (xllm_hip_stream_t)c10::hip::getCurrentHIPStream(dev.index()).stream();
}

xllm_hip_kv_cache make_cache(const torch::Tensor& k, const torch::Tensor& v, const Maybe& k_scale, const Maybe& v_scale, bool nhd) {
  TREE_REQUIRE(k.dim() == 4, "cache must be 4-D, got ", k.dim(), "-D");
  TREE_REQUIRE(k.stride(3) == 1 || k.size(3) == 1, "head_dim of k_cache must be contiguous");
  TREE_REQUIRE(v.sizes() == k.sizes() && v.strides() == k.strides() && v.scalar_type() == k.scalar_type(),
               "v_cache must match k_cache in shape, dtype and strides");
  const int head = nhd ? 2 : 1, slot = nhd ? 1 : 2;
  xllm_hip_kv_cache c{};
  c.k_cache = k.data_ptr();
  c.v_cache = v.data_ptr();
  c.num_blocks = k.size(0);
  c.num_kv_heads = as_i32(k.size(head), "num_kv_heads");
  c.block_size = as_i32(k.size(slot), "block_size");
  c.head_dim = as_i32(k.size(3), "head_dim");
  c.dtype = dtype_code(k);
  c.stride_block = k.stride(0);
  c.stride_head = k.stride(head);
  c.stride_slot = k.stride(slot);
  TREE_REQUIRE(has(k_scale) == has(v_scale), "the k and v cache scales go together");
  if (has(k_scale)) {
    const torch::Tensor& ks = *k_scale;
    TREE_REQUIRE(ks.scalar_type() == torch::kFloat && ks.dim() == 3 && ks.size(0) == k.size(0) && ks.size(1) == k.size(1) &&
                     ks.size(2) == k.size(2),
                 "k_cache_scale must be float32, the cache's shape minus head_dim");
    TREE_REQUIRE(v_scale->sizes() == ks.sizes() && v_scale->strides() == ks.strides() && v_scale->scalar_type() == torch::kFloat,
                 "v_cache_scale must match k_cache_scale");
    c.k_scale = (float*)ks.data_ptr();
    c.v_scale = (float*)v_scale->data_ptr();
    c.scale_stride_block = ks.stride(0);
    c.scale_stride_head = ks.stride(head);
    c.scale_stride_slot = ks.stride(slot);
  }
  return c;
}

// int64 [rows, words], rows contiguous
void mask_words(const torch::Tensor& t, int64_t rows) {
  TREE_REQUIRE(t.scalar_type() == torch::kLong && t.dim() == 2 && t.size(0) == rows && t.size(1) >= 1 &&
                   (t.stride(1) == 1 || t.size(1) == 1),
               "tree_mask must be int64 [", rows, ", words], rows contiguous");
}

// One buffer per (device, stream) for eager calls, grown to the largest call's need: the buffer that is outgrown goes
// back to torch's allocator, which hands it out again in the order of the stream.
StreamScratch<torch::Tensor>& tree_scratch() {
  static auto* scratch = new StreamScratch<torch::Tensor>();  // (outlives the allocator's teardown)
  return *scratch;
}

bool is_capturing(xllm_hip_stream_t stream) {
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  (void)hipStreamIsCapturing((hipStream_t)stream, &status);
  return status != hipStreamCaptureStatusNone;
}

}  // namespace

void build_step_indices(const torch::Tensor& cached_lens, const torch::Tensor& block_pool, int64_t block_size,
                        const torch::Tensor& block_table, const torch::Tensor& seq_lens, const torch::Tensor& q_indptr,
                        const torch::Tensor& slot_mapping, const torch::Tensor& positions, const Maybe& new_lens, int64_t q_per_seq,
                        const Maybe& request_ids, const Maybe& held_blocks, const Maybe& free_blocks, const Maybe& free_head,
                        const Maybe& held_blocks_out, const Maybe& free_head_out, const Maybe& paged_kv_indptr,
                        const Maybe& paged_kv_indices, const Maybe& paged_kv_last_page_len) {
  const int64_t batch = cached_lens.numel();
  vec32(cached_lens, batch, "cached_lens");
  vec32(seq_lens, batch, "seq_lens");
  vec32(q_indptr, batch + 1, "q_indptr");
  vec32(new_lens, batch, "new_lens");
  vec32(request_ids, batch, "request_ids");
  vec32(held_blocks, batch, "held_blocks");
  vec32(held_blocks_out, batch, "held_blocks_out");
  vec32(paged_kv_last_page_len, batch, "paged_kv_last_page_len");
  matrix32(block_pool, "block_pool");
  matrix32(block_table, "block_table");
  TREE_REQUIRE(block_pool.size(0) >= 1, "block_pool holds no rows");
  TREE_REQUIRE(has(request_ids) || block_pool.size(0) >= batch, "block_pool has ", block_pool.size(0), " rows for ", batch, " sequences");
  TREE_REQUIRE(block_table.size(0) == batch, "block_table has ", block_table.size(0), " rows for ", batch, " sequences");
  vec32(slot_mapping, slot_mapping.numel(), "slot_mapping");
  TREE_REQUIRE((positions.scalar_type() == torch::kInt || positions.scalar_type() == torch::kLong) && positions.dim() == 1 &&
                   positions.is_contiguous() && positions.numel() == slot_mapping.numel(),
               "positions must be int32 or int64, one entry per slot");
  TREE_REQUIRE(has(free_blocks) == has(free_head), "free_blocks and free_head go together");
  TREE_REQUIRE(!has(free_blocks) || has(held_blocks), "free_blocks needs held_blocks");
  TREE_REQUIRE(has(held_blocks) == has(held_blocks_out) && has(held_blocks) == has(free_head_out),
               "held_blocks, held_blocks_out and free_head_out go together");
  if (has(free_blocks)) vec32(free_blocks, free_blocks->numel(), "free_blocks");
  vec32(free_head, 1, "free_head");
  vec32(free_head_out, 2, "free_head_out");
  TREE_REQUIRE(has(paged_kv_indptr) == has(paged_kv_indices) && has(paged_kv_indptr) == has(paged_kv_last_page_len),
               "the paged_kv arrays go together");
  vec32(paged_kv_indptr, batch + 1, "paged_kv_indptr");
  if (has(paged_kv_indices)) vec32(paged_kv_indices, paged_kv_indices->numel(), "paged_kv_indices");
  const c10::Device dev =
      one_gpu(cached_lens, block_pool, block_table, seq_lens, q_indptr, slot_mapping, positions, new_lens, request_ids, held_blocks,
              free_blocks, free_head, held_blocks_out, free_head_out, paged_kv_indptr, paged_kv_indices, paged_kv_last_page_len);
  xllm_hip_step_args a{};
  a.cached_lens = (const int32_t*)cached_lens.data_ptr();
  a.new_lens = i32(new_lens);
  a.request_ids = i32(request_ids);
  a.held_blocks = i32(held_blocks);
  a.block_pool = (int32_t*)block_pool.data_ptr();
  a.pool_stride = row_stride(block_pool);
  a.free_blocks = i32(free_blocks);
  a.free_head = i32(free_head);
  a.num_free = has(free_blocks) ? as_i32(free_blocks->numel(), "free_blocks") : 0;
  a.pool_rows = as_i32(block_pool.size(0), "block_pool rows");
  a.pool_width = as_i32(block_pool.size(1), "block_pool width");
  a.batch = as_i32(batch, "batch");
  a.q_per_seq = as_i32(q_per_seq, "q_per_seq");
  a.block_size = as_i32(block_size, "block_size");
  a.table_width = as_i32(block_table.size(1), "block_table width");
  a.positions_int32 = positions.scalar_type() == torch::kInt;
  a.block_table = (int32_t*)block_table.data_ptr();
  a.table_stride = row_stride(block_table);
  a.seq_lens = (int32_t*)seq_lens.data_ptr();
  a.q_indptr = (int32_t*)q_indptr.data_ptr();
  a.slot_mapping = (int32_t*)slot_mapping.data_ptr();
  a.positions = positions.data_ptr();
  a.num_rows = slot_mapping.numel();
  a.kv_indptr = i32_out(paged_kv_indptr);
  a.kv_indices = i32_out(paged_kv_indices);
  a.kv_last_page_len = i32_out(paged_kv_last_page_len);
  a.kv_indices_capacity = has(paged_kv_indices) ? paged_kv_indices->numel() : 0;
  a.held_blocks_out = i32_out(held_blocks_out);
  a.free_head_out = i32_out(free_head_out);
  const c10::DeviceGuard guard(dev);
  check(xllm_hip_build_step_indices(&a, stream_of(dev)));
}

void tree_masks(const torch::Tensor& parents, const torch::Tensor& tree_mask, const Maybe& positions, const Maybe& base,
                const Maybe& q_indptr, int64_t q_per_seq) {
  const int64_t rows = parents.numel();
  vec32(parents, rows, "parents");
  TREE_REQUIRE(has(q_indptr) != (q_per_seq >= 0), "either q_indptr or q_per_seq");
  int64_t batch;
  if (has(q_indptr)) {
    TREE_REQUIRE(q_indptr->numel() >= 1, "q_indptr must be [batch + 1]");
    vec32(q_indptr, q_indptr->numel(), "q_indptr");
    batch = q_indptr->numel() - 1;
    q_per_seq = 0;
  } else {
    TREE_REQUIRE(q_per_seq >= 1 && rows % q_per_seq == 0, "rows not divisible by q_per_seq");
    batch = rows / q_per_seq;
  }
  mask_words(tree_mask, rows);
  int64_t axes = 1, axis_stride = 0;
  if (has(positions)) {
    const torch::Tensor& p = *positions;
    TREE_REQUIRE((p.scalar_type() == torch::kInt || p.scalar_type() == torch::kLong) && (p.dim() == 1 || p.dim() == 2) &&
                     p.size(-1) == rows && (rows <= 1 || p.stride(-1) == 1),
                 "positions must be int32 or int64 [rows] or [axes, rows]");
    if (p.dim() == 2) {
      axes = p.size(0);
      axis_stride = row_stride(p);
    }
  }
  vec32(base, batch, "base");
  const c10::Device dev = one_gpu(parents, tree_mask, positions, base, q_indptr);
  const c10::DeviceGuard guard(dev);
  check(xllm_hip_tree_masks((const int32_t*)parents.data_ptr(), i32(q_indptr), i32(base), as_i32(batch, "batch"),
                            as_i32(q_per_seq, "q_per_seq"), rows, (uint64_t*)tree_mask.data_ptr(), row_stride(tree_mask),
                            as_i32(tree_mask.size(1), "mask words"), has(positions) ? positions->data_ptr() : nullptr,
                            has(positions) && positions->scalar_type() == torch::kInt, as_i32(axes, "axes"), axis_stride, stream_of(dev)));
}

void mrope_kv_write(const torch::Tensor& qkv, int64_t num_heads_q, int64_t num_heads_kv, int64_t head_dim,
                    const torch::Tensor& cos_sin_cache, const torch::Tensor& position_ids, const std::vector<int64_t>& mrope_section,
                    const Maybe& k_cache, const Maybe& v_cache, const Maybe& slot_mapping, bool mrope_interleaved, const Maybe& q_weight,
                    const Maybe& k_weight, double eps, bool interleaved, bool round_each_op, const Maybe& k_cache_scale,
                    const Maybe& v_cache_scale, bool nhd) {
  TREE_REQUIRE(qkv.dim() == 2 && qkv.stride(1) == 1, "qkv must be 2-D, rows contiguous");
  const int64_t tokens = qkv.size(0);
  TREE_REQUIRE(num_heads_q >= 0 && num_heads_kv >= 0 && head_dim >= 1 && qkv.size(1) >= (num_heads_q + 2 * num_heads_kv) * head_dim,
               "qkv rows do not hold the heads");
  TREE_REQUIRE((position_ids.scalar_type() == torch::kLong || position_ids.scalar_type() == torch::kInt) && position_ids.dim() == 2 &&
                   position_ids.size(1) == tokens && (tokens <= 1 || position_ids.stride(1) == 1),
               "position_ids must be int64 or int32 [axes, tokens], rows contiguous");
  TREE_REQUIRE((int64_t)mrope_section.size() == position_ids.size(0) && mrope_section.size() >= 1 && mrope_section.size() <= 4,
               "mrope_section needs one entry for each of 1 to 4 axes");
  TREE_REQUIRE(cos_sin_cache.dim() == 2 && cos_sin_cache.is_contiguous(), "cos_sin_cache must be [max_position, rotary_dim]");
  TREE_REQUIRE(has(q_weight) == has(k_weight), "q_weight and k_weight go together");
  for (const Maybe* w : {&q_weight, &k_weight}) {
    TREE_REQUIRE(!has(*w) || ((*w)->scalar_type() == qkv.scalar_type() && (*w)->dim() == 1 && (*w)->numel() == head_dim &&
                              (*w)->is_contiguous()),
                 "norm weights must be [head_dim] of qkv's dtype");
  }
  xllm_hip_kv_cache cache{};
  if (has(k_cache)) {
    TREE_REQUIRE(has(v_cache) && has(slot_mapping), "k_cache needs v_cache and slot_mapping");
    vec32(slot_mapping, tokens, "slot_mapping");
    cache = make_cache(*k_cache, *v_cache, k_cache_scale, v_cache_scale, nhd);
  } else {
    TREE_REQUIRE(!has(v_cache) && !has(slot_mapping), "v_cache or slot_mapping given without k_cache");
  }
  xllm_hip_rope_args a{};
  a.qkv = qkv.data_ptr();
  a.token_stride = tokens > 1 ? qkv.stride(0) : qkv.size(1);
  a.num_tokens = tokens;
  a.dtype = dtype_code(qkv);
  a.num_q_heads = as_i32(num_heads_q, "num_heads_q");
  a.num_k_heads = a.num_v_heads = as_i32(num_heads_kv, "num_heads_kv");
  a.head_dim = as_i32(head_dim, "head_dim");
  a.rotary_dim = as_i32(cos_sin_cache.size(1), "rotary_dim");
  a.q_weight = has(q_weight) ? q_weight->data_ptr() : nullptr;
  a.k_weight = has(k_weight) ? k_weight->data_ptr() : nullptr;
  a.eps = (float)eps;
  a.cos_sin_dtype = dtype_code(cos_sin_cache);
  a.cos_sin_cache = cos_sin_cache.data_ptr();
  a.max_position = cos_sin_cache.size(0);
  a.positions = position_ids.data_ptr();
  a.positions_int32 = position_ids.scalar_type() == torch::kInt;
  a.interleave = interleaved;
  a.round_each_op = round_each_op;
  xllm_hip_mrope m{};
  m.num_axes = (int32_t)mrope_section.size();
  m.dealt = mrope_interleaved;
  m.axis_stride = row_stride(position_ids);
  for (size_t i = 0; i < mrope_section.size(); ++i) m.sections[i] = as_i32(mrope_section[i], "mrope_section");
  const c10::Device dev = one_gpu(qkv, cos_sin_cache, position_ids, k_cache, v_cache, slot_mapping, q_weight, k_weight, k_cache_scale,
                                  v_cache_scale);
  const c10::DeviceGuard guard(dev);
  check(xllm_hip_mrope_kv_write(&a, &m, has(k_cache) ? &cache : nullptr, i32(slot_mapping), stream_of(dev)));
}

void batch_tree_decode(const torch::Tensor& query, const torch::Tensor& k_cache, const torch::Tensor& v_cache,
                       const torch::Tensor& output, const Maybe& block_table, const Maybe& seq_lens, const torch::Tensor& tree_mask,
                       double scale, const Maybe& q_indptr, int64_t q_per_seq, const Maybe& output_lse, const Maybe& k_cache_quant_scale,
                       const Maybe& v_cache_quant_scale, bool nhd, int64_t max_seq_len, int64_t total_kv_len, const Maybe& workspace,
                       const Maybe& paged_kv_indptr, const Maybe& paged_kv_indices, const Maybe& paged_kv_last_page_len) {
  TREE_REQUIRE(query.dim() == 3 && output.dim() == 3, "query and output must be [tokens, heads, dim]");
  TREE_REQUIRE(q_per_seq >= 1, "q_per_seq (the most query tokens of a sequence) is required");
  const int64_t rows = query.size(0);
  mask_words(tree_mask, rows);
  const bool csr = has(paged_kv_indptr);
  TREE_REQUIRE(csr == has(paged_kv_indices) && csr == has(paged_kv_last_page_len) && csr != has(block_table) && csr != has(seq_lens),
               "either block_table and seq_lens, or csr");
  TREE_REQUIRE(output.sizes() == query.sizes() && output.scalar_type() == query.scalar_type(), "output must match query");
  for (const torch::Tensor* t : {&query, &output}) {
    TREE_REQUIRE((t->stride(2) == 1 || t->size(2) == 1) && (t->stride(1) == t->size(2) || t->size(1) == 1),
                 "query/output heads and head_dim must be contiguous");
  }
  const xllm_hip_kv_cache cache = make_cache(k_cache, v_cache, k_cache_quant_scale, v_cache_quant_scale, nhd);
  TREE_REQUIRE(query.size(2) == cache.head_dim, "query head_dim ", query.size(2), " != cache head_dim ", cache.head_dim);
  xllm_hip_decode_args a{};
  if (has(q_indptr)) {
    TREE_REQUIRE(q_indptr->numel() >= 1, "q_indptr must be [batch + 1]");
    vec32(q_indptr, q_indptr->numel(), "q_indptr");
    a.batch = as_i32(q_indptr->numel() - 1, "batch");
  } else {
    TREE_REQUIRE(rows % q_per_seq == 0, "query tokens not divisible by q_per_seq");
    a.batch = as_i32(rows / q_per_seq, "batch");
  }
  a.q = query.data_ptr();
  a.out = output.data_ptr();
  const int64_t row = query.size(1) * query.size(2);
  a.q_token_stride = rows > 1 ? query.stride(0) : row;
  a.out_token_stride = rows > 1 ? output.stride(0) : row;
  a.q_dtype = dtype_code(query);
  a.q_indptr = i32(q_indptr);
  a.q_per_seq = as_i32(q_per_seq, "q_per_seq");
  a.num_q_heads = as_i32(query.size(1), "num_q_heads");
  a.sm_scale = (float)scale;
  a.window_left = -1;
  if (has(output_lse)) {
    TREE_REQUIRE(output_lse->scalar_type() == torch::kFloat && output_lse->is_contiguous() && output_lse->numel() == rows * query.size(1),
                 "output_lse must be contiguous float32 [tokens, heads]");
    a.lse = (float*)output_lse->data_ptr();
  }
  if (csr) {
    vec32(paged_kv_indptr, (int64_t)a.batch + 1, "paged_kv_indptr");
    vec32(paged_kv_indices, paged_kv_indices->numel(), "paged_kv_indices");
    vec32(paged_kv_last_page_len, a.batch, "paged_kv_last_page_len");
    a.kv_indptr = i32(paged_kv_indptr);
    a.kv_indices = i32(paged_kv_indices);
    a.kv_last_page_len = i32(paged_kv_last_page_len);
  } else {
    matrix32(*block_table, "block_table");
    TREE_REQUIRE(block_table->size(0) == a.batch, "block_table has ", block_table->size(0), " rows for ", a.batch, " sequences");
    vec32(seq_lens, a.batch, "seq_lens");
    a.block_table = i32(block_table);
    a.block_table_stride = row_stride(*block_table);
    a.max_blocks_per_seq = as_i32(block_table->size(1), "block_table width");
    a.seq_lens = i32(seq_lens);
  }
  a.max_seq_len = as_i32(max_seq_len, "max_seq_len");
  a.total_kv_len = total_kv_len;
  const c10::Device dev = one_gpu(query, k_cache, v_cache, output, block_table, seq_lens, tree_mask, q_indptr, output_lse,
                                  k_cache_quant_scale, v_cache_quant_scale, workspace, paged_kv_indptr, paged_kv_indices,
                                  paged_kv_last_page_len);
  if (rows == 0) return;
  const c10::DeviceGuard guard(dev);
  const xllm_hip_stream_t stream = stream_of(dev);
  const auto attend = [&](const torch::Tensor& ws) {
    check(xllm_hip_tree_attention(&cache, &a, (const uint64_t*)tree_mask.data_ptr(), row_stride(tree_mask),
                                  as_i32(tree_mask.size(1), "mask words"), ws.defined() ? ws.data_ptr() : nullptr,
                                  ws.defined() ? (size_t)ws.nbytes() : 0, stream));
  };
  if (has(workspace)) {
    TREE_REQUIRE(workspace->is_contiguous(), "workspace must be contiguous");
    return attend(*workspace);
  }
  const size_t need = xllm_hip_tree_attention_workspace_bytes(a.batch, a.q_per_seq, a.num_q_heads, cache.num_kv_heads, cache.head_dim);
  if (need == 0) return attend(torch::Tensor());
  const auto options = torch::TensorOptions().dtype(torch::kUInt8).device(dev);
  if (is_capturing(stream)) return attend(torch::empty({(int64_t)need}, options));
  const auto held = tree_scratch().hold(dev.index(), stream);  // until both launches are enqueued
  torch::Tensor& ws = *held;
  if (!ws.defined() || (size_t)ws.numel() < need) ws = torch::empty({(int64_t)need}, options);
  attend(ws);
}

void move_accepted_tokens(const torch::Tensor& k_cache, const torch::Tensor& v_cache, const torch::Tensor& block_table,
                          const torch::Tensor& cached_lens, const torch::Tensor& accepted, const torch::Tensor& num_accepted,
                          const Maybe& new_lens, const Maybe& k_cache_scale, const Maybe& v_cache_scale, bool nhd) {
  const int64_t batch = cached_lens.numel();
  vec32(cached_lens, batch, "cached_lens");
  vec32(num_accepted, batch, "num_accepted");
  vec32(new_lens, batch, "new_lens");
  matrix32(block_table, "block_table");
  TREE_REQUIRE(block_table.size(0) == batch, "block_table has ", block_table.size(0), " rows for ", batch, " sequences");
  TREE_REQUIRE(accepted.scalar_type() == torch::kInt && accepted.dim() == 2 && accepted.size(0) == batch &&
                   (accepted.size(1) <= 1 || accepted.stride(1) == 1),
               "accepted must be int32 [batch, width], rows contiguous");
  const xllm_hip_kv_cache cache = make_cache(k_cache, v_cache, k_cache_scale, v_cache_scale, nhd);
  const c10::Device dev = one_gpu(k_cache, v_cache, block_table, cached_lens, accepted, num_accepted, new_lens, k_cache_scale, v_cache_scale);
  const c10::DeviceGuard guard(dev);
  check(xllm_hip_move_accepted_tokens(&cache, i32(block_table), row_stride(block_table), as_i32(block_table.size(1), "block_table width"),
                                      i32(cached_lens), i32(accepted), row_stride(accepted), as_i32(accepted.size(1), "accepted width"),
                                      i32(num_accepted), as_i32(batch, "batch"), i32_out(new_lens), stream_of(dev)));
}

}  // namespace xllm::kernel::hip
