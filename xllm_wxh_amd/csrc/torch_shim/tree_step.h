// libtorch host side of the operators of a speculative step over a tree of drafted tokens (the C ABI's section of that
// name).  They have no counterpart in the reference; names, argument order and error behaviour follow the operators of
// ops_api.h beside them: tensors are only checked and passed on, outputs are pre-allocated by the caller, everything is
// enqueued on torch's current stream of the tensors' device, and a contract violation throws (StatusError, which carries
// the C ABI's status).  The Python functions of ops.py are these.
#pragma once

#include <torch/torch.h>

#include <optional>
#include <string>
#include <vector>

namespace xllm::kernel::hip {

class StatusError : public c10::Error {
 public:
  StatusError(int status, const std::string& message) : c10::Error(c10::SourceLocation{"", "", 0}, message), status_(status) {}
  int status() const { return status_; }

 private:
  int status_;
};

// Cache tensors in the HND logical shape [num_blocks, num_kv_heads, block_size, head_dim] of any strides, or with `nhd`
// as [num_blocks, block_size, num_kv_heads, head_dim]; scales are the shape minus the last dimension.

// xllm_hip_build_step_indices
void build_step_indices(const torch::Tensor& cached_lens,
                        const torch::Tensor& block_pool,
                        int64_t block_size,
                        const torch::Tensor& block_table,
                        const torch::Tensor& seq_lens,
                        const torch::Tensor& q_indptr,
                        const torch::Tensor& slot_mapping,
                        const torch::Tensor& positions,
                        const std::optional<torch::Tensor>& new_lens,
                        int64_t q_per_seq,
                        const std::optional<torch::Tensor>& request_ids,
                        const std::optional<torch::Tensor>& held_blocks,
                        const std::optional<torch::Tensor>& free_blocks,
                        const std::optional<torch::Tensor>& free_head,
                        const std::optional<torch::Tensor>& held_blocks_out,
                        const std::optional<torch::Tensor>& free_head_out,
                        const std::optional<torch::Tensor>& paged_kv_indptr,
                        const std::optional<torch::Tensor>& paged_kv_indices,
                        const std::optional<torch::Tensor>& paged_kv_last_page_len);

// xllm_hip_tree_masks; q_per_seq < 0: q_indptr is given
void tree_masks(const torch::Tensor& parents,
                const torch::Tensor& tree_mask,
                const std::optional<torch::Tensor>& positions,
                const std::optional<torch::Tensor>& base,
                const std::optional<torch::Tensor>& q_indptr,
                int64_t q_per_seq);

// xllm_hip_mrope_kv_write; without k_cache only q and k are rewritten
void mrope_kv_write(const torch::Tensor& qkv,
                    int64_t num_heads_q,
                    int64_t num_heads_kv,
                    int64_t head_dim,
                    const torch::Tensor& cos_sin_cache,
                    const torch::Tensor& position_ids,
                    const std::vector<int64_t>& mrope_section,
                    const std::optional<torch::Tensor>& k_cache,
                    const std::optional<torch::Tensor>& v_cache,
                    const std::optional<torch::Tensor>& slot_mapping,
                    bool mrope_interleaved,
                    const std::optional<torch::Tensor>& q_weight,
                    const std::optional<torch::Tensor>& k_weight,
                    double eps,
                    bool interleaved,
                    bool round_each_op,
                    const std::optional<torch::Tensor>& k_cache_scale,
                    const std::optional<torch::Tensor>& v_cache_scale,
                    bool nhd);

// xllm_hip_tree_attention.  block_table and seq_lens, or the three csr arrays.  Without `workspace` the scratch is one
// buffer per (device, stream), grown to the largest call's need and held while the call's launches are enqueued, so that
// several host threads may use one stream; under stream capture it is memory of the graph's own pool, so that no two
// graphs, and no graph and no eager call, share one.  A `workspace` of the caller's serves one call at a time.
void batch_tree_decode(const torch::Tensor& query,
                       const torch::Tensor& k_cache,
                       const torch::Tensor& v_cache,
                       const torch::Tensor& output,
                       const std::optional<torch::Tensor>& block_table,
                       const std::optional<torch::Tensor>& seq_lens,
                       const torch::Tensor& tree_mask,
                       double scale,
                       const std::optional<torch::Tensor>& q_indptr,
                       int64_t q_per_seq,
                       const std::optional<torch::Tensor>& output_lse,
                       const std::optional<torch::Tensor>& k_cache_quant_scale,
                       const std::optional<torch::Tensor>& v_cache_quant_scale,
                       bool nhd,
                       int64_t max_seq_len,
                       int64_t total_kv_len,
                       const std::optional<torch::Tensor>& workspace,
                       const std::optional<torch::Tensor>& paged_kv_indptr,
                       const std::optional<torch::Tensor>& paged_kv_indices,
                       const std::optional<torch::Tensor>& paged_kv_last_page_len);

// xllm_hip_move_accepted_tokens
void move_accepted_tokens(const torch::Tensor& k_cache,
                          const torch::Tensor& v_cache,
                          const torch::Tensor& block_table,
                          const torch::Tensor& cached_lens,
                          const torch::Tensor& accepted,
                          const torch::Tensor& num_accepted,
                          const std::optional<torch::Tensor>& new_lens,
                          const std::optional<torch::Tensor>& k_cache_scale,
                          const std::optional<torch::Tensor>& v_cache_scale,
                          bool nhd);

}  // namespace xllm::kernel::hip
