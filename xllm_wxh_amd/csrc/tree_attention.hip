// Paged attention of drafted trees for gfx950: the verify step of tree speculation.  Every query token sees the whole
// context and, among the drafted tokens at the end of its sequence, those its mask names (see
// xllm_hip_tree_attention in the header for the exact statement).
//
//   x_t = scale * q.k_t,   out = sum_t 2^(x_t - m) v_t / sum_t 2^(x_t - m)      (x in units of log 2)
//
// Long sequences are cut into chunks of whole tiles, a workgroup each; a chunk leaves a normalised partial and its
// base-2 log-sum-exp, and tree_merge_kernel joins them.  How a sequence is cut follows from its own length, read on
// the device, and two numbers from the host (tokens per chunk, chunks a sequence may have), so any hints, stale ones
// of a captured graph included, give the same result.
#include "device_utils.h"
#include "host_utils.h"
#include "tree_generic.h"
#include "tree_params.h"

#include <math.h>

namespace xllm_hip {

constexpr int kTreeMaxNodes = 512;
constexpr int kTreeMaxWords = 8;
constexpr int kTreeMaxSlots = 64;    // chunks per sequence: a lane each in the merge
constexpr int kTreeMinChunk = 256;   // tokens: a shorter chunk costs more in its partial than it saves

// Chunks a sequence may have: enough that the launch has 2048 items, no more than the merge holds, and no more than
// 64 MiB of partials.  Sizes only, so that one workspace serves every step of these sizes.
static int tree_slots(int64_t batch, int64_t n, int64_t hq, int64_t hkv, int64_t d) {
  const int64_t items = batch * hkv;
  int64_t s = items > 0 ? (2048 + items - 1) / items : 1;
  const int64_t row_bytes = batch * n * hq * (d + 1) * 4;
  const int64_t fit = row_bytes > 0 ? ((int64_t)64 << 20) / row_bytes : kTreeMaxSlots;
  s = s < fit ? s : fit;
  s = s < kTreeMaxSlots ? s : kTreeMaxSlots;
  return s > 1 ? (int)s : 1;
}

static size_t tree_lse_bytes(int64_t batch, int64_t n, int64_t hq, int64_t slots) {
  return (size_t)((batch * slots * n * hq * 4 + 255) & ~(int64_t)255);
}

template <int Q_DT>
static void launch_tree_generic(int kv_dt, const TreeParams& p, unsigned grid, hipStream_t st) {
  switch (kv_dt) {
    case XLLM_HIP_BF16:
      tree_generic_kernel<Q_DT, XLLM_HIP_BF16><<<grid, 64, 0, st>>>(p);
      break;
    case XLLM_HIP_FP16:
      tree_generic_kernel<Q_DT, XLLM_HIP_FP16><<<grid, 64, 0, st>>>(p);
      break;
    case XLLM_HIP_FP32:
      tree_generic_kernel<Q_DT, XLLM_HIP_FP32><<<grid, 64, 0, st>>>(p);
      break;
    case XLLM_HIP_FP8_E4M3:
      tree_generic_kernel<Q_DT, XLLM_HIP_FP8_E4M3><<<grid, 64, 0, st>>>(p);
      break;
    default:
      tree_generic_kernel<Q_DT, XLLM_HIP_INT8><<<grid, 64, 0, st>>>(p);
      break;
  }
}

}  // namespace xllm_hip

using namespace xllm_hip;

extern "C" size_t xllm_hip_tree_attention_workspace_bytes(int32_t batch, int32_t q_per_seq, int32_t num_q_heads,
                                                          int32_t num_kv_heads, int32_t head_dim) {
  if (batch < 1 || q_per_seq < 1 || num_q_heads < 1 || num_kv_heads < 1 || head_dim < 1) return 0;
  const int64_t s = tree_slots(batch, q_per_seq, num_q_heads, num_kv_heads, head_dim);
  if (s == 1) return 0;
  return tree_lse_bytes(batch, q_per_seq, num_q_heads, s) + (size_t)(batch * s * q_per_seq * num_q_heads * head_dim * 4);
}

extern "C" int xllm_hip_tree_attention(const xllm_hip_kv_cache* c,
                                       const xllm_hip_decode_args* a,
                                       const uint64_t* tree_mask,
                                       int64_t mask_stride,
                                       int32_t mask_words,
                                       void* workspace,
                                       size_t workspace_bytes,
                                       xllm_hip_stream_t stream) {
  XLLM_HIP_REQUIRE(c != nullptr && a != nullptr, "cache or args is NULL");
  XLLM_HIP_REQUIRE(c->k_cache != nullptr && c->v_cache != nullptr, "k_cache or v_cache is NULL");
  XLLM_HIP_REQUIRE(c->num_blocks > 0 && c->num_blocks <= 0x7fffffff && c->block_size > 0 && c->num_kv_heads > 0 && c->head_dim > 0,
                   "cache sizes must be positive");
  XLLM_HIP_REQUIRE(elem_bytes(c->dtype) > 0, "unknown cache dtype %d", c->dtype);
  XLLM_HIP_REQUIRE(a->batch >= 0 && a->q_per_seq >= 1 && a->num_q_heads >= 1, "bad batch/q_per_seq/num_q_heads");
  XLLM_HIP_REQUIRE(a->num_q_heads % c->num_kv_heads == 0, "num_q_heads %d is not a multiple of num_kv_heads %d",
                   a->num_q_heads, c->num_kv_heads);
  XLLM_HIP_REQUIRE(a->q_dtype == XLLM_HIP_BF16 || a->q_dtype == XLLM_HIP_FP16 || a->q_dtype == XLLM_HIP_FP32,
                   "query dtype must be BF16/FP16/FP32, got %d", a->q_dtype);
  const bool quant = c->dtype == XLLM_HIP_FP8_E4M3 || c->dtype == XLLM_HIP_INT8;
  XLLM_HIP_REQUIRE(!quant || (c->k_scale != nullptr && c->v_scale != nullptr),
                   "a quantised cache needs k_scale and v_scale");
  XLLM_HIP_REQUIRE(c->stride_block >= 0 && c->stride_head >= 0 && c->stride_slot >= 0 &&
                       (!quant || (c->scale_stride_block >= 0 && c->scale_stride_head >= 0 && c->scale_stride_slot >= 0)),
                   "cache strides must not be negative");
  if (a->window_left >= 0) return fail(XLLM_HIP_UNSUPPORTED, "a sliding window is not supported under a tree mask");
  if (a->host_plan != 0) return fail(XLLM_HIP_UNSUPPORTED, "host_plan is not supported under a tree mask");
  if (c->head_dim > 256) return fail(XLLM_HIP_UNSUPPORTED, "head_dim %d is larger than 256", c->head_dim);
  if (a->q_per_seq > kTreeMaxNodes) {
    return fail(XLLM_HIP_UNSUPPORTED, "q_per_seq %d is larger than %d", a->q_per_seq, kTreeMaxNodes);
  }
  XLLM_HIP_REQUIRE(mask_words >= 1 && mask_stride >= mask_words, "mask rows need at least one word");
  if (mask_words > kTreeMaxWords) {
    return fail(XLLM_HIP_UNSUPPORTED, "mask_words %d is larger than %d", mask_words, kTreeMaxWords);
  }
  XLLM_HIP_REQUIRE(a->max_seq_len >= 0 && a->total_kv_len >= 0, "max_seq_len or total_kv_len is negative");
  if (a->batch == 0) return XLLM_HIP_OK;
  XLLM_HIP_REQUIRE(a->q != nullptr && a->out != nullptr && tree_mask != nullptr, "q, out or tree_mask is NULL");
  if (a->block_table != nullptr) {
    XLLM_HIP_REQUIRE(a->seq_lens != nullptr, "block_table form needs seq_lens");
    XLLM_HIP_REQUIRE(a->max_blocks_per_seq >= 1 && a->block_table_stride >= a->max_blocks_per_seq, "bad block_table shape");
  } else {
    XLLM_HIP_REQUIRE(a->kv_indptr != nullptr && a->kv_indices != nullptr && a->kv_last_page_len != nullptr,
                     "neither block_table nor the CSR arrays were given");
  }
  const int64_t rowlen = (int64_t)a->num_q_heads * c->head_dim;
  XLLM_HIP_REQUIRE(a->q_token_stride >= rowlen && a->out_token_stride >= rowlen,
                   "q/out token stride smaller than num_q_heads*head_dim");
  const size_t need = xllm_hip_tree_attention_workspace_bytes(a->batch, a->q_per_seq, a->num_q_heads, c->num_kv_heads, c->head_dim);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need)) {
    return fail(XLLM_HIP_WORKSPACE_TOO_SMALL, "workspace has %zu bytes, need %zu", workspace_bytes, need);
  }
  XLLM_HIP_REQUIRE(need == 0 || ((uintptr_t)workspace & 255) == 0, "workspace must be 256-byte aligned");

  TreeParams p{};
  p.q = a->q;
  p.out = a->out;
  p.lse = a->lse;
  p.k_cache = (const uint8_t*)c->k_cache;
  p.v_cache = (const uint8_t*)c->v_cache;
  p.k_scale = c->k_scale;
  p.v_scale = c->v_scale;
  if (a->block_table != nullptr) {
    p.block_ids = a->block_table;
    p.seq_lens = a->seq_lens;
    p.bt_stride = a->block_table_stride;
    p.len_cap = (int64_t)a->max_blocks_per_seq * c->block_size;
  } else {
    p.block_ids = a->kv_indices;
    p.kv_indptr = a->kv_indptr;
    p.kv_last_page_len = a->kv_last_page_len;
  }
  p.q_indptr = a->q_indptr;
  p.mask = tree_mask;
  p.mask_stride = mask_stride;
  p.mask_words = mask_words;
  p.q_token_stride = a->q_token_stride;
  p.out_token_stride = a->out_token_stride;
  p.stride_block = c->stride_block;
  p.stride_head = c->stride_head;
  p.stride_slot = c->stride_slot;
  p.sc_stride_block = c->scale_stride_block;
  p.sc_stride_head = c->scale_stride_head;
  p.sc_stride_slot = c->scale_stride_slot;
  p.batch = a->batch;
  p.n = a->q_per_seq;
  p.num_q_heads = a->num_q_heads;
  p.num_kv_heads = c->num_kv_heads;
  p.group = a->num_q_heads / c->num_kv_heads;
  p.head_dim = c->head_dim;
  p.block_size = c->block_size;
  p.log2_bs = is_pow2(c->block_size) ? ilog2(c->block_size) : -1;
  p.last_block = (int32_t)(c->num_blocks - 1);
  p.q_dtype = a->q_dtype;
  p.scale_log2 = (float)((double)a->sm_scale * 1.4426950408889634);
  const int64_t slots = tree_slots(a->batch, p.n, p.num_q_heads, p.num_kv_heads, p.head_dim);
  p.slots = (int32_t)slots;
  if (slots > 1) {
    p.partial_lse = (float*)workspace;
    p.partial_out = (float*)((uint8_t*)workspace + tree_lse_bytes(a->batch, p.n, p.num_q_heads, slots));
  }
  p.tile = 64;
  p.chunk = kTreeMinChunk;
  // Chunk slots no sequence can reach by the host's hint are not launched (a longer sequence than the hint says gets
  // longer chunks).
  if (a->max_seq_len > 0) {
    const int64_t most = ((int64_t)a->max_seq_len + p.chunk - 1) / p.chunk;
    if (most < p.slots) p.slots = (int32_t)most;
  }
  p.row_groups = p.n * p.group;
  const int64_t items = (int64_t)p.batch * p.slots * p.num_kv_heads * p.row_groups;
  XLLM_HIP_REQUIRE(items <= 0x7fffffff, "too many work items: %lld", (long long)items);
  hipStream_t st = (hipStream_t)stream;
  if (p.q_dtype == XLLM_HIP_BF16) {
    launch_tree_generic<XLLM_HIP_BF16>(c->dtype, p, (unsigned)items, st);
  } else if (p.q_dtype == XLLM_HIP_FP16) {
    launch_tree_generic<XLLM_HIP_FP16>(c->dtype, p, (unsigned)items, st);
  } else {
    launch_tree_generic<XLLM_HIP_FP32>(c->dtype, p, (unsigned)items, st);
  }
  int rc = check_launch("tree attention kernel");
  if (rc != XLLM_HIP_OK || p.slots == 1) return rc;
  const unsigned merge_grid = (unsigned)(((int64_t)p.batch * p.n * p.num_q_heads + 3) / 4);
  if (p.q_dtype == XLLM_HIP_BF16) {
    tree_merge_kernel<XLLM_HIP_BF16><<<merge_grid, 256, 0, st>>>(p);
  } else if (p.q_dtype == XLLM_HIP_FP16) {
    tree_merge_kernel<XLLM_HIP_FP16><<<merge_grid, 256, 0, st>>>(p);
  } else {
    tree_merge_kernel<XLLM_HIP_FP32><<<merge_grid, 256, 0, st>>>(p);
  }
  return check_launch("tree_merge_kernel");
}
