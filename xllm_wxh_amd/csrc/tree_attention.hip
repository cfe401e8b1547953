// Paged attention of drafted trees for gfx950: the verify step of tree speculation.  Every query token sees the whole
// context and, among the drafted tokens at the end of its sequence, those its mask names (see
// xllm_hip_tree_attention in the header for the exact statement).
//
//   x_t = scale * q.k_t,   out = sum_t 2^(x_t - m) v_t / sum_t 2^(x_t - m)      (x in units of log 2)
//
// Long sequences are cut into chunks of whole tiles, a workgroup each; a chunk leaves a normalised partial and its
// base-2 log-sum-exp, and tree_merge_kernel joins them.  How a sequence is cut follows from its own length, read on
// the device, and two numbers from the host (tokens per chunk, chunks a sequence may have), so any hints, stale ones
// of a captured graph included, give the same result up to the rounding of sums that are formed in another order.
#include "device_utils.h"
#include "host_utils.h"
#include "tree_generic.h"
#include "tree_mfma.h"
#include "tree_params.h"

#include <math.h>

namespace xllm_hip {

constexpr int kTreeMaxNodes = 512;
constexpr int kTreeMaxWords = 8;
constexpr int kTreeMaxSlots = 64;    // chunks per sequence: a lane each in the merge
constexpr int kTreeMinChunk = 256;   // tokens: a shorter chunk costs more in its partial than it saves

// Chunks a sequence may have: enough that the launch has 2048 items (and four, for lengths that differ), no more than
// the merge holds, and no more than 512 MiB of partials.  Sizes only, so that one workspace serves every step of these
// sizes.
static int tree_slots(int64_t batch, int64_t n, int64_t hq, int64_t hkv, int64_t d) {
  const int64_t items = batch * hkv;
  int64_t s = items > 0 ? (2048 + items - 1) / items : 1;
  s = s > 4 ? s : 4;
  const int64_t row_bytes = batch * n * hq * (d + 1) * 4;
  const int64_t fit = row_bytes > 0 ? ((int64_t)512 << 20) / row_bytes : kTreeMaxSlots;
  s = s < fit ? s : fit;
  s = s < kTreeMaxSlots ? s : kTreeMaxSlots;
  return s > 1 ? (int)s : 1;
}

// Where the sequences lie on the line (see TreeLine), for the merge.
static size_t tree_line_bytes(int64_t batch) {
  return batch <= kTreeLineBatch ? (size_t)(((batch + 1) * 8 + 255) & ~(int64_t)255) : 0;
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

// How the matrix kernels would run a call; rows_per_item 0: they do not serve it.
struct TreeForm {
  int rows_per_item;
  int slots;  // workgroups that run at a time on 256 CUs
};

static TreeForm tree_form(const xllm_hip_kv_cache* c, const xllm_hip_decode_args* a) {
  TreeForm none{0, 0};
  const int eb = elem_bytes(c->dtype);
  const bool quant = c->dtype == XLLM_HIP_FP8_E4M3 || c->dtype == XLLM_HIP_INT8;
  if (a->q_dtype != XLLM_HIP_BF16 && a->q_dtype != XLLM_HIP_FP16) return none;
  if (!quant && c->dtype != a->q_dtype) return none;
  if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256) return none;
  // (a wave's load instruction covers rows of one group of 16 tokens, which must lie in one block)
  if (!is_pow2(c->block_size) || c->block_size < 16) return none;
  if (!(a->sm_scale >= 0.0f)) return none;  // (the running maximum is taken before the scale)
  const int64_t vec = 16 / eb, lim = (int64_t)1 << 31;
  if (c->stride_block % vec != 0 || c->stride_head % vec != 0 || c->stride_slot % vec != 0) return none;
  if (c->stride_block >= lim || c->stride_slot * c->block_size >= lim) return none;
  // (a lane's scale lies within 32 bits of bytes from its block's first: TreeLoader::sc_off)
  if (quant && (c->scale_stride_block >= lim || c->scale_stride_slot * c->block_size >= lim / 2)) return none;
  if ((((uintptr_t)c->k_cache | (uintptr_t)c->v_cache | (uintptr_t)a->q | (uintptr_t)a->out) & 15) != 0) return none;
  if (a->q_token_stride % 8 != 0 || a->out_token_stride % 8 != 0) return none;
  const int64_t rows = (int64_t)a->q_per_seq * (a->num_q_heads / c->num_kv_heads);
  const int rb = c->head_dim * eb;
  TreeForm f;
  f.rows_per_item = rows <= 32 ? 32 : (rows <= 64 || c->head_dim == 256) ? 64 : 128;
  f.slots = rb == 512 ? 256 : 512;
  return f;
}

// Tokens per chunk and chunks per sequence (at most p.slots of them on entry), or pieces of a line.  Without the host's
// lengths: from 64 (sequence, kv head, row group)s on the line where it serves, else chunks of at least kTreeMinChunk tokens, as
// many to a sequence as make 1024 items (with 2048, 32 x 8192 fp8 tokens and 512 query rows to a kv head take 848 us against
// 673).  Where the two meet, bf16, 8 kv heads of 128, 8 drafts, ragged, us in chunks / on the line:
//   up to 1000 tokens   32 items 13.8 / 17.3   64 items 14.8 / 18.5   128 items 18.6 / 22.2   256 items  31.7 /  29.7
//             4000               17.5 / 22.0            29.0 / 26.3             45.2 / 42.3              76.6 /  70.1
//            16000               46.2 / 41.8            76.0 / 70.0            138.2 / 122.8
// (head_dim 256 and 128 query rows gain more from it: 64 items of 4000 tokens 61.1 / 45.0 and 45.2 / 38.1.)
// With them, the cut whose step is predicted to end first, from what a token costs where all workgroups run (`slots` of
// them): its K and V at the memory's rate, or its products at that of the matrix kernels, whichever is more,
//   nearly equal lengths   rounds of equal items:  ceil(items / slots) * (chunk + start)
//   ragged lengths         the longest chunk while all items run together; else the items' tokens over `slots`, and
//                          half a chunk until the last one ends
//   on a line (TreeLine)   a piece, one more start, and laying the line
// plus, where sequences are cut, the merge's launch and the partial results, written once and read once.
// The line serves 16-bit caches: 40 sequences of 800 to 16384 tokens, 8 drafts, 272 -> 246 us; 24 of 800 to 8192, 16
// drafts, 110 -> 99; 103 of up to 2208, 31 drafts, head_dim 256, 263 -> 198.  Over 8-bit caches the kernels have no
// register left for the loop over a piece's items, and what it takes from the loop over the tokens costs more than the
// even pieces save (100 int8 sequences 217 -> 220 us).
static void choose_chunks(const xllm_hip_decode_args* a, const TreeForm& form, int eb, TreeParams& p) {
  auto whole = [&](int64_t tokens) { return (tokens + p.tile - 1) / p.tile * p.tile; };
  const int64_t longest = a->max_seq_len;
  const bool can_line = form.rows_per_item > 0 && eb == 2 && p.batch <= kTreeLineBatch && p.slots > 1 && p.num_kv_heads <= form.slots;
  const int32_t pieces = can_line ? form.slots / p.num_kv_heads : 0;
  if (longest <= 0 && can_line && (int64_t)p.batch * p.num_kv_heads * p.row_groups >= 64) {
    p.pieces = pieces;
    return;
  }
  if (longest <= 0 || form.rows_per_item == 0) {
    p.chunk = (int32_t)whole(kTreeMinChunk);
    if (longest <= 0 && form.rows_per_item > 0) {
      const int64_t lanes = (int64_t)p.batch * p.num_kv_heads * p.row_groups, cuts = (1024 + lanes - 1) / lanes;
      if (cuts < p.slots) p.slots = (int32_t)cuts;
    }
    if (longest > 0) {  // (chunk slots no sequence reaches are not launched)
      const int64_t most = (longest + p.chunk - 1) / p.chunk;
      if (most < p.slots) p.slots = (int32_t)most;
    }
    return;
  }
  int64_t total = a->total_kv_len;
  if (total <= 0 || total > longest * p.batch) total = longest * p.batch;
  const bool equal = longest * p.batch * 4 <= total * 5;
  const double lanes = (double)p.num_kv_heads * p.row_groups;
  const double rows = (double)p.n * p.group < form.rows_per_item ? (double)p.n * p.group : (double)form.rows_per_item;
  // ns (6.5 kB or 850 kflop in one)
  const double bytes = 2.0 * p.head_dim * eb * form.slots / 6.5e3;
  const double flops = 4.0 * p.head_dim * form.rows_per_item * form.slots / 850e3;
  const double token = bytes > flops ? bytes : flops;
  const double partial = rows * 8.0 * p.head_dim / 6.5e3;
  constexpr double kStart = 5000.0, kMerge = 5000.0, kLine = 5000.0;
  double best = 0.0;
  int best_cut = 0;
  for (int cut = 1; cut <= p.slots; ++cut) {
    const int64_t chunk = whole((longest + cut - 1) / cut);
    if (cut > 1 && chunk < kTreeMinChunk) break;
    const double item = (double)chunk * token + kStart;
    double items, t;
    if (equal) {
      items = lanes * p.batch * (double)((longest + chunk - 1) / chunk);
      t = ceil(items / form.slots) * item;
    } else {
      items = lanes * ((double)total / (double)chunk + 0.5 * p.batch);
      t = items <= (double)form.slots ? item : (lanes * (double)total * token + items * kStart) / form.slots + 0.5 * (double)chunk * token;
    }
    if (cut > 1) t += items * partial + kMerge;
    if (best_cut == 0 || t < best) {
      best = t;
      best_cut = cut;
    }
  }
  if (can_line) {
    const double wgs = (double)pieces * p.num_kv_heads;
    double t = lanes * ((double)total * token + p.batch * kStart) / wgs;
    const double least = (double)longest / (double)(p.slots - 1), piece = (least > kTreeMinChunk ? least : (double)kTreeMinChunk) * token;
    t = (t > piece ? t : piece) + kStart + kLine + 1.5 * wgs * partial + kMerge;
    if (t < best) {
      p.pieces = pieces;
      return;
    }
  }
  p.chunk = (int32_t)whole((longest + best_cut - 1) / best_cut);
  p.slots = best_cut;
}

template <int Q_DT, int COLS, bool LINE>
static void launch_tree_merge_rows(const TreeParams& p, hipStream_t st) {
  const int rows = p.n * p.num_q_heads;  // (p.n <= kTreeMaxNodes)
  if ((int64_t)p.batch * rows <= 8192) {  // two waves to a CU's SIMD
    tree_merge_kernel<Q_DT, COLS, 1, LINE><<<dim3((unsigned)((rows + 3) / 4), (unsigned)p.batch), 256, 0, st>>>(p);
  } else {
    tree_merge_kernel<Q_DT, COLS, 4, LINE><<<dim3((unsigned)((rows + 15) / 16), (unsigned)p.batch), 256, 0, st>>>(p);
  }
}

template <int Q_DT, int COLS>
static void launch_tree_merge_cols(const TreeParams& p, hipStream_t st) {
  if (p.pieces == 0) {
    launch_tree_merge_rows<Q_DT, COLS, false>(p, st);
  } else if constexpr (Q_DT != XLLM_HIP_FP32) {
    launch_tree_merge_rows<Q_DT, COLS, true>(p, st);
  }
}

template <int Q_DT>
static void launch_tree_merge(const TreeParams& p, hipStream_t st) {
  if (p.head_dim <= 64) {
    launch_tree_merge_cols<Q_DT, 16>(p, st);
  } else if (p.head_dim <= 128) {
    launch_tree_merge_cols<Q_DT, 32>(p, st);
  } else {
    launch_tree_merge_cols<Q_DT, 64>(p, st);
  }
}

template <int QT, int KV, int D, int RTW, int TS, bool STREAM>
static void launch_tree_mfma_form(const TreeParams& p, unsigned grid, hipStream_t st) {
  if (p.pieces == 0) {
    tree_mfma_kernel<QT, KV, D, RTW, TS, STREAM><<<grid, 256, 0, st>>>(p);
  } else if constexpr (!tree_quant(KV)) {
    tree_mfma_line_kernel<QT, KV, D, RTW, TS, STREAM><<<grid, 256, 0, st>>>(p);
  }
}

template <int QT, int KV, int D>
static void launch_tree_mfma_d(int rows_per_item, const TreeParams& p, unsigned grid, hipStream_t st) {
  const bool stream = p.row_groups == 1;  // nobody else reads an item's K and V
  constexpr bool kBoth = tree_quant(KV) && D <= 128;  // (two row tiles of head_dim 256 do not fit the registers)
  if (rows_per_item == 32) {
    launch_tree_mfma_form<QT, KV, D, kBoth ? 2 : 1, kBoth ? 4 : 2, true>(p, grid, st);
  } else if (rows_per_item == 64) {
    if (D < 256 || stream) {
      launch_tree_mfma_form<QT, KV, D, kBoth ? 2 : 1, kBoth ? 2 : 1, true>(p, grid, st);
    } else {
      if constexpr (D == 256) launch_tree_mfma_form<QT, KV, D, 1, 1, false>(p, grid, st);
    }
  } else {
    if constexpr (D <= 128) {
      if (stream) {
        launch_tree_mfma_form<QT, KV, D, 2, 1, true>(p, grid, st);
      } else {
        launch_tree_mfma_form<QT, KV, D, 2, 1, false>(p, grid, st);
      }
    }
  }
}

template <int QT, int KV>
static void launch_tree_mfma_kv(int rows_per_item, const TreeParams& p, unsigned grid, hipStream_t st) {
  if (p.head_dim == 64) {
    launch_tree_mfma_d<QT, KV, 64>(rows_per_item, p, grid, st);
  } else if (p.head_dim == 128) {
    launch_tree_mfma_d<QT, KV, 128>(rows_per_item, p, grid, st);
  } else {
    launch_tree_mfma_d<QT, KV, 256>(rows_per_item, p, grid, st);
  }
}

template <int QT>
static void launch_tree_mfma(int kv_dt, int rows_per_item, const TreeParams& p, unsigned grid, hipStream_t st) {
  if (kv_dt == XLLM_HIP_FP8_E4M3) {
    launch_tree_mfma_kv<QT, XLLM_HIP_FP8_E4M3>(rows_per_item, p, grid, st);
  } else if (kv_dt == XLLM_HIP_INT8) {
    launch_tree_mfma_kv<QT, XLLM_HIP_INT8>(rows_per_item, p, grid, st);
  } else {
    launch_tree_mfma_kv<QT, QT>(rows_per_item, p, grid, st);
  }
}

// How a call is run: the form, and in `p` the sizes, how its sequences are cut and the items of the launch that follow.
static TreeForm lay_out_tree(const xllm_hip_kv_cache* c, const xllm_hip_decode_args* a, TreeParams& p) {
  p.batch = a->batch;
  p.n = a->q_per_seq;
  p.num_q_heads = a->num_q_heads;
  p.num_kv_heads = c->num_kv_heads;
  p.group = a->num_q_heads / c->num_kv_heads;
  p.head_dim = c->head_dim;
  p.slots = (int32_t)tree_slots(a->batch, p.n, p.num_q_heads, p.num_kv_heads, p.head_dim);
  const TreeForm form = tree_form(c, a);
  p.tile = form.rows_per_item > 0 ? 32 : 64;  // (what the kernels take at a time)
  const int64_t rows = (int64_t)p.n * p.group;
  p.row_groups = (int32_t)(form.rows_per_item > 0 ? (rows + form.rows_per_item - 1) / form.rows_per_item : rows);
  p.rows_per_item = form.rows_per_item;
  choose_chunks(a, form, elem_bytes(c->dtype), p);
  return form;
}

// Workgroups of the attention launch.
static int64_t tree_workgroups(const TreeForm& form, const TreeParams& p) {
  int64_t items = (int64_t)p.batch * p.slots * p.num_kv_heads * p.row_groups;
  if (p.pieces > 0) {
    items = (int64_t)p.pieces * p.num_kv_heads;
  } else if (form.rows_per_item > 0 && p.row_groups > 1) {  // whole rounds of the XCDs (see the kernel)
    items = (items + kTreeXcds * p.row_groups - 1) / (kTreeXcds * p.row_groups) * (kTreeXcds * p.row_groups);
  }
  return items;
}

// What can be said of a call without its query, output, mask and workspace.
static int check_tree_sizes(const xllm_hip_kv_cache* c, const xllm_hip_decode_args* a) {
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
  if (a->batch > 65535) return fail(XLLM_HIP_UNSUPPORTED, "batch %d is larger than 65535", a->batch);
  XLLM_HIP_REQUIRE(a->max_seq_len >= 0 && a->total_kv_len >= 0, "max_seq_len or total_kv_len is negative");
  return XLLM_HIP_OK;
}

// The lists and strides of a call with sequences.
static int check_tree_lists(const xllm_hip_kv_cache* c, const xllm_hip_decode_args* a) {
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
  return XLLM_HIP_OK;
}

}  // namespace xllm_hip

using namespace xllm_hip;

extern "C" size_t xllm_hip_tree_attention_workspace_bytes(int32_t batch, int32_t q_per_seq, int32_t num_q_heads,
                                                          int32_t num_kv_heads, int32_t head_dim) {
  if (batch < 1 || q_per_seq < 1 || num_q_heads < 1 || num_kv_heads < 1 || head_dim < 1) return 0;
  const int64_t s = tree_slots(batch, q_per_seq, num_q_heads, num_kv_heads, head_dim);
  if (s == 1) return 0;
  return tree_line_bytes(batch) + tree_lse_bytes(batch, q_per_seq, num_q_heads, s) + (size_t)(batch * s * q_per_seq * num_q_heads * head_dim * 4);
}

extern "C" int xllm_hip_tree_attention(const xllm_hip_kv_cache* c,
                                       const xllm_hip_decode_args* a,
                                       const uint64_t* tree_mask,
                                       int64_t mask_stride,
                                       int32_t mask_words,
                                       void* workspace,
                                       size_t workspace_bytes,
                                       xllm_hip_stream_t stream) {
  int rc = check_tree_sizes(c, a);
  if (rc != XLLM_HIP_OK) return rc;
  XLLM_HIP_REQUIRE(mask_words >= 1 && mask_stride >= mask_words, "mask rows need at least one word");
  if (mask_words > kTreeMaxWords) {
    return fail(XLLM_HIP_UNSUPPORTED, "mask_words %d is larger than %d", mask_words, kTreeMaxWords);
  }
  if (a->batch == 0) return XLLM_HIP_OK;
  XLLM_HIP_REQUIRE(a->q != nullptr && a->out != nullptr && tree_mask != nullptr, "q, out or tree_mask is NULL");
  rc = check_tree_lists(c, a);
  if (rc != XLLM_HIP_OK) return rc;
  const size_t need = xllm_hip_tree_attention_workspace_bytes(a->batch, a->q_per_seq, a->num_q_heads, c->num_kv_heads, c->head_dim);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need)) {
    return fail(XLLM_HIP_WORKSPACE_TOO_SMALL, "workspace has %zu bytes, need %zu", workspace_bytes, need);
  }
  XLLM_HIP_REQUIRE(need == 0 || ((uintptr_t)workspace & 255) == 0, "workspace must be 256-byte aligned");

  TreeParams p{};
  const int64_t slots = tree_slots(a->batch, a->q_per_seq, a->num_q_heads, c->num_kv_heads, c->head_dim);  // the workspace's
  const TreeForm form = lay_out_tree(c, a, p);
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
  p.block_size = c->block_size;
  p.log2_bs = is_pow2(c->block_size) ? ilog2(c->block_size) : -1;
  p.last_block = (int32_t)(c->num_blocks - 1);
  p.q_dtype = a->q_dtype;
  p.scale_log2 = (float)((double)a->sm_scale * 1.4426950408889634);
  if (slots > 1) {
    p.line = (int64_t*)workspace;
    p.partial_lse = (float*)((uint8_t*)workspace + tree_line_bytes(a->batch));
    p.partial_out = (float*)((uint8_t*)p.partial_lse + tree_lse_bytes(a->batch, p.n, p.num_q_heads, slots));
  }
  const int64_t items = tree_workgroups(form, p);
  XLLM_HIP_REQUIRE(items <= 0x7fffffff, "too many work items: %lld", (long long)items);
  hipStream_t st = (hipStream_t)stream;
  const unsigned grid = (unsigned)items;
  if (form.rows_per_item > 0) {
    if (p.q_dtype == XLLM_HIP_BF16) {
      launch_tree_mfma<XLLM_HIP_BF16>(c->dtype, form.rows_per_item, p, grid, st);
    } else {
      launch_tree_mfma<XLLM_HIP_FP16>(c->dtype, form.rows_per_item, p, grid, st);
    }
  } else if (p.q_dtype == XLLM_HIP_BF16) {
    launch_tree_generic<XLLM_HIP_BF16>(c->dtype, p, grid, st);
  } else if (p.q_dtype == XLLM_HIP_FP16) {
    launch_tree_generic<XLLM_HIP_FP16>(c->dtype, p, grid, st);
  } else {
    launch_tree_generic<XLLM_HIP_FP32>(c->dtype, p, grid, st);
  }
  rc = check_launch("tree attention kernel");
  if (rc != XLLM_HIP_OK || (p.slots == 1 && p.pieces == 0)) return rc;
  if (p.q_dtype == XLLM_HIP_BF16) {
    launch_tree_merge<XLLM_HIP_BF16>(p, st);
  } else if (p.q_dtype == XLLM_HIP_FP16) {
    launch_tree_merge<XLLM_HIP_FP16>(p, st);
  } else {
    launch_tree_merge<XLLM_HIP_FP32>(p, st);
  }
  return check_launch("tree_merge_kernel");
}

extern "C" int xllm_hip_tree_attention_describe(const xllm_hip_kv_cache* c, const xllm_hip_decode_args* a, int64_t* out, int32_t count) {
  XLLM_HIP_REQUIRE(out != nullptr && count >= 0, "out is NULL or count negative");
  int rc = check_tree_sizes(c, a);
  if (rc != XLLM_HIP_OK) return rc;
  int64_t values[6] = {};
  if (a->batch > 0) {
    rc = check_tree_lists(c, a);
    if (rc != XLLM_HIP_OK) return rc;
    TreeParams p{};
    const TreeForm form = lay_out_tree(c, a, p);
    values[0] = form.rows_per_item;
    values[1] = tree_workgroups(form, p);
    values[2] = p.row_groups;
    values[3] = p.pieces;
    values[4] = p.pieces > 0 ? 0 : p.chunk;
    values[5] = p.slots;
  }
  for (int i = 0; i < count; ++i) out[i] = i < 6 ? values[i] : 0;
  return XLLM_HIP_OK;
}
