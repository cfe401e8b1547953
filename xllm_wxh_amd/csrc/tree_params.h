// Arguments of the tree-attention kernels, and what a workgroup works on.
#pragma once

#include "device_utils.h"

#include <stdint.h>

namespace xllm_hip {

struct TreeParams {
  const void* q;
  void* out;
  float* lse;
  const uint8_t* k_cache;
  const uint8_t* v_cache;
  const float* k_scale;
  const float* v_scale;
  const int32_t* block_ids;  // block_table, or kv_indices in CSR form
  const int32_t* kv_indptr;  // non-NULL selects the CSR form
  const int32_t* seq_lens;
  const int32_t* kv_last_page_len;
  const int32_t* q_indptr;
  const uint64_t* mask;
  float* partial_out;  // [batch * slots][n * Hq][head_dim], each row normalised
  float* partial_lse;  // [batch * slots][n * Hq], base 2
  int64_t* line;       // pieces > 0: where the sequences start on the line, [batch]; behind them the tokens of a piece
  int64_t mask_stride;
  int64_t q_token_stride;
  int64_t out_token_stride;
  int64_t stride_block;
  int64_t stride_head;
  int64_t stride_slot;
  int64_t sc_stride_block;
  int64_t sc_stride_head;
  int64_t sc_stride_slot;
  int64_t bt_stride;
  int64_t len_cap;     // tokens a table row can hold
  int32_t mask_words;
  int32_t batch;
  int32_t n;           // most query tokens of a sequence
  int32_t num_q_heads;
  int32_t num_kv_heads;
  int32_t group;       // q heads per kv head
  int32_t head_dim;
  int32_t block_size;
  int32_t log2_bs;     // or -1
  int32_t last_block;  // num_blocks - 1: block ids are taken within 0 .. last_block
  int32_t row_groups;  // items a (sequence, chunk, kv head)'s query rows are cut into
  int32_t slots;       // chunks a sequence may have
  int32_t chunk;       // tokens per chunk of a sequence that needs no more than `slots` of them
  int32_t tile;        // chunks are multiples of it
  int32_t pieces;      // > 0: the work is laid on a line and cut into so many pieces per kv head (see TreeLine)
  int32_t rows_per_item;
  int32_t q_dtype;
  float scale_log2;    // sm_scale * log2(e)
};

struct TreeItem {
  int b, hk, rg;
  int chunk, chunks;   // this item's chunk; 1: it is the whole sequence
  int len;             // kv length
  int t_begin, t_end;  // tokens of the chunk
  int prefix;          // tokens every row sees: len - (query tokens of the sequence); may be negative
  int n;               // query tokens that are computed
  int64_t q0;          // index of the first of them
  const int32_t* ids;  // block list
  int nblk;            // entries of it that may be read (>= 1)
};

// kv length: never negative and never beyond what the sequence's block list holds.
__device__ inline int tree_kv_length(const TreeParams& p, int b) {
  if (p.kv_indptr != nullptr) {
    const int64_t nb = (int64_t)p.kv_indptr[b + 1] - p.kv_indptr[b];
    int last = p.kv_last_page_len[b];
    last = last < 0 ? 0 : (last < p.block_size ? last : p.block_size);
    const int64_t len = nb > 0 ? (nb - 1) * p.block_size + last : 0;
    return (int)(len < 0x7fffff00 ? len : 0x7fffff00);
  }
  int64_t len = p.seq_lens[b];
  len = len < p.len_cap ? len : p.len_cap;
  len = len < 0x7fffff00 ? len : 0x7fffff00;  // (tile ends past the length stay within 32 bits)
  return len > 0 ? (int)len : 0;
}

// Tokens per chunk of a sequence of `len`: p.chunk, or what `slots` chunks of whole tiles cover it with.
__device__ inline int tree_chunk_tokens(const TreeParams& p, int len) {
  int per = (int)(((int64_t)len + p.slots - 1) / p.slots);
  per = (per + p.tile - 1) / p.tile * p.tile;
  return per > p.chunk ? per : p.chunk;
}
__device__ inline int tree_chunks(const TreeParams& p, int len) {
  const int c = tree_chunk_tokens(p, len);
  return len > 0 ? (int)(((int64_t)len + c - 1) / c) : 1;
}

__device__ inline void tree_rows(const TreeParams& p, int b, int64_t& q0, int& count) {
  if (p.q_indptr != nullptr) {
    q0 = p.q_indptr[b];
    count = p.q_indptr[b + 1] - (int)q0;
    count = count > 0 ? count : 0;
  } else {
    q0 = (int64_t)b * p.n;
    count = p.n;
  }
}

constexpr int kTreeXcds = 8;  // workgroup x runs on XCD x % 8

// The sequence's block list; its length is known.
__device__ inline void tree_blocks(const TreeParams& p, TreeItem& it) {
  int64_t listed;
  if (p.kv_indptr != nullptr) {
    it.ids = p.block_ids + p.kv_indptr[it.b];
    listed = (int64_t)p.kv_indptr[it.b + 1] - p.kv_indptr[it.b];
  } else {
    it.ids = p.block_ids + (int64_t)it.b * p.bt_stride;
    listed = p.len_cap / p.block_size;
  }
  const int64_t need = ((int64_t)it.len + p.block_size - 1) / p.block_size;
  it.nblk = (int)(need < listed ? need : listed);
  if (it.nblk < 1) it.nblk = 1;
}

// Items in their natural order are (chunk slot, sequence, kv head, row group), row group fastest: the row groups of one
// (chunk, kv head) read the same K and V, and the sequences' last chunks, which are the short ones, run last.
__device__ inline bool tree_item(const TreeParams& p, int id, int rows_per_item, TreeItem& it) {
  it.rg = id % p.row_groups;
  int rest = id / p.row_groups;
  it.hk = rest % p.num_kv_heads;
  rest /= p.num_kv_heads;
  it.b = rest % p.batch;
  it.chunk = rest / p.batch;
  if (it.chunk >= p.slots) return false;
  int count;
  tree_rows(p, it.b, it.q0, count);
  it.n = count < p.n ? count : p.n;
  if (it.rg * rows_per_item >= it.n * p.group) return false;
  it.len = tree_kv_length(p, it.b);
  it.prefix = it.len - count;
  const int per = tree_chunk_tokens(p, it.len);
  it.chunks = it.len > 0 ? (int)(((int64_t)it.len + per - 1) / per) : 1;
  if (it.chunk >= it.chunks) return false;
  it.t_begin = it.chunk * per;
  const int64_t end = (int64_t)it.t_begin + per;
  it.t_end = end < it.len ? (int)end : it.len;
  tree_blocks(p, it);
  return true;
}

// Ragged lengths: the work of a kv head laid on a line, in units of 32 tokens: sequence after sequence, each as often as
// it has row groups, kTreeStart units for the start of an item and then its tokens.  The line is cut into `pieces` equal
// pieces, a workgroup each, that run at the same time and end together, whatever the lengths are; a sequence that lies
// in several pieces leaves a partial in each.  Which piece holds what is computed from the lengths on the device.
constexpr int kTreeStart = 4;
constexpr int kTreeLineBatch = 1024;  // sequences: four to a thread that lays the line

__device__ inline int tree_line_groups(const TreeParams& p, int b) {
  int64_t q0;
  int count;
  tree_rows(p, b, q0, count);
  const int rows = (count < p.n ? count : p.n) * p.group;
  return (rows + p.rows_per_item - 1) / p.rows_per_item;
}
// Units of a sequence; one without tokens has a unit too (its rows are written).
__device__ inline int tree_line_units(int len) { return kTreeStart + (len > 32 ? (len - 1) / 32 + 1 : 1); }

// Chunks of the row group that starts at `at` on the line: pieces from the one with its first token to the one with its last.
__device__ inline int tree_line_chunks(int64_t at, int units, int64_t piece) {
  return (int)((at + units - 1) / piece - (at + kTreeStart) / piece) + 1;
}

struct TreeLine {
  int64_t left;  // units of the piece from the start of the current item's sequence on

  // This workgroup's first item; every thread of 256 takes part.  False: there is none.
  __device__ inline bool start(const TreeParams& p, int id, TreeItem& it) {
    __shared__ int64_t sums[4];
    __shared__ int most[4];
    __shared__ int64_t found[3];  // the sequence, its row group and the units of it before the piece
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    it.hk = id % p.num_kv_heads;
    const int64_t i = id / p.num_kv_heads;
    const int per = (p.batch + 255) / 256;
    int64_t sum = 0;
    int longest = 0;
    for (int e = 0; e < per; ++e) {
      const int b = tid * per + e;
      if (b >= p.batch) break;
      const int units = tree_line_units(tree_kv_length(p, b));
      sum += (int64_t)units * tree_line_groups(p, b);
      longest = units > longest ? units : longest;
    }
    int64_t upto = sum;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int64_t other = __shfl_up(upto, d);
      if (lane >= d) upto += other;
      longest = max(longest, __shfl_xor(longest, d));
    }
    if (lane == 63) sums[wave] = upto;
    if (lane == 0) most[wave] = longest;
    if (tid == 0) found[0] = -1;
    __syncthreads();
    int64_t total = 0, at = upto - sum;
    for (int w = 0; w < 4; ++w) {
      if (w < wave) at += sums[w];
      total += sums[w];
      longest = max(longest, most[w]);
    }
    // equal pieces; no sequence in more of them than it has slots for partials; none that a partial would outweigh
    int64_t piece = (int64_t)(((uint64_t)total + (uint32_t)p.pieces - 1) / (uint32_t)p.pieces);
    const int64_t least = ((int64_t)longest + p.slots - 2) / (p.slots - 1);
    piece = piece > least ? piece : least;
    piece = piece > 8 ? piece : 8;
    piece = (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(piece >> 32)) << 32 |
                      (uint32_t)__builtin_amdgcn_readfirstlane((int)piece));
    const int64_t from = i * piece;
    for (int e = 0; e < per; ++e) {
      const int b = tid * per + e;
      if (b >= p.batch) break;
      if (id == 0) p.line[b] = at;
      const int units = tree_line_units(tree_kv_length(p, b));
      const int64_t all = (int64_t)units * tree_line_groups(p, b);
      if (from >= at && from < at + all) {
        found[1] = (from - at) / units;
        found[2] = (from - at) % units;
        found[0] = b;
      }
      at += all;
    }
    if (id == 0 && tid == 0) p.line[p.batch] = piece;
    __syncthreads();
    it.b = __builtin_amdgcn_readfirstlane((int)found[0]);
    if (it.b < 0) return false;
    it.rg = __builtin_amdgcn_readfirstlane((int)found[1]);
    const int skip = __builtin_amdgcn_readfirstlane((int)found[2]);  // (units of a sequence: below 2^27)
    sequence(p, it);
    it.chunk = skip > kTreeStart ? (int)(i - (from - skip + kTreeStart) / piece) : 0;
    left = piece + skip;
    it.t_begin = skip > kTreeStart ? (skip - kTreeStart) * 32 : 0;
    set_end(it);
    return true;
  }

  // The next item of the piece.
  __device__ inline bool next(const TreeParams& p, TreeItem& it) {
    left -= tree_line_units(it.len);
    if (left <= kTreeStart) return false;
    if ((++it.rg) * p.rows_per_item >= it.n * p.group) {
      it.rg = 0;
      do {
        if (++it.b >= p.batch) return false;
      } while (tree_line_groups(p, it.b) == 0);
      sequence(p, it);
    }
    it.chunk = 0;
    it.t_begin = 0;
    set_end(it);
    return true;
  }

 private:
  __device__ static inline void sequence(const TreeParams& p, TreeItem& it) {
    int count;
    tree_rows(p, it.b, it.q0, count);
    it.n = count < p.n ? count : p.n;
    it.len = tree_kv_length(p, it.b);
    it.prefix = it.len - count;
    tree_blocks(p, it);
  }
  // The item ends with the sequence or with the piece.
  __device__ inline void set_end(TreeItem& it) const {
    const int units = tree_line_units(it.len);
    const bool whole = left >= units;
    it.t_end = whole ? it.len : (int)((left - kTreeStart) * 32);
    it.chunks = whole && it.t_begin == 0 ? 1 : 2;
  }
};

// A block id as the kernels use it: within the cache, whatever the table holds.
__device__ inline int tree_block(const TreeParams& p, int id) {
  id = id > 0 ? id : 0;
  return id < p.last_block ? id : p.last_block;
}

// Whether a row with mask words `m` sees key t of its sequence (t < len).
__device__ inline bool tree_sees(const TreeParams& p, const uint64_t* m, int prefix, int t) {
  const int u = t - prefix;
  if (u < 0) return true;
  const int w = u >> 6;
  return w < p.mask_words && ((m[w] >> (u & 63)) & 1) != 0;
}

}  // namespace xllm_hip
