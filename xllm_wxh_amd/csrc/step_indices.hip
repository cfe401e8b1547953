// The index arrays of a step built on the device from the requests' lengths, and the ancestor masks of drafted
// trees.  What the batch builder does on the host (xllm/core/framework/batch/batch_input_builder.cpp:438-560) for a
// step whose lengths are on the device: after a speculative step the accepted counts are, and a read-back would
// hold the stream up.
//
// Both are launch-bound: the arrays of a decode step are kilobytes, those of a large mixed step a megabyte.  So
// each is one launch in which no workgroup waits for another: a workgroup that needs sums over the sequences in
// front of its own forms them itself from the lengths (4096 sequences at most: 48 KiB, from L2).  8 sequences of 4096
// tokens, one new token each: 5.0 us; 255 sequences of up to 9001 tokens and 700 new ones: 7.3, the loads of the
// lengths, the scan, the search for a row's sequence and the load of its block one after another.
#include "device_utils.h"
#include "host_utils.h"

#include <limits.h>

namespace xllm_hip {

constexpr int kStepMaxBatch = 4096;   // the offsets of all sequences fit a workgroup's LDS
constexpr int kStepThreads = 256;
constexpr int kStepTile = 1024;       // table columns or token rows per workgroup: four per thread

struct StepParams {
  xllm_hip_step_args a;
  int32_t log2_bs;       // of block_size, or -1 where it is no power of two
  int32_t seqs_per_wg;   // sequences a table workgroup walks
  int32_t col_tiles;     // column tiles of a table row
  int32_t table_wgs;     // workgroups of the table part; the token part follows
};

// What sequence b needs and owns before the sums over the sequences in front of it enter.
struct SeqNeed {
  int64_t cached, n, need;  // need: blocks of cached + n tokens
  int32_t row;              // its row of the block pool, -1: none
  int32_t held;             // blocks the row holds
  int32_t width;            // blocks it may have: min(need, pool and table width)
  int32_t grow;             // blocks to take from the free list
};

__device__ inline int64_t blocks_of(const StepParams& p, int64_t tokens) {
  if (p.log2_bs >= 0) return (tokens + p.a.block_size - 1) >> p.log2_bs;
  return (tokens + p.a.block_size - 1) / p.a.block_size;
}

__device__ inline SeqNeed seq_need(const StepParams& p, int b) {
  const xllm_hip_step_args& a = p.a;
  SeqNeed s;
  const int c = a.cached_lens[b];
  const int n = a.new_lens != nullptr ? a.new_lens[b] : a.q_per_seq;
  const int r = a.request_ids != nullptr ? a.request_ids[b] : b;
  const int h = a.held_blocks != nullptr ? a.held_blocks[b] : a.pool_width;
  s.cached = c > 0 ? c : 0;
  s.n = n > 0 ? n : 0;
  s.need = blocks_of(p, s.cached + s.n);
  s.row = r >= 0 && r < a.pool_rows ? r : -1;
  s.held = s.row < 0 ? 0 : (h < 0 ? 0 : (h < a.pool_width ? h : a.pool_width));
  const int w = a.pool_width < a.table_width ? a.pool_width : a.table_width;
  s.width = s.need < w ? (int)s.need : w;
  s.grow = s.row >= 0 && a.free_blocks != nullptr && s.width > s.held ? s.width - s.held : 0;
  return s;
}

// Blocks of the sequence that exist after the step: those held and those the free list still had.
__device__ inline int blocks_available(const StepParams& p, const SeqNeed& s, int64_t first_free) {
  int64_t got = (int64_t)p.a.num_free - first_free;
  got = got < 0 ? 0 : (got < s.grow ? got : s.grow);
  const int64_t have = s.held + got;
  return have < s.width ? (int)have : s.width;
}

__device__ inline int block_id(const StepParams& p, const SeqNeed& s, int i, int64_t first_free) {
  return i < s.held ? p.a.block_pool[(int64_t)s.row * p.a.pool_stride + i] : p.a.free_blocks[first_free + (i - s.held)];
}

__device__ inline int32_t clip32(int64_t v) { return v < INT_MAX ? (int32_t)v : INT_MAX; }

__device__ inline int64_t free_start(const StepParams& p) {
  if (p.a.free_head == nullptr) return 0;
  const int h = *p.a.free_head;
  return h > 0 ? h : 0;
}

__device__ inline int64_t wave_sum64(int64_t v) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o);
  return v;
}

// Rows of the table (and of the CSR list), the per-sequence scalars, the request's row of the pool.
__device__ inline void table_part(const StepParams& p, int wg, int64_t* lds) {
  const xllm_hip_step_args& a = p.a;
  const int group = wg / p.col_tiles, tile = wg - group * p.col_tiles;
  const int b0 = group * p.seqs_per_wg;
  const int tid = threadIdx.x;
  int64_t tokens = 0, grown = 0, listed = 0, taken = 0, missing = 0;
  const int64_t head = free_start(p);
  SeqNeed next = b0 < a.batch ? seq_need(p, b0) : SeqNeed{};  // (on its way while the sums are formed)
  for (int b = tid; b < b0; b += kStepThreads) {
    const SeqNeed s = seq_need(p, b);
    tokens += s.n;
    grown += s.grow;
    listed += s.need < a.table_width ? s.need : a.table_width;
  }
  // (a workgroup of the first sequences has nothing in front of it)
  if (b0 > 0) {
    tokens = wave_sum64(tokens);
    grown = wave_sum64(grown);
    listed = wave_sum64(listed);
    if ((tid & 63) == 0) {
      lds[(tid >> 6) * 3] = tokens;
      lds[(tid >> 6) * 3 + 1] = grown;
      lds[(tid >> 6) * 3 + 2] = listed;
    }
    __syncthreads();
    tokens = lds[0] + lds[3] + lds[6] + lds[9];
    grown = lds[1] + lds[4] + lds[7] + lds[10];
    listed = lds[2] + lds[5] + lds[8] + lds[11];
  }
  const int b1 = b0 + p.seqs_per_wg < a.batch ? b0 + p.seqs_per_wg : a.batch;
  for (int b = b0; b < b1; ++b) {
    const SeqNeed s = next;
    if (b + 1 < b1) next = seq_need(p, b + 1);
    const int64_t first = head + grown;
    const int avail = blocks_available(p, s, first);
    const int rows = s.need < a.table_width ? (int)s.need : a.table_width;  // listed blocks
    const int c1 = (tile + 1) * kStepTile < a.table_width ? (tile + 1) * kStepTile : a.table_width;
#pragma unroll 4
    for (int i = tile * kStepTile + tid; i < c1; i += kStepThreads) {
      const int id = i < avail ? block_id(p, s, i, first) : 0;
      a.block_table[(int64_t)b * a.table_stride + i] = id;
      if (i >= s.held && i < avail) a.block_pool[(int64_t)s.row * a.pool_stride + i] = id;
      if (a.kv_indptr != nullptr && i < rows && listed + i < a.kv_indices_capacity) a.kv_indices[listed + i] = id;
    }
    if (tile == 0 && tid == 0) {
      a.seq_lens[b] = clip32(s.cached + s.n);
      a.q_indptr[b] = clip32(tokens);
      if (a.kv_indptr != nullptr) {
        a.kv_indptr[b] = clip32(listed);
        const int64_t last = (s.cached + s.n) - (s.need - 1) * a.block_size;
        a.kv_last_page_len[b] = s.need == 0 ? 0 : (s.need > a.table_width ? a.block_size : (int)last);
      }
      if (a.held_blocks_out != nullptr) a.held_blocks_out[b] = s.held > avail ? s.held : avail;
    }
    tokens += s.n;
    grown += s.grow;
    listed += rows;
  }
  if (b1 == a.batch && tile == 0) {  // the last sequences' workgroup: the ends of the lists
    if (tid == 0) {
      a.q_indptr[a.batch] = clip32(tokens);
      if (a.kv_indptr != nullptr) a.kv_indptr[a.batch] = clip32(listed);
    }
    if (a.free_head_out != nullptr) {
      // blocks that could not be had, over all sequences (first of each: needs the sums again, which a thread's
      // own stretch of sequences does not give: one thread walks them, only when something can be missing)
      const int64_t end = head + grown;
      taken = end < a.num_free ? grown : (head < a.num_free ? a.num_free - head : 0);
      for (int b = tid; b < a.batch; b += kStepThreads) {
        const SeqNeed s = seq_need(p, b);
        const int have = s.held < s.width ? s.held : s.width;
        missing += s.need - have;
      }
      missing = wave_sum64(missing);
      __syncthreads();
      if ((tid & 63) == 0) lds[tid >> 6] = missing;
      __syncthreads();
      if (tid == 0) {
        a.free_head_out[0] = clip32(head + taken);
        a.free_head_out[1] = clip32(lds[0] + lds[1] + lds[2] + lds[3] - taken);
      }
    }
  }
}

// What the token rows need of the sequences: exclusive sums of token counts and of blocks taken; up to 512 sequences
// also what seq_need fetched, so that a row does not wait for it again (255 sequences: a tenth less time; the 96 KiB of 4096
// sequences would leave a CU one workgroup: 2000 sequences 16.9 -> 22.5 us).
template <int N>
struct StepSums {
  static constexpr bool kKept = N <= 512;
  int32_t q[N + 1];
  int32_t grow[N];
  int32_t cached[kKept ? N : 1];
  int32_t held[kKept ? N : 1];
  int32_t row[kKept ? N : 1];
  int32_t avail[kKept ? N : 1];
};

// Slots and positions of kStepTile token rows.
template <int N>
__device__ inline void token_part(const StepParams& p, int wg, StepSums<N>& of, int64_t* lds) {
  const xllm_hip_step_args& a = p.a;
  const int tid = threadIdx.x;
  const int wave = tid >> 6, lane = tid & 63;
  // Exclusive sums of the token counts and of the blocks taken: a thread sums its stretch of sequences, the
  // threads' sums are scanned over the workgroup, the thread then writes its stretch.
  const int per = (a.batch + kStepThreads - 1) / kStepThreads;
  const int s0 = tid * per, s1 = s0 + per < a.batch ? s0 + per : a.batch;
  int64_t n = 0, g = 0;
  for (int b = s0; b < s1; ++b) {
    const SeqNeed s = seq_need(p, b);
    n += s.n;
    g += s.grow;
  }
  int64_t ni = n, gi = g;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int64_t nu = __shfl_up(ni, o), gu = __shfl_up(gi, o);
    if (lane >= o) {
      ni += nu;
      gi += gu;
    }
  }
  if (lane == 63) {
    lds[2 * wave] = ni;
    lds[2 * wave + 1] = gi;
  }
  __syncthreads();
  int64_t nb = ni - n, gb = gi - g;
  for (int w = 0; w < wave; ++w) {
    nb += lds[2 * w];
    gb += lds[2 * w + 1];
  }
  const int64_t head = free_start(p);
  for (int b = s0; b < s1; ++b) {
    const SeqNeed s = seq_need(p, b);
    of.q[b] = clip32(nb);
    of.grow[b] = clip32(gb);
    if constexpr (StepSums<N>::kKept) {
      of.cached[b] = (int32_t)s.cached;
      of.held[b] = s.held;
      of.row[b] = s.row;
      of.avail[b] = blocks_available(p, s, head + gb);
    }
    nb += s.n;
    gb += s.grow;
    if (b == a.batch - 1) of.q[a.batch] = clip32(nb);
  }
  if (a.batch == 0 && tid == 0) of.q[0] = 0;
  __syncthreads();
  const int64_t total = of.q[a.batch];
#pragma unroll
  for (int u = 0; u < kStepTile / kStepThreads; ++u) {
    const int64_t t = (int64_t)wg * kStepTile + u * kStepThreads + tid;
    if (t >= a.num_rows) break;
    int64_t slot = -1, pos = 0;
    if (t < total) {
      int lo = 0, hi = a.batch;  // the last sequence whose offset is <= t (behind empty ones)
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (of.q[mid] <= t) {
          lo = mid;
        } else {
          hi = mid;
        }
      }
      const int64_t first = head + of.grow[lo];
      SeqNeed s;
      int avail;
      if constexpr (StepSums<N>::kKept) {
        s.cached = of.cached[lo];
        s.held = of.held[lo];
        s.row = of.row[lo];
        avail = of.avail[lo];
      } else {
        s = seq_need(p, lo);
        avail = blocks_available(p, s, first);
      }
      pos = s.cached + (t - of.q[lo]);
      const int64_t i = p.log2_bs >= 0 ? pos >> p.log2_bs : pos / a.block_size;
      if (i < avail) {
        const int id = block_id(p, s, (int)i, first);
        slot = (int64_t)id * a.block_size + (pos - i * a.block_size);
        if (id < 0 || slot > INT_MAX) slot = -1;
      }
    }
    a.slot_mapping[t] = (int32_t)slot;
    if (a.positions_int32) {
      ((int32_t*)a.positions)[t] = clip32(pos);
    } else {
      ((int64_t*)a.positions)[t] = pos;
    }
  }
}

// N: sequences at most.
template <int N>
__global__ void __launch_bounds__(kStepThreads) step_indices_kernel(StepParams p) {
  __shared__ StepSums<N> sums;
  __shared__ int64_t lds[12];
  if ((int)blockIdx.x < p.table_wgs) {
    table_part(p, blockIdx.x, lds);
  } else {
    token_part(p, blockIdx.x - p.table_wgs, sums, lds);
  }
}

// ---------------------------------------------------------------------------------
// Ancestor masks.  Pointer doubling: with A(v) = {v} and J(v) = parent(v), the step
//   A(v) <- A(v) U A(J(v)),  J(v) <- J(J(v))
// doubles the stretch of ancestors A(v) covers, so ceil(log2 (depth + 1)) steps finish any tree (a chain of 512 nodes
// takes nine; a walk up it would take 511 dependent reads; a random tree of 300 nodes takes four).  One workgroup per
// sequence, one thread per node, the words of all nodes in LDS; the depth is the number of bits set, less the node
// itself.  Bound by the launch, two dependent loads (offsets, parents), the doubling's barriers and the load of the base
// behind them (192 trees of up to 300 nodes: 5.4 us; 6.0 with eight words and nine steps for all of them).
// ---------------------------------------------------------------------------------
struct TreeMaskParams {
  const int32_t* parents;
  const int32_t* q_indptr;
  const int32_t* base;
  uint64_t* mask;
  void* positions;
  int64_t num_rows;
  int64_t mask_stride;
  int64_t axis_stride;
  int32_t q_per_seq;
  int32_t positions_int32;
  int32_t num_axes;
  int32_t mask_words;
};

template <int W>
__global__ void __launch_bounds__(64 * W) tree_masks_kernel(TreeMaskParams p) {
  constexpr int kNodes = 64 * W;
  __shared__ uint64_t words[W][kNodes];  // (word-major: neighbouring nodes in neighbouring banks)
  __shared__ int16_t jump[kNodes];
  const int b = blockIdx.x;
  const int v = threadIdx.x;
  int64_t row0;
  int64_t count;
  if (p.q_indptr != nullptr) {
    row0 = p.q_indptr[b];
    count = p.q_indptr[b + 1] - row0;
  } else {
    row0 = (int64_t)b * p.q_per_seq;
    count = p.q_per_seq;
  }
  if (row0 < 0 || row0 > p.num_rows) return;
  if (count > p.num_rows - row0) count = p.num_rows - row0;
  if (count <= 0) return;
  const int nodes = count < kNodes ? (int)count : kNodes;  // (the rest gets empty masks below)
  const int limit = nodes < 64 * p.mask_words ? nodes : 64 * p.mask_words;
  uint64_t mine[W];
#pragma unroll
  for (int w = 0; w < W; ++w) mine[w] = (v >> 6) == w && v < limit ? 1ull << (v & 63) : 0ull;
  int j = v < limit ? p.parents[row0 + v] : -1;
  j = j >= 0 && j < limit ? j : -1;
  int steps = 0;
  while ((1 << steps) < limit) ++steps;
  for (int k = 0; k < steps; ++k) {
#pragma unroll
    for (int w = 0; w < W; ++w) words[w][v] = mine[w];
    jump[v] = (int16_t)j;
    if (!__syncthreads_or(j >= 0)) break;  // every chain has reached the context
    if (j >= 0) {
#pragma unroll
      for (int w = 0; w < W; ++w) mine[w] |= words[w][j];
      j = jump[j];
    }
    __syncthreads();
  }
  int depth = -1;
#pragma unroll
  for (int w = 0; w < W; ++w) depth += __popcll(mine[w]);
  depth = depth > 0 ? depth : 0;
  const int start = p.base != nullptr ? p.base[b] : 0;
  for (int64_t u = v; u < count; u += kNodes) {
    const int64_t row = row0 + u;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      if (w < p.mask_words) p.mask[row * p.mask_stride + w] = u == v ? mine[w] : 0ull;
    }
    if (p.positions != nullptr) {
      const int64_t pos = (int64_t)start + (u == v ? depth : 0);
      for (int a = 0; a < p.num_axes; ++a) {
        if (p.positions_int32) {
          ((int32_t*)p.positions)[a * p.axis_stride + row] = (int32_t)pos;
        } else {
          ((int64_t*)p.positions)[a * p.axis_stride + row] = pos;
        }
      }
    }
  }
}

// Whether [a, a + an) and [b, b + bn) share a byte.
static bool overlaps(const void* a, int64_t an, const void* b, int64_t bn) {
  if (a == nullptr || b == nullptr || an <= 0 || bn <= 0) return false;
  const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
  return x < y + (uintptr_t)bn && y < x + (uintptr_t)an;
}

}  // namespace xllm_hip

using namespace xllm_hip;

extern "C" int xllm_hip_build_step_indices(const xllm_hip_step_args* a, xllm_hip_stream_t stream) {
  XLLM_HIP_REQUIRE(a != nullptr, "step args are NULL");
  XLLM_HIP_REQUIRE(a->batch >= 0 && a->num_rows >= 0, "batch or num_rows is negative");
  if (a->batch > kStepMaxBatch) {
    return fail(XLLM_HIP_UNSUPPORTED, "batch %d is larger than %d sequences", a->batch, kStepMaxBatch);
  }
  XLLM_HIP_REQUIRE(a->block_size >= 1 && a->pool_width >= 1 && a->pool_rows >= 1 && a->table_width >= 1,
                   "block_size, pool_width, pool_rows and table_width must be positive");
  XLLM_HIP_REQUIRE(a->pool_stride >= a->pool_width && a->table_stride >= a->table_width,
                   "pool_stride or table_stride smaller than the row");
  XLLM_HIP_REQUIRE(a->q_per_seq >= 0, "q_per_seq is negative");
  XLLM_HIP_REQUIRE(a->num_free >= 0 && a->kv_indices_capacity >= 0, "num_free or kv_indices_capacity is negative");
  XLLM_HIP_REQUIRE(a->q_indptr != nullptr, "q_indptr is NULL");
  XLLM_HIP_REQUIRE(a->num_rows == 0 || (a->slot_mapping != nullptr && a->positions != nullptr),
                   "slot_mapping or positions is NULL");
  XLLM_HIP_REQUIRE(a->batch == 0 || (a->cached_lens != nullptr && a->block_pool != nullptr && a->block_table != nullptr &&
                                     a->seq_lens != nullptr),
                   "cached_lens, block_pool, block_table or seq_lens is NULL");
  // (arrays without entries may be NULL)
  XLLM_HIP_REQUIRE((a->kv_indptr == nullptr || ((a->kv_indices != nullptr || a->kv_indices_capacity == 0) &&
                                                (a->kv_last_page_len != nullptr || a->batch == 0))) &&
                       (a->kv_indptr != nullptr || (a->kv_indices == nullptr && a->kv_last_page_len == nullptr)),
                   "kv_indptr, kv_indices and kv_last_page_len go together");
  XLLM_HIP_REQUIRE((a->free_blocks == nullptr || a->free_head != nullptr) &&
                       (a->free_head == nullptr || a->free_blocks != nullptr || a->num_free == 0),
                   "free_blocks and free_head go together");
  XLLM_HIP_REQUIRE(a->free_blocks == nullptr || a->held_blocks != nullptr || a->batch == 0, "free_blocks needs held_blocks");
  XLLM_HIP_REQUIRE(a->batch == 0 || ((a->held_blocks == nullptr) == (a->held_blocks_out == nullptr) &&
                                     (a->held_blocks == nullptr) == (a->free_head_out == nullptr)),
                   "held_blocks, held_blocks_out and free_head_out go together");
  // Every workgroup reads the inputs while others write the outputs.
  const int64_t B = a->batch, pb = a->positions_int32 ? 4 : 8;
  const struct { const void* p; int64_t n; } in[] = {
      {a->cached_lens, 4 * B}, {a->new_lens, 4 * B}, {a->request_ids, 4 * B}, {a->held_blocks, 4 * B},
      {a->free_blocks, 4 * (int64_t)a->num_free}, {a->free_head, 4},
      {B > 0 ? a->block_pool : nullptr, 4 * ((a->pool_rows - 1) * a->pool_stride + a->pool_width)}};
  const struct { const void* p; int64_t n; } out[] = {
      {B > 0 ? a->block_table : nullptr, 4 * ((B - 1) * a->table_stride + a->table_width)}, {a->seq_lens, 4 * B},
      {a->q_indptr, 4 * (B + 1)}, {a->slot_mapping, 4 * a->num_rows}, {a->positions, pb * a->num_rows},
      {a->kv_indptr, 4 * (B + 1)}, {a->kv_indices, 4 * a->kv_indices_capacity}, {a->kv_last_page_len, 4 * B},
      {a->held_blocks_out, 4 * B}, {a->free_head_out, 8}};
  for (const auto& o : out) {
    for (const auto& i : in) XLLM_HIP_REQUIRE(!overlaps(o.p, o.n, i.p, i.n), "an output overlaps an input");
  }
  StepParams p{};
  p.a = *a;
  p.log2_bs = is_pow2(a->block_size) ? ilog2(a->block_size) : -1;
  // (at most 512 groups: the sums in front of a group cost each of them a pass over the lengths before it)
  p.seqs_per_wg = (a->batch + 511) / 512 > 1 ? (a->batch + 511) / 512 : 1;
  p.col_tiles = (a->table_width + kStepTile - 1) / kStepTile;
  const int64_t groups = a->batch > 0 ? (a->batch + p.seqs_per_wg - 1) / p.seqs_per_wg : 1;
  const int64_t table_wgs = groups * p.col_tiles;
  const int64_t token_wgs = (a->num_rows + kStepTile - 1) / kStepTile;
  XLLM_HIP_REQUIRE(table_wgs + token_wgs <= 0x7fffffff, "too many rows");
  p.table_wgs = (int32_t)table_wgs;
  const unsigned grid = (unsigned)(table_wgs + token_wgs);
  if (a->batch <= 512) {
    step_indices_kernel<512><<<grid, kStepThreads, 0, (hipStream_t)stream>>>(p);
  } else {
    step_indices_kernel<kStepMaxBatch><<<grid, kStepThreads, 0, (hipStream_t)stream>>>(p);
  }
  return check_launch("step_indices_kernel");
}

extern "C" int xllm_hip_tree_masks(const int32_t* parents,
                                   const int32_t* q_indptr,
                                   const int32_t* base,
                                   int32_t batch,
                                   int32_t q_per_seq,
                                   int64_t num_rows,
                                   uint64_t* mask,
                                   int64_t mask_stride,
                                   int32_t mask_words,
                                   void* positions,
                                   int32_t positions_int32,
                                   int32_t num_axes,
                                   int64_t axis_stride,
                                   xllm_hip_stream_t stream) {
  XLLM_HIP_REQUIRE(batch >= 0 && num_rows >= 0 && q_per_seq >= 0, "batch, num_rows or q_per_seq is negative");
  XLLM_HIP_REQUIRE(mask_words >= 1 && mask_stride >= mask_words, "mask rows need at least one word");
  if (mask_words > 8) return fail(XLLM_HIP_UNSUPPORTED, "mask_words %d is larger than 8 (512 nodes)", mask_words);
  if (batch == 0 || num_rows == 0) return XLLM_HIP_OK;
  XLLM_HIP_REQUIRE(parents != nullptr && mask != nullptr, "parents or mask is NULL");
  XLLM_HIP_REQUIRE(q_indptr != nullptr || (int64_t)batch * q_per_seq <= num_rows, "batch * q_per_seq exceeds num_rows");
  XLLM_HIP_REQUIRE(positions == nullptr || (num_axes >= 1 && num_axes <= 4 && (num_axes == 1 || axis_stride >= num_rows)),
                   "positions need 1 to 4 axes, at least num_rows apart");
  TreeMaskParams p{parents,   q_indptr,    base,      mask,            positions, num_rows, mask_stride,
                   axis_stride, q_per_seq, positions_int32, num_axes, mask_words};
  hipStream_t st = (hipStream_t)stream;
  switch (mask_words) {
#define TREE_MASKS_CASE(W)                                   \
  case W:                                                    \
    tree_masks_kernel<W><<<batch, 64 * W, 0, st>>>(p);       \
    break;
    TREE_MASKS_CASE(1)
    TREE_MASKS_CASE(2)
    TREE_MASKS_CASE(3)
    TREE_MASKS_CASE(4)
    TREE_MASKS_CASE(5)
    TREE_MASKS_CASE(6)
    TREE_MASKS_CASE(7)
    default:
    TREE_MASKS_CASE(8)
#undef TREE_MASKS_CASE
  }
  return check_launch("tree_masks_kernel");
}
