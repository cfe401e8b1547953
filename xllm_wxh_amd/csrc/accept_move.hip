// The cache rows of an accepted path moved to the front of the drafted range of their sequences (K, V and, for a
// quantised cache, the two scale tensors), and the sequences' new lengths.
//
// Every source row is read before any destination is written — a destination is often another row's source: the
// path 2, 5, 6 writes row 2 from row 6 after row 0 was to receive row 2.  A workgroup owns a set of columns (pieces
// of 16 bytes, or of one element where the strides do not allow that) of all path rows of one sequence and one
// array, holds them in registers, and meets at a barrier between its loads and its stores; no other workgroup
// touches those bytes.
//
// Little memory traffic behind a chain of three dependent loads (length, path and table entry, row), so what counts is
// how many chains run side by side: one launch for K, V and the scales, as few pieces to a thread as keep K and V near
// two thousand workgroups (more only queue; the scales' have little to do), and few registers (512 sequences, paths of
// 13 rows of fp8: 27 us with eight pieces to every thread and the scales in a launch of their own, 9 so).
#include "device_utils.h"
#include "host_utils.h"

namespace xllm_hip {

constexpr int kMoveThreads = 256;
constexpr int kMovePieces = 8;     // most pieces a thread holds
constexpr int kMoveMaxPath = 1024;

struct AcceptParams {
  // array a: 0 = K, 1 = V, 2 = K scales, 3 = V scales
  uint8_t* base[4];
  int64_t stride_block[4];  // bytes
  int64_t stride_head[4];
  int64_t stride_slot[4];
  int32_t pieces[4];        // pieces of one (head, token) row
  int32_t cols[4];          // columns: num_kv_heads * pieces
  int32_t cols_per_wg[4];
  const int32_t* table;
  const int32_t* cached;
  const int32_t* accepted;
  const int32_t* count;
  int32_t* new_lens;
  int64_t table_stride;
  int64_t accepted_stride;
  int64_t num_blocks;
  int64_t capacity;         // tokens a table row holds
  int32_t path;
  int32_t block_size;
  int32_t log2_bs;          // or -1
};

// Byte offset of token `tok`'s row (head 0) in array a, or -1 where the table does not reach it.
__device__ inline int64_t token_offset(const AcceptParams& p, int a, int b, int64_t tok) {
  if (tok < 0 || tok >= p.capacity) return -1;
  const int64_t i = p.log2_bs >= 0 ? tok >> p.log2_bs : tok / p.block_size;
  const int64_t blk = p.table[(int64_t)b * p.table_stride + i];
  if (blk < 0 || blk >= p.num_blocks) return -1;
  return blk * p.stride_block[a] + (tok - i * p.block_size) * p.stride_slot[a];
}

// One workgroup's columns of array a; PIECES to a thread, cnt * cols <= kMoveThreads * PIECES (see the host side).
template <typename VecT, int PIECES>
__device__ inline void move_columns(const AcceptParams& p, int a, int b, int col0, int64_t c, int cnt, int64_t* src, int64_t* dst) {
  const int tid = threadIdx.x;
  for (int i = tid; i < cnt; i += kMoveThreads) {
    const int k = p.accepted[(int64_t)b * p.accepted_stride + i];
    int64_t from = -1, to = -1;
    if (k >= 0 && k != i) {
      from = token_offset(p, a, b, c + k);
      to = token_offset(p, a, b, c + i);
    }
    src[i] = to >= 0 ? from : -1;  // (-1: nothing to move)
    dst[i] = to;
  }
  __syncthreads();
  const int cols = p.cols[a] - col0 < p.cols_per_wg[a] ? p.cols[a] - col0 : p.cols_per_wg[a];
  const int items = cnt * cols;
  VecT v[PIECES];
  int64_t to[PIECES];
#pragma unroll
  for (int u = 0; u < PIECES; ++u) {
    const int x = u * kMoveThreads + tid;
    to[u] = -1;
    if (x < items) {
      const int i = (int)((unsigned)x / (unsigned)cols);
      const int col = col0 + (x - i * cols);
      const int h = (int)((unsigned)col / (unsigned)p.pieces[a]);
      const int64_t off = (int64_t)h * p.stride_head[a] + (int64_t)(col - h * p.pieces[a]) * (int64_t)sizeof(VecT);
      if (src[i] >= 0) {
        v[u] = *(const VecT*)(p.base[a] + src[i] + off);
        to[u] = dst[i] + off;
      }
    }
  }
  // The stores of the others may only start when these loads have returned.
  __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0)
  __syncthreads();
#pragma unroll
  for (int u = 0; u < PIECES; ++u) {
    if (to[u] >= 0) *(VecT*)(p.base[a] + to[u]) = v[u];
  }
}

// grid (columns, sequence, array).  LDS: two offsets per path row.
template <typename VecT, int PIECES>
__global__ void __launch_bounds__(kMoveThreads, PIECES == 1 ? 8 : 4) accept_move_kernel(AcceptParams p) {
  extern __shared__ int64_t offsets[];
  const int b = blockIdx.y;
  const int a = blockIdx.z;
  const int col0 = blockIdx.x * p.cols_per_wg[a];
  const int64_t c = p.cached[b];
  int cnt = p.count[b];
  cnt = cnt < 0 ? 0 : (cnt < p.path ? cnt : p.path);
  if (blockIdx.x == 0 && a == 0 && threadIdx.x == 0 && p.new_lens != nullptr) p.new_lens[b] = (int32_t)(c + cnt);
  if (col0 >= p.cols[a]) return;
  if (a < 2) {
    move_columns<VecT, PIECES>(p, a, b, col0, c, cnt, offsets, offsets + p.path);
  } else {
    move_columns<uint32_t, PIECES>(p, a, b, col0, c, cnt, offsets, offsets + p.path);
  }
}

template <typename VecT>
static void launch_accept_move(int pieces, const AcceptParams& p, dim3 grid, hipStream_t st) {
  const size_t lds = (size_t)(2 * (p.path > 0 ? p.path : 1)) * sizeof(int64_t);  // <= 16 KiB
  if (pieces == 1) {
    accept_move_kernel<VecT, 1><<<grid, kMoveThreads, lds, st>>>(p);
  } else if (pieces == 2) {
    accept_move_kernel<VecT, 2><<<grid, kMoveThreads, lds, st>>>(p);
  } else if (pieces == 4) {
    accept_move_kernel<VecT, 4><<<grid, kMoveThreads, lds, st>>>(p);
  } else {
    accept_move_kernel<VecT, 8><<<grid, kMoveThreads, lds, st>>>(p);
  }
}

}  // namespace xllm_hip

using namespace xllm_hip;

extern "C" int xllm_hip_move_accepted_tokens(const xllm_hip_kv_cache* cache,
                                             const int32_t* block_table,
                                             int64_t block_table_stride,
                                             int32_t max_blocks_per_seq,
                                             const int32_t* cached_lens,
                                             const int32_t* accepted,
                                             int64_t accepted_stride,
                                             int32_t path_width,
                                             const int32_t* num_accepted,
                                             int32_t batch,
                                             int32_t* new_lens,
                                             xllm_hip_stream_t stream) {
  XLLM_HIP_REQUIRE(cache != nullptr, "cache is NULL");
  XLLM_HIP_REQUIRE(batch >= 0 && path_width >= 0, "batch or path_width is negative");
  if (batch == 0) return XLLM_HIP_OK;
  if (path_width > kMoveMaxPath) {
    return fail(XLLM_HIP_UNSUPPORTED, "path_width %d is larger than %d", path_width, kMoveMaxPath);
  }
  XLLM_HIP_REQUIRE(batch <= 65535, "batch %d is larger than 65535", batch);
  XLLM_HIP_REQUIRE(cache->k_cache != nullptr && cache->v_cache != nullptr, "k_cache or v_cache is NULL");
  XLLM_HIP_REQUIRE(cache->num_blocks > 0 && cache->block_size > 0 && cache->num_kv_heads > 0 && cache->head_dim > 0,
                   "cache sizes must be positive");
  const int eb = elem_bytes(cache->dtype);
  XLLM_HIP_REQUIRE(eb > 0, "unknown cache dtype %d", cache->dtype);
  const bool quant = cache->dtype == XLLM_HIP_FP8_E4M3 || cache->dtype == XLLM_HIP_INT8;
  XLLM_HIP_REQUIRE(!quant || (cache->k_scale != nullptr && cache->v_scale != nullptr),
                   "a quantised cache needs k_scale and v_scale");
  XLLM_HIP_REQUIRE(cache->stride_block > 0 && cache->stride_head > 0 && cache->stride_slot > 0,
                   "cache strides must be positive");
  XLLM_HIP_REQUIRE(cached_lens != nullptr && num_accepted != nullptr && block_table != nullptr,
                   "cached_lens, num_accepted or block_table is NULL");
  XLLM_HIP_REQUIRE(max_blocks_per_seq >= 1 && block_table_stride >= max_blocks_per_seq, "bad block_table shape");
  XLLM_HIP_REQUIRE(path_width == 0 || (accepted != nullptr && accepted_stride >= path_width), "bad accepted shape");
  // (every workgroup reads the inputs while one writes the new lengths)
  auto apart = [&](const int32_t* in, int64_t n) {
    return new_lens == nullptr || (uintptr_t)(new_lens + batch) <= (uintptr_t)in || (uintptr_t)(in + n) <= (uintptr_t)new_lens;
  };
  XLLM_HIP_REQUIRE(apart(cached_lens, batch), "new_lens overlaps cached_lens");
  XLLM_HIP_REQUIRE(apart(num_accepted, batch), "new_lens overlaps num_accepted");
  XLLM_HIP_REQUIRE(path_width == 0 || apart(accepted, (int64_t)(batch - 1) * accepted_stride + path_width), "new_lens overlaps accepted");
  XLLM_HIP_REQUIRE(apart(block_table, (int64_t)(batch - 1) * block_table_stride + max_blocks_per_seq), "new_lens overlaps block_table");

  AcceptParams p{};
  const int64_t row = (int64_t)cache->head_dim * eb;
  // the widest piece every address is a multiple of
  uintptr_t bits = (uintptr_t)cache->k_cache | (uintptr_t)cache->v_cache | (uintptr_t)(cache->stride_block * eb) |
                   (uintptr_t)(cache->stride_head * eb) | (uintptr_t)(cache->stride_slot * eb) | (uintptr_t)row;
  const int piece = (bits & 15) == 0 ? 16 : eb;
  for (int a = 0; a < 4; ++a) {
    const bool scale = a >= 2;
    const int64_t unit = scale ? 4 : eb;
    p.base[a] = (uint8_t*)(a == 0 ? cache->k_cache : a == 1 ? cache->v_cache : a == 2 ? (void*)cache->k_scale : (void*)cache->v_scale);
    p.stride_block[a] = (scale ? cache->scale_stride_block : cache->stride_block) * unit;
    p.stride_head[a] = (scale ? cache->scale_stride_head : cache->stride_head) * unit;
    p.stride_slot[a] = (scale ? cache->scale_stride_slot : cache->stride_slot) * unit;
    p.pieces[a] = scale ? 1 : (int32_t)(row / piece);
    const int64_t cols = (int64_t)cache->num_kv_heads * p.pieces[a];
    XLLM_HIP_REQUIRE(cols <= 0x7fffffff, "too many kv heads");
    p.cols[a] = (int32_t)cols;
  }
  // Pieces to a thread: as few as make at most 2048 workgroups for K and V, kMovePieces at most; a workgroup takes a path's
  // whole columns.
  const int arrays = quant ? 4 : 2;
  const int path = path_width > 0 ? path_width : 1;
  int pieces = 1;
  unsigned columns = 1;
  for (;; pieces *= 2) {
    const int most = kMoveThreads * pieces / path;
    columns = 1;
    for (int a = 0; a < arrays; ++a) {
      p.cols_per_wg[a] = most > 1 ? most : 1;
      const unsigned wgs = (unsigned)((p.cols[a] + p.cols_per_wg[a] - 1) / p.cols_per_wg[a]);
      columns = wgs > columns ? wgs : columns;
    }
    if (pieces == kMovePieces || (most >= 1 && (int64_t)columns * batch * 2 <= 2048)) break;
  }
  p.table = block_table;
  p.cached = cached_lens;
  p.accepted = accepted;
  p.count = num_accepted;
  p.new_lens = new_lens;
  p.table_stride = block_table_stride;
  p.accepted_stride = accepted_stride;
  p.num_blocks = cache->num_blocks;
  p.capacity = (int64_t)max_blocks_per_seq * cache->block_size;
  p.path = path_width;
  p.block_size = cache->block_size;
  p.log2_bs = is_pow2(cache->block_size) ? ilog2(cache->block_size) : -1;
  hipStream_t st = (hipStream_t)stream;
  const dim3 grid(columns, batch, arrays);
  if (piece == 16) {
    launch_accept_move<u32x4>(pieces, p, grid, st);
  } else if (piece == 4) {
    launch_accept_move<uint32_t>(pieces, p, grid, st);
  } else if (piece == 2) {
    launch_accept_move<uint16_t>(pieces, p, grid, st);
  } else {
    launch_accept_move<uint8_t>(pieces, p, grid, st);
  }
  return check_launch("accept_move_kernel");
}
