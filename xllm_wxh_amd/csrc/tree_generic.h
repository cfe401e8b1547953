// Tree attention for any head_dim up to 256, any type, layout and block size; and the merge of cut sequences.
#pragma once

#include "device_utils.h"
#include "tree_params.h"

#include <math.h>

namespace xllm_hip {

// One wave per (sequence, chunk, kv head, query row): lanes are tokens for q.k, head-dim columns for p.v.  One pass
// over the chunk with the running maximum m and sum l of the softmax,
//   m' = max(m, max_t x_t),  l' = l 2^(m - m') + sum_t 2^(x_t - m'),  o' = o 2^(m - m') + sum_t 2^(x_t - m') v_t,
// in floats; a token the row does not see is given x = -inf and its V is never read.  Not tuned (one dependent
// cache row per lane): it serves the shapes the matrix kernels do not.
template <int Q_DT, int KV_DT>
__global__ void __launch_bounds__(64) tree_generic_kernel(TreeParams p) {
  __shared__ __attribute__((aligned(16))) float qs[256];
  TreeItem it;
  if (!tree_item(p, blockIdx.x, 1, it)) return;
  const int lane = threadIdx.x;
  const int D = p.head_dim;
  const float neg_inf = -INFINITY;
  constexpr bool kQuant = KV_DT == XLLM_HIP_FP8_E4M3 || KV_DT == XLLM_HIP_INT8;
  const int j = it.rg / p.group;
  const int head = it.hk * p.group + (it.rg - j * p.group);
  const int64_t row = it.q0 + j;
  const uint64_t* mask = p.mask + row * p.mask_stride;
  for (int d = lane; d < D; d += 64) qs[d] = Elem<Q_DT>::load(p.q, row * p.q_token_stride + (int64_t)head * D + d);
  __syncthreads();

  float m_run = neg_inf, l_run = 0.0f;
  float o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int tb = it.t_begin; tb < it.t_end; tb += 64) {
    const int tok = tb + lane;
    const bool vis = tok < it.t_end && tree_sees(p, mask, it.prefix, tok);
    float x = neg_inf, vscale = 1.0f;
    int64_t vrow = -1;
    if (vis) {
      const int bi = p.log2_bs >= 0 ? tok >> p.log2_bs : tok / p.block_size;
      const int64_t blk = tree_block(p, it.ids[bi < it.nblk ? bi : it.nblk - 1]);
      const int slot = tok - bi * p.block_size;
      vrow = blk * p.stride_block + (int64_t)it.hk * p.stride_head + (int64_t)slot * p.stride_slot;
      float dot = 0.0f;
      for (int d = 0; d < D; ++d) dot += qs[d] * Elem<KV_DT>::load(p.k_cache, vrow + d);
      if (kQuant) {
        const int64_t srow = blk * p.sc_stride_block + (int64_t)it.hk * p.sc_stride_head + (int64_t)slot * p.sc_stride_slot;
        dot *= p.k_scale[srow];
        vscale = p.v_scale[srow];
      }
      x = dot * p.scale_log2;
    }
    const float m_new = fmaxf(m_run, wave_max(x));
    const float m_safe = m_new == neg_inf ? 0.0f : m_new;
    const float alpha = __builtin_amdgcn_exp2f(m_run - m_safe);
    const float e = __builtin_amdgcn_exp2f(x - m_safe);
    l_run = l_run * alpha + wave_sum(e);
    m_run = m_new;
    const float pw = e * vscale;
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] *= alpha;
    const int cnt = it.t_end - tb < 64 ? it.t_end - tb : 64;
    for (int tt = 0; tt < cnt; ++tt) {
      const float pt = __shfl(pw, tt);
      const int64_t rw = __shfl(vrow, tt);
      if (rw < 0) continue;  // (uniform: the row does not see this token)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int d = lane + 64 * i;
        if (d < D) o[i] += pt * Elem<KV_DT>::load(p.v_cache, rw + d);
      }
    }
  }
  const float inv = l_run == 0.0f ? 0.0f : 1.0f / l_run;  // (a NaN stays one)
  const float lse2 = l_run == 0.0f ? neg_inf : m_run + __builtin_amdgcn_logf(l_run);
  if (it.chunks == 1) {
    if (lane == 0 && p.lse != nullptr) p.lse[row * p.num_q_heads + head] = lse2;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int d = lane + 64 * i;
      if (d < D) Elem<Q_DT>::store(p.out, row * p.out_token_stride + (int64_t)head * D + d, l_run == 0.0f ? 0.0f : o[i] * inv);
    }
    return;
  }
  const int64_t prow = ((int64_t)it.b * p.slots + it.chunk) * ((int64_t)p.n * p.num_q_heads) + (int64_t)j * p.num_q_heads + head;
  if (lane == 0) p.partial_lse[prow] = lse2;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int d = lane + 64 * i;
    if (d < D) p.partial_out[prow * D + d] = l_run == 0.0f ? 0.0f : o[i] * inv;
  }
}

// Rows of cut sequences: out = sum_c 2^(lse_c - lse) partial_c, lse = log2 sum_c 2^lse_c; a chunk that saw nothing has
// lse -inf, weight 0 and a partial of zeros.  Bound by the partials' bytes and by the latency of their loads, so four
// floats to a lane, D / 4 lanes to a chunk's row (a wave has 64 / (D / 4) chunks' rows at a time), and ROWS query rows
// to a wave, all of whose loads go out before the first is used: four where there are rows enough, else one, with more
// of its chunks at a time.
template <int Q_DT, int COLS, int ROWS, bool LINE>
__global__ void __launch_bounds__(256) tree_merge_kernel(TreeParams p) {
  static_assert(COLS == 16 || COLS == 32 || COLS == 64, "lanes that share a chunk's row, four columns each");
  constexpr int kAtOnce = 64 / COLS;
  constexpr int kRows = ROWS;
  constexpr int kUnroll = (ROWS == 1 ? 8 : 2) * (COLS == 64 ? 2 : 1);  // loads per query row in flight
  const int lane = threadIdx.x & 63;
  // (grid: rows of a sequence, sequences; the workgroups of a sequence that was not cut end here)
  const int b = blockIdx.y;
  const int len = tree_kv_length(p, b);
  int chunks = LINE ? 2 : tree_chunks(p, len);
  if (chunks == 1) return;  // written by the attention kernel
  const int per_seq = p.n * p.num_q_heads;
  int64_t q0;
  int count;
  tree_rows(p, b, q0, count);
  const int rows = (count < p.n ? count : p.n) * p.num_q_heads;
  const int r0 = ((int)blockIdx.x * 4 + (int)(threadIdx.x >> 6)) * kRows;
  if (r0 >= rows) return;
  int cut[LINE ? kRows : 1];  // chunks of a row: row groups of one sequence may be cut differently
  if constexpr (LINE) {
    const int64_t at = p.line[b], piece = p.line[p.batch];
    const int units = tree_line_units(len);
    chunks = 1;
#pragma unroll
    for (int k = 0; k < kRows; ++k) {
      cut[k] = 1;
      if (r0 + k < rows) {
        const int j = (r0 + k) / p.num_q_heads;
        const int row = j * p.group + (r0 + k - j * p.num_q_heads) % p.group;
        cut[k] = tree_line_chunks(at + (int64_t)(row / p.rows_per_item) * units, units, piece);
      }
      chunks = cut[k] > chunks ? cut[k] : chunks;
    }
    if (chunks == 1) return;
  }
  // Chunks to read: none of a row that the attention kernel has written.
  auto parts = [&](int k) {
    if constexpr (LINE) return cut[k] > 1 ? cut[k] : 0;
    return chunks;
  };
  const int D = p.head_dim;
  const float neg_inf = -INFINITY;
  const int64_t first = (int64_t)b * p.slots * per_seq;  // row r of chunk c: + c * per_seq + r
  const int col = (lane % COLS) * 4;
  const int mine = lane / COLS;
  const bool vec = (D & 3) == 0;
  f32x4 v[kRows][kUnroll];
  float l[kRows];
  auto load = [&](int c0) {
#pragma unroll
    for (int k = 0; k < kRows; ++k) {
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const int c = c0 + u * kAtOnce + mine;
        v[k][u] = f32x4{0, 0, 0, 0};
        if (c < parts(k) && col < D && r0 + k < rows) {
          const float* src = p.partial_out + (first + (int64_t)c * per_seq + r0 + k) * D + col;
          if (vec) {
            v[k][u] = *(const f32x4*)src;
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) v[k][u][e] = col + e < D ? src[e] : 0.0f;
          }
        }
      }
    }
  };
  // slots <= 64: a chunk to a lane
#pragma unroll
  for (int k = 0; k < kRows; ++k) {
    l[k] = lane < parts(k) && r0 + k < rows ? p.partial_lse[first + (int64_t)lane * per_seq + r0 + k] : neg_inf;
  }
  load(0);  // (on their way while the weights are formed)
  float e[kRows], m[kRows], total[kRows];
#pragma unroll
  for (int k = 0; k < kRows; ++k) {
    m[k] = wave_max(l[k]);
    e[k] = __builtin_amdgcn_exp2f(l[k] - (m[k] == neg_inf ? 0.0f : m[k]));
    total[k] = wave_sum(e[k]);
  }
  f32x4 o[kRows];
#pragma unroll
  for (int k = 0; k < kRows; ++k) o[k] = f32x4{0, 0, 0, 0};
  for (int c0 = 0; c0 < chunks; c0 += kAtOnce * kUnroll) {
    if (c0 > 0) load(c0);
#pragma unroll
    for (int k = 0; k < kRows; ++k) {
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) o[k] += __shfl(e[k], (c0 + u * kAtOnce + mine) & 63) * v[k][u];
    }
  }
#pragma unroll
  for (int k = 0; k < kRows; ++k) {
    if (r0 + k >= rows) break;
    if (LINE && parts(k) == 0) continue;
#pragma unroll
    for (int s = COLS; s < 64; s <<= 1) {
#pragma unroll
      for (int x = 0; x < 4; ++x) o[k][x] += __shfl_xor(o[k][x], s);
    }
    const float inv = total[k] == 0.0f ? 0.0f : 1.0f / total[k];
    const int j = (r0 + k) / p.num_q_heads;
    const int head = r0 + k - j * p.num_q_heads;
    const int64_t row = q0 + j;
    if (lane == 0 && p.lse != nullptr) {
      p.lse[row * p.num_q_heads + head] = total[k] == 0.0f ? neg_inf : m[k] + __builtin_amdgcn_logf(total[k]);
    }
    if (mine == 0) {
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        if (col + x < D) Elem<Q_DT>::store(p.out, row * p.out_token_stride + (int64_t)head * D + col + x, o[k][x] * inv);
      }
    }
  }
}

}  // namespace xllm_hip
