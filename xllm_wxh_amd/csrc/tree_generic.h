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
// cache row per lane): it serves the shapes the matrix kernels do not, and checks them.
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

// Rows of cut sequences: out = sum_c 2^(lse_c - lse) partial_c, lse = log2 sum_c 2^lse_c.  One wave per row, four rows
// to a workgroup; a chunk that saw nothing has lse -inf, weight 0 and a partial of zeros.
template <int Q_DT>
__global__ void __launch_bounds__(256) tree_merge_kernel(TreeParams p) {
  const int lane = threadIdx.x & 63;
  const int64_t unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int64_t per_seq = (int64_t)p.n * p.num_q_heads;
  const int64_t b64 = unit / per_seq;
  if (b64 >= p.batch) return;
  const int b = (int)b64;
  const int rem = (int)(unit - b64 * per_seq);
  const int j = rem / p.num_q_heads;
  const int head = rem - j * p.num_q_heads;
  int64_t q0;
  int count;
  tree_rows(p, b, q0, count);
  if (j >= count) return;
  const int chunks = tree_chunks(p, tree_kv_length(p, b));
  if (chunks == 1) return;  // written by the attention kernel
  const int D = p.head_dim;
  const float neg_inf = -INFINITY;
  const int64_t first = (int64_t)b * p.slots * per_seq + rem;  // chunk c: + c * per_seq
  // slots <= 64: a chunk to a lane
  const float l = lane < chunks ? p.partial_lse[first + lane * per_seq] : neg_inf;
  const float m = wave_max(l);
  const float m_safe = m == neg_inf ? 0.0f : m;
  const float e = __builtin_amdgcn_exp2f(l - m_safe);
  const float total = wave_sum(e);
  float o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int c = 0; c < chunks; ++c) {
    const float w = __shfl(e, c);
    const float* src = p.partial_out + (first + c * per_seq) * D;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int d = lane + 64 * i;
      if (d < D) o[i] += w * src[d];
    }
  }
  const float inv = total == 0.0f ? 0.0f : 1.0f / total;
  const int64_t row = q0 + j;
  if (lane == 0 && p.lse != nullptr) {
    p.lse[row * p.num_q_heads + head] = total == 0.0f ? neg_inf : m + __builtin_amdgcn_logf(total);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int d = lane + 64 * i;
    if (d < D) Elem<Q_DT>::store(p.out, row * p.out_token_stride + (int64_t)head * D + d, o[i] * inv);
  }
}

}  // namespace xllm_hip
