// Norm, rotary embedding with positions of several axes, and the KV write, in one pass over the fused qkv buffer:
// rope_kv_write.hip's step for models whose tokens have a position in time, height and width.
//
//   x <- x / sqrt(mean x^2 + eps) * weight                         (q and k heads, optional)
//   pair j, axis a = axis(j), p = positions[a][t]:
//   x' = x cos - y sin,  y' = y cos + x sin,   cos = table[p][j], sin = table[p][rotary_dim/2 + j]
//
// in float with one rounding to the element type at the end (or, round_each_op, after every operation).
//
// The table row of a token is mixed from one row per axis.  A workgroup belongs to one token and mixes that row once,
// into LDS, for all of the token's heads (each head fetching it by itself asks the caches for the row 40 times and
// picks the axis 40 times).  Then D / 8 lanes to a head, eight elements (16 bytes of a 16-bit type) to a lane; a
// rotation partner is a shuffle away.  The bound is memory: q and k heads read and written, v heads read, K and V
// rows written (8191 bf16 tokens of 32 + 8 + 8 heads of 128, norm, 16-bit cache: 51 us for 223 MB, 4.3 TB/s where a
// large copy runs at 5.0; 136 drafted tokens of 14 + 2 + 2 heads of 64: 4.6 us, a launch).  Other head sizes, strides
// and rotary dims take a wave per head, an element to a lane.
#include "device_utils.h"
#include "host_utils.h"
#include "rope_common.h"

#include <float.h>

namespace xllm_hip {

struct MropeParams {
  RopeParams r;
  int64_t axis_stride;
  int32_t num_axes;
  int32_t dealt;
  int32_t sections[4];
  int32_t heads;         // heads to walk: without a cache the v heads are left alone
  int32_t cache_vec_ok;  // cache rows can be written in the lanes' vectors
};

__device__ inline int axis_of_pair(const MropeParams& p, int j) {
  if (p.dealt) {
    const int a = j % p.num_axes;
    return j / p.num_axes < p.sections[a] ? a : 0;
  }
  int a = 0, end = p.sections[0];
  while (a < p.num_axes - 1 && j >= end) end += p.sections[++a];
  return a;
}

__device__ inline int64_t position_of(const MropeParams& p, int a, int64_t t) {
  const int64_t i = a * p.axis_stride + t;
  const int64_t pos = p.r.positions_int32 ? (int64_t)((const int32_t*)p.r.positions)[i] : ((const int64_t*)p.r.positions)[i];
  return pos < 0 ? 0 : (pos >= p.r.max_position ? p.r.max_position - 1 : pos);  // never read outside the table
}

// Element x < rotary_dim of token t's mixed table row: cos of pair x, or sin of pair x - rotary_dim/2.
template <int DT>
__device__ inline float table_value(const MropeParams& p, int64_t t, int x) {
  const int half = p.r.rotary_dim >> 1;
  const int64_t pos = position_of(p, axis_of_pair(p, x < half ? x : x - half), t);
  const float v = load_any(p.r.cos_sin, pos * p.r.rotary_dim + x, p.r.cos_sin_dtype);
  return p.r.per_op ? rounded<DT>(v) : v;
}

// Eight elements as floats and back.
template <int DT>
struct Eight {
  u32x4 raw[DT == XLLM_HIP_FP32 ? 2 : 1];
  __device__ inline void load(const void* p, int64_t i) {
    if constexpr (DT == XLLM_HIP_FP32) {
      raw[0] = *(const u32x4*)((const float*)p + i);
      raw[1] = *(const u32x4*)((const float*)p + i + 4);
    } else {
      raw[0] = *(const u32x4*)((const uint16_t*)p + i);
    }
  }
  __device__ inline void store(void* p, int64_t i) const {
    if constexpr (DT == XLLM_HIP_FP32) {
      *(u32x4*)((float*)p + i) = raw[0];
      *(u32x4*)((float*)p + i + 4) = raw[1];
    } else {
      *(u32x4*)((uint16_t*)p + i) = raw[0];
    }
  }
  __device__ inline void get(float (&x)[8]) const {
    if constexpr (DT == XLLM_HIP_FP32) {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = __uint_as_float(raw[e >> 2][e & 3]);
    } else {
      unpack8<DT>(raw[0], x);
    }
  }
  __device__ inline void set(const float (&x)[8]) {
    if constexpr (DT == XLLM_HIP_FP32) {
#pragma unroll
      for (int e = 0; e < 8; ++e) raw[e >> 2][e & 3] = __float_as_uint(x[e]);
    } else {
      raw[0] = pack8<DT>(x);
    }
  }
  // element by element, for rows that are not 16-byte aligned
  __device__ inline void store_elements(void* p, int64_t i) const {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if constexpr (DT == XLLM_HIP_FP32) {
        ((uint32_t*)p)[i + e] = raw[e >> 2][e & 3];
      } else {
        ((uint16_t*)p)[i + e] = (uint16_t)(raw[0][e >> 1] >> (16 * (e & 1)));
      }
    }
  }
};

// LANES lanes to a head of 8 * LANES elements.  grid (token, part): a part is PASSES * 256 / LANES heads.
template <int DT, int LANES, int CACHE, int PASSES>
__global__ void __launch_bounds__(256) mrope_kv_write_kernel(MropeParams p) {
  constexpr int kD = 8 * LANES;
  constexpr int kHeads = 256 / LANES;  // per pass
  __shared__ __attribute__((aligned(16))) float table[kD];  // cos of the pairs, then sin
  const int tid = threadIdx.x;
  const int sub = tid & (LANES - 1);
  const int64_t t = blockIdx.x;
  const int first_head = blockIdx.y * (PASSES * kHeads) + tid / LANES;
  const int R = p.r.rotary_dim;
  const int64_t base = t * p.r.token_stride + 8 * sub;

  // every pass's row is on its way before the table is mixed
  Eight<DT> in[PASSES];
#pragma unroll
  for (int u = 0; u < PASSES; ++u) {
    const int hh = first_head + u * kHeads;
    if (hh < p.heads) {
      in[u].load(p.r.qkv, base + (int64_t)hh * kD);
    } else {
      in[u].raw[0] = u32x4{0, 0, 0, 0};
      if constexpr (DT == XLLM_HIP_FP32) in[u].raw[1] = u32x4{0, 0, 0, 0};
    }
  }
  const int64_t slot = CACHE != kNoCache ? (int64_t)p.r.slots[t] : -1;
  if (tid < R) table[tid] = table_value<DT>(p, t, tid);
  __syncthreads();

  // this lane's factors: the same for every head
  const int half = R >> 1;
  const bool rotates = 8 * sub < R;
  const int hl = R >> 4;  // lanes per half of the rotated range
  float c[8], sn[8];
  bool lower = false;  // the lane holds the x of its pairs (pairs side by side in a lane: decided by element)
  if (p.r.interleave) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      c[e] = table[rotates ? 4 * sub + (e >> 1) : 0];
      sn[e] = table[rotates ? half + 4 * sub + (e >> 1) : 0];
    }
  } else {
    lower = sub < hl;
    const int f = rotates ? 8 * (lower ? sub : sub - hl) : 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      c[e] = table[f + e];
      sn[e] = table[rotates ? half + f + e : 0];
    }
  }
  const bool writes = slot >= 0 && slot < p.r.num_slots;
  const int64_t block = writes ? slot / p.r.block_size : 0;
  const int64_t off = writes ? slot - block * p.r.block_size : 0;
  const int lane = tid & 63;
  const int partner = rotates && !p.r.interleave ? (lower ? lane + hl : lane - hl) : lane;

#pragma unroll
  for (int u = 0; u < PASSES; ++u) {
    const int hh = first_head + u * kHeads;
    const bool live = hh < p.heads;  // idle groups still take part in the shuffles
    const bool is_q = hh < p.r.num_q_heads;
    const bool is_v = hh >= p.r.num_q_heads + p.r.num_k_heads;
    float x[8];
    in[u].get(x);
    if (!is_v) {
      const void* w = is_q ? p.r.q_weight : p.r.k_weight;
      if (w != nullptr) {
        float ss = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) ss += x[e] * x[e];
        ss = group_sum<LANES>(ss);
        const float rms = 1.0f / sqrtf(ss / (float)kD + p.r.eps);
        Eight<DT> wr;
        float wv[8];
        wr.load(w, 8 * sub);
        wr.get(wv);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          x[e] *= rms * wv[e];
          if (p.r.per_op) x[e] = rounded<DT>(x[e]);
        }
      }
      float y[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = p.r.interleave ? x[e ^ 1] : __shfl(x[e], partner);
      if (rotates) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const bool first = p.r.interleave ? (e & 1) == 0 : lower;
          const float a = x[e], b = y[e];
          if (p.r.per_op) {
            const float ac = rounded<DT>(a * c[e]), bs = rounded<DT>(b * sn[e]);
            x[e] = rounded<DT>(first ? ac - bs : ac + bs);
          } else {
            x[e] = first ? a * c[e] - b * sn[e] : b * sn[e] + a * c[e];
          }
        }
      }
      in[u].set(x);
      if (live) in[u].store(p.r.qkv, base + (int64_t)hh * kD);
      in[u].get(x);  // the cache receives what a reader of qkv would see
    }
    if (CACHE == kNoCache) continue;
    const int h = is_v ? hh - p.r.num_q_heads - p.r.num_k_heads : hh - p.r.num_q_heads;
    const int64_t row = block * p.r.stride_block + (int64_t)h * p.r.stride_head + off * p.r.stride_slot + 8 * sub;
    uint8_t* cache = is_v ? p.r.v_cache : p.r.k_cache;
    if (CACHE == kVerbatim) {
      if (!live || is_q || !writes) continue;
      if (p.cache_vec_ok) {
        in[u].store(cache, row);
      } else {
        in[u].store_elements(cache, row);
      }
      continue;
    }
    float amax = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) amax = fmaxf(amax, fabsf(x[e]));
    amax = group_max<LANES>(amax);
    if (!live || is_q || !writes) continue;
    constexpr float kQmax = CACHE == kInt8 ? 127.0f : 448.0f;
    constexpr float kMinScale = CACHE == kInt8 ? FLT_EPSILON : 1.0f / (448.0f * 512.0f);
    const float scale = fmaxf(amax / kQmax, kMinScale);
    uint32_t q2[2] = {0, 0};
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float yv = x[e] / scale;
      const uint32_t q = CACHE == kInt8 ? quantise_int8(yv) : quantise_fp8_e4m3(yv);
      q2[e >> 2] |= q << (8 * (e & 3));
    }
    if (p.cache_vec_ok) {
      *(u32x2*)(cache + row) = u32x2{q2[0], q2[1]};
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) cache[row + e] = (uint8_t)(q2[e >> 2] >> (8 * (e & 3)));
    }
    if (sub == 0) {
      float* sc = is_v ? p.r.v_scale : p.r.k_scale;
      sc[block * p.r.sc_stride_block + (int64_t)h * p.r.sc_stride_head + off * p.r.sc_stride_slot] = scale;
    }
  }
}

// Any head_dim up to 512, any rotary_dim: one wave per (token, head), elements lane, lane + 64, ... to a lane; the
// head's values pass through LDS so that an element finds its partner.
template <int DT, int CACHE>
__global__ void __launch_bounds__(256) mrope_kv_write_any_kernel(MropeParams p) {
  constexpr int kPer = 8;
  __shared__ float stage[4][512];
  const int lane = threadIdx.x & 63;
  const int wave = threadIdx.x >> 6;
  const int64_t unit = (int64_t)blockIdx.x * 4 + wave;
  const bool live = unit < p.r.num_tokens * p.heads;
  const int64_t t = live ? unit / p.heads : 0;
  const int hh = live ? (int)(unit - t * p.heads) : 0;
  const bool is_q = hh < p.r.num_q_heads;
  const bool is_v = hh >= p.r.num_q_heads + p.r.num_k_heads;
  const int D = p.r.head_dim, R = p.r.rotary_dim, half = R >> 1;
  const int64_t base = t * p.r.token_stride + (int64_t)hh * D;
  float x[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int d = lane + 64 * i;
    x[i] = live && d < D ? Elem<DT>::load(p.r.qkv, base + d) : 0.0f;
  }
  const void* w = is_q ? p.r.q_weight : p.r.k_weight;
  if (!is_v && w != nullptr) {
    float ss = 0.0f;
#pragma unroll
    for (int i = 0; i < kPer; ++i) ss += x[i] * x[i];
    ss = wave_sum(ss);
    const float rms = 1.0f / sqrtf(ss / (float)D + p.r.eps);
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int d = lane + 64 * i;
      if (d < D) {
        x[i] *= rms * Elem<DT>::load(w, d);
        if (p.r.per_op) x[i] = rounded<DT>(x[i]);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < kPer; ++i) stage[wave][lane + 64 * i] = x[i];
  __syncthreads();
  if (!live) return;
  if (!is_v) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int d = lane + 64 * i;
      if (d < R) {
        const bool first = p.r.interleave ? (d & 1) == 0 : d < half;
        const int j = p.r.interleave ? d >> 1 : (first ? d : d - half);
        const int partner = p.r.interleave ? d ^ 1 : (first ? d + half : d - half);
        const float c = table_value<DT>(p, t, j), s = table_value<DT>(p, t, half + j);
        const float a = x[i], b = stage[wave][partner];
        if (p.r.per_op) {
          const float ac = rounded<DT>(a * c), bs = rounded<DT>(b * s);
          x[i] = rounded<DT>(first ? ac - bs : ac + bs);
        } else {
          x[i] = first ? a * c - b * s : b * s + a * c;
        }
      }
    }
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int d = lane + 64 * i;
      if (d < D) {
        Elem<DT>::store(p.r.qkv, base + d, x[i]);
        x[i] = rounded<DT>(x[i]);
      }
    }
  }
  if (CACHE == kNoCache || is_q) return;
  const int64_t slot = p.r.slots[t];
  if (slot < 0 || slot >= p.r.num_slots) return;
  const int64_t block = slot / p.r.block_size;
  const int64_t off = slot - block * p.r.block_size;
  const int h = is_v ? hh - p.r.num_q_heads - p.r.num_k_heads : hh - p.r.num_q_heads;
  const int64_t row = block * p.r.stride_block + (int64_t)h * p.r.stride_head + off * p.r.stride_slot;
  uint8_t* cache = is_v ? p.r.v_cache : p.r.k_cache;
  if (CACHE == kVerbatim) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int d = lane + 64 * i;
      if (d < D) {
        if (is_v) {  // value rows are copied bit for bit
          ((typename Elem<DT>::T*)cache)[row + d] = ((const typename Elem<DT>::T*)p.r.qkv)[base + d];
        } else {
          Elem<DT>::store(cache, row + d, x[i]);
        }
      }
    }
    return;
  }
  float amax = 0.0f;
#pragma unroll
  for (int i = 0; i < kPer; ++i) amax = fmaxf(amax, fabsf(x[i]));
  amax = wave_max(amax);
  constexpr float kQmax = CACHE == kInt8 ? 127.0f : 448.0f;
  constexpr float kMinScale = CACHE == kInt8 ? FLT_EPSILON : 1.0f / (448.0f * 512.0f);
  const float scale = fmaxf(amax / kQmax, kMinScale);
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int d = lane + 64 * i;
    if (d < D) {
      const float y = x[i] / scale;
      cache[row + d] = CACHE == kInt8 ? quantise_int8(y) : quantise_fp8_e4m3(y);
    }
  }
  if (lane == 0) {
    float* sc = is_v ? p.r.v_scale : p.r.k_scale;
    sc[block * p.r.sc_stride_block + (int64_t)h * p.r.sc_stride_head + off * p.r.sc_stride_slot] = scale;
  }
}

template <int DT, int LANES, int CACHE>
static void launch_mrope(const MropeParams& p, hipStream_t st) {
  constexpr int kHeads = 256 / LANES;
  // Few tokens: a workgroup per 256 / LANES heads, for the launch's latency; from about two rounds of the CUs on the
  // table row is mixed once for four times as many.
  const int64_t parts = (p.heads + kHeads - 1) / kHeads;
  if (p.r.num_tokens * parts <= 2048) {
    mrope_kv_write_kernel<DT, LANES, CACHE, 1><<<dim3((unsigned)p.r.num_tokens, (unsigned)parts), 256, 0, st>>>(p);
  } else {
    mrope_kv_write_kernel<DT, LANES, CACHE, 4>
        <<<dim3((unsigned)p.r.num_tokens, (unsigned)((p.heads + 4 * kHeads - 1) / (4 * kHeads))), 256, 0, st>>>(p);
  }
}

template <int DT, int CACHE>
static void launch_mrope_dim(const MropeParams& p, bool vec, hipStream_t st) {
  if (vec && p.r.head_dim == 64) return launch_mrope<DT, 8, CACHE>(p, st);
  if (vec && p.r.head_dim == 128) return launch_mrope<DT, 16, CACHE>(p, st);
  if (vec && p.r.head_dim == 256) return launch_mrope<DT, 32, CACHE>(p, st);
  mrope_kv_write_any_kernel<DT, CACHE><<<(unsigned)((p.r.num_tokens * p.heads + 3) / 4), 256, 0, st>>>(p);
}

template <int DT>
static void launch_mrope_kind(int kind, const MropeParams& p, bool vec, hipStream_t st) {
  switch (kind) {
    case kNoCache:
      return launch_mrope_dim<DT, kNoCache>(p, vec, st);
    case kVerbatim:
      return launch_mrope_dim<DT, kVerbatim>(p, vec, st);
    case kInt8:
      return launch_mrope_dim<DT, kInt8>(p, vec, st);
    default:
      return launch_mrope_dim<DT, kFp8>(p, vec, st);
  }
}

}  // namespace xllm_hip

using namespace xllm_hip;

extern "C" int xllm_hip_mrope_kv_write(const xllm_hip_rope_args* a,
                                       const xllm_hip_mrope* axes,
                                       const xllm_hip_kv_cache* cache,
                                       const int32_t* slot_mapping,
                                       xllm_hip_stream_t stream) {
  XLLM_HIP_REQUIRE(a != nullptr && axes != nullptr, "rope args or axes are NULL");
  XLLM_HIP_REQUIRE(a->num_tokens >= 0, "num_tokens is negative");
  XLLM_HIP_REQUIRE(axes->num_axes >= 1 && axes->num_axes <= 4, "num_axes must be 1 to 4, got %d", axes->num_axes);
  int64_t pairs = 0;
  for (int i = 0; i < axes->num_axes; ++i) {
    XLLM_HIP_REQUIRE(axes->sections[i] >= 0, "section %d is negative", i);
    pairs += axes->sections[i];
  }
  XLLM_HIP_REQUIRE(pairs * 2 == a->rotary_dim, "the sections hold %lld pairs, rotary_dim / 2 is %d", (long long)pairs,
                   a->rotary_dim / 2);
  if (a->num_tokens == 0) return XLLM_HIP_OK;
  XLLM_HIP_REQUIRE(axes->num_axes == 1 || axes->axis_stride >= a->num_tokens, "axis_stride smaller than num_tokens");
  MropeParams p{};
  int kind;
  const int rc = fill_rope_params(a, cache, slot_mapping, p.r, kind);
  if (rc != XLLM_HIP_OK) return rc;
  p.axis_stride = axes->axis_stride;
  p.num_axes = axes->num_axes;
  p.dealt = axes->dealt != 0;
  for (int i = 0; i < 4; ++i) p.sections[i] = i < axes->num_axes ? axes->sections[i] : 0;
  p.heads = a->num_q_heads + a->num_k_heads + (cache != nullptr ? a->num_v_heads : 0);
  if (p.heads == 0) return XLLM_HIP_OK;
  XLLM_HIP_REQUIRE((a->num_tokens * p.heads + 3) / 4 <= 0x7fffffff, "too many (token, head) pairs");
  // The vector kernel: whole lanes of eight rotated elements, rows on 16-byte boundaries.  It never depends on the
  // cache, so a call with and one without a cache compute the same q and k.
  const int eb = elem_bytes(a->dtype);
  const bool vec = (((uintptr_t)a->qkv | (uintptr_t)a->q_weight | (uintptr_t)a->k_weight | (uintptr_t)(a->token_stride * eb)) & 15) == 0 &&
                   a->rotary_dim % (a->interleave ? 8 : 16) == 0;
  if (cache != nullptr) {
    const int ceb = elem_bytes(cache->dtype);
    const int need = ceb == 1 ? 8 : 16;  // bytes a lane stores at once
    p.cache_vec_ok = (((uintptr_t)cache->k_cache | (uintptr_t)cache->v_cache | (uintptr_t)(cache->stride_block * ceb) |
                       (uintptr_t)(cache->stride_head * ceb) | (uintptr_t)(cache->stride_slot * ceb)) &
                      (uintptr_t)(need - 1)) == 0;
  }
  hipStream_t st = (hipStream_t)stream;
  if (a->dtype == XLLM_HIP_BF16) {
    launch_mrope_kind<XLLM_HIP_BF16>(kind, p, vec, st);
  } else if (a->dtype == XLLM_HIP_FP16) {
    launch_mrope_kind<XLLM_HIP_FP16>(kind, p, vec, st);
  } else {
    launch_mrope_kind<XLLM_HIP_FP32>(kind, p, vec, st);
  }
  return check_launch("mrope_kv_write_kernel");
}
