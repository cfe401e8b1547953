// What the rotary-embedding kernels share: their arguments, element conversions, reductions over the lanes of a head,
// and the host-side checks that fill the arguments in.
#pragma once

#include "device_utils.h"
#include "host_utils.h"

namespace xllm_hip {

struct RopeParams {
  uint8_t* qkv;  // [tokens, (Hq + Hk + Hv) * D], q and k heads rewritten in place
  const void* q_weight;
  const void* k_weight;
  const void* cos_sin;  // [max_position, rotary_dim]: cos of the rotary_dim/2 frequencies, then sin
  const void* positions;
  int32_t positions_int32;  // nonzero: positions holds int32 entries, else int64
  const int32_t* slots;  // NULL: no cache write
  uint8_t* k_cache;
  uint8_t* v_cache;
  float* k_scale;
  float* v_scale;
  int64_t token_stride;  // elements
  int64_t stride_block;  // cache strides, elements
  int64_t stride_head;
  int64_t stride_slot;
  int64_t sc_stride_block;
  int64_t sc_stride_head;
  int64_t sc_stride_slot;
  int64_t num_tokens;
  int64_t num_slots;
  int64_t max_position;
  int32_t num_q_heads;
  int32_t num_k_heads;
  int32_t num_v_heads;
  int32_t head_dim;
  int32_t rotary_dim;
  int32_t block_size;
  int32_t cos_sin_dtype;
  int32_t interleave;   // pairs (2j, 2j+1) instead of (j, j + rotary_dim/2)
  int32_t per_op;       // round after every multiply and add, as arithmetic on scalar_t operands does
  float eps;
};

__device__ inline float load_any(const void* p, int64_t i, int dtype) {
  switch (dtype) {
    case XLLM_HIP_BF16:
      return Elem<XLLM_HIP_BF16>::load(p, i);
    case XLLM_HIP_FP16:
      return Elem<XLLM_HIP_FP16>::load(p, i);
    default:
      return Elem<XLLM_HIP_FP32>::load(p, i);
  }
}

// x as the element type DT holds it.
template <int DT>
__device__ inline float rounded(float x) {
  if (DT == XLLM_HIP_BF16) return bf16_bits_to_float(float_to_bf16_bits(x));
  if (DT == XLLM_HIP_FP16) return (float)(_Float16)x;
  return x;
}

enum { kNoCache = 0, kVerbatim = 1, kInt8 = 2, kFp8 = 3 };

template <int G>
__device__ inline float group_sum(float v) {  // over G consecutive lanes (G a power of two)
#pragma unroll
  for (int o = G / 2; o >= 1; o >>= 1) v += __shfl_xor(v, o);
  return v;
}
template <int G>
__device__ inline float group_max(float v) {
#pragma unroll
  for (int o = G / 2; o >= 1; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
  return v;
}

template <int DT>
__device__ inline void unpack8(const u32x4 raw, float (&x)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const uint32_t w = raw[e >> 1];
    if (DT == XLLM_HIP_BF16) {
      x[e] = __uint_as_float((e & 1) ? (w & 0xffff0000u) : (w << 16));
    } else {
      x[e] = (float)__builtin_bit_cast(_Float16, (uint16_t)((e & 1) ? (w >> 16) : (w & 0xffffu)));
    }
  }
}
template <int DT>
__device__ inline u32x4 pack8(const float (&x)[8]) {
  u32x4 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t lo, hi;
    if (DT == XLLM_HIP_BF16) {
      lo = float_to_bf16_bits(x[2 * i]);
      hi = float_to_bf16_bits(x[2 * i + 1]);
    } else {
      lo = __builtin_bit_cast(uint16_t, (_Float16)x[2 * i]);
      hi = __builtin_bit_cast(uint16_t, (_Float16)x[2 * i + 1]);
    }
    r[i] = lo | (hi << 16);
  }
  return r;
}

// Checks a rope call (num_tokens > 0) and fills in what every kernel needs; `kind`: how the cache is written.
static int fill_rope_params(const xllm_hip_rope_args* a, const xllm_hip_kv_cache* cache, const int32_t* slot_mapping,
                            RopeParams& p, int& kind) {
  XLLM_HIP_REQUIRE(a->qkv != nullptr && a->cos_sin_cache != nullptr && a->positions != nullptr,
                   "qkv, cos_sin_cache or positions is NULL");
  XLLM_HIP_REQUIRE(a->dtype == XLLM_HIP_BF16 || a->dtype == XLLM_HIP_FP16 || a->dtype == XLLM_HIP_FP32,
                   "qkv must be BF16/FP16/FP32, got dtype %d", a->dtype);
  XLLM_HIP_REQUIRE(a->cos_sin_dtype == XLLM_HIP_BF16 || a->cos_sin_dtype == XLLM_HIP_FP16 ||
                       a->cos_sin_dtype == XLLM_HIP_FP32,
                   "cos_sin_cache must be BF16/FP16/FP32, got dtype %d", a->cos_sin_dtype);
  XLLM_HIP_REQUIRE(a->num_q_heads >= 0 && a->num_k_heads >= 0 && a->num_v_heads >= 0 &&
                       a->num_q_heads + a->num_k_heads + a->num_v_heads > 0,
                   "head counts must be non-negative and not all zero");
  XLLM_HIP_REQUIRE(a->head_dim > 0 && a->head_dim <= 512, "head_dim must be in 1..512, got %d", a->head_dim);
  XLLM_HIP_REQUIRE(a->rotary_dim >= 0 && a->rotary_dim <= a->head_dim && a->rotary_dim % 2 == 0,
                   "rotary_dim must be even and at most head_dim, got %d", a->rotary_dim);
  XLLM_HIP_REQUIRE(a->max_position > 0, "max_position must be positive");
  XLLM_HIP_REQUIRE((a->q_weight == nullptr) == (a->k_weight == nullptr), "q_weight and k_weight go together");
  const int64_t row = (int64_t)(a->num_q_heads + a->num_k_heads + a->num_v_heads) * a->head_dim;
  XLLM_HIP_REQUIRE(a->token_stride >= row, "token stride smaller than the heads it holds");

  p = RopeParams{};
  p.qkv = (uint8_t*)a->qkv;
  p.q_weight = a->q_weight;
  p.k_weight = a->k_weight;
  p.cos_sin = a->cos_sin_cache;
  p.positions = a->positions;
  p.positions_int32 = a->positions_int32;
  p.token_stride = a->token_stride;
  p.num_tokens = a->num_tokens;
  p.max_position = a->max_position;
  p.num_q_heads = a->num_q_heads;
  p.num_k_heads = a->num_k_heads;
  p.num_v_heads = a->num_v_heads;
  p.head_dim = a->head_dim;
  p.rotary_dim = a->rotary_dim;
  p.cos_sin_dtype = a->cos_sin_dtype;
  p.interleave = a->interleave;
  p.per_op = a->round_each_op;
  p.eps = a->eps;

  kind = kNoCache;
  if (cache != nullptr) {
    XLLM_HIP_REQUIRE(slot_mapping != nullptr, "a cache is given but slot_mapping is NULL");
    XLLM_HIP_REQUIRE(cache->k_cache != nullptr && cache->v_cache != nullptr, "k_cache or v_cache is NULL");
    XLLM_HIP_REQUIRE(cache->num_blocks > 0 && cache->block_size > 0, "cache sizes must be positive");
    XLLM_HIP_REQUIRE(cache->head_dim == a->head_dim && cache->num_kv_heads == a->num_k_heads &&
                         a->num_v_heads == a->num_k_heads,
                     "cache is [%d heads, dim %d], qkv holds %d k / %d v heads of dim %d", cache->num_kv_heads,
                     cache->head_dim, a->num_k_heads, a->num_v_heads, a->head_dim);
    XLLM_HIP_REQUIRE(cache->stride_block > 0 && cache->stride_head > 0 && cache->stride_slot > 0,
                     "cache strides must be positive");
    if (cache->dtype == XLLM_HIP_INT8 || cache->dtype == XLLM_HIP_FP8_E4M3) {
      XLLM_HIP_REQUIRE(cache->k_scale != nullptr && cache->v_scale != nullptr,
                       "a quantised cache needs k_scale and v_scale");
      kind = cache->dtype == XLLM_HIP_INT8 ? kInt8 : kFp8;
    } else {
      XLLM_HIP_REQUIRE(cache->dtype == a->dtype, "cache dtype %d differs from qkv dtype %d", cache->dtype, a->dtype);
      kind = kVerbatim;
    }
    p.slots = slot_mapping;
    p.k_cache = (uint8_t*)cache->k_cache;
    p.v_cache = (uint8_t*)cache->v_cache;
    p.k_scale = cache->k_scale;
    p.v_scale = cache->v_scale;
    p.stride_block = cache->stride_block;
    p.stride_head = cache->stride_head;
    p.stride_slot = cache->stride_slot;
    p.sc_stride_block = cache->scale_stride_block;
    p.sc_stride_head = cache->scale_stride_head;
    p.sc_stride_slot = cache->scale_stride_slot;
    p.num_slots = cache->num_blocks * cache->block_size;
    p.block_size = cache->block_size;
  }
  return XLLM_HIP_OK;
}

}  // namespace xllm_hip
