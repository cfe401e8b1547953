// Tree attention on the matrix cores: head_dim 64, 128 and 256, 16-bit queries, 16-bit and 8-bit caches.
//
// One workgroup of four waves per (sequence chunk, kv head, group of query rows); query row r = j * group + gq (token
// j, head gq of the kv head's group).  The products are taken transposed, 16 query rows to a matrix tile,
//   S^T[t][r]  = sum_d K[t][d] Q[r][d]        A = K from LDS,    B = Q^T in registers
//   O^T[d][r] += sum_t V[t][d] P[r][t]        A = V^T from LDS,  B = P^T, the softmax weights as S^T left them
// so that a query row stays in one lane column from the scores to the output, and its running maximum and sum are a
// lane's own numbers.  K and V go from memory straight into LDS (16 bytes a lane, no registers on the way), the tile
// after the one in use always in flight; an 8-bit cache stays bytes there — half the LDS traffic — and becomes 16-bit
// operands in the registers that feed the matrix instructions:
//   fp8   K to the queries' type, V to fp16, both exact
//   int8  x ^ 0x80 = x + 128.  V: behind 0x64 it is the fp16 number 1024 + 128 + x; minus 1152 it is x, exactly.  K: behind
//         0 it is the subnormal (x + 128) 2^-24, and the row takes back 128 times the sum of its query's elements with
//         the factor that its scores get anyway.  (Twice 128 is the most that this adds to a product, so the fp32 sums
//         lose about a bit.  V has no such end: there the 128 would pile up over the tokens.)
// Both operands of a matrix instruction have one type.  So with V in fp16 the weights of an fp16 or 8-bit cache are rounded to
// 11 bits — how fp16's range is kept from cutting into them stands at TreeRows::kFollow — and those over a bf16 cache to 8: a
// bf16 V has no exact fp16 form, and two bf16 numbers to a weight would double the second product.
//
// How the waves share an item: 128 rows to a workgroup are 32 to each wave, which then reads all of the tile, and 64 rows
// over a 16-bit cache 16.  Up to 32 rows are two tiles of 16: over a 16-bit cache two waves share a row tile, taking
// alternate 32-token pieces.  Over an 8-bit cache every wave has two row tiles, and two (64 rows) or all four (32 rows)
// share the pieces, because a piece is widened once per wave that takes it (64 x 8192 tokens: int8, 64 rows, 315 -> 258
// us; 32 rows 225 -> 187; fp8 268 -> 237 and 186 -> 176).  The second half of a narrow item's arithmetic is often unused
// (16 rows or fewer): a step this narrow is bound by memory.
//
// Measured, kernel and merge, bf16 queries, head_dim 128, block_size 16 unless stated:
//   16-bit cache, 8 or 16 drafts of 4 heads to a kv head, 64 x 4096 or 8192 tokens   165 / 335 us   6.5 TB/s: memory
//   512 rows to a kv head, 32 x 8192 tokens   bf16 652 us, 843 TFLOP/s; fp8 661 us, 831; int8 760 us, 723: the softmax's
//   and the widening's vector instructions, which the matrix instructions of one wave only partly cover for another
//
// Only the last tokens of a sequence are drafted ones, so only the last pieces are masked.  There a row takes from its
// mask the 32 bits of the piece; scores of unseen tokens are replaced by -inf whatever they were.  An unseen V may
// hold anything, and 0 * NaN in a matrix product would reach every row, so the V rows of a masked tile are looked
// through: rows past the length are zeroed, and where another holds a NaN or an infinity the piece is accumulated
// token by token under each row's own bits.
#pragma once

#include "decode_mfma.h"
#include "tree_params.h"

#include <float.h>

namespace xllm_hip {

// 16 bytes a lane from memory into LDS.  STREAM: lines that nobody reads again are not kept (64 x 4096 tokens of bf16, 8
// drafts: 184 -> 164 us); an item whose neighbour on the XCD reads the same K and V keeps them (32 x 8192, 512 query
// rows to a kv head: 654 us kept, 697 streamed).
template <bool STREAM>
__device__ __forceinline__ void tree_to_lds(const uint8_t* from, uint8_t* to) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)from, (__attribute__((address_space(3))) void*)to, 16, 0,
                                   STREAM ? 2 : 0);
}

constexpr bool tree_quant(int kv) { return kv == XLLM_HIP_FP8_E4M3 || kv == XLLM_HIP_INT8; }

template <int QT, int KV, int D>
struct TreeShape {
  static constexpr bool kQuant = tree_quant(KV);
  static constexpr bool kInt8 = KV == XLLM_HIP_INT8;
  static constexpr int kEB = kQuant ? 1 : 2;
  static constexpr int kRB = D * kEB;                  // bytes of a cache row
  static constexpr int kPPR = kRB / 16;                // 16-byte pieces of a row
  static constexpr int kRPI = 64 / kPPR;               // rows a load instruction of a wave covers
  static constexpr int kTT = kRB >= 256 ? 64 : 128;    // tokens per tile
  static constexpr int kRW = kTT / 4;                  // tokens of a tile that one wave fetches
  static constexpr int kLoads = kRW / kRPI;            // load instructions a wave needs for them (K; as many for V)
  static constexpr int kArray = kTT * kRB;             // bytes of a tile's K or V
  static constexpr int kFactors = 2 * kArray;          // three per-token factors of an 8-bit cache behind them
  static constexpr int kStage = 2 * kArray + (kQuant ? 3 * kTT * 4 : 0);
  static constexpr bool kQF16 = QT == XLLM_HIP_FP16;
  static constexpr bool kKF16 = kQF16 || kInt8;        // type of the first product: fp16, else bf16
  static constexpr bool kVF16 = kQF16 || kQuant;       // type of the second
  static constexpr bool kNormQ = kInt8 && !kQF16;      // bf16 queries that become fp16: see init
  static constexpr int kChunks = D / 32;
  static constexpr int kDT = D / 16;
};

// LDS placement: the 16-byte pieces of a row are permuted by an XOR that depends on the row, so that the lanes the LDS
// serves together (8 of a 16-byte access, 16 of an 8-byte one: 128 bytes) meet all 8 pieces (mod 8):
//   K: 8 consecutive rows, same piece;   V, 16-bit: 4 rows x 2 pieces;   V, 8-bit: rows r..r+3 and r+16.., same piece.
// A 64-byte row (head_dim 64, 8-bit) is half a line: there the row's parity is one of the three bits already.
template <int RB>
__device__ inline int tree_swz_k(int row) {
  return RB == 64 ? (row >> 1) & 3 : row & 7;
}
template <int RB, bool QUANT>
__device__ inline int tree_swz_v(int row) {
  if (!QUANT) return (row & 3) << 1;
  return RB == 64 ? ((row >> 1) & 1) | (((row >> 4) & 1) << 1) : (row & 3) | (((row >> 4) & 1) << 2);
}

// Eight bytes of an 8-bit cache as eight 16-bit numbers.
template <int KV, bool F16>
__device__ inline u32x4 tree_widen(uint32_t a, uint32_t b) {
  u32x4 o;
  const uint32_t in[2] = {a, b};
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    if constexpr (KV == XLLM_HIP_INT8) {
      static_assert(KV != XLLM_HIP_INT8 || F16, "int8 operands are fp16");
      const uint32_t t = in[w] ^ 0x80808080u;
      const f16x2 off = {(_Float16)1152.0f, (_Float16)1152.0f};
      const f16x2 lo = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, t, 0x04010400u)) - off;
      const f16x2 hi = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, t, 0x04030402u)) - off;
      o[2 * w] = __builtin_bit_cast(uint32_t, lo);
      o[2 * w + 1] = __builtin_bit_cast(uint32_t, hi);
    } else if constexpr (F16) {
      o[2 * w] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(in[w], 1.0f, false));
      o[2 * w + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(in[w], 1.0f, true));
    } else {
      o[2 * w] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)in[w], 1.0f, false));
      o[2 * w + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)in[w], 1.0f, true));
    }
  }
  return o;
}

// The same for the K operand of the scores; int8: (x + 128) 2^-24, see TreeRows::q_bias.
template <int KV, bool F16>
__device__ inline u32x4 tree_widen_k(uint32_t a, uint32_t b) {
  if constexpr (KV == XLLM_HIP_INT8) {
    const uint32_t ta = a ^ 0x80808080u, tb = b ^ 0x80808080u;
    return u32x4{__builtin_amdgcn_perm(0u, ta, 0x0c010c00u), __builtin_amdgcn_perm(0u, ta, 0x0c030c02u),
                 __builtin_amdgcn_perm(0u, tb, 0x0c010c00u), __builtin_amdgcn_perm(0u, tb, 0x0c030c02u)};
  } else {
    return tree_widen<KV, F16>(a, b);
  }
}

// Any non-finite value among the 16 bytes?
template <int KV>
__device__ inline bool tree_not_finite(u32x4 v) {
  uint32_t hit = 0;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    if constexpr (KV == XLLM_HIP_FP8_E4M3) {
      // a byte is a NaN if its low seven bits are all set: adding one to them carries into bit 7
      hit |= ((v[w] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
    } else {
      const uint32_t e = KV == XLLM_HIP_BF16 ? 0x7f807f80u : 0x7c007c00u;
      const uint32_t one = KV == XLLM_HIP_BF16 ? 0x00800080u : 0x04000400u;
      hit |= ((v[w] & e) + one) & 0x80008000u;  // an exponent of all ones carries into the sign's place
    }
  }
  return hit != 0;
}

// One wave's share of the loads: where its rows lie, and the loads of a tile.
template <class SH, int KV>
struct TreeLoader {
  // Byte offset of this lane's piece from the first row of a load instruction.  The rows of further instructions differ
  // in the swizzle by few bits, so few of these are distinct: K's in the row's low three bits (kVarK instructions in
  // turn), V's in the low two, or over an 8-bit cache in the group of 16.
  static constexpr int kGroups = SH::kRW > 16 ? SH::kRW / 16 : 1;
  static constexpr int kPer = SH::kLoads / kGroups;  // load instructions per group of 16 tokens
  static constexpr int kVarK = SH::kRPI >= 8 ? 1 : 8 / SH::kRPI;
  static constexpr int kVarV = SH::kQuant ? kGroups : SH::kRPI >= 4 ? 1 : 4 / SH::kRPI;
  uint32_t off_k[kVarK], off_v[kVarV];
  int wave, lane;
  uint32_t sc_off;

  __device__ inline void init(const TreeParams& p, int w, int l) {
    wave = w;
    lane = l;
    const int pos = l % SH::kPPR, lr = l / SH::kPPR;
    const uint32_t at = (uint32_t)(lr * p.stride_slot) * SH::kEB;
#pragma unroll
    for (int v = 0; v < kVarK; ++v) off_k[v] = at + ((pos ^ tree_swz_k<SH::kRB>(w * SH::kRW + v * SH::kRPI + lr)) << 4);
#pragma unroll
    for (int v = 0; v < kVarV; ++v) {
      off_v[v] = at + ((pos ^ tree_swz_v<SH::kRB, SH::kQuant>(w * SH::kRW + v * (SH::kQuant ? 16 : SH::kRPI) + lr)) << 4);
    }
    sc_off = 0;
    if (SH::kQuant) sc_off = (uint32_t)((l & (SH::kRW < 16 ? SH::kRW - 1 : 15)) * p.sc_stride_slot) * 4;
  }

  // The block that holds the wave's group g (16 tokens) of the tile at tb, by a scalar load; past the sequence's list
  // its last block.
  __device__ static inline int block(const TreeParams& p, const TreeItem& it, int tok) {
    int bi = tok >> p.log2_bs;
    bi = bi < it.nblk ? bi : it.nblk - 1;
    return tree_block(p, ((const __attribute__((address_space(4))) int32_t*)it.ids)[bi]);
  }

  // The wave's loads of the tile at tb, in flight on return.  Past the sequence's end they read its last block.  `sc`:
  // lanes 0..31 the K scales of the wave's tokens, 32..63 the V scales.
  template <bool STREAM>
  __device__ inline void issue(const TreeParams& p, const TreeItem& it, int tb, uint8_t* stage, float& sc) const {
    const int first = tb + wave * SH::kRW;
    uint8_t* kl = stage + wave * (SH::kRW * SH::kRB);
    uint8_t* vl = kl + SH::kArray;
    int64_t sbase[kGroups];
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      const int tok = first + 16 * g;
      const int blk = block(p, it, tok);
      const uint32_t slot = (uint32_t)(tok & (p.block_size - 1));
      const int64_t elem = (int64_t)((uint64_t)(uint32_t)blk * (uint32_t)p.stride_block) + (int64_t)it.hk * p.stride_head +
                           (int64_t)(slot * (uint32_t)p.stride_slot);
      if (SH::kQuant) {
        sbase[g] = (int64_t)((uint64_t)(uint32_t)blk * (uint32_t)p.sc_stride_block) + (int64_t)it.hk * p.sc_stride_head +
                   (int64_t)(slot * (uint32_t)p.sc_stride_slot);
      }
      const uint8_t* kb = p.k_cache + elem * SH::kEB;
      const uint8_t* vb = p.v_cache + elem * SH::kEB;
      const int64_t next = (int64_t)SH::kRPI * p.stride_slot * SH::kEB;  // from one instruction's rows to the next's
#pragma unroll
      for (int q = 0; q < kPer; ++q) tree_to_lds<STREAM>(kb + q * next + off_k[q % kVarK], kl + (g * kPer + q) * 1024);
#pragma unroll
      for (int q = 0; q < kPer; ++q) {
        tree_to_lds<STREAM>(vb + q * next + off_v[SH::kQuant ? g : q % kVarV], vl + (g * kPer + q) * 1024);
      }
    }
    if constexpr (SH::kQuant) {
      // lane = (array, token among the wave's, several times where there are fewer than 32)
      const int64_t sb = kGroups > 1 && (lane & 16) != 0 ? sbase[kGroups - 1] : sbase[0];
      const float* arr = (lane & 32) != 0 ? p.v_scale : p.k_scale;
      sc = *(const float*)((const uint8_t*)(arr + sb) + sc_off);
    }
  }

  // The per-token factors of the tile whose scales have arrived:
  //   kscl = k_scale * sm_scale * log2 e       x = s * kscl + lv
  //   lv   = log2 v_scale                      weight 2^(x - max x): the V scale rides in the exponent, so the 16-bit
  //   rvs  = 1 / v_scale                       weights use their whole range; a weight's share of the sum is w * rvs
  // A V scale of 0 counts as 2^-100: its tokens keep their share of the sum and add nothing.
  __device__ inline void factors(const TreeParams& p, uint8_t* stage, float sc) const {
    if constexpr (SH::kQuant) {
      float* f = (float*)(stage + SH::kFactors);
      const int i = lane & 31;
      if (i < SH::kRW) {
        const int t = wave * SH::kRW + i;
        if (lane < 32) {
          f[t] = sc * p.scale_log2;
        } else {
          const float vs = sc < 0x1p-100f ? 0x1p-100f : sc;  // (a NaN stays one)
          f[SH::kTT + t] = __builtin_amdgcn_logf(vs);
          f[2 * SH::kTT + t] = __builtin_amdgcn_rcpf(vs);
        }
      }
    }
  }

  // The wave's V rows of a masked tile, landed: zeros over the rows past the length; whether a drafted token's holds
  // something that is not finite.
  __device__ inline bool look_through(int tb, int prefix, int len, uint8_t* stage) const {
    bool bad = false;
    if constexpr (KV != XLLM_HIP_INT8) {
#pragma unroll
      for (int q = 0; q < SH::kLoads; ++q) {
        const int tok = tb + wave * SH::kRW + q * SH::kRPI + lane / SH::kPPR;
        u32x4* at = (u32x4*)(stage + SH::kArray + wave * (SH::kRW * SH::kRB) + q * 1024 + lane * 16);
        if (tok >= len) {
          *at = u32x4{0, 0, 0, 0};
        } else if (tok >= prefix) {
          bad = bad || tree_not_finite<KV>(*at);
        }
      }
    }
    return __builtin_amdgcn_ballot_w64(bad) != 0;
  }
};

// The lane's query row among the item's, in the row tile that starts at first_row; -1: none.
__device__ inline int tree_row(const TreeParams& p, const TreeItem& it, int first_row, int lane) {
  const int row = first_row + (lane & 15);
  return row < it.n * p.group ? row : -1;
}

// The mask of the lane's row.  KEEP: its first word is held in registers (fetched while the last tiles are in flight);
// otherwise, and for the further words of trees of more than 64 nodes, words are fetched by the pieces that need them.
template <bool KEEP>
struct TreeRowMask {
  uint64_t word0;

  __device__ static inline uint64_t word(const TreeParams& p, const TreeItem& it, int first_row, int lane, int w) {
    const int row = tree_row(p, it, first_row, lane);
    if (row < 0 || w >= p.mask_words) return 0;
    return p.mask[(it.q0 + row / p.group) * p.mask_stride + w];
  }
  __device__ inline void init(const TreeParams& p, const TreeItem& it, int first_row, int lane) {
    if (KEEP) word0 = word(p, it, first_row, lane, 0);
  }
  // Bits of the 32 tokens from t0 on that the row sees.
  __device__ inline uint32_t bits(const TreeParams& p, const TreeItem& it, int first_row, int lane, int t0) const {
    uint32_t b;
    const int u = t0 - it.prefix;
    if (u <= -32) {
      b = ~0u;
    } else if (u < 0) {  // the context's last tokens, then the first drafted ones
      b = (uint32_t)((KEEP ? word0 : word(p, it, first_row, lane, 0)) << -u) | ((1u << -u) - 1u);
    } else {
      const int w = u >> 6, s = u & 63;
      uint64_t v = (KEEP && w == 0 ? word0 : word(p, it, first_row, lane, w)) >> s;
      if (s > 32) v |= word(p, it, first_row, lane, w + 1) << (64 - s);
      b = (uint32_t)v;
    }
    const int left = it.len - t0;
    if (left < 32) b &= left > 0 ? (1u << left) - 1u : 0u;
    return b;
  }
};

// 16 query rows of one wave.
template <class SH, int KV>
struct TreeRows {
  typedef typename MmaOps<SH::kKF16>::Op OpK;
  typedef typename MmaOps<SH::kVF16>::Op OpV;
  OpK qf[SH::kChunks];
  f32x4 acc[SH::kDT];
  float m_run, l_run;
  float q_scale, q_bias;  // int8: the row's scores are s * q_scale + q_bias
  __device__ inline void init(const TreeParams& p, const TreeItem& it, int first_row, int lane) {
    const int kg = lane >> 4;
    const int row = tree_row(p, it, first_row, lane);
    const int r = row < 0 ? 0 : row;
    const int j = r / p.group;
    const int64_t token = it.q0 + j;
    const uint16_t* q = (const uint16_t*)p.q + token * p.q_token_stride + (int64_t)(it.hk * p.group + (r - j * p.group)) * (SH::kDT * 16);
    q_scale = 1.0f;
    u32x4 raw[SH::kChunks];
#pragma unroll
    for (int c = 0; c < SH::kChunks; ++c) {
      // elements of chunk c this lane feeds: as the K bytes lie (an 8-bit K piece of 16 elements feeds two chunks)
      const int at = SH::kQuant ? 64 * (c >> 1) + 16 * kg + 8 * (c & 1) : 32 * c + 8 * kg;
      raw[c] = u32x4{0, 0, 0, 0};
      if (row >= 0) raw[c] = *(const u32x4*)(q + at);
    }
    if constexpr (SH::kNormQ) {
      // bf16 queries become fp16: the row is first brought to a largest magnitude in [2^14, 2^15) by a power of two,
      // exactly, so that neither end of fp16's range cuts into what bf16 holds (elements 2^28 below the largest lose
      // bits); the scores take the factor back.
      float top = 0.0f;
#pragma unroll
      for (int c = 0; c < SH::kChunks; ++c) {
#pragma unroll
        for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf((float)__builtin_bit_cast(bf16x8, raw[c])[e]));
      }
      top = kg_max(top);
      int e2 = (int)((__builtin_bit_cast(uint32_t, top) >> 23) & 0xffu) - 126 - 15;
      e2 = e2 < -100 ? -100 : (e2 > 100 ? 100 : e2);
      const float down = __builtin_amdgcn_ldexpf(1.0f, -e2);
      q_scale = __builtin_amdgcn_ldexpf(1.0f, e2);
#pragma unroll
      for (int c = 0; c < SH::kChunks; ++c) {
#pragma unroll
        for (int e = 0; e < 8; ++e) qf[c][e] = (_Float16)((float)__builtin_bit_cast(bf16x8, raw[c])[e] * down);
      }
    } else {
#pragma unroll
      for (int c = 0; c < SH::kChunks; ++c) qf[c] = __builtin_bit_cast(OpK, raw[c]);
    }
    if constexpr (SH::kInt8) {
      float sum = 0.0f;
#pragma unroll
      for (int c = 0; c < SH::kChunks; ++c) {
#pragma unroll
        for (int e = 0; e < 8; ++e) sum += (float)qf[c][e];
      }
      q_bias = -128.0f * kg_sum(sum) * q_scale;
      q_scale *= 0x1p24f;
    }
    m_run = SH::kQuant ? -FLT_MAX : -INFINITY;
    l_run = 0.0f;
#pragma unroll
    for (int dt = 0; dt < SH::kDT; ++dt) acc[dt] = f32x4{0, 0, 0, 0};
  }

  // Where the largest weight of a piece may lie (log 2).  Where V is fp16 so are the weights, and one far enough below the
  // reference point would be rounded to few bits, or to 0, while its share stays in the sum: a key that dominates a row but
  // has a tiny V would hide what the others add.
  //   fp16 cache    the reference point follows the pieces, down too (kFollow): a piece's largest weight stays within
  //                 2^kLow .. 2^kTop, so what fp16's end at 2^-25 costs is at most 2^-12 of that weight; of the row's
  //                 largest, which is at least 2^(kTop - 5), 2^-35.  (64 x 8192 tokens, 128 rows: 409 us before and after;
  //                 430 where scores scatter by 6 nats and the point moves often)
  //   8-bit cache   a weight holds its token's V scale, so it says what the token can add; the largest is between 2^kHead
  //                 and 2^(kHead + kLazyRescale), a smaller one costs 2^-29 of it at most.  (Following the pieces took 4 to 6 %
  //                 from the forms that vector instructions bound.)
  //   bf16 cache    bf16 weights have a float's range.
  static constexpr bool kFollow = SH::kVF16 && !SH::kQuant;
  static constexpr float kTop = 15.0f, kLow = -13.0f, kMost = 60.0f;
  static constexpr float kHead = SH::kQuant ? 4.0f : 0.0f;

  // The scale rides in the FMA that forms the exponent where nothing else needs the scaled score.
  template <bool MASKED>
  static constexpr bool kFold = !SH::kQuant && !MASKED;

  // Scores of 32 tokens (s[h][rr]: token 16h + 4kg + rr), scaled and masked, in x (index 4h + rr).
  template <bool MASKED>
  __device__ __forceinline__ void scaled(const f32x4 (&s)[2], const f32x4 (&kscl)[2], const f32x4 (&lv)[2], float scale_log2, uint32_t vis,
                                         int kg, float (&x)[8]) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float v = s[i >> 2][i & 3];
      if constexpr (SH::kInt8) v = __builtin_fmaf(v, q_scale, q_bias);
      if constexpr (SH::kQuant) {
        v = __builtin_fmaf(v, kscl[i >> 2][i & 3], lv[i >> 2][i & 3]);
      } else if constexpr (!kFold<MASKED>) {
        v *= scale_log2;
      }
      if (MASKED) v = (vis >> (16 * (i >> 2) + 4 * kg + (i & 3))) & 1 ? v : -INFINITY;
      x[i] = v;
    }
  }

  // Scores to weights, in place; returns whether the reference point of some row moved.
  template <bool MASKED>
  __device__ __forceinline__ bool weights(float (&x)[8], const f32x4 (&rvs)[2], float scale_log2, uint32_t vis, int kg, float& alpha) {
    const float neg_inf = -INFINITY;
    float mt = neg_inf;
#pragma unroll
    for (int i = 0; i < 8; ++i) mt = fmaxf(mt, x[i]);
    mt = kg_max(mt);
    if (kFold<MASKED>) mt *= scale_log2;
    // The reference point of the exponents follows the scores lazily, so that the accumulators are seldom rescaled.  (It
    // begins at -FLT_MAX over an 8-bit cache, where a guard against -inf - -inf would cost two instructions a piece.)
    float m_new, m_safe;
    bool moved;
    if constexpr (kFollow) {
      const float d = mt - m_run;
      moved = __builtin_amdgcn_ballot_w64(!(fabsf(d - (kTop + kLow) * 0.5f) <= (kTop - kLow) * 0.5f)) != 0;
      m_new = m_run;
      if (moved) {
        // (not so far down that what has been summed up could pass 2^kMost; of a row that has seen a token l_run is above 1)
        const float low = m_run + (__builtin_amdgcn_logf(kg_max(l_run)) - kMost);
        if (d > kTop) m_new = mt - kTop + 5.0f;
        if (d < kLow && mt > neg_inf) m_new = fmaxf(mt - kLow - 5.0f, fminf(m_run, low));
      }
      m_safe = m_new == neg_inf ? 0.0f : m_new;
      alpha = __builtin_amdgcn_exp2f(m_run - m_safe);
    } else {
      // It moves when a row's maximum has grown by more than kLazyRescale (in log 2).
      const float m_top = fmaxf(m_run, mt);
      moved = __builtin_amdgcn_ballot_w64(m_top > m_run + kLazyRescale) != 0;
      m_new = moved ? m_top : m_run;
      if constexpr (SH::kQuant) {
        m_safe = m_new - kHead;
        alpha = __builtin_amdgcn_exp2f(m_run - m_new);
      } else {
        m_safe = m_new == neg_inf ? 0.0f : m_new;
        alpha = __builtin_amdgcn_exp2f(m_run - m_safe);
      }
    }
    l_run *= alpha;
    m_run = m_new;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float e = __builtin_amdgcn_exp2f(kFold<MASKED> ? __builtin_fmaf(x[i], scale_log2, -m_safe) : x[i] - m_safe);
      x[i] = e;
      if constexpr (SH::kQuant) {
        const float share = e * rvs[i >> 2][i & 3];
        // (an unseen token's scale may be anything: 0 * NaN must not reach the sum)
        l_run += MASKED ? ((vis >> (16 * (i >> 2) + 4 * kg + (i & 3))) & 1 ? share : 0.0f) : share;
      } else {
        l_run += e;
      }
    }
    return moved;
  }

  __device__ static inline OpV pack(const float (&w)[8]) {
    typedef MmaOps<SH::kVF16> M;
    return __builtin_bit_cast(OpV, u32x4{M::pack(w[0], w[1]), M::pack(w[2], w[3]), M::pack(w[4], w[5]), M::pack(w[6], w[7])});
  }
};

// Where the lane's row goes: the output, or (cut sequences) a normalised partial and its base-2 log-sum-exp.
struct TreeOut {
  float* partial;
  uint16_t* out;
  float inv;

  // `l`, `m`: the row's sum and reference point.  False: the lane has no row.
  __device__ inline bool init(const TreeParams& p, const TreeItem& it, int first_row, int lane, float l, float m, bool writes_lse) {
    const int row = tree_row(p, it, first_row, lane);
    if (row < 0) return false;
    inv = l == 0.0f ? 0.0f : 1.0f / l;  // (a NaN stays one)
    const float lse2 = l == 0.0f ? -INFINITY : m + __builtin_amdgcn_logf(l);
    const int j = row / p.group;
    const int head = it.hk * p.group + (row - j * p.group);
    partial = nullptr;
    if (it.chunks == 1) {
      const int64_t token = it.q0 + j;
      if (writes_lse && p.lse != nullptr) p.lse[token * p.num_q_heads + head] = lse2;
      out = (uint16_t*)p.out + token * p.out_token_stride + (int64_t)head * p.head_dim;
    } else {
      const int64_t prow = ((int64_t)it.b * p.slots + it.chunk) * ((int64_t)p.n * p.num_q_heads) + (int64_t)j * p.num_q_heads + head;
      if (writes_lse) p.partial_lse[prow] = lse2;
      partial = p.partial_out + prow * p.head_dim;
    }
    return true;
  }
  template <bool F16>
  __device__ inline void store(int d, f32x4 o) const {
    o *= inv;
    if (partial != nullptr) {
      *(f32x4*)(partial + d) = o;
    } else {
      typedef MmaOps<F16> M;
      *(u32x2*)(out + d) = u32x2{M::pack(o[0], o[1]), M::pack(o[2], o[3])};
    }
  }
};

// RTW: row tiles per wave; TS: waves that share the tokens of a set of row tiles, a 32-token piece each in turn; STREAM:
// see tree_to_lds (one row group; a template argument, because a branch in the loop costs the compiler its schedule: 24
// fp8 sequences, 61 drafts, 379 against 353 us); LINE: the item is one of several of its workgroup.
template <int QT, int KV, int D, int RTW, int TS, bool STREAM, bool LINE>
__device__ __forceinline__ void tree_mfma_item(const TreeParams& p, const TreeItem& it, int wave) {
  typedef TreeShape<QT, KV, D> SH;
  static_assert(TS == 1 || (TS == 2 && RTW == 1) || RTW == 2, "how the end of the item joins the waves' sums");
  constexpr int kApart = 4 / TS;  // sets of row tiles: wave w has set w % kApart, and share w / kApart of its tokens
  constexpr int kRowsPerItem = 16 * RTW * 4 / TS;
  constexpr int kSums = RTW * SH::kDT * 1024;  // bytes of a wave's accumulators
  __shared__ __attribute__((aligned(16))) uint8_t stage0[SH::kStage];
  __shared__ __attribute__((aligned(16))) uint8_t stage1[SH::kStage];
  __shared__ int found[2][4];  // per stage and wave: a masked tile's V rows hold something that is not finite
  __shared__ float lds_ml[TS > 1 && RTW == 2 ? 4 * RTW * 32 : 1];
  static_assert(TS == 1 || (RTW == 1 ? SH::kDT * 1024 + 512 : 2 * kSums) <= SH::kStage, "the exchange of the waves must fit the stages");

  int lane = threadIdx.x & 63;
  if constexpr (LINE) {  // formed anew for every item, like the arguments
    lane = lane_id();
    asm volatile("" : "+v"(lane));
    lane &= 63;
  }
  const int mi = lane & 15, kg = lane >> 4;
  // (TS == 1 spelled out: the compiler does not know that there are four waves; fp8, 512 rows, 670 against 662 us)
  const int tg = TS == 1 ? 0 : wave / kApart;  // which of the waves that share the tokens
  const int first_row = it.rg * kRowsPerItem + (TS == 1 ? wave : wave % kApart) * RTW * 16;

  TreeLoader<SH, KV> ld;
  ld.init(p, wave, lane);
  const int t0 = it.t_begin;
  const int iters = it.t_end > t0 ? (it.t_end - t0 + SH::kTT - 1) / SH::kTT : 0;
  float sc = 0.0f;  // the scales in flight (8-bit caches)
  if (iters > 0) ld.template issue<STREAM>(p, it, t0, stage0, sc);

  TreeRows<SH, KV> rows[RTW];
#pragma unroll
  for (int a = 0; a < RTW; ++a) rows[a].init(p, it, first_row + 16 * a, lane);
  const bool has_rows = first_row < it.n * p.group;

  // LDS offsets of the operand reads: lane constants, tiles and pieces XORed or added in
  const uint32_t k_off = (uint32_t)(mi * SH::kRB + ((kg ^ tree_swz_k<SH::kRB>(mi)) << 4));
  uint32_t v_off;
  if constexpr (SH::kQuant) {
    const int r = mi >> 1;  // eight rows to sixteen lanes: tokens 4kg .. 4kg+3 and 16 + 4kg ..
    const int row = r < 4 ? 4 * kg + r : 16 + 4 * kg + (r - 4);
    v_off = (uint32_t)(SH::kArray + row * SH::kRB + (tree_swz_v<SH::kRB, true>(row) << 4) + (mi & 1) * 8);
  } else {
    const int row = 4 * kg + (mi >> 2);
    v_off = (uint32_t)(SH::kArray + row * SH::kRB + ((((mi & 3) >> 1) ^ tree_swz_v<SH::kRB, false>(row)) << 4) + (mi & 1) * 8);
  }

  typedef TreeRows<SH, KV> Rows;
  typedef typename Rows::OpK OpK;
  typedef typename Rows::OpV OpV;

  // Two row tiles, or head_dim 256, leave no registers for the operands' XORed offsets: there they are formed anew for
  // every 32 tokens (an opaque copy of the first keeps the compiler from holding them through the loop).
  auto fresh = [](uint32_t off) {
    if (RTW > 1 || D == 256) asm volatile("" : "+v"(off));
    return off;
  };
  // The operands of 32 tokens: K rows 16h + mi, elements of chunk c (16-bit), or chunks 2c and 2c + 1 (8-bit) ...
  auto k_operand = [&](const uint8_t* tile, uint32_t ko, int c, int h) { return *(const u32x4*)(tile + (ko ^ (uint32_t)(c << 6)) + h * 16 * SH::kRB); };
  // ... and V^T, head-dim tile dt.
  typedef __attribute__((ext_vector_type(2))) int i32x2;
  auto v_bytes = [&](const uint8_t* tile, uint32_t vo, int dt) {
    return __builtin_amdgcn_ds_read_tr8_b64_v2i32((__attribute__((address_space(3))) i32x2*)(tile + (vo ^ (uint32_t)(dt << 4))));
  };
  auto v_operand = [&](const uint8_t* tile, uint32_t vo, int dt) {
    if constexpr (SH::kQuant) {
      const i32x2 raw = v_bytes(tile, vo, dt);
      return __builtin_bit_cast(OpV, tree_widen<KV, SH::kVF16>((uint32_t)raw[0], (uint32_t)raw[1]));
    } else {
      const uint32_t at = vo ^ (uint32_t)(dt << 5);
      const s16x4 a0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(tile + at));
      const s16x4 a1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(tile + at + 16 * SH::kRB));
      return __builtin_bit_cast(OpV, __builtin_shufflevector(a0, a1, 0, 1, 2, 3, 4, 5, 6, 7));
    }
  };
  // S^T of N row tiles from `a` on over 32 tokens: every K operand serves all of them.
  auto scores = [&](const uint8_t* tile, auto count, int a, f32x4 (&s)[decltype(count)::value][2]) {
    constexpr int N = decltype(count)::value;
    const uint32_t ko = fresh(k_off);
#pragma unroll
    for (int n = 0; n < N; ++n) s[n][0] = s[n][1] = f32x4{0, 0, 0, 0};
#pragma unroll
    for (int c = 0; c < (SH::kQuant ? SH::kChunks / 2 : SH::kChunks); ++c) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const u32x4 raw = k_operand(tile, ko, c, h);
        if constexpr (SH::kQuant) {
          const OpK f0 = __builtin_bit_cast(OpK, tree_widen_k<KV, SH::kKF16>(raw[0], raw[1]));
          const OpK f1 = __builtin_bit_cast(OpK, tree_widen_k<KV, SH::kKF16>(raw[2], raw[3]));
#pragma unroll
          for (int n = 0; n < N; ++n) {
            s[n][h] = MmaOps<SH::kKF16>::run(f0, rows[a + n].qf[2 * c], s[n][h]);
            s[n][h] = MmaOps<SH::kKF16>::run(f1, rows[a + n].qf[2 * c + 1], s[n][h]);
          }
        } else {
          const OpK f = __builtin_bit_cast(OpK, raw);
#pragma unroll
          for (int n = 0; n < N; ++n) s[n][h] = MmaOps<SH::kKF16>::run(f, rows[a + n].qf[c], s[n][h]);
        }
      }
    }
  };
  // One of the three per-token factors of 32 tokens (8-bit caches): 0 kscl, 1 lv, 2 rvs.
  auto factor = [&](const uint8_t* stage, int piece, int which, f32x4 (&f)[2]) {
    if constexpr (SH::kQuant) {
      const float* src = (const float*)(stage + SH::kFactors) + which * SH::kTT + piece + 4 * kg;
      f[0] = *(const f32x4*)src;
      f[1] = *(const f32x4*)(src + 16);
    }
  };

  // 32 tokens: those every row sees, or (MASKED) under the rows' bits.
  TreeRowMask<RTW == 1> masks[RTW];
  auto attend = [&](const uint8_t* stage, int tb, int piece, auto masked) {
    constexpr bool MASKED = decltype(masked)::value;
    const uint8_t* tile = stage + piece * SH::kRB;
    f32x4 s[RTW][2];
    // Matrix instructions before the other workgroup's softmax: fp8, 512 rows to a kv head, 2 % faster.  (The forms that
    // are bound by memory or latency lose half a microsecond to what it does to their schedule.)
    constexpr bool kFirst = SH::kQuant || RTW > 1;
    if constexpr (kFirst) __builtin_amdgcn_s_setprio(1);
    scores(tile, std::integral_constant<int, RTW>{}, 0, s);
    if constexpr (kFirst) __builtin_amdgcn_s_setprio(0);
    uint32_t vis[RTW];
#pragma unroll
    for (int a = 0; a < RTW; ++a) vis[a] = MASKED ? masks[a].bits(p, it, first_row + 16 * a, lane, tb + piece) : 0u;
    float x[RTW][8];
    {
      f32x4 kscl[2], lv[2];
      factor(stage, piece, 0, kscl);
      factor(stage, piece, 1, lv);
#pragma unroll
      for (int a = 0; a < RTW; ++a) rows[a].template scaled<MASKED>(s[a], kscl, lv, p.scale_log2, vis[a], kg, x[a]);
    }
    // Two row tiles over an 8-bit cache leave no register to spare: the factors live as briefly as they can, and the
    // registers they leave take V's bytes, which are on their way while the weights are formed.
    constexpr bool kAhead = SH::kQuant && RTW > 1;
    if (kAhead) __builtin_amdgcn_sched_barrier(0);
    f32x4 rvs[2];
    factor(stage, piece, 2, rvs);
    const uint32_t vo = fresh(v_off);
    constexpr int kFetched = TS == 1 ? SH::kDT - 1 : SH::kDT;  // (all of them would spill)
    i32x2 vraw[kAhead ? SH::kDT : 1];
    if constexpr (kAhead) {
#pragma unroll
      for (int dt = 0; dt < kFetched; ++dt) vraw[dt] = v_bytes(tile, vo, dt);
      __builtin_amdgcn_sched_barrier(0);
    }
    OpV pf[RTW];
    float alpha[RTW];
    bool moved = false;
#pragma unroll
    for (int a = 0; a < RTW; ++a) {
      moved |= rows[a].template weights<MASKED>(x[a], rvs, p.scale_log2, vis[a], kg, alpha[a]);
      pf[a] = Rows::pack(x[a]);
    }
    if (moved) {
#pragma unroll
      for (int a = 0; a < RTW; ++a) {
#pragma unroll
        for (int dt = 0; dt < SH::kDT; ++dt) rows[a].acc[dt] *= alpha[a];
      }
    }
    if constexpr (kFirst) __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int dt = 0; dt < SH::kDT; ++dt) {
      OpV vf;
      if (kAhead && dt < kFetched) {
        vf = __builtin_bit_cast(OpV, tree_widen<KV, SH::kVF16>((uint32_t)vraw[dt][0], (uint32_t)vraw[dt][1]));
      } else {
        vf = v_operand(tile, vo, dt);
      }
#pragma unroll
      for (int a = 0; a < RTW; ++a) rows[a].acc[dt] = MmaOps<SH::kVF16>::run(vf, pf[a], rows[a].acc[dt]);
    }
    if constexpr (kFirst) __builtin_amdgcn_s_setprio(0);
  };

  // The same where V holds something that is not finite: token by token, each row under its own bits, a row tile after
  // the other (see the head of the file).
  auto attend_exact = [&](const uint8_t* stage, int tb, int piece) {
    const uint8_t* tile = stage + piece * SH::kRB;
#pragma unroll
    for (int a = 0; a < RTW; ++a) {
      f32x4 s[1][2];
      scores(tile, std::integral_constant<int, 1>{}, a, s);
      const uint32_t vis = masks[a].bits(p, it, first_row + 16 * a, lane, tb + piece);
      float w[8], alpha;
      {
        f32x4 kscl[2], lv[2];
        factor(stage, piece, 0, kscl);
        factor(stage, piece, 1, lv);
        rows[a].template scaled<true>(s[0], kscl, lv, p.scale_log2, vis, kg, w);
      }
      f32x4 rvs[2];
      factor(stage, piece, 2, rvs);
      if (rows[a].template weights<true>(w, rvs, p.scale_log2, vis, kg, alpha)) {
#pragma unroll
        for (int dt = 0; dt < SH::kDT; ++dt) rows[a].acc[dt] *= alpha;
      }
#pragma unroll
      for (int dt = 0; dt < SH::kDT; ++dt) {
        f32x4 o = rows[a].acc[dt];
#pragma unroll 1
        for (int t = 0; t < 32; ++t) {
          // the weight of token t lies with lane kg' = (t >> 2) & 3 of the row's four, as its number 4 (t >> 4) + (t & 3)
          const int idx = 4 * (t >> 4) + (t & 3);
          float mine = 0.0f;
#pragma unroll
          for (int i = 0; i < 8; ++i) mine = idx == i ? w[i] : mine;
          const float wt = __shfl(mine, ((t >> 2) & 3) * 16 + mi);
          const int row = piece + t, at = (dt * 16 + 4 * kg) * SH::kEB;
          const uint8_t* v = stage + SH::kArray + row * SH::kRB + (((at >> 4) ^ tree_swz_v<SH::kRB, SH::kQuant>(row)) << 4) + (at & 15);
#pragma unroll
          for (int e = 0; e < 4; ++e) o[e] = (vis >> t) & 1 ? __builtin_fmaf(wt, Elem<KV>::load(v, e), o[e]) : o[e];
        }
        rows[a].acc[dt] = o;
      }
    }
  };

  // Tile i from `here`: its loads have landed (every wave waits for its own), the waves meet — nobody reads `next` any
  // more — tile i + 1 goes in flight into `next`, tile i is attended.  The two stages are LDS arrays of their own and
  // the loop over tiles that every row sees is written out for both, so that the compiler can tell the loads in
  // flight from the tile being read and does not wait for them.  (Four stages of half the tokens, three of them in
  // flight, were slower: 24 fp8 sequences, 61 drafts, 413 against 353 us; 64 x 4096 bf16 tokens 193 against 184: what
  // a step costs beside its tokens outweighs the deeper queue.)
  auto step = [&](int i, uint8_t* here, uint8_t* next) {
    __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0)
    ld.factors(p, here, sc);
    __syncthreads();
    if (i + 1 < iters) ld.template issue<STREAM>(p, it, t0 + (i + 1) * SH::kTT, next, sc);
    if (!has_rows) return;
#pragma unroll 1
    for (int piece = 32 * tg; piece < SH::kTT; piece += 32 * TS) attend(here, 0, piece, std::false_type{});
  };
  // Tiles of the chunk whose tokens all lie in the context.
  const int whole = max(min(it.prefix, it.t_end) - t0, 0) / SH::kTT;
  int i = 0;
  for (; i + 2 <= whole; i += 2) {
    step(i, stage0, stage1);
    step(i + 1, stage1, stage0);
  }
  // The rest: an odd tile of the context, the last of the context with the drafted tokens behind it, and so on.
  if (i < iters) {
#pragma unroll
    for (int a = 0; a < RTW; ++a) masks[a].init(p, it, first_row + 16 * a, lane);
  }
  for (; i < iters; ++i) {
    uint8_t* here = (i & 1) != 0 ? stage1 : stage0;
    const int tb = t0 + i * SH::kTT;
    __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0)
    ld.factors(p, here, sc);
    const bool masked = tb + SH::kTT > it.prefix;
    if (KV != XLLM_HIP_INT8 && masked) {
      const bool bad = ld.look_through(tb, it.prefix, it.len, here);
      if (lane == 0) found[i & 1][wave] = bad;
    }
    __syncthreads();  // (factors, zeros and findings are in LDS too)
    if (i + 1 < iters) ld.template issue<STREAM>(p, it, tb + SH::kTT, (i & 1) != 0 ? stage0 : stage1, sc);
    if (!has_rows) continue;
    bool exact = false;
    if (KV != XLLM_HIP_INT8 && masked) {
      const int* f = found[i & 1];
      exact = __builtin_amdgcn_readfirstlane(f[0] | f[1] | f[2] | f[3]) != 0;
    }
#pragma unroll 1
    for (int piece = 32 * tg; piece < SH::kTT && tb + piece < it.t_end; piece += 32 * TS) {
      if (tb + piece + 32 <= it.prefix) {
        attend(here, tb, piece, std::false_type{});
      } else if (KV != XLLM_HIP_INT8 && exact) {
        attend_exact(here, tb, piece);
      } else {
        attend(here, tb, piece, std::true_type{});
      }
    }
  }

  // End of the item.  (The lane's number is formed anew: held through the loops it costs a register.)
  const int end_lane = lane_id(), end_kg = end_lane >> 4;
  const float neg_inf = -INFINITY;
  if constexpr (TS == 2 && RTW == 1) {
    // the second wave of a row tile hands over its sums; nothing is in flight any more
    __syncthreads();
    uint8_t* xch = (wave & 1) != 0 ? stage1 : stage0;
    float* ml = (float*)(xch + SH::kDT * 1024);
    Rows& r = rows[0];
    if (tg == 1) {
      ml[end_lane] = r.m_run;
      ml[64 + end_lane] = r.l_run;
#pragma unroll
      for (int dt = 0; dt < SH::kDT; ++dt) *(f32x4*)(xch + dt * 1024 + end_lane * 16) = r.acc[dt];
    }
    __syncthreads();
    if (tg == 1) return;
    const float m2 = ml[end_lane], l2 = ml[64 + end_lane];
    const float m = fmaxf(r.m_run, m2);
    const float m_safe = m == neg_inf ? 0.0f : m;
    const float a1 = __builtin_amdgcn_exp2f(r.m_run - m_safe), a2 = __builtin_amdgcn_exp2f(m2 - m_safe);
    r.m_run = m;
    r.l_run = r.l_run * a1 + l2 * a2;
#pragma unroll
    for (int dt = 0; dt < SH::kDT; ++dt) {
      const f32x4 o = *(const f32x4*)(xch + dt * 1024 + end_lane * 16);
      r.acc[dt] = r.acc[dt] * a1 + o * a2;
    }
  }
  if constexpr (TS > 1 && RTW == 2) {
    // All hand over their sums; each finishes its part of the head's columns.
    __syncthreads();
    const int end_mi = end_lane & 15;
    uint8_t* mine = (wave < 2 ? stage0 : stage1) + (wave & 1) * kSums;
#pragma unroll
    for (int a = 0; a < RTW; ++a) {
      const float l = kg_sum(rows[a].l_run);
      if (end_kg == 0) {
        lds_ml[(wave * RTW + a) * 32 + end_mi] = rows[a].m_run;
        lds_ml[(wave * RTW + a) * 32 + 16 + end_mi] = l;
      }
#pragma unroll
      for (int dt = 0; dt < SH::kDT; ++dt) *(f32x4*)(mine + (a * SH::kDT + dt) * 1024 + end_lane * 16) = rows[a].acc[dt];
    }
    __syncthreads();
#pragma unroll
    for (int a = 0; a < RTW; ++a) {
      float m = neg_inf, l = 0.0f, w[TS];
      const float* ml = lds_ml + ((wave % kApart) * RTW + a) * 32 + end_mi;  // (of share x: + x * kApart * RTW * 32)
#pragma unroll
      for (int x = 0; x < TS; ++x) m = fmaxf(m, ml[x * kApart * RTW * 32]);
      const float m_safe = m == neg_inf ? 0.0f : m;
#pragma unroll
      for (int x = 0; x < TS; ++x) {
        w[x] = __builtin_amdgcn_exp2f(ml[x * kApart * RTW * 32] - m_safe);
        l += w[x] * ml[x * kApart * RTW * 32 + 16];
      }
      TreeOut out;
      if (!out.init(p, it, first_row + 16 * a, end_lane, l, m - Rows::kHead, tg == 0 && end_kg == 0)) continue;
#pragma unroll
      for (int q = 0; q < SH::kDT / TS; ++q) {
        const int dt = tg * (SH::kDT / TS) + q;
        f32x4 o = {0, 0, 0, 0};
#pragma unroll
        for (int x = 0; x < TS; ++x) {
          const int from = x * kApart + wave % kApart;
          o += w[x] * *(const f32x4*)((from < 2 ? stage0 : stage1) + (from & 1) * kSums + (a * SH::kDT + dt) * 1024 + end_lane * 16);
        }
        out.template store<SH::kQF16>(dt * 16 + 4 * end_kg, o);
      }
    }
    return;
  }
  if (!has_rows) return;
#pragma unroll
  for (int a = 0; a < RTW; ++a) {
    Rows& r = rows[a];
    const float l = kg_sum(r.l_run);
    TreeOut out;
    if (!out.init(p, it, first_row + 16 * a, end_lane, l, r.m_run - Rows::kHead, end_kg == 0)) continue;
#pragma unroll
    for (int dt = 0; dt < SH::kDT; ++dt) out.template store<SH::kQF16>(dt * 16 + 4 * end_kg, r.acc[dt]);
  }
}

template <int QT, int KV, int D, int RTW, int TS, bool STREAM>
__global__ void __launch_bounds__(256, (TreeShape<QT, KV, D>::kStage > 40000 ? 1 : 2)) tree_mfma_kernel(TreeParams p) {
  TreeItem it;
  int id = blockIdx.x;
  if (p.row_groups > 1) {
    // the row groups of one (chunk, kv head) read the same K and V: neighbours on one XCD, whose L2 they share
    const int on = id / kTreeXcds;
    id = ((on / p.row_groups) * kTreeXcds + id % kTreeXcds) * p.row_groups + on % p.row_groups;
  }
  if (!tree_item(p, id, 16 * RTW * 4 / TS, it)) return;
  tree_mfma_item<QT, KV, D, RTW, TS, STREAM, false>(p, it, __builtin_amdgcn_readfirstlane(threadIdx.x >> 6));
}

template <int QT, int KV, int D, int RTW, int TS, bool STREAM>
__global__ void __launch_bounds__(256, (TreeShape<QT, KV, D>::kStage > 40000 ? 1 : 2)) tree_mfma_line_kernel(TreeParams p) {
  TreeItem it;
  TreeLine line;
  if (!line.start(p, blockIdx.x, it)) return;
  // The arguments are read anew for every item: held in registers from one to the next they are too many.
  typedef const __attribute__((address_space(4))) TreeParams* Args;
  Args args = (Args)__builtin_amdgcn_kernarg_segment_ptr();
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  for (;;) {
    asm volatile("" : "+s"(args));
    tree_mfma_item<QT, KV, D, RTW, TS, STREAM, true>(*(const TreeParams*)args, it, wave);
    asm volatile("" : "+s"(args));
    if (!line.next(*(const TreeParams*)args, it)) return;
    __syncthreads();  // (nobody reads the stages any more)
  }
}

}  // namespace xllm_hip
