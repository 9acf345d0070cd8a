// Attention of a few new tokens per sequence over a cache of keys and values, the cache 16-bit or quantised (token_cache.h), with an
// optional prefix that all sequences share.  Kernel templates; the instantiations are split over cache_attention_{plain,mx}.hip.
//
//   o_r = sum_j w_rj v_j / sum_j w_rj,   w_rj = exp(s_rj),   s = scale q.k, then cap tanh(s / cap), then - slope_h (pos_r - pos_j)
//
// The rows r that read one key head are the T new tokens times the G query heads of the group: 1 to 16 of them for nearly every
// call, so a key row of D values feeds at most 16 dot products and the call is bound by the bytes of the cache.  What follows from it:
//
//  * One wave streams blocks of 32 keys from memory STRAIGHT into the operand layout of v_mfma_f32_16x16x32: no LDS, no barrier in
//    the loop, every byte is loaded once.  All layouts below work because the order of a contraction index is free as long as both operands use
//    the same one.
//      scores   S^T = K Q^T  (A = K: lane (key i, g) holds the D / 4 values from g D / 4 on, in D / 32 slices of 8; B = Q, same slices)
//               -> lane (row i, g) holds the scores of keys 4 g + 0..3 of both 16-key tiles
//      values   O^T = V^T P^T (B = P straight from those registers: contraction slot 8 g + j is key 4 g + j, j < 4, resp. 16 + 4 g + j - 4;
//               A = V: lane (i, g) loads elements [i E, (i + 1) E) of exactly those 8 keys, E = 16, 8, 4, 2 by head dimension, and
//               turns its 8 x E block around with v_perm_b32, half an instruction an element)
//               -> lane (row i, g) holds output elements [4 g E, 4 (g + 1) E) of its OWN row: the softmax statistics need no exchange.
//  * The running maximum is raised only when a score exceeds it by more than 2^8: the weights stay below 2^8, the sums are fp32, and
//    the cross-lane reduction and the rescaling of O leave the loop after the first blocks.
//  * Quantised codes are converted with their scale into bf16, which holds code * 2^e exactly (at most 4 significant bits and an 8-bit
//    exponent).  fp16 queries become TWO bf16 operands whose sum is exact; the weights become two bf16 operands (16 significant
//    bits) wherever the values are bf16: the matrix pipe idles in this kernel, the second product is free, and the result carries no
//    rounding but the output's.  fp16 caches: the weights are one fp16 operand (11 bits, the output's own precision).
//  * The keys are split over workgroups (and over the four waves of one); parts are joined by k_cache_attn_join with fp32 weights.
//  * The shared prefix is one matrix of keys for ALL rows B T G of a key head: its workgroups take 4 waves of different rows over the
//    same keys, so the prefix is read from HBM once and from L2 once per 64 or 128 rows, not once per sequence.
#pragma once
#include "token_cache.h"

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));

struct CacheAttnArgs {
  const char* q;                 // 16-bit elements
  int64_t q_b, q_t, q_h;         // strides in bytes
  char* out;                     // [B,T,Hq,D] contiguous
  const uint8_t *k, *v, *ks, *vs, *pk, *pv, *pks, *pvs;
  int64_t k_b, k_h, v_b, v_h, ks_b, ks_h, vs_b, vs_h, pk_h, pv_h, pks_h, pvs_h;   // strides in bytes
  unsigned k_c, v_c, ks_c, vs_c, pk_c, pv_c, pks_c, pvs_c;                        // bytes from a token to the next
  const int32_t* lens;
  const float* slopes;
  int B, T, Hq, Hkv, G, D, C, P;
  float scale, cap;
  int own_chunk, own_parts, own_groups;    // keys per workgroup, parts per sequence, row groups per key head
  int pre_chunk, pre_parts, pre_groups;    // the same for the prefix (pre_groups workgroup row groups)
  int pre_rows;                            // 1: the four waves of a prefix workgroup hold different rows; 0: different keys
  int pre_blocks;                          // workgroups [0, pre_blocks) work on the prefix
  float* part_o;                           // [parts][B T Hq][D]; null: one part, written out at once
  f32x2_t* part_ml;                        // [parts][B T Hq]
};

#define DS2_LOG2E 1.44269504088896340736f

template <bool F16>
__device__ __forceinline__ f32x4 ds2_mfma16(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (F16) return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}

// NB bytes (1, 2, 4, 8, 16, 32) into words
template <int NB>
__device__ __forceinline__ void ds2_load_bytes(unsigned* to, const uint8_t* p) {
  if constexpr (NB == 1) to[0] = *p;
  else if constexpr (NB == 2) to[0] = *(const uint16_t*)p;
  else if constexpr (NB == 4) to[0] = *(const unsigned*)p;
  else if constexpr (NB == 8) {
    const u32x2 w = *(const u32x2*)p;
    to[0] = w[0], to[1] = w[1];
  } else {
#pragma unroll
    for (int i = 0; i < NB / 16; ++i) {
      const u32x4 w = ((const u32x4*)p)[i];
#pragma unroll
      for (int j = 0; j < 4; ++j) to[4 * i + j] = w[j];
    }
  }
}

// 8 codes (2 words of e4m3 or 1 word of e2m1) times their scale -> 8 bf16 values, exact.  The conversion takes the scale's exponent
// field: byte 255 gives NaN, byte 0 gives 2^-127 (both measured).
template <int FORMAT>
__device__ __forceinline__ u32x4 ds2_decode8(const unsigned* w, float s) {
  u32x4 r;
  if constexpr (FORMAT == DS2_CACHE_MXFP8) {
    r[0] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[0], s, false));
    r[1] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[0], s, true));
    r[2] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[1], s, false));
    r[3] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[1], s, true));
  } else {
    r[0] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[0], s, 0));
    r[1] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[0], s, 1));
    r[2] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[0], s, 2));
    r[3] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[0], s, 3));
  }
  return r;
}

__device__ __forceinline__ float ds2_operand_scale(unsigned s) { return __builtin_bit_cast(float, max(s << 23, 0x00400000u)); }

// 16-bit pair: which halves are infinities or NaNs, as a mask over the word
template <bool F16>
__device__ __forceinline__ unsigned ds2_not_finite16(unsigned w) {
  constexpr unsigned EXP = F16 ? 0x7c00u : 0x7f80u;
  return ((w & EXP) == EXP ? 0xffffu : 0u) | (((w >> 16) & EXP) == EXP ? 0xffff0000u : 0u);
}

// one stream of keys of a head, as its kernel argument lists it
struct CacheRows {
  const uint8_t *k, *v, *ks, *vs;
  unsigned k_c, v_c, ks_c, vs_c;
};

// E: values a lane holds of a value row (D <= 16 E; FULL: D == 16 E); RT: tiles of 16 query rows of a wave
template <int FORMAT, bool QF16, int E, int RT, bool FULL>
struct CacheStream {
  static constexpr bool QUANT = FORMAT != DS2_CACHE_PLAIN;
  static constexpr bool F16 = QF16 && !QUANT;            // operand type of both products
  static constexpr bool QLO = QF16 && QUANT;             // queries as two bf16 operands
  static constexpr bool PLO = !F16;                      // weights as two bf16 operands
  static constexpr int KS = E / 2;                       // slices of 8 values a lane holds of a key row, at most
  static constexpr int SB = FORMAT == DS2_CACHE_PLAIN ? 16 : FORMAT == DS2_CACHE_MXFP8 ? 8 : 4;          // bytes of a slice
  static constexpr int VB = FORMAT == DS2_CACHE_PLAIN ? 2 * E : FORMAT == DS2_CACHE_MXFP8 ? E : E / 2;   // bytes of a lane's value row
  static constexpr int SW = SB / 4, VW = VB < 4 ? 1 : VB / 4;

  u32x4 q[RT][KS], ql[QLO ? RT : 1][QLO ? KS : 1];
  f32x4 o[RT][E];
  float m[RT], l[RT];
  float slope[RT];          // * log2 e
  int pos[RT], sees[RT];    // position of the row and how many keys it sees, both counted in the keys of this stream

  __device__ __forceinline__ void start(int rt, const char* row, bool live, int g, int ksr) {
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      u32x4 w = {0, 0, 0, 0};
      if (live && (FULL || s < ksr)) w = *(const u32x4*)(row + (g * ksr + s) * 16);
      if constexpr (QLO) {
        u32x4 hi, lo;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float x = ds2_low16<true>(w[j]), y = ds2_high16<true>(w[j]);
          hi[j] = ds2_pack16<false>(x, y);
          lo[j] = ds2_pack16<false>(x - ds2_low16<false>(hi[j]), y - ds2_high16<false>(hi[j]));
          // (an infinite query has no remainder: inf - inf would be NaN)
          lo[j] &= ~ds2_not_finite16<false>(lo[j]);
        }
        q[rt][s] = hi, ql[rt][s] = lo;
      } else q[rt][s] = w;
    }
#pragma unroll
    for (int t = 0; t < E; ++t) o[rt][t] = f32x4{0, 0, 0, 0};
    m[rt] = -INFINITY, l[rt] = 0.f;
  }

  // Blocks first, first + step, ... of the keys [k0, k1); every key below `common` is seen by all rows.  nrt: row tiles in use.
  __device__ __forceinline__ void run(const CacheAttnArgs& a, const CacheRows& c, int k0, int k1, int first, int step, int common,
                                      int nrt, int lane) {
    const int i = lane & 15, g = lane >> 4;
    const int ksr = FULL ? KS : a.D >> 5;
    const int vi = FULL || i * E < a.D ? i : 0;            // lanes beyond the head dimension repeat the first one's elements
    const unsigned k_lane = g * ksr * SB, v_lane = vi * VB, vs_lane = (vi * E) >> 5;
    const float sc = a.scale * DS2_LOG2E, cap2 = a.cap * DS2_LOG2E;
    const float in_cap = a.cap > 0.f ? 2.f * DS2_LOG2E * a.scale / a.cap : 0.f;
    for (int blk = k0 + first * 32; blk < k1; blk += step * 32) {
      const int last = k1 - 1 - blk;                       // rows behind the end repeat the last key: their weight is zero
      const uint8_t *kb = c.k + (int64_t)blk * c.k_c, *vb = c.v + (int64_t)blk * c.v_c;
      const uint8_t *ksb = c.ks + (int64_t)blk * c.ks_c, *vsb = c.vs + (int64_t)blk * c.vs_c;
      // ---- all loads of the block
      unsigned kw[2][KS * SW], vw[8][VW], kscale[2][KS], vscale[8];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const unsigned row = min(16 * t + i, last);
        const uint8_t* p = kb + (row * c.k_c + k_lane);
        if constexpr (FULL) ds2_load_bytes<KS * SB>(kw[t], p);
        else {
#pragma unroll
          for (int s = 0; s < KS; ++s)
            if (s < ksr) ds2_load_bytes<SB>(kw[t] + s * SW, p + s * SB);
        }
        if constexpr (QUANT) {
#pragma unroll
          for (int s = 0; s < KS; ++s) {
            if constexpr (FULL) {                          // KS slices are D / 4 values: 4 slices lie in one group
              if (s % 4 == 0) kscale[t][s] = ksb[row * c.ks_c + ((g * KS + s) >> 2)];
              else kscale[t][s] = kscale[t][s - 1];
            } else kscale[t][s] = s < ksr ? ksb[row * c.ks_c + ((g * ksr + s) >> 2)] : 127u;
          }
        }
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const unsigned row = min((j < 4 ? 0 : 12) + 4 * g + j, last);
        ds2_load_bytes<VB>(vw[j], vb + (row * c.v_c + v_lane));
        if constexpr (QUANT) vscale[j] = vsb[row * c.vs_c + vs_lane];
      }
      // ---- operands
      u32x4 kf[2][KS];
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int s = 0; s < KS; ++s) {
          if (!FULL && s >= ksr) continue;
          if constexpr (QUANT) kf[t][s] = ds2_decode8<FORMAT>(kw[t] + s * SW, ds2_operand_scale(kscale[t][s]));
          else kf[t][s] = u32x4{kw[t][4 * s], kw[t][4 * s + 1], kw[t][4 * s + 2], kw[t][4 * s + 3]};
        }
      u32x4 vf[E];
      {
        unsigned vv[8][E < 8 && QUANT ? 4 : E / 2];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if constexpr (QUANT) {
            const float f = ds2_operand_scale(vscale[j]);
            unsigned w[4] = {};
#pragma unroll
            for (int x = 0; x < VW; ++x) w[x] = vw[j][x];
#pragma unroll
            for (int x = 0; x < (E + 7) / 8; ++x) {
              const u32x4 r = ds2_decode8<FORMAT>(w + x * SW, f);
#pragma unroll
              for (int y = 0; y < 4; ++y) vv[j][4 * x + y] = r[y];
            }
          } else {
#pragma unroll
            for (int x = 0; x < E / 2; ++x) vv[j][x] = vw[j][x];
          }
        }
#pragma unroll
        for (int t = 0; t < E; ++t)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            vf[t][j] = __builtin_amdgcn_perm(vv[2 * j + 1][t >> 1], vv[2 * j][t >> 1], (t & 1) ? 0x07060302u : 0x05040100u);
      }
      // A key that a row does not see has weight 0, but 0 times an infinity or a NaN is not 0.  Where rows of the block may see
      // different keys, values that are not finite leave the product and go to the rows that do see them, one by one.
      const bool edge = blk + 32 > common;
      bool apart = false;
      if (edge) {
        unsigned bad = 0;
#pragma unroll
        for (int t = 0; t < E; ++t)
#pragma unroll
          for (int j = 0; j < 4; ++j) bad |= ds2_not_finite16<F16>(vf[t][j]);
        apart = __any(bad != 0);
        if (apart) {
#pragma unroll
          for (int t = 0; t < E; ++t)
#pragma unroll
            for (int j = 0; j < 4; ++j) vf[t][j] &= ~ds2_not_finite16<F16>(vf[t][j]);
        }
      }
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        if (RT > 1 && rt >= nrt) break;
        float p[8];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          f32x4 acc = {0, 0, 0, 0};
#pragma unroll
          for (int s = 0; s < KS; ++s) {
            if (!FULL && s >= ksr) continue;
            acc = ds2_mfma16<F16>(kf[t][s], q[rt][s], acc);
            if constexpr (QLO) acc = ds2_mfma16<F16>(kf[t][s], ql[rt][s], acc);
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) p[4 * t + j] = acc[j];
        }
        if (a.cap > 0.f) {
          // cap tanh(x / cap) = cap - 2 cap / (1 + exp(2 x / cap)): no branch, saturates by itself; off by a few 2^-24 of cap
#pragma unroll
          for (int j = 0; j < 8; ++j)
            p[j] = cap2 - 2.f * cap2 * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(p[j] * in_cap));
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) p[j] *= sc;
        }
        if (a.slopes) {
#pragma unroll
          for (int j = 0; j < 8; ++j) p[j] -= slope[rt] * (float)(pos[rt] - (blk + (j < 4 ? 0 : 12) + 4 * g + j));
        }
        if (edge) {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (blk + (j < 4 ? 0 : 12) + 4 * g + j >= sees[rt]) p[j] = -INFINITY;
        }
        float top = fmaxf(fmaxf(fmaxf(p[0], p[1]), fmaxf(p[2], p[3])), fmaxf(fmaxf(p[4], p[5]), fmaxf(p[6], p[7])));
        if (__any(top > m[rt] + 8.f)) {
          top = fmaxf(top, __shfl_xor(top, 16));
          top = fmaxf(top, __shfl_xor(top, 32));
          const float mn = fmaxf(m[rt], top);
          const float al = m[rt] == mn ? 1.f : __builtin_amdgcn_exp2f(m[rt] - mn);
          l[rt] *= al;
#pragma unroll
          for (int t = 0; t < E; ++t) o[rt][t] *= al;
          m[rt] = mn;
        }
        const float ref = m[rt] == -INFINITY ? 0.f : m[rt];
        u32x4 ph, pl;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          p[j] = __builtin_amdgcn_exp2f(p[j] - ref);
          l[rt] += p[j];
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          ph[j] = ds2_pack16<F16>(p[2 * j], p[2 * j + 1]);
          if constexpr (PLO) pl[j] = ds2_pack16<F16>(p[2 * j] - ds2_low16<F16>(ph[j]), p[2 * j + 1] - ds2_high16<F16>(ph[j]));
        }
        if (apart) add_apart(rt, a, p, vb, vsb, c, blk, last, i, g);
#pragma unroll
        for (int t = 0; t < E; ++t) {
          o[rt][t] = ds2_mfma16<F16>(vf[t], ph, o[rt][t]);
          if constexpr (PLO) o[rt][t] = ds2_mfma16<F16>(vf[t], pl, o[rt][t]);
        }
      }
    }
  }

  // the values of a block that are not finite, to the rows that see their keys (rare: speed does not matter)
  __device__ __forceinline__ void add_apart(int rt, const CacheAttnArgs& a, const float (&p)[8], const uint8_t* vb, const uint8_t* vsb,
                                            const CacheRows& c, int blk, int last, int i, int g) {
#pragma unroll 1
    for (int key = 0; key < 32; ++key) {
      if (key > last) break;
      const int j = (key & 3) | (key >> 4) << 2, from = (key >> 2) & 3;
      float mine = p[0];
#pragma unroll
      for (int x = 1; x < 8; ++x) mine = j == x ? p[x] : mine;
      const float w = __shfl(mine, i | from << 4);
      if (blk + key >= sees[rt]) continue;
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int t = 0; t < E; ++t) {
          const int d = (4 * g + r) * E + t;
          if (!FULL && d >= a.D) continue;
          float x;
          if constexpr (FORMAT == DS2_CACHE_PLAIN) x = ds2_low16<F16>(*(const uint16_t*)(vb + ((int64_t)key * c.v_c + 2 * d)));
          else {
            const float f = ds2_operand_scale(vsb[(int64_t)key * c.vs_c + (d >> 5)]);
            unsigned code[2] = {FORMAT == DS2_CACHE_MXFP8 ? vb[(int64_t)key * c.v_c + d] : (unsigned)vb[(int64_t)key * c.v_c + (d >> 1)] >> 4 * (d & 1), 0u};
            x = ds2_low16<false>(ds2_decode8<FORMAT>(code, f)[0]);
          }
          if (!__builtin_isfinite(x)) o[rt][t][r] += w * x;
        }
    }
  }
};

template <int FORMAT, bool QF16, int E, int RT, bool FULL>
__global__ __launch_bounds__(256, 2) __attribute__((amdgpu_num_vgpr(256))) void k_cache_attn(CacheAttnArgs a) {
  typedef CacheStream<FORMAT, QF16, E, RT, FULL> Stream;
  constexpr bool HALF = QF16;
  __shared__ float join[3][RT * E * 4 + 2 * RT][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int i = lane & 15, g = lane >> 4;
  const bool prefix = (int)blockIdx.x < a.pre_blocks;
  int id = prefix ? blockIdx.x : blockIdx.x - a.pre_blocks;
  int part, head, group, seq = 0;
  if (prefix) {                                            // row groups over the same keys are far apart in id: same chiplet, one L2
    group = id / (a.Hkv * a.pre_parts), id -= group * a.Hkv * a.pre_parts;
    part = id / a.Hkv, head = id - part * a.Hkv;
  } else {
    const int x = id / a.own_parts;
    part = id - x * a.own_parts;
    const int y = x / a.own_groups;
    group = x - y * a.own_groups;
    seq = y / a.Hkv, head = y - seq * a.Hkv;
  }
  const int chunk = prefix ? a.pre_chunk : a.own_chunk;
  const int len = prefix ? a.P : max(0, min(a.lens[seq], a.C));
  const int k0 = part * chunk, k1 = min(len, k0 + chunk);
  const bool by_rows = prefix && a.pre_rows;               // the four waves hold different rows, or the same rows and different keys
  const int rows = prefix ? a.B * a.T * a.G : a.T * a.G;
  const int base = (by_rows ? group * 4 + wave : group) * RT * 16;
  if (a.part_o && k0 >= k1) return;                        // the join does not read this part
  if (by_rows && base >= rows) return;

  Stream st;
  const int ksr = a.D >> 5;
  int row_id[RT];                                          // (b T + t) Hq + query head; -1: no row, or one that sees nothing at all
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int r = base + rt * 16 + i;
    const bool live = r < rows;
    const int rr = live ? r : 0;
    const int b = prefix ? rr / (a.T * a.G) : seq, tg = prefix ? rr - b * a.T * a.G : rr;
    const int t = tg / a.G, hq = head * a.G + (tg - t * a.G);
    const int at = max(0, min(a.lens[b], a.C)) - a.T + t;  // position in the sequence's own keys
    row_id[rt] = live ? (b * a.T + t) * a.Hq + hq : -1;
    st.pos[rt] = at + (prefix ? a.P : 0);
    st.sees[rt] = prefix ? a.P : at + 1;
    st.slope[rt] = a.slopes ? a.slopes[hq] * DS2_LOG2E : 0.f;
    st.start(rt, a.q + b * a.q_b + t * a.q_t + hq * a.q_h, live, g, ksr);
    if (live && at < 0) st.sees[rt] = prefix ? a.P : 0;
  }
  const int nrt = min(RT, (rows - base + 15) >> 4);
  const CacheRows c = prefix ? CacheRows{a.pk + head * a.pk_h, a.pv + head * a.pv_h, a.pks + head * a.pks_h, a.pvs + head * a.pvs_h, a.pk_c, a.pv_c, a.pks_c, a.pvs_c}
                             : CacheRows{a.k + seq * a.k_b + head * a.k_h, a.v + seq * a.v_b + head * a.v_h, a.ks + seq * a.ks_b + head * a.ks_h,
                                         a.vs + seq * a.vs_b + head * a.vs_h, a.k_c, a.v_c, a.ks_c, a.vs_c};
  st.run(a, c, k0, k1, by_rows ? 0 : wave, by_rows ? 1 : 4, prefix ? a.P : len - a.T + 1, nrt, lane);

  if (!by_rows) {                                          // join the four waves' keys: the same rows in the same lanes
    if (wave) {
      float(&to)[RT * E * 4 + 2 * RT][64] = join[wave - 1];
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
        for (int t = 0; t < E; ++t)
#pragma unroll
          for (int j = 0; j < 4; ++j) to[(rt * E + t) * 4 + j][lane] = st.o[rt][t][j];
        to[RT * E * 4 + 2 * rt][lane] = st.m[rt], to[RT * E * 4 + 2 * rt + 1][lane] = st.l[rt];
      }
    }
    __syncthreads();
    if (wave) return;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      float mm = st.m[rt], f[3];
#pragma unroll
      for (int w = 0; w < 3; ++w) mm = fmaxf(mm, join[w][RT * E * 4 + 2 * rt][lane]);
      const float f0 = st.m[rt] == mm ? 1.f : __builtin_amdgcn_exp2f(st.m[rt] - mm);      // (equal also covers -inf and -inf)
      st.l[rt] *= f0;
#pragma unroll
      for (int w = 0; w < 3; ++w) {
        const float mw = join[w][RT * E * 4 + 2 * rt][lane];
        f[w] = mw == mm ? 1.f : __builtin_amdgcn_exp2f(mw - mm);
        st.l[rt] += f[w] * join[w][RT * E * 4 + 2 * rt + 1][lane];
      }
      st.m[rt] = mm;
#pragma unroll
      for (int t = 0; t < E; ++t)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float x = st.o[rt][t][j] * f0;
#pragma unroll
          for (int w = 0; w < 3; ++w) x += f[w] * join[w][(rt * E + t) * 4 + j][lane];
          st.o[rt][t][j] = x;
        }
    }
  }
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    float l = st.l[rt];
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    if (row_id[rt] < 0) continue;
    if (a.part_o) {
      const int64_t at = (int64_t)(prefix ? part : a.pre_parts + part) * a.B * a.T * a.Hq + row_id[rt];
      if (g == 0) a.part_ml[at] = f32x2_t{st.m[rt], l};
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int d = (4 * g + r) * E;
        if (!FULL && d >= a.D) break;
        float* to = a.part_o + at * a.D + d;
        if constexpr (E >= 4) {
#pragma unroll
          for (int t = 0; t < E; t += 4) *(f32x4*)(to + t) = f32x4{st.o[rt][t][r], st.o[rt][t + 1][r], st.o[rt][t + 2][r], st.o[rt][t + 3][r]};
        } else *(f32x2_t*)to = f32x2_t{st.o[rt][0][r], st.o[rt][1][r]};
      }
    } else {
      const bool none = st.m[rt] == -INFINITY && l == 0.f;  // nothing seen: zeros
      const float f = none ? 0.f : 1.f / l;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int d = (4 * g + r) * E;
        if (!FULL && d >= a.D) break;
        unsigned* to = (unsigned*)(a.out + ((int64_t)row_id[rt] * a.D + d) * 2);
#pragma unroll
        for (int t = 0; t < E; t += 2)
          to[t >> 1] = none ? 0u : ds2_pack16<HALF>(st.o[rt][t][r] * f, st.o[rt][t + 1][r] * f);
      }
    }
  }
}

int launch_cache_attn_plain(const CacheAttnArgs& a, bool f16, bool two_tiles, unsigned blocks, hipStream_t st);
int launch_cache_attn_mxfp8(const CacheAttnArgs& a, bool f16, bool two_tiles, unsigned blocks, hipStream_t st);
int launch_cache_attn_mxfp4(const CacheAttnArgs& a, bool f16, bool two_tiles, unsigned blocks, hipStream_t st);

// two_tiles only with D <= 128 (E <= 8): at E = 16 a second tile's accumulators leave one wave a SIMD
template <int FORMAT, bool QF16>
int launch_cache_attn_of(const CacheAttnArgs& a, bool two_tiles, unsigned blocks, hipStream_t st) {
#define DS2_GO(E, FULL)                                                                                                  \
  {                                                                                                                      \
    if (two_tiles && E <= 8) k_cache_attn<FORMAT, QF16, E, E <= 8 ? 2 : 1, FULL><<<dim3(blocks), 256, 0, st>>>(a);       \
    else k_cache_attn<FORMAT, QF16, E, 1, FULL><<<dim3(blocks), 256, 0, st>>>(a);                                        \
  }
  if (a.D == 32) DS2_GO(2, true)
  else if (a.D == 64) DS2_GO(4, true)
  else if (a.D == 96) DS2_GO(8, false)
  else if (a.D == 128) DS2_GO(8, true)
  else DS2_GO(16, true)
#undef DS2_GO
  DS2_CHECK_LAUNCH();
  return DS2_OK;
}
