// Attention of a few new tokens per sequence over a cache of keys and values, the cache 16-bit or quantised (token_cache.h), with an
// optional prefix that all sequences share.  Kernel templates; the instantiations are split over cache_attention_{plain,mx}*.hip.
//
//   o_r = sum_j w_rj v_j / sum_j w_rj,   w_rj = exp(s_rj),   s = scale q.k, then cap tanh(s / cap), then - slope_h (pos_r - pos_j)
//
// The rows r that read one key head are the T new tokens times the G query heads of the group: 1 to 16 of them for nearly every
// call, so a key row of D values feeds at most 16 dot products and the call is bound by the bytes of the cache.  What follows from it:
//
//  * One wave streams blocks of 32 keys from memory into the operand layout of v_mfma_f32_16x16x32 without a barrier; every byte is
//    loaded once.  The layouts work because the order of a contraction index is free as long as both operands use the same one.
//      scores   S^T = K Q^T  (A = K: lane (key i, g) holds the D / 4 values from g D / 4 on, in D / 32 slices of 8; B = Q, same slices)
//               -> lane (row i, g) holds the scores of keys 4 g + 0..3 of both 16-key tiles.  This operand has neighbouring lanes in
//               different rows; loaded like that, the address unit takes a cycle a lane.  So keys go whole rows at a time into
//               LDS that belongs to the wave alone (buffer loads to LDS, 16-byte pieces exchanged within a row so that the reads
//               meet all banks) and are read from there.
//      values   O^T = V^T P^T (B = P straight from those registers: contraction slot 8 g + j is key 4 g + j, j < 4, resp. 16 + 4 g + j - 4;
//               A = V: lane (i, g) loads elements [i E, (i + 1) E) of exactly those 8 keys, E = 8, 4, 2 by head dimension, and
//               turns its 8 x E block around with v_perm_b32, half an instruction an element)
//               -> lane (row i, g) holds output elements [4 g E, 4 (g + 1) E) of its OWN row: the softmax statistics need no exchange.
//    At D = 256 two waves share the rows and keys, each with half of the values (both compute the scores).
//  * The loads are buffer loads: offsets are lane constants, the block is the descriptor's (scalar) base, keys behind the end cost
//    nothing.  The next block's keys are asked for as soon as this one's scores are done, its values after the value product.
//  * The running reference of a row is raised only when a weight would exceed a fixed power of 2 (DS2_LIMIT): the weights stay bounded, the
//    sums are fp32, and the cross-lane reduction and the rescaling of O leave the loop after the first blocks.
//  * Quantised codes are converted with their scale into bf16, which holds code * 2^e exactly (at most 4 significant bits and an 8-bit
//    exponent).  fp16 queries become TWO bf16 operands whose sum is exact; the weights become two bf16 operands (16 significant
//    bits) wherever the values are bf16: the matrix pipe idles in this kernel, the second product is free, and the result carries no
//    rounding but the output's.  fp16 caches: the weights are one fp16 operand (11 bits, the output's own precision, down to 2^-25
//    of the row's largest; DS2_SHIFT).
//  * The work is cut into equal shares, not into sequences: all keys of all (sequence, key head) streams are laid end to end in units of 128
//    and every workgroup takes the same number of units, wherever streams begin and end (the lengths are read on the device).  A
//    share's part of a stream is a segment; k_attn_join joins a stream's segments with fp32 weights.  Beginning a stream costs about as
//    much as a unit (queries, lengths, the first loads, the join of the waves): each counts one unit more than its keys.  Short streams
//    get a workgroup each (cache_attention.hip has the rule).
//  * The shared prefix is one matrix of keys for ALL rows B T G of a key head: it comes from HBM once, not once per sequence.  Its
//    workgroups are in one launch with the sequences' own; a large product over a 16-bit prefix goes to the kernel of whole prompts
//    instead.
//
// Measured: 32 sequences of 8192 tokens, 8 key heads of 128: 16 bits 194 us, 5.5 TB/s of cache; 8 bits 109 us, 5.1 TB/s; 4 bits 67 us, 4.2
// TB/s (64 sequences, heads of 64: 188, 108, 77 us).  A large copy makes 4.9 TB/s, a sum over a large tensor 6.0.  Ragged, 65 to 8192
// tokens, 8 bits: 65 us, 4.3 TB/s with the join.  Four bits are bound by the vector pipe (60 % busy at D = 64: 215 instructions a block
// of 32 keys, mostly conversions and the turning of values), the others by memory.  One sequence of 2048 tokens, 8 key heads: 8 us and
// 3.5 for the join, all of it latency.  64 sequences of 33 to 512 tokens behind 8192 (16 bits, 8 heads of 128, 4 query heads each): 46 us and
// 4.5 for the join; no pipe is full (vector 30 % of cycles, matrix 11 %, vector memory 33 %): the 16 row groups of a head's 256 rows take the
// prefix's 33.5 MB through L1 16 times, and on average half of the waves that fit are resident.
#pragma once
#include <algorithm>

#include "token_cache.h"

constexpr int CACHE_UNIT = 128;  // keys of a unit of work: a block of 32 for each of the four waves

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
  int shares;                              // workgroups that share the sequences' own keys; 0: one workgroup a stream
  bool direct;                             // ... and nothing to join: results are written at once
  int own_rows, own_groups;                // rows of a workgroup, row groups of a key head
  int pre_chunk, pre_parts;                // prefix keys of a workgroup, parts
  int pre_blocks;                          // workgroups [0, pre_blocks) work on the prefix
  int by_rows, pre_by_rows;                // the waves of a workgroup hold different rows over the same keys, or the same rows and different keys
  float* seg_o;                            // [shares + streams][own_rows][D]: segment share + stream (stream, where shares is 0)
  f32x2_t* seg_ml;                         // [shares + streams][own_rows]
  int2* seg_of;                            // [streams]: first and last share of a stream
  float* pre_o;                            // [pre_parts][B T Hq][D]
  f32x2_t* pre_ml;
};

#define DS2_LOG2E 1.44269504088896340736f

template <bool F16>
__device__ __forceinline__ f32x4 ds2_mfma16(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (F16) return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}

// NB bytes (1, 2, 4, 8, 16, 32, 64) into words; zeros beyond the buffer's end
template <int NB>
__device__ __forceinline__ void ds2_load_bytes(unsigned* to, __amdgpu_buffer_rsrc_t from, unsigned at) {
  if constexpr (NB == 1) to[0] = __builtin_amdgcn_raw_buffer_load_b8(from, at, 0, 0);
  else if constexpr (NB == 2) to[0] = __builtin_amdgcn_raw_buffer_load_b16(from, at, 0, 0);
  else if constexpr (NB == 4) to[0] = __builtin_amdgcn_raw_buffer_load_b32(from, at, 0, 0);
  else if constexpr (NB == 8) {
    const u32x2 w = __builtin_amdgcn_raw_buffer_load_b64(from, at, 0, 0);
    to[0] = w[0], to[1] = w[1];
  } else {
#pragma unroll
    for (int i = 0; i < NB / 16; ++i) {
      const u32x4 w = __builtin_amdgcn_raw_buffer_load_b128(from, at + 16 * i, 0, 0);
#pragma unroll
      for (int j = 0; j < 4; ++j) to[4 * i + j] = w[j];
    }
  }
}
// rows [0, n) of a tensor as a buffer
__device__ __forceinline__ __amdgpu_buffer_rsrc_t ds2_rows(const uint8_t* p, int64_t at, unsigned stride, int n, int row_bytes) {
  const int bytes = (int)((unsigned)(min(n, 32) - 1) * stride + row_bytes) & ~((n - 1) >> 31);       // 0 behind the end, without a branch
  return __builtin_amdgcn_make_buffer_rsrc((void*)(p + at * stride), 0, bytes, 0x00020000);
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

// the keys and values of a head
struct CacheRows {
  const uint8_t *k, *v, *ks, *vs;
  unsigned k_c, v_c, ks_c, vs_c;
};

// KS: slices of 8 values a lane holds of a key row (D = 32 KS); E: values it holds of a value row, of every VS-th part of it
template <int FORMAT, bool QF16, int KS, int E, int VS>
struct CacheStream {
  static constexpr bool QUANT = FORMAT != DS2_CACHE_PLAIN;
  static constexpr bool F16 = QF16 && !QUANT;            // operand type of both products
  static constexpr bool QLO = QF16 && QUANT;             // queries as two bf16 operands
  static constexpr bool PLO = !F16;                      // weights as two bf16 operands
  static constexpr int D = 32 * KS;
  static constexpr bool FULL = D == 16 * E * VS;         // else the last lanes hold no values
  static constexpr int SB = FORMAT == DS2_CACHE_PLAIN ? 16 : FORMAT == DS2_CACHE_MXFP8 ? 8 : 4;          // bytes of a slice
  static constexpr int VB = FORMAT == DS2_CACHE_PLAIN ? 2 * E : FORMAT == DS2_CACHE_MXFP8 ? E : E / 2;   // bytes of a lane's value row
  static constexpr int SW = SB / 4, VW = VB < 4 ? 1 : VB / 4;
  static constexpr int ROW = 4 * KS * SB, PIECES = ROW / 16;             // bytes and 16-byte pieces of a row
  static constexpr int ISSUES = (PIECES + 1) / 2;                        // loads to LDS of 64 pieces for 32 rows
  static constexpr int LDS = ISSUES * 1024;                              // a wave's key block
  // pieces of a row change places by row: 16 rows of one piece cover the 64 banks
  static constexpr bool MIX = KS * SB % 16 == 0 && (PIECES & (PIECES - 1)) == 0 && PIECES >= 4;
  static __device__ __forceinline__ int mixed(int row, int piece) {
    return !MIX ? piece : piece ^ (PIECES >= 16 ? row & 15 : PIECES == 8 ? row >> 1 & 7 : row >> 2 & 3);
  }
  static constexpr int SG = KS == 3 ? 3 : (KS + 3) / 4;  // scale bytes a lane needs of a key row (its 8 KS values begin at 8 KS g)

  u32x4 q[KS], ql[QLO ? KS : 1];
  f32x4 o[E];
  float m, l;               // reference and sum of the weights
  float slope;              // * log2 e
  int pos, sees;            // position of the lane's row and how many keys it sees, both counted in the keys of this stream
  unsigned vw[8][VW], kscale[2][SG], vscale[8];

  __device__ __forceinline__ void start(const char* row, bool live, int g) {
#pragma unroll
    for (int s = 0; s < KS; ++s) q[s] = live ? *(const u32x4*)(row + (g * KS + s) * 16) : u32x4{0, 0, 0, 0};
#pragma unroll
    for (int t = 0; t < E; ++t) o[t] = f32x4{0, 0, 0, 0};
    m = -INFINITY, l = 0.f;
  }
  // fp16 queries as the sum of two bf16 operands
  __device__ __forceinline__ void split_queries() {
    if constexpr (QLO) {
#pragma unroll
      for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float x = ds2_low16<true>(q[s][j]), y = ds2_high16<true>(q[s][j]);
          const unsigned hi = ds2_pack16<false>(x, y), lo = ds2_pack16<false>(x - ds2_low16<false>(hi), y - ds2_high16<false>(hi));
          q[s][j] = hi, ql[s][j] = lo & ~ds2_not_finite16<false>(lo);     // (an infinite query has no remainder: inf - inf would be NaN)
        }
    }
  }

  // 32 keys to the wave's LDS (rows behind the end: whatever is there, their scores are replaced) and their scales to registers
  // (`stride` and `scale_stride` pass through an empty asm statement: offsets made from them are an addition a load, not two dozen
  // registers kept through the loop)
  __device__ __forceinline__ void load_keys(const CacheRows& c, int blk, int k1, unsigned char* lds, int lane) {
    unsigned stride = c.k_c, scale_stride = c.ks_c;
    asm volatile("" : "+s"(stride), "+s"(scale_stride));
    const __amdgpu_buffer_rsrc_t r = ds2_rows(c.k, blk, c.k_c, k1 - blk, ROW);
#pragma unroll
    for (int n = 0; n < ISSUES; ++n) {
      const int p = n * 64 + lane, row = p / PIECES;
      const unsigned at = PIECES * 32 % 64 && p >= PIECES * 32 ? 0x80000000u : row * stride + mixed(row, p - row * PIECES) * 16;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)(lds + n * 1024), 16, at, 0, 0, 0);
    }
    if constexpr (QUANT) {
      const int i = lane & 15, g = lane >> 4;
      const __amdgpu_buffer_rsrc_t rs = ds2_rows(c.ks, blk, c.ks_c, k1 - blk, KS);
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int x = 0; x < SG; ++x)
          kscale[t][x] = __builtin_amdgcn_raw_buffer_load_b8(rs, (16 * t + i) * scale_stride + ((KS == 3 ? g * 3 + x : g * KS + 4 * x) >> 2), 0, 0);
    }
  }
  // Loads to LDS are not followed by hipcc: the reads wait for them here.  Loads return in order and the block's value loads were asked
  // for after its keys, so at most they may be outstanding.
  __device__ __forceinline__ void wait_keys() {
    constexpr int LATER = 8 * (QUANT ? 2 : 1);
    static_assert(VB <= 16, "one load a value row");
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(LATER) : "memory");
  }
  // slices of key 16 t + i from the wave's LDS
  __device__ __forceinline__ void read_keys(unsigned (&w)[KS * SW], const unsigned char* lds, int t, int i, int g) {
    const unsigned char* row = lds + (16 * t + i) * ROW;
    if constexpr (KS * SB % 16 == 0) {
#pragma unroll
      for (int x = 0; x < KS * SB / 16; ++x) {
        const u32x4 y = *(const u32x4*)(row + mixed(i, g * (KS * SB / 16) + x) * 16);
#pragma unroll
        for (int j = 0; j < 4; ++j) w[4 * x + j] = y[j];
      }
    } else {
#pragma unroll
      for (int s = 0; s < KS * SW; ++s) w[s] = *(const unsigned*)(row + g * KS * SB + 4 * s);
    }
  }
  __device__ __forceinline__ void load_values(const CacheRows& c, int blk, int k1, unsigned v_lane, unsigned vs_lane, int g) {
    unsigned stride = c.v_c, scale_stride = c.vs_c;
    asm volatile("" : "+s"(stride), "+s"(scale_stride));
    const __amdgpu_buffer_rsrc_t r = ds2_rows(c.v, blk, c.v_c, k1 - blk, ROW);
    const __amdgpu_buffer_rsrc_t rs = ds2_rows(c.vs, blk, c.vs_c, k1 - blk, KS);
    const unsigned first = 4 * g * stride + v_lane, scale_first = 4 * g * scale_stride + vs_lane;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const unsigned row = (j < 4 ? 0 : 12) + j;           // + 4 g
      ds2_load_bytes<VB>(vw[j], r, first + row * stride);
      if constexpr (QUANT) vscale[j] = __builtin_amdgcn_raw_buffer_load_b8(rs, scale_first + row * scale_stride, 0, 0);
    }
  }

  // Blocks first, first + step, ... of the keys [k0, k1); every key below `common` is seen by all rows; vh: the wave's part of the values
  __device__ __forceinline__ void run(const CacheAttnArgs& a, const CacheRows& c, int k0, int k1, int first, int step, int common, int vh,
                                      unsigned char* lds, int lane) {
    const int i = lane & 15, g = lane >> 4;
    const int d0 = (vh * 16 + i) * E;                      // the lane's first value element
    const bool none = !FULL && d0 >= D;                    // lanes beyond the head dimension load zeros
    const unsigned v_lane = none ? 0x80000000u : d0 / E * VB, vs_lane = none ? 0x80000000u : (unsigned)d0 >> 5;
    const float sc = a.scale * DS2_LOG2E, cap2 = a.cap * DS2_LOG2E;
    const float in_cap = a.cap > 0.f ? 2.f * DS2_LOG2E * a.scale / a.cap : 0.f;
    int blk = k0 + first * 32;
    if (blk >= k1) return;
    load_keys(c, blk, k1, lds, lane);
    asm volatile("" ::: "memory");                         // (keys before values: wait_keys counts on it)
    load_values(c, blk, k1, v_lane, vs_lane, g);
    split_queries();                                       // (after the loads have been asked for)
    for (; blk < k1; blk += step * 32) {
      const int next = blk + step * 32;
      // ---- scores
      wait_keys();
      float p[8];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        unsigned w[KS * SW];
        read_keys(w, lds, t, i, g);
        f32x4 x = {0, 0, 0, 0};
#pragma unroll
        for (int s = 0; s < KS; ++s) {
          u32x4 kf;
          if constexpr (QUANT) kf = ds2_decode8<FORMAT>(w + s * SW, ds2_operand_scale(kscale[t][KS == 3 ? s : s / 4]));
          else kf = u32x4{w[4 * s], w[4 * s + 1], w[4 * s + 2], w[4 * s + 3]};
          x = ds2_mfma16<F16>(kf, q[s], x);
          if constexpr (QLO) x = ds2_mfma16<F16>(kf, ql[s], x);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) p[4 * t + j] = x[j];
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // the block has left LDS: the next one may come
      load_keys(c, next, k1, lds, lane);                   // (behind the end: no traffic)
      asm volatile("" ::: "memory");
      // ---- weights
      const bool edge = blk + 32 > common;                 // some row may not see all of the block's keys (uniform)
      if (a.cap > DS2_CAP_WIDE) {
#pragma unroll
        for (int j = 0; j < 8; ++j) p[j] = ds2_capped_wide(p[j], in_cap, cap2, sc);
      } else if (a.cap > 0.f) {
#pragma unroll
        for (int j = 0; j < 8; ++j) p[j] = ds2_capped(p[j], in_cap, cap2);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) p[j] *= sc;
      }
      if (a.slopes) {
#pragma unroll
        for (int j = 0; j < 8; ++j) p[j] -= slope * (float)(pos - (blk + (j < 4 ? 0 : 12) + 4 * g + j));
      }
      if (edge) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (blk + (j < 4 ? 0 : 12) + 4 * g + j >= sees) p[j] = -INFINITY;
      }
      float top = fmaxf(fmaxf(fmaxf(p[0], p[1]), fmaxf(p[2], p[3])), fmaxf(fmaxf(p[4], p[5]), fmaxf(p[6], p[7])));
      if (__any(top - fmaxf(m, -3e38f) > DS2_LIMIT<F16>)) {
        top = fmaxf(top, __shfl_xor(top, 16));
        top = fmaxf(top, __shfl_xor(top, 32));
        float mn = fmaxf(m, top - DS2_SHIFT<F16>);
        if (top - mn > DS2_LIMIT<F16>) mn = top;           // (scores so large that fp32 does not hold the difference)
        const float al = m == mn ? 1.f : __builtin_amdgcn_exp2f(m - mn);
        l *= al;
#pragma unroll
        for (int t = 0; t < E; ++t) o[t] *= al;
        m = mn;
      }
      const float ref = fmaxf(m, -3e38f);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        p[j] = __builtin_amdgcn_exp2f(p[j] - ref);
        l += p[j];
      }
      // ---- values: as 16-bit rows, then turned around
      unsigned vv[8][E < 8 && QUANT ? 4 : E / 2];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if constexpr (QUANT) {
          const float f = ds2_operand_scale(vscale[j]);
          unsigned w[2] = {vw[j][0], VW > 1 ? vw[j][VW - 1] : 0u};
          const u32x4 r = ds2_decode8<FORMAT>(w, f);
#pragma unroll
          for (int y = 0; y < 4; ++y) vv[j][y] = r[y];
        } else {
#pragma unroll
          for (int x = 0; x < E / 2; ++x) vv[j][x] = vw[j][x];
        }
      }
      // A key that a row does not see has weight 0, but 0 times an infinity or a NaN is not 0.  Where rows of the block may see
      // different keys, values that are not finite leave the product and go to the rows that do see them, one by one.
      if (edge) {
        unsigned bad = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
          for (int x = 0; x < E / 2; ++x) bad |= ds2_not_finite16<F16>(vv[j][x]);
        if (__any(bad != 0)) {
#pragma unroll
          for (int j = 0; j < 8; ++j)
#pragma unroll
            for (int x = 0; x < E / 2; ++x) vv[j][x] &= ~ds2_not_finite16<F16>(vv[j][x]);
          add_apart(a, p, c, blk, k1, i, g, vh);
        }
      }
      u32x4 ph, pl;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        ph[j] = ds2_pack16<F16>(p[2 * j], p[2 * j + 1]);
        if constexpr (PLO) pl[j] = ds2_pack16<F16>(p[2 * j] - ds2_low16<F16>(ph[j]), p[2 * j + 1] - ds2_high16<F16>(ph[j]));
      }
#pragma unroll
      for (int t = 0; t < E; ++t) {
        u32x4 vf;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          vf[j] = __builtin_amdgcn_perm(vv[2 * j + 1][t >> 1], vv[2 * j][t >> 1], (t & 1) ? 0x07060302u : 0x05040100u);
        o[t] = ds2_mfma16<F16>(vf, ph, o[t]);
        if constexpr (PLO) o[t] = ds2_mfma16<F16>(vf, pl, o[t]);
      }
      load_values(c, next, k1, v_lane, vs_lane, g);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");       // (nothing of this wave reaches LDS later)
  }

  // the values of a block that are not finite, to the rows that see their keys (rare: speed does not matter)
  __device__ __forceinline__ void add_apart(const CacheAttnArgs& a, const float (&p)[8], const CacheRows& c, int blk, int k1, int i, int g,
                                            int vh) {
#pragma unroll 1
    for (int key = 0; key < 32; ++key) {
      if (blk + key >= k1) break;
      const int j = (key & 3) | (key >> 4) << 2, from = (key >> 2) & 3;
      float mine = p[0];
#pragma unroll
      for (int x = 1; x < 8; ++x) mine = j == x ? p[x] : mine;
      const float w = __shfl(mine, i | from << 4);
      if (blk + key >= sees) continue;
      const uint8_t *row = c.v + (int64_t)(blk + key) * c.v_c, *row_scale = c.vs + (int64_t)(blk + key) * c.vs_c;
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int t = 0; t < E; ++t) {
          const int d = (vh * 16 + 4 * g + r) * E + t;
          if (!FULL && d >= D) continue;
          float x;
          if constexpr (FORMAT == DS2_CACHE_PLAIN) x = ds2_low16<F16>(*(const uint16_t*)(row + 2 * d));
          else {
            const unsigned code[2] = {FORMAT == DS2_CACHE_MXFP8 ? row[d] : (unsigned)row[d >> 1] >> 4 * (d & 1), 0u};
            x = ds2_low16<false>(ds2_decode8<FORMAT>(code, ds2_operand_scale(row_scale[d >> 5]))[0]);
          }
          o[t][r] += __builtin_isfinite(x) ? 0.f : w * x;
          asm volatile("" ::: "memory");                   // (one at a time: this path must not widen the kernel's registers)
          __builtin_amdgcn_sched_barrier(0);
        }
    }
  }
};

constexpr int cache_value_split(int D) { return D > 128 ? 2 : 1; }
// rows of a workgroup: its waves share 16 rows and split the keys, or each holds 16 rows of its own over the same keys
constexpr int cache_rows(int D, bool by_rows) { return by_rows ? 4 / cache_value_split(D) * 16 : 16; }

// workgroups (and waves a SIMD) that a CU holds, by registers; the shares of the keys are as many as fit the chip
constexpr int cache_residents(int D) { return D > 128 ? 2 : D > 64 ? 3 : 4; }

template <int FORMAT, bool QF16, int KS, int E, int VS>
__global__ __launch_bounds__(256, cache_residents(32 * KS)) void k_cache_attn(CacheAttnArgs a) {
  ds2_ask_args(a);
  typedef CacheStream<FORMAT, QF16, KS, E, VS> Stream;
  constexpr bool FULL = Stream::FULL;
  constexpr int KW = 4 / VS;                               // waves of a workgroup that share its keys (or hold different rows)
  typedef float Joined[E * 4 + 2][64];                     // what a wave hands over, by lane
  __shared__ __attribute__((aligned(16))) unsigned char lds[std::max((int)sizeof(Joined) * (KW - 1) * VS, 4 * Stream::LDS)];
  Joined* const join = (Joined*)lds;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int kw = wave % KW, vh = wave / KW;
  const int i = lane & 15, g = lane >> 4;
  const bool prefix = (int)blockIdx.x < a.pre_blocks;
  const bool by_rows = prefix ? a.pre_by_rows : a.by_rows;

  // ---- the share: [at, end) of the units of all streams, or one stream, or prefix keys
  const int heads = a.Hkv * a.own_groups;                  // streams of a sequence
  int part = 0, head = 0, group = 0, b = 0, at = 0, end = 1, base = 0, units = 1;
  const int share = blockIdx.x - a.pre_blocks;
  const int len0 = lane < a.B ? max(0, min(a.lens[lane], a.C)) : 0;        // of the first 64 sequences, kept
  auto len_of = [&](int x) { return x < 64 ? __builtin_amdgcn_readlane(len0, x) : max(0, min(a.lens[x], a.C)); };
  auto units_of = [&](int n) { return n ? (n + CACHE_UNIT - 1) / CACHE_UNIT + 1 : 0; };                  // one for the stream's beginning
  if (prefix) {                                            // row groups over the same keys are far apart in id: same chiplet, one L2
    int id = blockIdx.x;
    group = id / (a.Hkv * a.pre_parts), id -= group * a.Hkv * a.pre_parts;
    part = id / a.Hkv, head = id - part * a.Hkv;
  } else if (a.shares == 0) {
    b = share / heads;
  } else {
    int sum = units_of(len0);
    for (int x = lane + 64; x < a.B; x += 64) sum += units_of(max(0, min(a.lens[x], a.C)));
#pragma unroll 1
    for (int s = 1; s < 64 && s < a.B; s <<= 1) sum += __shfl_xor(sum, s);           // (lanes from B on hold zeros)
    const int total = __builtin_amdgcn_readfirstlane(sum) * heads, each = max(1, (total + a.shares - 1) / a.shares);
    at = share * each, end = min(total, at + each);
    if (at >= end) return;
    for (int b0 = 0;; b0 += 64) {                          // the sequence in which the share begins
      int x = (b0 == 0 ? units_of(len0) : b0 + lane < a.B ? units_of(max(0, min(a.lens[b0 + lane], a.C))) : 0) * heads;
      const int mine = x;
#pragma unroll 1
      for (int s = 1; s < 64 && s < a.B; s <<= 1) {
        const int y = __shfl_up(x, s);
        x += lane >= s ? y : 0;
      }
      const unsigned long long past = __ballot(base + x > at);
      if (past) {
        const int w = __builtin_ctzll(past);
        b = b0 + w;
        base += __builtin_amdgcn_readlane(x, w) - __builtin_amdgcn_readlane(mine, w);
        units = __builtin_amdgcn_readlane(mine, w) / heads;
        break;
      }
      base += __builtin_amdgcn_readlane(x, 63);
    }
  }

  while (true) {                                           // ---- one segment: the part of the share that lies in one stream
    int len, k0, k1, hg = 0, n = 0;
    bool last = false;                                     // ... and ends it
    if (prefix) {
      len = a.P, k0 = part * a.pre_chunk, k1 = min(len, k0 + a.pre_chunk);
    } else {
      len = len_of(b);
      if (a.shares == 0) hg = share - b * heads, k0 = 0, k1 = len;
      else {
        hg = (at - base) / units;
        const int from = at - base - hg * units;
        n = min(end - at, units - from), last = from + n == units;
        k0 = max(0, from - 1) * CACHE_UNIT, k1 = min(len, (from + n - 1) * CACHE_UNIT);
      }
      head = hg / a.own_groups, group = hg - head * a.own_groups;
    }
    if (k0 < k1 || a.shares == 0) {                        // (a share may end with a stream's beginning: the next one counts as its first)
      const int rows = prefix ? a.B * a.T * a.G : a.T * a.G;
      const int own_row = (by_rows ? kw * 16 : 0) + i;     // the lane's row in the workgroup's
      const int r = group * (by_rows ? KW * 16 : 16) + own_row;
      const bool live = r < rows;
      const int rr = live ? r : 0, rb = prefix ? rr / (a.T * a.G) : b, tg = prefix ? rr - rb * a.T * a.G : rr;
      const int t = tg / a.G, hq = head * a.G + (tg - t * a.G);
      const int own = (prefix ? max(0, min(a.lens[rb], a.C)) : len) - a.T + t;        // position in the sequence's own keys
      const int row_id = (rb * a.T + t) * a.Hq + hq;
      Stream st;
      st.pos = own + (prefix ? a.P : 0);
      st.sees = prefix ? a.P : max(0, own + 1);
      st.slope = a.slopes ? a.slopes[hq] * DS2_LOG2E : 0.f;
      st.start(a.q + rb * a.q_b + t * a.q_t + hq * a.q_h, live, g);
      const CacheRows c = prefix ? CacheRows{a.pk + head * a.pk_h, a.pv + head * a.pv_h, a.pks + head * a.pks_h, a.pvs + head * a.pvs_h, a.pk_c, a.pv_c, a.pks_c, a.pvs_c}
                                 : CacheRows{a.k + b * a.k_b + head * a.k_h, a.v + b * a.v_b + head * a.v_h, a.ks + b * a.ks_b + head * a.ks_h,
                                             a.vs + b * a.vs_b + head * a.vs_h, a.k_c, a.v_c, a.ks_c, a.vs_c};
      if (r - i < rows)                                    // (a wave without rows only keeps the barriers)
        st.run(a, c, k0, k1, by_rows ? 0 : kw, by_rows ? 1 : KW, prefix ? a.P : len - a.T + 1, vh, lds + wave * Stream::LDS, lane);

      if (!by_rows) {                                      // join the waves' keys: the same rows in the same lanes
        __syncthreads();                                   // (the waves are through with their keys)
        if (kw) {
          Joined& to = join[(kw - 1) * VS + vh];
#pragma unroll
          for (int t = 0; t < E; ++t)
#pragma unroll
            for (int j = 0; j < 4; ++j) to[t * 4 + j][lane] = st.o[t][j];
          to[E * 4][lane] = st.m, to[E * 4 + 1][lane] = st.l;
        }
        __syncthreads();
        if (kw == 0) {
          float mm = st.m, f[KW - 1];
#pragma unroll
          for (int w = 0; w < KW - 1; ++w) mm = fmaxf(mm, join[w * VS + vh][E * 4][lane]);
          const float f0 = st.m == mm ? 1.f : __builtin_amdgcn_exp2f(st.m - mm);      // (equal also covers -inf and -inf)
          st.l *= f0;
#pragma unroll
          for (int w = 0; w < KW - 1; ++w) {
            const float mw = join[w * VS + vh][E * 4][lane];
            f[w] = mw == mm ? 1.f : __builtin_amdgcn_exp2f(mw - mm);
            st.l += f[w] * join[w * VS + vh][E * 4 + 1][lane];
          }
          st.m = mm;
#pragma unroll
          for (int t = 0; t < E; ++t)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              float x = st.o[t][j] * f0;
#pragma unroll
              for (int w = 0; w < KW - 1; ++w) x += f[w] * join[w * VS + vh][t * 4 + j][lane];
              st.o[t][j] = x;
            }
        }
      }
      if (by_rows || kw == 0) {
        const int stream = b * heads + hg;
        if (!prefix && a.shares && wave == 0 && lane == 0) {
          if (k0 == 0) a.seg_of[stream].x = share;
          if (last) a.seg_of[stream].y = share;
        }
        float l = st.l;
        l += __shfl_xor(l, 16);
        l += __shfl_xor(l, 32);
        if (live && (prefix || !a.direct)) {
          const int64_t to = prefix ? (int64_t)part * a.B * a.T * a.Hq + row_id : (int64_t)((a.shares ? share : 0) + stream) * a.own_rows + own_row;
          if (g == 0 && vh == 0) (prefix ? a.pre_ml : a.seg_ml)[to] = f32x2_t{st.m, l};
          float* out = (prefix ? a.pre_o : a.seg_o) + to * Stream::D;
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int d = (vh * 16 + 4 * g + r) * E;
            if (!FULL && d >= Stream::D) break;
            if constexpr (E >= 4) {
#pragma unroll
              for (int t = 0; t < E; t += 4) *(f32x4*)(out + d + t) = f32x4{st.o[t][r], st.o[t + 1][r], st.o[t + 2][r], st.o[t + 3][r]};
            } else *(f32x2_t*)(out + d) = f32x2_t{st.o[0][r], st.o[1][r]};
          }
        } else if (live) {
          const bool none = st.m == -INFINITY && l == 0.f;  // nothing seen: zeros
          const float f = none ? 0.f : 1.f / l;
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int d = (vh * 16 + 4 * g + r) * E;
            if (!FULL && d >= Stream::D) break;
            unsigned* to = (unsigned*)(a.out + ((int64_t)row_id * Stream::D + d) * 2);
#pragma unroll
            for (int t = 0; t < E; t += 2) to[t >> 1] = none ? 0u : ds2_pack16<QF16>(st.o[t][r] * f, st.o[t + 1][r] * f);
          }
        }
      }
    }
    if (prefix || a.shares == 0) break;
    at += n;
    if (at >= end) break;
    if (!by_rows) __syncthreads();                         // (what the waves handed over has been read)
    while (at >= base + units * heads) {                   // the next sequence that holds tokens
      base += units * heads;
      units = units_of(len_of(++b));
    }
  }
}

int launch_cache_attn_plain(const CacheAttnArgs& a, bool f16, unsigned blocks, hipStream_t st);
int launch_cache_attn_mxfp8(const CacheAttnArgs& a, bool f16, unsigned blocks, hipStream_t st);
int launch_cache_attn_mxfp4(const CacheAttnArgs& a, bool f16, unsigned blocks, hipStream_t st);

template <int FORMAT, bool QF16>
int launch_cache_attn_of(const CacheAttnArgs& a, unsigned blocks, hipStream_t st) {
  if (a.D == 32) k_cache_attn<FORMAT, QF16, 1, 2, 1><<<dim3(blocks), 256, 0, st>>>(a);
  else if (a.D == 64) k_cache_attn<FORMAT, QF16, 2, 4, 1><<<dim3(blocks), 256, 0, st>>>(a);
  else if (a.D == 96) k_cache_attn<FORMAT, QF16, 3, 8, 1><<<dim3(blocks), 256, 0, st>>>(a);
  else if (a.D == 128) k_cache_attn<FORMAT, QF16, 4, 8, 1><<<dim3(blocks), 256, 0, st>>>(a);
  else k_cache_attn<FORMAT, QF16, 8, 8, 2><<<dim3(blocks), 256, 0, st>>>(a);
  DS2_CHECK_LAUNCH();
  return DS2_OK;
}
