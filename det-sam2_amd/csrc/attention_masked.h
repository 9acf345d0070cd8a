// Masked attention of whole prompts, 16-bit operands, fp32 statistics (kernel templates; instantiated per type in
// attention_masked_{bf16,f16}.hip):
//
//   o_r = sum_j w_rj v_j / sum_j w_rj,  w_rj = exp(s_rj) where row r sees key j, else 0
//   s = scale q.k, then cap tanh(s / cap), then - slope_h |pos_r - j|
//
// One pass with a running maximum and sum.  The rows of a key head are its G Lq (query head, position) pairs, position-major, so that
// the G heads of a group share every key tile and a tile of rows spans few positions (few edge tiles under the causal mask).
//
//  * A wave holds 32 rows: S^T = K Q^T with v_mfma_f32_32x32x16 (A = K from LDS, B = Q in registers) leaves a row's scores in one lane
//    pair, so maximum and sum cost one exchange.  P^T is the B operand of O^T = V^T P^T straight from the score registers: contraction
//    slots are free to be permuted, slot j of lane half h is key 8 (j / 4) + 4 h + j % 4 of a block of 16; the A operand
//    follows with two transposing LDS reads (ds_read_b64_tr_b16: 4 keys of one column a lane).
//  * Steps of 32 keys, software pipelined: the score products of step i + 1 are issued among the exponentials of step i, the value
//    products of step i among the scaling (tanh, distance) of step i + 1, so that matrix and vector pipe both have work from one wave.
//  * Key tiles (64 keys; 32 at head dims over 128) go through registers into one of THREE LDS buffers: loads fly for two tiles, one
//    barrier a tile.  Rows behind the last key come as zeros from the buffer descriptor's bounds.  K rows are padded by 16 bytes (16 rows
//    of a ds_read_b128 quarter cover all 64 banks), V rows to 64 bytes modulo 256 (the four rows of a transposing read do).
//  * causal, prefix and length masks are one number a row: the keys it sees are those below `limit`.  Tiles beyond every row's limit are
//    not visited, steps below every row's limit are not masked.  Documents: a small kernel notes the smallest and largest document of
//    each key tile; a wave-wide vote over 64 tiles at a time finds the tiles that can hold a visible pair.
//  * The running reference of a row is raised only when a weight would exceed a fixed power of 2 (DS2_LIMIT): the weights stay bounded and the
//    rescaling of O is rare.
//  * Where 256 rows a workgroup would leave CUs idle or unevenly loaded, the eight waves hold 128 rows twice (KG = 2): each takes every
//    other step of the tiles, and the two halves are joined through LDS at the end (attention_masked.hip has the rule).
//  * Weights are rounded to the operands' 16-bit type before the value product, while their sum takes them as they are: half a step of each term
//    w |v|, like the output's own rounding (fp16: down to 2^-25 of the row's largest weight; DS2_SHIFT).  Two bf16 operands (WIDE) leave 2^-16 and
//    take up to a fifth more time (8 key heads, 2048 rows a head behind 8192 tokens: D = 64 69 -> 84 us, D = 128 105 -> 127).  A prefix that
//    sequences share has them, as their own tokens do; whole prompts have one.
//
// Measured (fp16 / bf16 operands, normal values, TFLOP/s over the visible pairs): D = 128, 32 over 8 heads, 8192 tokens: full 962 / 1014, causal 928 /
// 974, capped 817 / 851, distance bias 871 / 900; a plain library product of such matrices makes 1035 / 1096 on the same card.  D = 64, 16 heads, 8190
// tokens: 865 / 902, causal 671 / 690, bias 702 / 739; D = 256, 8 over 2 heads, 4096 tokens: 592 / 619 (both waves of a row compute its scores: three
// units of matrix work in place of two).  At D = 128 the matrix pipes are busy 44 % of the cycles, the vector pipe 39 %, LDS 27 %; other orders
// of a step, priorities, and halves of the workgroup in opposite phases all took the same time or more.  At D = 64 the exponentials (a quarter of the
// vector rate) carry more weight: vector pipe 67 %, matrix pipes 41 %.
#pragma once
#include "token_cache.h"

namespace {

typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4_t* lds_s16x4;

// Over 128 output elements a row, two waves take half of them each and both compute the scores: 128 accumulators and 64 query
// registers a wave leave no room for the pipeline.
constexpr int masked_value_split(int D) { return D > 128 ? 2 : 1; }
// rows of a workgroup
constexpr int masked_rows(int D, int key_groups) { return 256 / masked_value_split(D) / key_groups; }
constexpr int masked_tile(int D) { return D > 128 ? 32 : 64; }   // keys of a tile
constexpr float LOG2E = 1.44269504088896340736f;
// How scores become exponents.  LINEAR: distance bias without a cap, by what the products start from; GENERAL: cap and bias, or a scale
// or cap that the others do not take.  (D = 64, 16 heads, 8190 tokens, fp16 / bf16 TFLOP/s: with a bias GENERAL 634 / 666, LINEAR 679 /
// 736; without GENERAL 725 / 754, PLAIN 833 / 881; capped GENERAL with a bias 490 / 503, CAP without 619 / 633.)
enum { MASKED_PLAIN = 0, MASKED_CAP = 1, MASKED_LINEAR = 2, MASKED_GENERAL = 3 };

}  // namespace

struct MaskedArgs {
  const char *q, *k, *v;
  char* out;
  int64_t q_b, q_t, q_h, k_b, k_t, k_h, v_b, v_t, v_h;    // bytes
  const float* slopes;
  const int32_t *lens, *q_start, *prefix, *q_doc, *k_doc;
  const int32_t* row_lens;                  // rows of sequences behind a shared prefix of Lk keys (cache_attention.hip): position i is token i % row_T
  int row_T, row_C;                         // of sequence i / row_T (B is 1) and stands at Lk + row_lens[sequence] - row_T + token, row_lens at
                                            // most row_C; null: at q_start + i
  const int2* tile_docs;                    // [B][tiles]: smallest (-1: a key of none among them) and largest document of a tile
  int B, Lq, Lk, Hq, Hkv, G, D, causal;
  float scale, cap;
  int key_groups;                           // waves that share rows and take every other step (masked_rows)
  int row_tiles, heads, parts, tiles, tiles_a_part, fold;
  float* part_o;                            // null: one part
  f32x2_t* part_ml;
};

static inline int masked_mode(float scale, float cap, const float* slopes) {
  if (cap > 0.f) return slopes || cap > DS2_CAP_WIDE ? MASKED_GENERAL : MASKED_CAP;
  if (!(scale >= 0x1p-60f)) return MASKED_GENERAL;               // (PLAIN needs a positive scale, LINEAR divides by it)
  return slopes ? MASKED_LINEAR : MASKED_PLAIN;
}
int launch_masked_bf16(const MaskedArgs& a, int mode, unsigned blocks, hipStream_t st);
int launch_masked_f16(const MaskedArgs& a, int mode, unsigned blocks, hipStream_t st);
int launch_masked_bf16_wide(const MaskedArgs& a, int mode, unsigned blocks, hipStream_t st);        // weights as two operands, one key group

namespace {

template <bool F16>
__device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
  if constexpr (F16) return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}
// 16-bit pair: which halves are infinities or NaNs, as a mask over the word
template <bool F16>
__device__ __forceinline__ unsigned not_finite(unsigned w) {
  constexpr unsigned EXP = F16 ? 0x7c00u : 0x7f80u;
  return ((w & EXP) == EXP ? 0xffffu : 0u) | (((w >> 16) & EXP) == EXP ? 0xffff0000u : 0u);
}

// The register limit keeps accumulators out of the AGPRs.  With them, and a divergent branch in the tile loop, hipcc placed copies into
// AGPRs in front of the restored lane mask; the loop below has wave-uniform branches only.
template <bool F16, int DP, int MODE, int KG, bool WIDE>
__global__ __launch_bounds__(512, DP > 64 ? 2 : 4) void k_attn_masked(MaskedArgs a) {
  ds2_ask_args(a);
  constexpr int NW = 8;                                          // waves (those without rows of their own stage keys for the others)
  constexpr int KT = masked_tile(DP), H = KT / 32, ST = H / KG;  // steps of a tile, a wave's
  constexpr int VS = masked_value_split(DP), RW = NW / VS / KG;  // waves that share rows (each takes 1 / VS of the output or 1 / KG of the keys), waves of other rows
  static_assert(KG == 1 || (VS == 1 && H == 2));
  constexpr bool BIAS = MODE >= MASKED_LINEAR;
  constexpr int KS = DP / 16, DB = DP / 32 / VS;                 // contraction steps of a score, a wave's blocks of 32 output elements
  constexpr int KROW = DP * 2 + 16, VROW = DP == 32 ? 64 : DP == 64 ? 192 : DP == 96 ? 192 : DP == 128 ? 320 : 576;
  constexpr int CH = DP / 8;                                     // 16-byte pieces of a row
  constexpr int NT = NW * 64, PER = (KT * CH + NT - 1) / NT;     // pieces a thread stages of a K (and of a V) tile
  constexpr int KBUF = KT * KROW + 16, VBUF = KT * VROW + 16;    // (+ 16: where threads without a piece write)
  typedef float Joined[DB * 16 + 2][64];                         // what a wave of the second key group hands over, by lane
  static_assert(KG == 1 || RW * sizeof(Joined) <= 3 * (KBUF + VBUF));
  __shared__ __attribute__((aligned(16))) unsigned char lds[3 * (KBUF + VBUF)];
  unsigned char(*const lk)[KBUF] = (unsigned char(*)[KBUF])lds;
  unsigned char(*const lv)[VBUF] = (unsigned char(*)[VBUF])(lds + 3 * KBUF);
  __shared__ int ldoc[3][64];
  __shared__ int wg_lim[NW][4];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 31, h = lane >> 5;

  // ---- which tile: the heads of a batch are spread over the chiplets (blockIdx % 8); row tiles in descending order, the longest
  // of a causal mask first.  (fold: all workgroups are resident at once, two a CU; the second half ascends, so that a long and a
  // short one meet.)
  int id = blockIdx.x, part = 0, head, rt;
  {
    const int nh = a.heads, total = nh * a.parts;
    if (nh % 8 == 0) {
      const int x = id & 7, y = id >> 3, per = total / 8;
      const int z = y % per;
      rt = y / per;
      head = x * (nh / 8) + z / a.parts, part = z % a.parts;
    } else {
      rt = id / total;
      const int z = id % total;
      head = z / a.parts, part = z % a.parts;
    }
    rt = a.fold && rt >= (a.row_tiles + 1) / 2 ? rt - (a.row_tiles + 1) / 2 : a.row_tiles - 1 - rt;
  }
  const int b = head / a.Hkv, kvh = head - b * a.Hkv;
  const int rows = a.G * a.Lq;
  const int row0 = rt * RW * 32 + wave % RW * 32;                // the wave's rows of this key head
  const int d0 = VS > 1 ? wave / RW * DB * 32 : 0;               // its first output element
  const int kg = KG > 1 ? wave / RW : 0;                         // its first step of a tile
  const int r = min(row0 + c, rows - 1);                         // rows behind the last repeat it and are not written
  const int i = r / a.G, hq = kvh * a.G + (r - i * a.G);
  const int len = a.lens ? max(0, min(a.lens[b], a.Lk)) : a.Lk;
  const int start = a.q_start ? max(-(1 << 30), min(a.q_start[b], 1 << 30)) : 0;
  int pos = start + i;
  int seq = b, token = i;
  if (a.row_lens) seq = i / a.row_T, token = i - seq * a.row_T;
  if (BIAS && a.row_lens) pos = a.Lk + max(0, min(a.row_lens[seq], a.row_C)) - a.row_T + token;
  float slope = BIAS && a.slopes ? a.slopes[hq] * LOG2E : 0.f;
  int limit = len;
  if (a.causal) {
    int n = pos + 1;
    if (a.prefix) n = max(n, a.prefix[b]);
    limit = max(0, min(len, n));
  }
  // A row before the first key or behind the last has part of every distance in common, which is no part of a softmax: for the bias it stands
  // at that key, so that no exponent is a small difference of large ones.  (At 10^6 behind the keys with a slope of 1/2 exponents have steps of 1/16.)
  // Rows behind a shared prefix keep their places: their parts are joined with those of their own keys.
  if (BIAS && !a.row_lens) pos = max(0, min(pos, len - 1));
  int qdoc = a.q_doc ? a.q_doc[(int64_t)b * a.Lq + i] : 0;
  qdoc = qdoc < 0 ? -2 : qdoc;                                   // of no document: equal to no key's (a key of none is -1 in LDS)

  // ---- queries
  u32x4 qf[KS];
  {
    const char* row = a.q + seq * a.q_b + (int64_t)token * a.q_t + hq * a.q_h;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int d = 16 * s + 8 * h;
      qf[s] = d < a.D ? *(const u32x4*)(row + d * 2) : u32x4{0, 0, 0, 0};
    }
  }

  // ---- staging
  const int2* td = a.tile_docs ? a.tile_docs + (int64_t)b * a.tiles : nullptr;
  const char *kb = a.k + b * a.k_b + kvh * a.k_h, *vb = a.v + b * a.v_b + kvh * a.v_h;
  unsigned k_off[PER], v_off[PER];                               // of the thread's pieces in a tile; beyond any bound where there are none
  int lds_k[PER], lds_v[PER];
#pragma unroll
  for (int u = 0; u < PER; ++u) {
    const int p = u * NT + tid, row = p / CH, piece = p - row * CH;
    const bool place = PER * NT == KT * CH || row < KT, live = place && piece * 8 < a.D;
    k_off[u] = live ? (unsigned)(row * (int)a.k_t + piece * 16) : 0x80000000u;
    v_off[u] = live ? (unsigned)(row * (int)a.v_t + piece * 16) : 0x80000000u;
    lds_k[u] = place ? row * KROW + piece * 16 : KT * KROW, lds_v[u] = place ? row * VROW + piece * 16 : KT * VROW;
  }
  struct Tile {
    u32x4 k[PER], v[PER];
    int doc, left;                                               // left: keys from the tile's first one on
  };
  Tile tile, second;
  auto fetch = [&](Tile& to, int t) {                            // a tile into registers; behind the last key: zeros
    const int left = len - t * KT;                               // > 0
    const int64_t kn = (int64_t)(min(left, KT) - 1) * a.k_t + a.D * 2, vn = (int64_t)(min(left, KT) - 1) * a.v_t + a.D * 2;
    const __amdgpu_buffer_rsrc_t kr = __builtin_amdgcn_make_buffer_rsrc((void*)(kb + (int64_t)t * KT * a.k_t), 0, (int)kn, 0x00020000);
    const __amdgpu_buffer_rsrc_t vr = __builtin_amdgcn_make_buffer_rsrc((void*)(vb + (int64_t)t * KT * a.v_t), 0, (int)vn, 0x00020000);
#pragma unroll
    for (int u = 0; u < PER; ++u) {
      to.k[u] = __builtin_amdgcn_raw_buffer_load_b128(kr, k_off[u], 0, 0);
      to.v[u] = __builtin_amdgcn_raw_buffer_load_b128(vr, v_off[u], 0, 0);
    }
    if (td) {                                                    // (every wave fetches and writes all of the tile's documents: no divergent branch)
      const __amdgpu_buffer_rsrc_t dr = __builtin_amdgcn_make_buffer_rsrc((void*)(a.k_doc + (int64_t)b * a.Lk + t * KT), 0, min(left, KT) * 4, 0x00020000);
      to.doc = __builtin_amdgcn_raw_buffer_load_b32(dr, lane * 4, 0, 0);
      to.left = left;
    }
  };
  auto stage = [&](const Tile& from, int buf) {
#pragma unroll
    for (int u = 0; u < PER; ++u) {
      *(u32x4*)(lk[buf] + lds_k[u]) = from.k[u];
      *(u32x4*)(lv[buf] + lds_v[u]) = from.v[u];
    }
    if (td) ldoc[buf][lane] = lane < from.left ? max(from.doc, -1) : -1;
  };

  // The first two tiles of an undocumented call are known before the limits of all rows are: they are asked for at once (a tile behind
  // every limit is not used).
  int t_begin = part * a.tiles_a_part;
  if (!td && t_begin * KT < len) {
    fetch(tile, t_begin);
    if ((t_begin + 1) * KT < len) fetch(second, t_begin + 1);
  }

  // ---- smallest and largest limit and document of the wave and of the workgroup (rows of no document do not widen the range).  Limits
  // ascend with the row; documents need not.
  const int lo = __builtin_amdgcn_readlane(limit, 0);
  int hi = __builtin_amdgcn_readlane(limit, 31), dlo = qdoc < 0 ? INT32_MAX : qdoc, dhi = qdoc, dmin = qdoc;
#pragma unroll
  for (int s = 1; s < 32; s <<= 1) dmin = min(dmin, __shfl_xor(dmin, s)), dlo = min(dlo, __shfl_xor(dlo, s)), dhi = max(dhi, __shfl_xor(dhi, s));
  dmin = __builtin_amdgcn_readfirstlane(dmin), dlo = __builtin_amdgcn_readfirstlane(dlo), dhi = __builtin_amdgcn_readfirstlane(dhi);
  if (lane == 0) wg_lim[wave][1] = hi, wg_lim[wave][2] = dlo, wg_lim[wave][3] = dhi;
  __syncthreads();
  int ghi = 0, gdlo = INT32_MAX, gdhi = -1;
#pragma unroll
  for (int w = 0; w < NW; ++w) ghi = max(ghi, wg_lim[w][1]), gdlo = min(gdlo, wg_lim[w][2]), gdhi = max(gdhi, wg_lim[w][3]);
  ghi = __builtin_amdgcn_readfirstlane(ghi), gdlo = __builtin_amdgcn_readfirstlane(gdlo), gdhi = __builtin_amdgcn_readfirstlane(gdhi);

  int t_end = (ghi + KT - 1) / KT;
  if (!td || a.parts == 1) t_end = min(t_end, t_begin + a.tiles_a_part);
  // next tile at or behind t that may hold a visible pair (the same answer in every wave); t_end: none.  64 tiles are looked at a time,
  // one a lane, and kept.
  int window = -64;
  unsigned long long window_on = 0;
  int2 mine = {-1, -1};
  auto next_tile = [&](int t) {
    if (!td) return min(t, t_end);
    while (t < t_end) {
      if (t >= window + 64) {
        window = t;
        mine = t + lane < t_end ? td[t + lane] : int2{-1, -1};
        window_on = __ballot(gdhi >= 0 && mine.x <= gdhi && mine.y >= gdlo);
      }
      const unsigned long long on = window_on >> (t - window);
      if (on) return t + __builtin_ctzll(on);
      t = window + 64;
    }
    return t_end;
  };
  if (td && a.parts > 1) {                                       // a part of what lies behind the first tile that counts, not of all keys
    const int from = next_tile(0), per = (t_end - from + a.parts - 1) / a.parts;
    t_begin = from + part * per, t_end = min(t_end, t_begin + per);
  }
  // the one document of the tile that next_tile has just found; -1: several, or keys of none; OTHER: none of the wave's rows
  constexpr int OTHER = -2;
  auto tile_doc = [&](int t) {
    if (!td || t >= t_end) return -1;
    const int x = __builtin_amdgcn_readlane(mine.x, t - window), y = __builtin_amdgcn_readlane(mine.y, t - window);
    return x > dhi || y < dlo ? OTHER : x == y ? x : -1;
  };

  // ---- pieces of a step
  const float sc = a.scale * LOG2E, cap2 = a.cap * LOG2E, in_cap = a.cap > 0.f ? 2.f * LOG2E * a.scale / a.cap : 0.f;
  const unsigned k_lane = c * KROW + h * 16;
  const unsigned v_lane = (4 * h + ((lane & 15) >> 2)) * VROW + ((lane >> 4 & 1) * 16 + 4 * (lane & 3) + d0) * 2;
  f32x16 o[DB];
  float m, l;                                                    // reference and sum of the weights
  auto clear = [&]() {
#pragma unroll
    for (int x = 0; x < DB; ++x)
#pragma unroll
      for (int y = 0; y < 16; ++y) o[x][y] = 0.f;
    m = -INFINITY, l = 0.f;
  };
  int pos_first = pos, pos_last = pos;                           // of the wave's rows
  float tilt = 0.f;
  if constexpr (BIAS) {
    if (a.row_lens) {
#pragma unroll
      for (int s = 1; s < 32; s <<= 1) pos_first = min(pos_first, __shfl_xor(pos_first, s)), pos_last = max(pos_last, __shfl_xor(pos_last, s));
    }
    pos_first = __builtin_amdgcn_readlane(pos_first, 0), pos_last = __builtin_amdgcn_readlane(pos_last, 31);
    // (a bias of 2^40 a token leaves the nearest key alone like any larger one: no division overflows)
    if constexpr (MODE == MASKED_LINEAR) slope = fmaxf(-0x1p100f * sc, fminf(slope, 0x1p100f * sc)), tilt = slope / sc;
  }
  // Scores of the 32 keys from key0 on.  LINEAR: the products are added to the bias over the scale, up to the bias of the lane's first
  // key, which is returned: where all keys lie on one side of all rows the bias is linear in the key.
  auto scores = [&](f32x16& s, int buf, int half, int key0) {
    float offset = 0.f;
    if constexpr (MODE == MASKED_LINEAR) {
      const float rel = (float)(pos - key0 - 4 * h);             // distance of the lane's first key
      if (key0 + 31 <= pos_first || key0 >= pos_last) {
        const bool before = key0 + 31 <= pos_first;
        const float up = before ? tilt : -tilt;
#pragma unroll
        for (int y = 0; y < 16; ++y) s[y] = up * (float)(8 * (y >> 2) + (y & 3));
        offset = (before ? -slope : slope) * rel;
      } else {
#pragma unroll
        for (int y = 0; y < 16; ++y) s[y] = -tilt * fabsf(rel - (float)(8 * (y >> 2) + (y & 3)));
      }
    } else {
#pragma unroll
      for (int y = 0; y < 16; ++y) s[y] = 0.f;
    }
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) s = mfma32<F16>(*(const u32x4*)(lk[buf] + half * 32 * KROW + k_lane + ks * 32), qf[ks], s);
    return offset;
  };
  // scores -> values whose exponent (base 2) is factor * value + offset: PLAIN and LINEAR the scores themselves; CAP 1 / (1 +
  // exp(2 x / cap)), the variable part of a capped score (ds2_capped); GENERAL exponents.
  constexpr bool DOWN = MODE == MASKED_CAP;                      // the largest exponent has the smallest value
  const float factor = MODE == MASKED_CAP ? -2.f * cap2 : MODE == MASKED_GENERAL ? 1.f : sc;
  auto exponents = [&](f32x16& s, int key0, float offset) {
    if constexpr (MODE == MASKED_CAP) {
#pragma unroll
      for (int y = 0; y < 16; ++y) s[y] = __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(s[y] * in_cap));
      return cap2;
    }
    if constexpr (MODE == MASKED_GENERAL) {
      if (a.cap > DS2_CAP_WIDE) {
#pragma unroll
        for (int y = 0; y < 16; ++y) s[y] = ds2_capped_wide(s[y], in_cap, cap2, sc);
      } else if (a.cap > 0.f) {
#pragma unroll
        for (int y = 0; y < 16; ++y) s[y] = ds2_capped(s[y], in_cap, cap2);
      } else {
#pragma unroll
        for (int y = 0; y < 16; ++y) s[y] *= sc;
      }
      const float rel = (float)(pos - key0 - 4 * h);             // distance of the lane's first key
      if (a.slopes) {
#pragma unroll
        for (int y = 0; y < 16; ++y) s[y] = __builtin_fmaf(-slope, fabsf(rel - (float)(8 * (y >> 2) + (y & 3))), s[y]);
      }
    }
    return offset;
  };
  auto hide = [&](f32x16& s, int key0, int buf, int half) {
    constexpr float NEVER = DOWN ? INFINITY : -INFINITY;
    if (key0 + 32 > lo) {
      const int rel = limit - key0 - 4 * h;
#pragma unroll
      for (int y = 0; y < 16; ++y)
        if (8 * (y >> 2) + (y & 3) >= rel) s[y] = NEVER;
    }
    if (td) {
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        const u32x4 d = *(const u32x4*)&ldoc[buf][32 * half + 8 * y + 4 * h];
#pragma unroll
        for (int z = 0; z < 4; ++z)
          if ((int)d[z] != qdoc) s[4 * y + z] = NEVER;
      }
    }
  };
  auto raise = [&](const f32x16& s, float offset) {
    float top = s[0];
#pragma unroll
    for (int y = 1; y < 16; ++y) top = DOWN ? fminf(top, s[y]) : fmaxf(top, s[y]);
    float off = offset - fmaxf(m, -3e38f);
    if (__any(__builtin_fmaf(top, factor, off) > DS2_LIMIT<F16>)) {
      float t = __builtin_fmaf(top, factor, offset);
      t = fmaxf(t, __shfl_xor(t, 32));
      float mn = fmaxf(m, t - DS2_SHIFT<F16>);
      float most = __builtin_fmaf(top, factor, offset - mn);
      most = fmaxf(most, __shfl_xor(most, 32));
      if (most > DS2_LIMIT<F16>) mn = fmaxf(m, t);                  // (scores so large that fp32 does not hold the difference)
      const float al = m == mn ? 1.f : __builtin_amdgcn_exp2f(m - mn);
      l *= al;
#pragma unroll
      for (int x = 0; x < DB; ++x)
#pragma unroll
        for (int y = 0; y < 16; ++y) o[x][y] *= al;
      m = mn;
      off = offset - fmaxf(m, -3e38f);
    }
    return off;
  };
  auto weights = [&](f32x16& s, float off) {                     // (off: what raise has returned)
#pragma unroll
    for (int y = 0; y < 16; ++y) {
      s[y] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[y], factor, off));
      l += s[y];
    }
  };
  auto packed = [&](const f32x16& s, int kk) {                   // weights of 16 keys as an operand
    u32x4 p;
#pragma unroll
    for (int y = 0; y < 4; ++y) p[y] = ds2_pack16<F16>(s[8 * kk + 2 * y], s[8 * kk + 2 * y + 1]);
    return p;
  };
  auto rest = [&](const f32x16& s, const u32x4& p, int kk) {     // WIDE: what that rounding left, as another
    u32x4 r;
#pragma unroll
    for (int y = 0; y < 4; ++y) r[y] = ds2_pack16<F16>(s[8 * kk + 2 * y] - ds2_low16<F16>(p[y]), s[8 * kk + 2 * y + 1] - ds2_high16<F16>(p[y]));
    return r;
  };
  auto value_operand = [&](int buf, int half, int kk, int x) {
    const unsigned char* at = lv[buf] + v_lane + (half * 32 + kk * 16) * VROW + x * 64;
    const u32x2 w0 = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)at));
    const u32x2 w1 = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(at + 8 * VROW)));
    return u32x4{w0[0], w0[1], w1[0], w1[1]};
  };
  auto is_edge = [&](int doc, int key0) {                        // some row of the wave may not see all of the step's keys
    return key0 + 32 > lo || (td && (doc < 0 || dmin != dhi || dmin != doc));
  };

  if (row0 >= rows) hi = 0;                                      // no rows of its own: stages keys for the others
  // ---- main loop: tile t0 in use, t1 in LDS, t2 in registers
  clear();
  bool edges = false;
  int t0 = next_tile(t_begin), doc0 = tile_doc(t0);
  if (t0 < t_end) {
    int t1 = next_tile(t0 + 1), doc1 = tile_doc(t1), t2 = next_tile(t1 + 1), doc2 = tile_doc(t2), t3 = t_end, doc3 = -1, buf = 0;
    if (td) {
      fetch(tile, t0);
      if (t1 < t_end) fetch(second, t1);
    }
    stage(tile, 0);
    if (t1 < t_end) stage(second, 1);
    if (t2 < t_end) fetch(tile, t2);
#pragma unroll
    for (int s = 0; s < KS; ++s) asm volatile("" : "+v"(qf[s])); // (arrived before the loop: a wait inside it would be for the tile loads too)
    __syncthreads();
    f32x16 s;
    float offset = scores(s, 0, kg, t0 * KT + kg * 32);
    offset = exponents(s, t0 * KT + kg * 32, offset);
    while (true) {
      const int next = buf == 2 ? 0 : buf + 1;
#pragma unroll
      for (int st = 0; st < ST; ++st) {
        const int half = kg + st, key0 = t0 * KT + half * 32;
        if (key0 < hi) {                                         // (keys ascend: a wave that is done stays done)
          // (The edge is decided before any product: no branch between score products and their first use - hipcc left out the wait
          // states in front of an accumulator read behind such a branch, and the last product's terms were missing.)
          if (is_edge(doc0, key0)) {
            edges = true;
            if (doc0 == OTHER) offset = -INFINITY;                // (no weight; a step that is left out would tear the pipeline)
            else hide(s, key0, buf, half);
          }
          const float off = raise(s, offset);
          f32x16 n;
          const int key1 = st + 1 < ST ? key0 + 32 : t1 * KT + kg * 32;          // (behind the last tile: not used)
          const float offset1 = scores(n, st + 1 < ST ? buf : next, st + 1 < ST ? half + 1 : kg, key1);
          weights(s, off);
          const u32x4 p0 = packed(s, 0), p1 = packed(s, 1);
          if constexpr (WIDE) {
            const u32x4 r0 = rest(s, p0, 0), r1 = rest(s, p1, 1);
#pragma unroll
            for (int x = 0; x < DB; ++x) {
              const u32x4 v0 = value_operand(buf, half, 0, x), v1 = value_operand(buf, half, 1, x);
              o[x] = mfma32<F16>(v0, p0, o[x]);
              o[x] = mfma32<F16>(v1, p1, o[x]);
              o[x] = mfma32<F16>(v0, r0, o[x]);
              o[x] = mfma32<F16>(v1, r1, o[x]);
            }
          } else {
#pragma unroll
            for (int x = 0; x < DB; ++x) o[x] = mfma32<F16>(value_operand(buf, half, 0, x), p0, o[x]);
#pragma unroll
            for (int x = 0; x < DB; ++x) o[x] = mfma32<F16>(value_operand(buf, half, 1, x), p1, o[x]);
          }
          offset = exponents(n, key1, offset1);
          s = n;
        }
        if (st == 0) {
          if (t2 < t_end) stage(tile, next == 2 ? 0 : next + 1);       // (that buffer was last read before this tile's barrier)
          t3 = next_tile(t2 + 1), doc3 = tile_doc(t3);
          if (t3 < t_end) fetch(tile, t3);
        }
      }
      if (t1 >= t_end) break;
      __syncthreads();
      t0 = t1, t1 = t2, t2 = t3, doc0 = doc1, doc1 = doc2, doc2 = doc3, buf = next;
    }
  }

  // ---- A hidden key has weight 0, but 0 times an infinity or a NaN is not 0.  Only edge steps can hide a key from some of the rows; if a
  // result is not finite after one, the tile is computed again, and values that are not finite go to the rows that see them one by
  // one (rare: speed does not matter).
  {
    float z = 0.f;
#pragma unroll
    for (int x = 0; x < DB; ++x)
#pragma unroll
      for (int y = 0; y < 16; ++y) z = __builtin_fmaf(o[x][y], 0.f, z);
    const bool bad = __any(!(z == 0.f)) && edges;
    __syncthreads();
    if (lane == 0) wg_lim[wave][0] = bad;
    __syncthreads();
    int again = 0;
#pragma unroll
    for (int w = 0; w < NW; ++w) again |= wg_lim[w][0];
    if (__builtin_amdgcn_readfirstlane(again)) {
      clear();
      window = -64, window_on = 0;
      for (int t = next_tile(t_begin); t < t_end; t = next_tile(t + 1)) {
        const int doc = tile_doc(t);
        __syncthreads();
        fetch(tile, t);
        stage(tile, 0);
        __syncthreads();
#pragma unroll 1
        for (int half = kg; half < kg + ST; ++half) {
          const int key0 = t * KT + half * 32;
          if (key0 >= hi) break;
          const bool edge = is_edge(doc, key0);
          f32x16 s;
          float offset = scores(s, 0, half, key0);
          offset = exponents(s, key0, offset);
          if (edge) hide(s, key0, 0, half);
          weights(s, raise(s, offset));
          if (edge) {
#pragma unroll 1
            for (int key = 0; key < 32; ++key) {
              const int want = (key & 3) | (key >> 3) << 2;
              float w = 0.f;
#pragma unroll
              for (int y = 0; y < 16; ++y) w = want == y ? s[y] : w;
              w = __shfl(w, c | (key >> 2 & 1) << 5);
              if (key0 + key >= limit || (td && ldoc[0][32 * half + key] != qdoc)) continue;
#pragma unroll
              for (int x = 0; x < DB; ++x)
#pragma unroll
                for (int y = 0; y < 16; ++y) {
                  const float v = ds2_low16<F16>(*(const uint16_t*)(lv[0] + (half * 32 + key) * VROW + (d0 + x * 32 + 8 * (y >> 2) + 4 * h + (y & 3)) * 2));
                  if (!__builtin_isfinite(v)) o[x][y] += w * v;
                }
            }
          }
#pragma unroll
          for (int kk = 0; kk < 2; ++kk) {
            const u32x4 p = packed(s, kk);
            u32x4 r;
            if constexpr (WIDE) r = rest(s, p, kk);
#pragma unroll
            for (int x = 0; x < DB; ++x) {
              u32x4 v = value_operand(0, half, kk, x);
#pragma unroll
              for (int y = 0; y < 4; ++y) v[y] &= edge ? ~not_finite<F16>(v[y]) : 0xffffffffu;
              o[x] = mfma32<F16>(v, p, o[x]);
              if constexpr (WIDE) o[x] = mfma32<F16>(v, r, o[x]);
            }
          }
        }
      }
    }
  }

  l += __shfl_xor(l, 32);
  if constexpr (KG > 1) {                                        // join the key groups: the same rows in the same lanes
    Joined& other = ((Joined*)lds)[wave % RW];
    __syncthreads();                                             // (the waves are through with their keys)
    if (kg) {
#pragma unroll
      for (int x = 0; x < DB; ++x)
#pragma unroll
        for (int y = 0; y < 16; ++y) other[x * 16 + y][lane] = o[x][y];
      other[DB * 16][lane] = m, other[DB * 16 + 1][lane] = l;
    }
    __syncthreads();
    if (kg) return;
    const float mo = other[DB * 16][lane], mn = fmaxf(m, mo);
    const float f = m == mn ? 1.f : __builtin_amdgcn_exp2f(m - mn), fo = mo == mn ? 1.f : __builtin_amdgcn_exp2f(mo - mn);
    l = l * f + fo * other[DB * 16 + 1][lane], m = mn;
#pragma unroll
    for (int x = 0; x < DB; ++x)
#pragma unroll
      for (int y = 0; y < 16; ++y) o[x][y] = o[x][y] * f + fo * other[x * 16 + y][lane];
  }
  if (row0 + c >= rows) return;
  int group = a.G;
  asm volatile("" : "+s"(group));                                // (position and head again: not kept in registers through the loop)
  const int at_i = r / group;
  const int64_t row = ((int64_t)b * a.Lq + at_i) * a.Hq + kvh * a.G + (r - at_i * group);
  const bool none = m == -INFINITY && l == 0.f;                  // nothing seen: zeros
  if (a.part_o) {
    const int64_t at = (int64_t)part * a.B * a.Lq * a.Hq + row;
    if (h == 0 && d0 == 0) a.part_ml[at] = f32x2_t{m, l};
    if (none) return;                                            // the join does not read such a row
#pragma unroll
    for (int x = 0; x < DB; ++x)
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        const int d = d0 + x * 32 + 8 * y + 4 * h;
        if (d < a.D) *(f32x4*)(a.part_o + at * a.D + d) = f32x4{o[x][4 * y], o[x][4 * y + 1], o[x][4 * y + 2], o[x][4 * y + 3]};
      }
  } else {
    const float f = none ? 0.f : 1.f / l;
#pragma unroll
    for (int x = 0; x < DB; ++x)
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        const int d = d0 + x * 32 + 8 * y + 4 * h;
        if (d < a.D)
          *(u32x2*)(a.out + (row * a.D + d) * 2) = none ? u32x2{0, 0}
                                                        : u32x2{ds2_pack16<F16>(o[x][4 * y] * f, o[x][4 * y + 1] * f), ds2_pack16<F16>(o[x][4 * y + 2] * f, o[x][4 * y + 3] * f)};
      }
  }
}

template <bool F16, int DP, int KG, bool WIDE>
void launch_masked_mode(const MaskedArgs& a, int mode, unsigned blocks, hipStream_t st) {
  if (mode == MASKED_PLAIN) k_attn_masked<F16, DP, MASKED_PLAIN, KG, WIDE><<<dim3(blocks), 512, 0, st>>>(a);
  else if (mode == MASKED_CAP) k_attn_masked<F16, DP, MASKED_CAP, KG, WIDE><<<dim3(blocks), 512, 0, st>>>(a);
  else if (mode == MASKED_LINEAR) k_attn_masked<F16, DP, MASKED_LINEAR, KG, WIDE><<<dim3(blocks), 512, 0, st>>>(a);
  else k_attn_masked<F16, DP, MASKED_GENERAL, KG, WIDE><<<dim3(blocks), 512, 0, st>>>(a);
}
template <bool F16, int DP, bool WIDE>
void launch_masked_groups(const MaskedArgs& a, int mode, unsigned blocks, hipStream_t st) {
  if constexpr (DP <= 128 && !WIDE) {
    if (a.key_groups == 2) return launch_masked_mode<F16, DP, 2, WIDE>(a, mode, blocks, st);
  }
  launch_masked_mode<F16, DP, 1, WIDE>(a, mode, blocks, st);
}
template <bool F16, bool WIDE = false>
int launch_masked(const MaskedArgs& a, int mode, unsigned blocks, hipStream_t st) {
  if (a.D <= 32) launch_masked_groups<F16, 32, WIDE>(a, mode, blocks, st);
  else if (a.D <= 64) launch_masked_groups<F16, 64, WIDE>(a, mode, blocks, st);
  else if (a.D <= 96) launch_masked_groups<F16, 96, WIDE>(a, mode, blocks, st);
  else if (a.D <= 128) launch_masked_groups<F16, 128, WIDE>(a, mode, blocks, st);
  else launch_masked_groups<F16, 256, WIDE>(a, mode, blocks, st);
  DS2_CHECK_LAUNCH();
  return DS2_OK;
}

}  // namespace
