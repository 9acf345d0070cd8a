// Masked attention of whole prompts, 16-bit operands, fp32 statistics:
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
//  * 64 keys a tile, two LDS buffers, staged through registers: the next tile's loads fly during this tile's products, one barrier a tile.
//    K rows are padded by 16 bytes (16 rows of a ds_read_b128 quarter cover all 64 banks), V rows to 64 bytes modulo 256 (the four rows
//    of a transposing read do).
//  * causal, prefix and length masks are one number a row: the keys it sees are those below `limit`.  Tiles beyond every row's limit are not
//    visited, tiles below every row's limit are not masked.  Documents: a small kernel notes the smallest and largest document of each
//    key tile; a wave-wide vote over 64 tiles at a time finds the tiles that can hold a visible pair.
#include <algorithm>
#include <cmath>

#include "attention_join.h"

namespace {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4_t* lds_s16x4;

constexpr int KT = 64;                      // keys of a tile
constexpr float LOG2E = 1.44269504088896340736f;

struct MaskedArgs {
  const char *q, *k, *v;
  char* out;
  int64_t q_b, q_t, q_h, k_b, k_t, k_h, v_b, v_t, v_h;    // bytes
  const float* slopes;
  const int32_t *lens, *q_start, *prefix, *q_doc, *k_doc;
  const int2* tile_docs;                    // [B][tiles]: smallest (-1: a key of none among them) and largest document of a tile
  int B, Lq, Lk, Hq, Hkv, G, D, causal;
  float scale, cap;
  int row_tiles, heads, parts, tiles, tiles_a_part;
  float* part_o;                            // null: one part
  f32x2_t* part_ml;
};

template <bool F16>
__device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
  if constexpr (F16) return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}
template <bool F16>
__device__ __forceinline__ unsigned not_finite(unsigned w) {
  constexpr unsigned EXP = F16 ? 0x7c00u : 0x7f80u;
  return ((w & EXP) == EXP ? 0xffffu : 0u) | (((w >> 16) & EXP) == EXP ? 0xffff0000u : 0u);
}

__global__ __launch_bounds__(64) void k_tile_docs(const int32_t* doc, int Lk, int tiles, int2* out) {
  const int b = blockIdx.x / tiles, t = blockIdx.x - b * tiles, j = t * KT + threadIdx.x;
  int lo = j < Lk ? max(-1, doc[(int64_t)b * Lk + j]) : -1, hi = lo;
#pragma unroll
  for (int s = 1; s < 64; s <<= 1) {
    lo = min(lo, __shfl_xor(lo, s));
    hi = max(hi, __shfl_xor(hi, s));
  }
  if (threadIdx.x == 0) out[(int64_t)b * tiles + t] = int2{lo, hi};
}

template <bool F16, int DP, int NW>
__global__ __launch_bounds__(NW * 64, DP > 128 ? 1 : 2) void k_attn_masked(MaskedArgs a) {
  constexpr int KS = DP / 16, DB = DP / 32;                      // contraction steps of a score, blocks of 32 output elements
  constexpr int KLD = DP * 2 + 16;
  constexpr int VROW = DP == 32 ? 64 : DP == 64 ? 192 : DP == 96 ? 192 : DP == 128 ? 320 : 576;
  constexpr int CH = DP / 8;                                     // 16-byte pieces of a row
  constexpr int NT = NW * 64, PER = (KT * CH + NT - 1) / NT;     // pieces a thread stages of a K (and of a V) tile
  __shared__ __attribute__((aligned(16))) unsigned char lk[2][KT * KLD];
  __shared__ __attribute__((aligned(16))) unsigned char lv[2][KT * VROW];
  __shared__ int ldoc[2][KT];
  __shared__ int wg_lim[NW][4];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 31, h = lane >> 5;

  // ---- which tile: the heads of a batch are spread over the chiplets (blockIdx % 8), long row tiles first
  int id = blockIdx.x, part = 0, head, rt;
  {
    const int nh = a.heads, total = nh * a.parts;
    if (nh % 8 == 0) {
      const int x = id & 7, y = id >> 3, per = total / 8;
      const int z = y % per;
      rt = a.row_tiles - 1 - y / per;
      head = x * (nh / 8) + z / a.parts, part = z % a.parts;
    } else {
      rt = a.row_tiles - 1 - id / total;
      const int z = id % total;
      head = z / a.parts, part = z % a.parts;
    }
  }
  const int b = head / a.Hkv, kvh = head - b * a.Hkv;
  const int rows = a.G * a.Lq;
  const int row0 = rt * NW * 32 + wave * 32;                     // the wave's rows of this key head
  const int r = min(row0 + c, rows - 1);                         // rows behind the last repeat it and are not written
  const int i = r / a.G, hq = kvh * a.G + (r - i * a.G);
  const int len = a.lens ? max(0, min(a.lens[b], a.Lk)) : a.Lk;
  const int64_t pos = (int64_t)(a.q_start ? a.q_start[b] : 0) + i;
  const float slope = a.slopes ? a.slopes[hq] * LOG2E : 0.f;
  int limit = len;
  if (a.causal) {
    int64_t n = pos + 1;
    if (a.prefix) n = max(n, (int64_t)a.prefix[b]);
    limit = (int)max((int64_t)0, min((int64_t)len, n));
  }
  const int qdoc = a.q_doc ? a.q_doc[(int64_t)b * a.Lq + i] : 0;

  // ---- smallest and largest limit and document of the wave and of the workgroup
  int lo = limit, hi = limit, dlo = qdoc, dhi = qdoc;
#pragma unroll
  for (int s = 1; s < 32; s <<= 1) {
    lo = min(lo, __shfl_xor(lo, s)), hi = max(hi, __shfl_xor(hi, s));
    dlo = min(dlo, __shfl_xor(dlo, s)), dhi = max(dhi, __shfl_xor(dhi, s));
  }
  lo = __builtin_amdgcn_readfirstlane(lo), hi = __builtin_amdgcn_readfirstlane(hi);
  dlo = __builtin_amdgcn_readfirstlane(dlo), dhi = __builtin_amdgcn_readfirstlane(dhi);
  if (lane == 0) wg_lim[wave][0] = lo, wg_lim[wave][1] = hi, wg_lim[wave][2] = dlo, wg_lim[wave][3] = dhi;
  __syncthreads();
  int ghi = 0, gdlo = INT32_MAX, gdhi = -1;
#pragma unroll
  for (int w = 0; w < NW; ++w) ghi = max(ghi, wg_lim[w][1]), gdlo = min(gdlo, wg_lim[w][2]), gdhi = max(gdhi, wg_lim[w][3]);
  ghi = __builtin_amdgcn_readfirstlane(ghi), gdlo = __builtin_amdgcn_readfirstlane(gdlo), gdhi = __builtin_amdgcn_readfirstlane(gdhi);

  const int t_end = min((ghi + KT - 1) / KT, (part + 1) * a.tiles_a_part);
  const int t_begin = part * a.tiles_a_part;
  // next tile at or behind t that may hold a visible pair (the same answer in every wave)
  const int2* td = a.tile_docs ? a.tile_docs + (int64_t)b * a.tiles : nullptr;
  auto next_tile = [&](int t) {
    if (!td) return t;
    while (t < t_end) {
      const int mine = t + lane;
      const int2 e = mine < t_end ? td[mine] : int2{-1, -1};
      const unsigned long long on = __ballot(gdhi >= 0 && e.x <= gdhi && e.y >= max(gdlo, 0));
      if (on) return t + __builtin_ctzll(on);
      t += 64;
    }
    return t_end;
  };

  // ---- queries
  u32x4 qf[KS];
  {
    const char* row = a.q + b * a.q_b + (int64_t)i * a.q_t + hq * a.q_h;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int d = 16 * s + 8 * h;
      qf[s] = d < a.D ? *(const u32x4*)(row + d * 2) : u32x4{0, 0, 0, 0};
    }
  }
  f32x16 o[DB];
#pragma unroll
  for (int x = 0; x < DB; ++x)
#pragma unroll
    for (int y = 0; y < 16; ++y) o[x][y] = 0.f;
  float m = -INFINITY, l = 0.f;

  const char *kb = a.k + b * a.k_b + kvh * a.k_h, *vb = a.v + b * a.v_b + kvh * a.v_h;
  u32x4 sk[PER], sv[PER];
  int sdoc = -1;
  auto fetch = [&](int t) {                                      // keys of the tile into registers; behind the last key: zeros
#pragma unroll
    for (int u = 0; u < PER; ++u) {
      const int p = u * NT + tid, row = p / CH, piece = p - row * CH, key = t * KT + row;
      const bool live = (PER * NT == KT * CH || row < KT) && key < len && piece * 8 < a.D;
      sk[u] = live ? *(const u32x4*)(kb + (int64_t)key * a.k_t + piece * 16) : u32x4{0, 0, 0, 0};
      sv[u] = live ? *(const u32x4*)(vb + (int64_t)key * a.v_t + piece * 16) : u32x4{0, 0, 0, 0};
    }
    if (a.k_doc && tid < KT) sdoc = t * KT + tid < len ? a.k_doc[(int64_t)b * a.Lk + t * KT + tid] : -1;
  };
  auto stage = [&](int buf) {
#pragma unroll
    for (int u = 0; u < PER; ++u) {
      const int p = u * NT + tid, row = p / CH, piece = p - row * CH;
      if (PER * NT != KT * CH && row >= KT) break;
      *(u32x4*)(lk[buf] + row * KLD + piece * 16) = sk[u];
      *(u32x4*)(lv[buf] + row * VROW + piece * 16) = sv[u];
    }
    if (a.k_doc && tid < KT) ldoc[buf][tid] = sdoc;
  };

  const float sc = a.scale * LOG2E, cap2 = a.cap * LOG2E, in_cap = a.cap > 0.f ? 2.f * LOG2E * a.scale / a.cap : 0.f;
  const bool plain = a.cap == 0.f && !a.slopes && a.scale > 0.f;
  int t = next_tile(t_begin), buf = 0;
  if (t < t_end) {
    fetch(t);
    stage(0);
  }
  __syncthreads();
  while (t < t_end) {
    const int next = next_tile(t + 1);
    if (next < t_end) fetch(next);
    const int key0 = t * KT;
    if (key0 < hi) {                                             // some row of the wave reaches this tile
      // (decided before the products: no branch between the score products and their first use - hipcc left out the wait states in
      // front of an accumulator read behind such a branch, and the last product's terms were missing)
      bool edge = key0 + KT > lo;
      if (td) {
        const int2 e = td[t];
        edge |= e.x != e.y || dlo != dhi || dlo != e.x;
      }
      f32x16 s[2];
#pragma unroll
      for (int x = 0; x < 2; ++x) {
#pragma unroll
        for (int y = 0; y < 16; ++y) s[x][y] = 0.f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
          s[x] = mfma32<F16>(*(const u32x4*)(lk[buf] + (x * 32 + c) * KLD + ks * 32 + h * 16), qf[ks], s[x]);
      }
      float f = sc;
      if (!plain) {
        f = 1.f;
        if (a.cap > 0.f) {
          // cap tanh(x / cap) = cap - 2 cap / (1 + exp(2 x / cap)): no branch, saturates by itself; off by a few 2^-24 of cap
#pragma unroll
          for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int y = 0; y < 16; ++y)
              s[x][y] = cap2 - 2.f * cap2 * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(s[x][y] * in_cap));
        } else {
#pragma unroll
          for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int y = 0; y < 16; ++y) s[x][y] *= sc;
        }
        if (a.slopes) {
          const int rel = (int)(pos - key0) - 4 * h;
#pragma unroll
          for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int y = 0; y < 16; ++y) s[x][y] -= slope * fabsf((float)(rel - (32 * x + 8 * (y >> 2) + (y & 3))));
        }
      }
      bool apart = false;
      if (edge) {
        const int rel = limit - key0 - 4 * h;
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int y = 0; y < 16; ++y)
            if (32 * x + 8 * (y >> 2) + (y & 3) >= rel) s[x][y] = -INFINITY;
        if (a.k_doc) {
#pragma unroll
          for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int y = 0; y < 4; ++y) {
              const u32x4 d = *(const u32x4*)&ldoc[buf][32 * x + 8 * y + 4 * h];
#pragma unroll
              for (int z = 0; z < 4; ++z)
                if ((int)d[z] != qdoc || qdoc < 0) s[x][4 * y + z] = -INFINITY;
            }
        }
        // A hidden key has weight 0, but 0 times an infinity or a NaN is not 0: values that are not finite leave the product of an
        // edge tile and go to the rows that see them one by one.
        unsigned bad = 0;
#pragma unroll 4
        for (int p = lane; p < KT * CH; p += 64) {
          const int row = p / CH;
          const u32x4 w = *(const u32x4*)(lv[buf] + row * VROW + (p - row * CH) * 16);
#pragma unroll
          for (int y = 0; y < 4; ++y) bad |= not_finite<F16>(w[y]);
        }
        apart = __any(bad != 0);
      }
      // ---- running maximum (raised only by more than 2^8: the weights stay small, the rescaling rare)
      float top = s[0][0];
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int y = 0; y < 16; ++y) top = fmaxf(top, s[x][y]);
      top *= f;
      if (__any(top > m + 8.f)) {
        top = fmaxf(top, __shfl_xor(top, 32));
        const float mn = fmaxf(m, top);
        const float al = m == mn ? 1.f : __builtin_amdgcn_exp2f(m - mn);
        l *= al;
#pragma unroll
        for (int x = 0; x < DB; ++x)
#pragma unroll
          for (int y = 0; y < 16; ++y) o[x][y] *= al;
        m = mn;
      }
      const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int y = 0; y < 16; ++y) {
          s[x][y] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[x][y], f, -ref));
          l += s[x][y];
        }
      if (apart) {
#pragma unroll 1
        for (int key = 0; key < KT; ++key) {
          const int want = (key & 3) | (key >> 3 & 3) << 2 | (key >> 5) << 4;
          float w = 0.f;
#pragma unroll
          for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int y = 0; y < 16; ++y) w = want == 16 * x + y ? s[x][y] : w;
          w = __shfl(w, c | (key >> 2 & 1) << 5);
          if (key0 + key >= limit || (a.k_doc && (ldoc[buf][key] != qdoc || qdoc < 0))) continue;
#pragma unroll
          for (int x = 0; x < DB; ++x)
#pragma unroll
            for (int y = 0; y < 16; ++y) {
              const float v = ds2_low16<F16>(*(const uint16_t*)(lv[buf] + key * VROW + (x * 32 + 8 * (y >> 2) + 4 * h + (y & 3)) * 2));
              if (!__builtin_isfinite(v)) o[x][y] += w * v;
            }
        }
      }
#pragma unroll
      for (int kk = 0; kk < 4; ++kk) {                           // 16 keys a step
        u32x4 p;
#pragma unroll
        for (int y = 0; y < 4; ++y) p[y] = ds2_pack16<F16>(s[kk >> 1][8 * (kk & 1) + 2 * y], s[kk >> 1][8 * (kk & 1) + 2 * y + 1]);
        const unsigned char* base = lv[buf] + (kk * 16 + 4 * h + ((lane & 15) >> 2)) * VROW + ((lane >> 4 & 1) * 16 + 4 * (lane & 3)) * 2;
#pragma unroll
        for (int x = 0; x < DB; ++x) {
          const s16x4_t v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(base + x * 64));
          const s16x4_t v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(base + x * 64 + 8 * VROW));
          const u32x2 w0 = __builtin_bit_cast(u32x2, v0), w1 = __builtin_bit_cast(u32x2, v1);
          u32x4 v = {w0[0], w0[1], w1[0], w1[1]};
          if (apart) {
#pragma unroll
            for (int y = 0; y < 4; ++y) v[y] &= ~not_finite<F16>(v[y]);
          }
          o[x] = mfma32<F16>(v, p, o[x]);
        }
      }
    }
    if (next < t_end) stage(buf ^ 1);
    __syncthreads();
    t = next, buf ^= 1;
  }

  l += __shfl_xor(l, 32);
  if (row0 + c >= rows) return;
  const int64_t row = ((int64_t)b * a.Lq + i) * a.Hq + hq;
  const bool none = m == -INFINITY && l == 0.f;                  // nothing seen: zeros
  if (a.part_o) {
    const int64_t at = (int64_t)part * a.B * a.Lq * a.Hq + row;
    if (h == 0) a.part_ml[at] = f32x2_t{m, l};
    if (none) return;                                            // the join does not read such a row
#pragma unroll
    for (int x = 0; x < DB; ++x)
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        const int d = x * 32 + 8 * y + 4 * h;
        if (d < a.D) *(f32x4*)(a.part_o + at * a.D + d) = f32x4{o[x][4 * y], o[x][4 * y + 1], o[x][4 * y + 2], o[x][4 * y + 3]};
      }
  } else {
    const float f = none ? 0.f : 1.f / l;
#pragma unroll
    for (int x = 0; x < DB; ++x)
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        const int d = x * 32 + 8 * y + 4 * h;
        if (d < a.D)
          *(u32x2*)(a.out + (row * a.D + d) * 2) = none ? u32x2{0, 0}
                                                        : u32x2{ds2_pack16<F16>(o[x][4 * y] * f, o[x][4 * y + 1] * f), ds2_pack16<F16>(o[x][4 * y + 2] * f, o[x][4 * y + 3] * f)};
      }
  }
}

struct Plan {
  int nw, row_tiles, heads, parts, tiles, tiles_a_part;
  int64_t blocks, doc_bytes, part_bytes;
};

Plan plan_of(const ds2_attention_masked_args& a) {
  Plan p{};
  const int64_t rows = (int64_t)(a.Hq / a.Hkv) * a.Lq;
  p.nw = rows <= 128 || a.D > 128 ? 4 : 8;
  p.row_tiles = (int)cdiv64(rows, p.nw * 32);
  p.heads = a.B * a.Hkv;
  p.tiles = cdiv(a.Lk, KT);
  // Fewer workgroups than CUs: the keys are split so that about two workgroups a CU result, at least 4 tiles each.
  const int64_t whole = (int64_t)p.row_tiles * p.heads;
  p.parts = 1;
  if (whole < 256) p.parts = (int)std::max<int64_t>(1, std::min<int64_t>(p.tiles / 4, 512 / whole));
  p.tiles_a_part = std::max(1, cdiv(p.tiles, p.parts));
  p.parts = std::max(1, cdiv(p.tiles, p.tiles_a_part));
  p.blocks = whole * p.parts;
  p.doc_bytes = a.q_doc ? (cdiv64((int64_t)a.B * p.tiles * 8, 16) * 16) : 0;
  p.part_bytes = p.parts > 1 ? (int64_t)p.parts * a.B * a.Lq * a.Hq * (a.D + 2) * 4 : 0;
  return p;
}

int check(const ds2_attention_masked_args& a) {
  DS2_REQUIRE(a.B >= 0 && a.Lq >= 0 && a.Lk >= 0, "attention_masked: negative size");
  DS2_REQUIRE(a.Hkv >= 1 && a.Hq >= a.Hkv && a.Hq % a.Hkv == 0, "attention_masked: %d query heads do not share %d key heads evenly", a.Hq, a.Hkv);
  DS2_REQUIRE(a.D >= 8 && a.D <= 256 && a.D % 8 == 0, "attention_masked: head dim %d is not a multiple of 8 up to 256", a.D);
  DS2_REQUIRE(a.type == DS2_TYPE_BF16 || a.type == DS2_TYPE_F16, "attention_masked: bf16 or fp16 expected, got type %d", a.type);
  DS2_REQUIRE(std::isfinite(a.scale) && std::isfinite(a.cap) && a.cap >= 0.f, "attention_masked: scale and cap must be finite, cap not negative");
  DS2_REQUIRE((!a.q_doc) == (!a.k_doc), "attention_masked: q_doc and k_doc go together");
  DS2_REQUIRE(a.causal || !a.prefix, "attention_masked: a prefix goes with the causal mask");
  DS2_REQUIRE(a.Lk < (1 << 30) && (int64_t)(a.Hq / a.Hkv) * a.Lq < (1ll << 31) - 512, "attention_masked: sequence too long");
  DS2_REQUIRE((int64_t)a.B * a.Hkv < (1 << 24) && (int64_t)a.B * a.Lq * a.Hq < (1ll << 32), "attention_masked: too many rows for one call");
  return DS2_OK;
}

int aligned(const ds2_strided& t, const char* name) {
  DS2_REQUIRE(t.p && (uintptr_t)t.p % 16 == 0 && t.s0 % 8 == 0 && t.s1 % 8 == 0 && t.s2 % 8 == 0, "attention_masked: rows of %s must be 16-byte aligned", name);
  return DS2_OK;
}

template <bool F16, int DP>
void launch(const MaskedArgs& a, int nw, unsigned blocks, hipStream_t st) {
  if (nw == 4 || DP > 128) k_attn_masked<F16, DP, 4><<<dim3(blocks), 256, 0, st>>>(a);
  else k_attn_masked<F16, DP, (DP > 128 ? 4 : 8)><<<dim3(blocks), 512, 0, st>>>(a);
}
template <bool F16>
void launch_of(const MaskedArgs& a, int nw, unsigned blocks, hipStream_t st) {
  if (a.D <= 32) launch<F16, 32>(a, nw, blocks, st);
  else if (a.D <= 64) launch<F16, 64>(a, nw, blocks, st);
  else if (a.D <= 96) launch<F16, 96>(a, nw, blocks, st);
  else if (a.D <= 128) launch<F16, 128>(a, nw, blocks, st);
  else launch<F16, 256>(a, nw, blocks, st);
}

}  // namespace

extern "C" int64_t ds2_op_attention_masked_work_bytes(const ds2_attention_masked_args* args) {
  if (!args || check(*args) || !args->B || !args->Lq) return 0;
  const Plan p = plan_of(*args);
  return p.doc_bytes + p.part_bytes;
}

extern "C" int ds2_op_attention_masked(const ds2_attention_masked_args* args, void* work, int64_t work_bytes, void* stream) {
  DS2_REQUIRE(args, "attention_masked: null argument");
  const ds2_attention_masked_args& x = *args;
  if (const int rc = check(x)) return rc;
  if (!x.B || !x.Lq) return DS2_OK;
  DS2_REQUIRE(x.out && (uintptr_t)x.out % 16 == 0, "attention_masked: output rows must be 16-byte aligned");
  if (const int rc = aligned(x.q, "q")) return rc;
  if (x.Lk) {
    if (const int rc = aligned(x.k, "k")) return rc;
    if (const int rc = aligned(x.v, "v")) return rc;
  }
  const Plan p = plan_of(x);
  DS2_REQUIRE(p.blocks < (1ll << 31), "attention_masked: too many rows for one call");
  const int64_t need = p.doc_bytes + p.part_bytes;
  DS2_REQUIRE(!need || (work && (uintptr_t)work % 16 == 0 && work_bytes >= need), "attention_masked: workspace too small");
  MaskedArgs a{};
  a.q = (const char*)x.q.p, a.k = (const char*)x.k.p, a.v = (const char*)x.v.p, a.out = (char*)x.out;
  a.q_b = x.q.s0 * 2, a.q_t = x.q.s1 * 2, a.q_h = x.q.s2 * 2;
  a.k_b = x.k.s0 * 2, a.k_t = x.k.s1 * 2, a.k_h = x.k.s2 * 2;
  a.v_b = x.v.s0 * 2, a.v_t = x.v.s1 * 2, a.v_h = x.v.s2 * 2;
  a.slopes = x.slopes, a.lens = x.lens, a.q_start = x.q_start, a.prefix = x.prefix, a.q_doc = x.q_doc, a.k_doc = x.k_doc;
  a.B = x.B, a.Lq = x.Lq, a.Lk = x.Lk, a.Hq = x.Hq, a.Hkv = x.Hkv, a.G = x.Hq / x.Hkv, a.D = x.D, a.causal = x.causal;
  a.scale = x.scale, a.cap = x.cap;
  a.row_tiles = p.row_tiles, a.heads = p.heads, a.parts = p.parts, a.tiles = p.tiles, a.tiles_a_part = p.tiles_a_part;
  hipStream_t st = (hipStream_t)stream;
  if (x.q_doc && p.tiles) {
    int2* docs = (int2*)work;
    k_tile_docs<<<dim3((unsigned)(x.B * p.tiles)), 64, 0, st>>>(x.k_doc, x.Lk, p.tiles, docs);
    DS2_CHECK_LAUNCH();
    a.tile_docs = docs;
  }
  const int64_t rows = (int64_t)x.B * x.Lq * x.Hq;
  if (p.parts > 1) {
    a.part_o = (float*)((char*)work + p.doc_bytes);
    a.part_ml = (f32x2_t*)(a.part_o + (int64_t)p.parts * rows * x.D);
  }
  const bool f16 = x.type == DS2_TYPE_F16;
  f16 ? launch_of<true>(a, p.nw, (unsigned)p.blocks, st) : launch_of<false>(a, p.nw, (unsigned)p.blocks, st);
  DS2_CHECK_LAUNCH();
  if (p.parts > 1) {
    AttnJoinArgs j{};
    j.o = a.part_o, j.ml = a.part_ml, j.out = a.out, j.rows = rows, j.D = x.D, j.parts = p.parts;
    return launch_attn_join(j, f16, p.parts, st);
  }
  return DS2_OK;
}
