// Joins the parts of an attention whose keys were split over workgroups: output row = sum of the parts' unnormalised rows, each
// times 2^(its maximum - the largest one), over the same sum of their weight sums (statistics and rows in fp32, one rounding at the end).
#pragma once
#include "token_cache.h"

namespace {

struct AttnJoinArgs {
  const float* o;             // [parts][rows][D]
  const f32x2_t* ml;          // [parts][rows]: maximum (base 2) and weight sum
  char* out;                  // [rows][D], 16 bits
  int64_t rows;
  int D, parts;
  // caches: segments of the row's stream besides (cache_attention.h); rows before a sequence's first token see nothing
  const float* seg_o;
  const f32x2_t* seg_ml;
  const int2* seg_of;
  const int32_t* lens;        // null: no segments
  int T, Hq, G, C, shares, own_rows, own_groups;
  int lanes;                  // of a reader, set at the launch
};

// Latency is what this kernel is made of (2 to 5 us for a few MB), so little of it is one after the other: D / 4 lanes (rounded up
// to a power of two) are a reader of parts, and every reader asks for statistics and rows of eight parts at once and weighs them against
// a running maximum.  A row of up to eight parts is one reader's (NARROW), one of more the readers' of a wave (ROW) or of four (WIDE),
// eight parts each as far as that reaches: it waits for memory twice, for where its parts are and for the parts.
enum { JOIN_NARROW = 0, JOIN_ROW = 1, JOIN_WIDE = 2 };
inline int attn_join_lanes(int D) { return D <= 32 ? 8 : D <= 64 ? 16 : D <= 128 ? 32 : 64; }

template <bool F16, int MODE>
__global__ __launch_bounds__(256) void k_attn_join(AttnJoinArgs a) {
  ds2_ask_args(a);
  constexpr bool WIDE = MODE == JOIN_WIDE;
  __shared__ __attribute__((aligned(16))) float sum[3][260];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int each = a.lanes, readers = 64 / each, reader = lane / each;
  const int64_t row = WIDE ? (int64_t)blockIdx.x : MODE == JOIN_ROW ? (int64_t)blockIdx.x * 4 + wave : ((int64_t)blockIdx.x * 4 + wave) * readers + reader;
  if (row >= a.rows) return;
  int parts = a.parts;
  int64_t seg = 0;                                           // index of part p, p >= a.parts, is seg + p own_rows
  bool none = false;
  if (a.lens) {
    const int b = (int)(row / ((int64_t)a.T * a.Hq)), rest = (int)(row - (int64_t)b * a.T * a.Hq), t = rest / a.Hq, hq = rest - t * a.Hq;
    const int head = hq / a.G, r = t * a.G + hq - head * a.G, group = r / a.own_rows;
    const int stream = (b * (a.Hq / a.G) + head) * a.own_groups + group;
    const int len = max(0, min(a.lens[b], a.C));
    const int2 of = a.shares ? a.seg_of[stream] : int2{0, 0};       // (not written where there is no token)
    if (len > 0) {
      parts += of.y - of.x + 1;
      seg = (int64_t)(of.x + stream - a.parts) * a.own_rows + r - group * a.own_rows;
    }
    none = len - a.T + t < 0;
  }
  const int first = MODE == JOIN_NARROW ? 0 : (WIDE ? wave * readers : 0) + reader, step = MODE == JOIN_NARROW ? 1 : (WIDE ? 4 : 1) * readers;
  const int d = (lane & (each - 1)) * 4;
  const bool live = d < a.D;
  f32x4 o = {0, 0, 0, 0};
  float l = 0.f, m = -INFINITY;
  auto add = [&](float mp, float lp, f32x4 op) {             // (one part, m is not below mp)
    const float g = mp == m ? 1.f : __builtin_amdgcn_exp2f(mp - m);
    l += g * lp;
    o += g * op;
  };
  auto raise = [&](float mn) {
    const float f = m == mn ? 1.f : __builtin_amdgcn_exp2f(m - mn);
    o *= f, l *= f, m = mn;
  };
  for (int p0 = first; p0 < parts; p0 += 8 * step) {
    f32x2_t ml[8];
    f32x4 x[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int p = p0 + u * step;
      ml[u] = f32x2_t{-INFINITY, 0.f}, x[u] = f32x4{0, 0, 0, 0};
      if (p < parts) {
        const bool own = p >= a.parts;
        const int64_t at = own ? seg + (int64_t)p * a.own_rows : p * a.rows + row;
        ml[u] = (own ? a.seg_ml : a.ml)[at];
        if (live) x[u] = *(const f32x4*)((own ? a.seg_o : a.o) + at * a.D + d);
      }
    }
    float mn = m;
#pragma unroll
    for (int u = 0; u < 8; ++u) mn = fmaxf(mn, ml[u][0]);
    raise(mn);
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (!(ml[u][0] == -INFINITY && ml[u][1] == 0.f)) add(ml[u][0], ml[u][1], x[u]);    // (a part that saw nothing may not have written its row)
  }
  for (int s = each; MODE != JOIN_NARROW && s < 64; s <<= 1) {       // the wave's readers
    const float mo = __shfl_xor(m, s), lo = __shfl_xor(l, s);
    const f32x4 oo = {__shfl_xor(o[0], s), __shfl_xor(o[1], s), __shfl_xor(o[2], s), __shfl_xor(o[3], s)};
    raise(fmaxf(m, mo));
    add(mo, lo, oo);
  }
  if constexpr (WIDE) {
    if (wave && lane < each) {
      *(f32x4*)&sum[wave - 1][d] = o;
      if (lane == 0) sum[wave - 1][256] = l, sum[wave - 1][257] = m;
    }
    __syncthreads();
    if (wave) return;
#pragma unroll
    for (int w = 0; w < 3; ++w) {
      raise(fmaxf(m, sum[w][257]));
      add(sum[w][257], sum[w][256], *(const f32x4*)&sum[w][d]);
    }
  }
  if (!live || (MODE != JOIN_NARROW && lane >= each)) return;
  none |= m == -INFINITY && l == 0.f;                        // nothing seen: zeros
  const float f = 1.f / l;
  *(u32x2*)(a.out + (row * a.D + d) * 2) =
      none ? u32x2{0, 0} : u32x2{ds2_pack16<F16>(o[0] * f, o[1] * f), ds2_pack16<F16>(o[2] * f, o[3] * f)};
}

// usual_parts: of a row, as far as the host knows
template <bool F16>
void launch_attn_join_of(const AttnJoinArgs& a, int64_t usual_parts, hipStream_t st) {
  const int readers = 64 / a.lanes;
  if (usual_parts <= 8) k_attn_join<F16, JOIN_NARROW><<<dim3((unsigned)cdiv64(a.rows, 4 * readers)), 256, 0, st>>>(a);
  else if (usual_parts <= 8 * readers) k_attn_join<F16, JOIN_ROW><<<dim3((unsigned)cdiv64(a.rows, 4)), 256, 0, st>>>(a);
  else k_attn_join<F16, JOIN_WIDE><<<dim3((unsigned)a.rows), 256, 0, st>>>(a);
}
inline int launch_attn_join(AttnJoinArgs a, bool f16, int64_t usual_parts, hipStream_t st) {
  a.lanes = attn_join_lanes(a.D);
  if (f16) launch_attn_join_of<true>(a, usual_parts, st);
  else launch_attn_join_of<false>(a, usual_parts, st);
  DS2_CHECK_LAUNCH();
  return DS2_OK;
}

}  // namespace
