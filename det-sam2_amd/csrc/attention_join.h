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
  int T, Hq, G, C, own_rows, own_groups;
};

// Latency is what this kernel is made of (2 to 5 us for a few MB): statistics and rows of eight parts are asked for at once and weighed
// against a running maximum, so a row with up to eight parts (32 in a WIDE one: four waves share the row's parts) waits for memory
// twice, for where its parts are and for the parts.
template <bool F16, bool WIDE>
__global__ __launch_bounds__(256) void k_attn_join(AttnJoinArgs a) {
  __shared__ float sum[4][260];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t row = WIDE ? (int64_t)blockIdx.x : (int64_t)blockIdx.x * 4 + wave;
  if (row >= a.rows) return;
  int parts = a.parts;
  int64_t seg = 0;                                           // index of part p, p >= a.parts, is seg + p own_rows
  bool none = false;
  if (a.lens) {
    const int b = (int)(row / ((int64_t)a.T * a.Hq)), rest = (int)(row - (int64_t)b * a.T * a.Hq), t = rest / a.Hq, hq = rest - t * a.Hq;
    const int head = hq / a.G, r = t * a.G + hq - head * a.G, group = r / a.own_rows;
    const int stream = (b * (a.Hq / a.G) + head) * a.own_groups + group;
    const int len = max(0, min(a.lens[b], a.C));
    const int2 of = a.seg_of[stream];                        // (not written where there is no token)
    if (len > 0) {
      parts += of.y - of.x + 1;
      seg = (int64_t)(of.x + stream - a.parts) * a.own_rows + r - group * a.own_rows;
    }
    none = len - a.T + t < 0;
  }
  const int first = WIDE ? wave : 0, step = WIDE ? 4 : 1;
  const int d = lane * 4;
  const bool live = d < a.D;
  f32x4 o = {0, 0, 0, 0};
  float l = 0.f, m = -INFINITY;
  for (int p0 = first; p0 < parts; p0 += 8 * step) {
    f32x2_t ml[8];
    f32x4 x[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int p = min(p0 + u * step, parts - 1);
      const bool own = p >= a.parts;
      const int64_t at = own ? seg + (int64_t)p * a.own_rows : p * a.rows + row;
      ml[u] = (own ? a.seg_ml : a.ml)[at];
      x[u] = live ? *(const f32x4*)((own ? a.seg_o : a.o) + at * a.D + d) : f32x4{0, 0, 0, 0};
      if (p0 + u * step >= parts) ml[u] = f32x2_t{-INFINITY, 0.f};
    }
    float mn = m;
#pragma unroll
    for (int u = 0; u < 8; ++u) mn = fmaxf(mn, ml[u][0]);
    const float f = m == mn ? 1.f : __builtin_amdgcn_exp2f(m - mn);
    o *= f, l *= f, m = mn;
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (!(ml[u][0] == -INFINITY && ml[u][1] == 0.f)) {     // (a part that saw nothing may not have written its row)
        const float g = ml[u][0] == m ? 1.f : __builtin_amdgcn_exp2f(ml[u][0] - m);
        l += g * ml[u][1];
        o += g * x[u];
      }
  }
  if constexpr (WIDE) {
#pragma unroll
    for (int j = 0; j < 4; ++j) sum[wave][d + j] = o[j];
    if (lane == 0) sum[wave][256] = l, sum[wave][257] = m;
    __syncthreads();
    if (wave) return;
    float mn = m;
#pragma unroll
    for (int w = 1; w < 4; ++w) mn = fmaxf(mn, sum[w][257]);
    const float f = m == mn ? 1.f : __builtin_amdgcn_exp2f(m - mn);
    o *= f, l *= f, m = mn;
#pragma unroll
    for (int w = 1; w < 4; ++w) {
      const float g = sum[w][257] == m ? 1.f : __builtin_amdgcn_exp2f(sum[w][257] - m);
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] += g * sum[w][d + j];
      l += g * sum[w][256];
    }
  }
  if (!live) return;
  none |= m == -INFINITY && l == 0.f;                        // nothing seen: zeros
  const float f = 1.f / l;
  *(u32x2*)(a.out + (row * a.D + d) * 2) =
      none ? u32x2{0, 0} : u32x2{ds2_pack16<F16>(o[0] * f, o[1] * f), ds2_pack16<F16>(o[2] * f, o[3] * f)};
}

// usual_parts: of a row, as far as the host knows; over eight of them four waves share a row
inline int launch_attn_join(const AttnJoinArgs& a, bool f16, int64_t usual_parts, hipStream_t st) {
  const bool wide = usual_parts > 8;
  const dim3 grid((unsigned)(wide ? a.rows : cdiv64(a.rows, 4)));
  if (f16) wide ? k_attn_join<true, true><<<grid, 256, 0, st>>>(a) : k_attn_join<true, false><<<grid, 256, 0, st>>>(a);
  else wide ? k_attn_join<false, true><<<grid, 256, 0, st>>>(a) : k_attn_join<false, false><<<grid, 256, 0, st>>>(a);
  DS2_CHECK_LAUNCH();
  return DS2_OK;
}

}  // namespace
