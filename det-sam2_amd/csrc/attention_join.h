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
  // caches: parts behind a sequence's last token were not written, and rows before its first token see nothing
  const int32_t* lens;        // null: all parts count
  int T, Hq, C, pre_parts, own_chunk;
};

// WIDE: four waves share the parts of a row (few rows with many parts); otherwise a wave has a row to itself.
template <bool F16, bool WIDE>
__global__ __launch_bounds__(256) void k_attn_join(AttnJoinArgs a) {
  __shared__ float sum[4][260];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t row = WIDE ? (int64_t)blockIdx.x : (int64_t)blockIdx.x * 4 + wave;
  if (row >= a.rows) return;
  int parts = a.parts;
  bool none = false;
  if (a.lens) {
    const int b = (int)(row / ((int64_t)a.T * a.Hq)), t = (int)(row / a.Hq - (int64_t)b * a.T);
    const int len = max(0, min(a.lens[b], a.C));
    parts = a.pre_parts + (int)(((int64_t)len + a.own_chunk - 1) / a.own_chunk);
    none = len - a.T + t < 0;
  }
  const int first = WIDE ? wave : 0, step = WIDE ? 4 : 1;
  float m = -INFINITY;
  for (int p = lane; p < parts; p += 64) m = fmaxf(m, a.ml[p * a.rows + row][0]);
#pragma unroll
  for (int s = 1; s < 64; s <<= 1) m = fmaxf(m, __shfl_xor(m, s));
  const int d = lane * 4;
  const bool live = d < a.D;
  f32x4 o = {0, 0, 0, 0};
  float l = 0.f;
  // four parts at a time: their loads do not wait for one another
  for (int p = first; p < parts; p += 4 * step) {
    f32x2_t ml[4];
    f32x4 x[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int64_t at = min(p + u * step, parts - 1) * a.rows + row;
      ml[u] = a.ml[at];
      x[u] = live ? *(const f32x4*)(a.o + at * a.D + d) : f32x4{0, 0, 0, 0};
    }
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (p + u * step < parts && !(ml[u][0] == -INFINITY && ml[u][1] == 0.f)) {
        const float f = ml[u][0] == m ? 1.f : __builtin_amdgcn_exp2f(ml[u][0] - m);
        l += f * ml[u][1];
        o += f * x[u];
      }
  }
  if constexpr (WIDE) {
#pragma unroll
    for (int j = 0; j < 4; ++j) sum[wave][d + j] = o[j];
    if (lane == 0) sum[wave][256] = l;
    __syncthreads();
    if (wave) return;
#pragma unroll
    for (int w = 1; w < 4; ++w) {
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] += sum[w][d + j];
      l += sum[w][256];
    }
  }
  if (!live) return;
  none |= m == -INFINITY && l == 0.f;                        // nothing seen: zeros
  const float f = 1.f / l;
  *(u32x2*)(a.out + (row * a.D + d) * 2) =
      none ? u32x2{0, 0} : u32x2{ds2_pack16<F16>(o[0] * f, o[1] * f), ds2_pack16<F16>(o[2] * f, o[3] * f)};
}

inline int launch_attn_join(const AttnJoinArgs& a, bool f16, int most_parts, hipStream_t st) {
  const bool wide = most_parts > 16;
  const dim3 grid((unsigned)(wide ? a.rows : cdiv64(a.rows, 4)));
  if (f16) wide ? k_attn_join<true, true><<<grid, 256, 0, st>>>(a) : k_attn_join<true, false><<<grid, 256, 0, st>>>(a);
  else wide ? k_attn_join<false, true><<<grid, 256, 0, st>>>(a) : k_attn_join<false, false><<<grid, 256, 0, st>>>(a);
  DS2_CHECK_LAUNCH();
  return DS2_OK;
}

}  // namespace
