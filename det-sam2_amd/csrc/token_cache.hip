// Token cache in 8 or 4 bits: rows are quantised as they are written and turned back into values as they are read (format:
// token_cache.h).  Both kernels are one pass over the data and bound by HBM; the arithmetic (about 6 operations a value) hides
// behind the loads.
#include "token_cache.h"

namespace {

struct WriteArgs {
  ds2_strided x[2], codes[2], scales[2];
  const int32_t *pos, *count;
  int T, H, D, capacity, BH, blocks_per_head;
};

// One thread holds 8 values, the 4 threads of a group of 32 are neighbours in a wave.  Threads run along the head dimension,
// then along the tokens: a wave reads whole rows of the token-major input (256 bytes at D = 128, 16 bits) and writes CONSECUTIVE rows
// of the head-major cache.  16 bits into mxfp8, 7 frames of 16 objects (28672 rows of 64 values, 16 sequences): 89 MB in 18.5 us,
// 4.8 TB/s; ragged prompts into mxfp4 (keys and values of 6 x 3001 tokens, 8 heads of 128): 70 MB in 18.8 us.  (All four units' loads
// before the first use: 20.8 and 19.6 us.)  One token of 16 sequences: 3 us, the launch.
template <int TYPE, int FORMAT>
__global__ __launch_bounds__(256) void k_cache_write(WriteArgs a) {
  ds2_ask_args(a);
  const unsigned blk = blockIdx.x, head = blk / a.blocks_per_head, part = blk - head * a.blocks_per_head;
  const int which = head >= (unsigned)a.BH;
  const int bh = head - which * a.BH, b = bh / a.H, h = bh - b * a.H;
  const ds2_strided X = a.x[which], K = a.codes[which], S = a.scales[which];
  const unsigned units = a.D >> 3;                              // 8-value units of a row
  const int first = a.pos[b];
  const int count = a.count ? min(a.count[b], a.T) : a.T;
  const char* xb = (const char*)X.p + (b * X.s0 + h * X.s2) * (TYPE == DS2_TYPE_F32 ? 4 : 2);
  uint8_t* kb = (uint8_t*)K.p + b * K.s0 + h * K.s1;
  uint8_t* sb = (uint8_t*)S.p + b * S.s0 + h * S.s1;
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const unsigned id = (part * 4 + u) * 256 + threadIdx.x;
    const unsigned t = id / units, c = id - t * units;
    const int64_t at = (int64_t)first + t;
    const bool live = (int)t < count && at >= 0 && at < a.capacity;     // whole groups live or not: units % 4 == 0
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = 0.f;
    if (live) {
      if constexpr (TYPE == DS2_TYPE_F32) {
        const float* p = (const float*)xb + (int64_t)t * X.s1 + c * 8;
        const f32x4 lo = *(const f32x4*)p, hi = *(const f32x4*)(p + 4);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = lo[j], v[4 + j] = hi[j];
      } else {
        const u32x4 w = *(const u32x4*)((const uint16_t*)xb + (int64_t)t * X.s1 + c * 8);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          v[2 * j] = ds2_low16<TYPE == DS2_TYPE_F16>(w[j]);
          v[2 * j + 1] = ds2_high16<TYPE == DS2_TYPE_F16>(w[j]);
        }
      }
    }
    // largest magnitude of the group on the bit patterns: ordered like the values, and a NaN is larger than all of them
    unsigned m = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) m = max(m, __builtin_bit_cast(unsigned, v[j]) & 0x7fffffffu);
    m = max(m, (unsigned)__shfl_xor((int)m, 1));
    m = max(m, (unsigned)__shfl_xor((int)m, 2));
    // 448 = 1.75 2^8, 6 = 1.5 2^2: one exponent more when the mantissa is beyond 0.75 resp. 0.5
    constexpr int EXP = FORMAT == DS2_CACHE_MXFP8 ? 8 : 2;
    constexpr unsigned MANT = FORMAT == DS2_CACHE_MXFP8 ? 0x600000u : 0x400000u;
    const bool poison = m >= 0x7f800000u;
    const int s = max(1, (int)(m >> 23) - EXP + ((m & 0x7fffffu) > MANT ? 1 : 0));
    const float inv = __builtin_bit_cast(float, (unsigned)(254 - (poison ? 127 : s)) << 23);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = poison ? 0.f : v[j] * inv;       // exact: a power of two
    if (!live) continue;
    if constexpr (FORMAT == DS2_CACHE_MXFP8) {
      int lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], 0, false), hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[4], v[5], 0, false);
      lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], lo, true);
      hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[6], v[7], hi, true);
      *(u32x2*)(kb + at * K.s2 + c * 8) = u32x2{(unsigned)lo, (unsigned)hi};
    } else {
      unsigned w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, v[0], v[1], 1.f, 0);
      w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[2], v[3], 1.f, 1);
      w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[4], v[5], 1.f, 2);
      w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[6], v[7], 1.f, 3);
      *(unsigned*)(kb + at * K.s2 + c * 4) = w;
    }
    if ((c & 3) == 0) sb[at * S.s2 + (c >> 2)] = (uint8_t)(poison ? 255 : s);
  }
}

struct ReadArgs {
  ds2_strided codes, scales, out;
  const int32_t* lens;
  int C, H, D, blocks_per_head, t_step, c_step;
};

// One thread turns 8 codes into 8 values, four times: the stores of a wave are 1 KB side by side at 16 bits.  The frames above: 89 MB
// in 13.9 us, 6.4 TB/s (with 16 codes a thread, whose stores leave gaps of 16 bytes between lanes, 15.1); the ragged prompts back, one
// tensor: 62 MB in 14.8 us (16.4).  Stores past the caches would make that 11.2, but the kernel that takes the values next would lose more
// (read and copy of 50 MB: 29.6 us so, 32.4 past the caches).
template <int TYPE, int FORMAT>
__global__ __launch_bounds__(256) void k_cache_read(ReadArgs a) {
  ds2_ask_args(a);
  const unsigned blk = blockIdx.x, bh = blk / a.blocks_per_head, part = blk - bh * a.blocks_per_head;
  const int b = bh / a.H, h = bh - b * a.H;
  const unsigned units = a.D >> 3;
  const int len = a.lens ? min(a.lens[b], a.C) : a.C;
  const uint8_t* kb = (const uint8_t*)a.codes.p + b * a.codes.s0 + h * a.codes.s1;
  const uint8_t* sb = (const uint8_t*)a.scales.p + b * a.scales.s0 + h * a.scales.s1;
  constexpr int SIZE = TYPE == DS2_TYPE_F32 ? 4 : 2, UNITS = 4;
  char* ob = (char*)a.out.p + (b * a.out.s0 + h * a.out.s1) * SIZE;
  unsigned t_of[UNITS], c_of[UNITS], scale[UNITS];
  u32x2 code[UNITS];
  {
    unsigned id = part * UNITS * 256 + threadIdx.x, t = id / units, c = id - t * units;
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {                           // all loads before the first use
      t_of[u] = t, c_of[u] = c, scale[u] = 127, code[u] = u32x2{0, 0};
      if ((int)t < len) {
        scale[u] = sb[(int64_t)t * a.scales.s2 + (c >> 2)];
        const uint8_t* p = kb + (int64_t)t * a.codes.s2;
        if constexpr (FORMAT == DS2_CACHE_MXFP8) code[u] = *(const u32x2*)(p + c * 8);
        else code[u][0] = *(const unsigned*)(p + c * 4);
      }
      t += a.t_step, c += a.c_step;                             // 256 units on
      if (c >= units) c -= units, ++t;
    }
  }
#pragma unroll
  for (int u = 0; u < UNITS; ++u) {
    if (t_of[u] >= (unsigned)a.C) continue;
    const float s = ds2_cache_scale(scale[u]);
    float v[8];
    if constexpr (FORMAT == DS2_CACHE_MXFP8) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)code[u][j], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)code[u][j], true);
        v[4 * j] = lo[0] * s, v[4 * j + 1] = lo[1] * s, v[4 * j + 2] = hi[0] * s, v[4 * j + 3] = hi[1] * s;
      }
    } else {
#define DS2_PAIR(i)                                                                  \
  {                                                                                  \
    const auto p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code[u][0], 1.f, i);     \
    v[2 * i] = p[0] * s, v[2 * i + 1] = p[1] * s;                                    \
  }
      DS2_PAIR(0) DS2_PAIR(1) DS2_PAIR(2) DS2_PAIR(3)
#undef DS2_PAIR
    }
    char* o = ob + ((int64_t)t_of[u] * a.out.s2 + c_of[u] * 8) * SIZE;
    if constexpr (TYPE == DS2_TYPE_F32) {
#pragma unroll
      for (int j = 0; j < 2; ++j) *(f32x4*)(o + 16 * j) = f32x4{v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]};
    } else {
      u32x4 w;
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = ds2_pack16<TYPE == DS2_TYPE_F16>(v[2 * j], v[2 * j + 1]);
      *(u32x4*)o = w;
    }
  }
}

bool aligned(const ds2_strided& t, int size, int to, int axes) {
  const int64_t s[3] = {t.s0, t.s1, t.s2};
  bool ok = ((uintptr_t)t.p % to) == 0;
  for (int i = 0; i < axes; ++i) ok = ok && (s[i] * size) % to == 0;
  return ok;
}

}  // namespace

extern "C" int ds2_op_cache_write(int32_t n, const ds2_strided* x, const ds2_strided* codes, const ds2_strided* scales, int32_t B,
                                  int32_t T, int32_t H, int32_t D, int32_t capacity, const int32_t* pos, const int32_t* count,
                                  int32_t type, int32_t format, void* stream) {
  DS2_REQUIRE((n == 1 || n == 2) && x && codes && scales, "cache_write: one or two tensors expected");
  DS2_REQUIRE(B >= 0 && T >= 0 && H >= 1 && capacity >= 0, "cache_write: bad sizes B %d T %d H %d capacity %d", B, T, H, capacity);
  DS2_REQUIRE(D >= DS2_CACHE_GROUP && D <= 4096 && D % DS2_CACHE_GROUP == 0, "cache_write: head dim %d is not a multiple of 32 up to 4096", D);
  DS2_REQUIRE(type == DS2_TYPE_BF16 || type == DS2_TYPE_F16 || type == DS2_TYPE_F32, "cache_write: unknown type %d", type);
  DS2_REQUIRE(format == DS2_CACHE_MXFP8 || format == DS2_CACHE_MXFP4, "cache_write: unknown format %d", format);
  if (!B || !T || !capacity) return DS2_OK;
  DS2_REQUIRE(pos, "cache_write: pos is missing");
  WriteArgs a{};
  for (int i = 0; i < n; ++i) {
    DS2_REQUIRE(x[i].p && codes[i].p && scales[i].p, "cache_write: null pointer");
    DS2_REQUIRE(aligned(x[i], type == DS2_TYPE_F32 ? 4 : 2, 16, 3), "cache_write: input rows must be 16-byte aligned");
    DS2_REQUIRE(aligned(codes[i], 1, 16, 3), "cache_write: code rows must be 16-byte aligned");
    a.x[i] = x[i], a.codes[i] = codes[i], a.scales[i] = scales[i];
  }
  a.pos = pos, a.count = count, a.T = T, a.H = H, a.D = D, a.capacity = capacity;
  DS2_REQUIRE((int64_t)T * (D / 8) < (1ll << 31) - 1024 && (int64_t)B * H < (1ll << 24), "cache_write: too many rows for one call");
  const int64_t per = cdiv64((int64_t)T * (D / 8), 1024), blocks = per * n * B * H;
  DS2_REQUIRE(ds2_launch_holds(blocks, 256), "cache_write: too many rows for one call");
  a.BH = B * H, a.blocks_per_head = (int)per;
  hipStream_t st = (hipStream_t)stream;
#define GO(TY, F) k_cache_write<TY, F><<<dim3((unsigned)blocks), 256, 0, st>>>(a)
#define GO2(TY) format == DS2_CACHE_MXFP8 ? (void)(GO(TY, DS2_CACHE_MXFP8)) : (void)(GO(TY, DS2_CACHE_MXFP4))
  if (type == DS2_TYPE_BF16) { GO2(DS2_TYPE_BF16); } else if (type == DS2_TYPE_F16) { GO2(DS2_TYPE_F16); } else { GO2(DS2_TYPE_F32); }
#undef GO
#undef GO2
  DS2_CHECK_LAUNCH();
  return DS2_OK;
}

extern "C" int ds2_op_cache_read(const ds2_strided* codes, const ds2_strided* scales, const ds2_strided* out, int32_t B, int32_t H,
                                 int32_t C, int32_t D, const int32_t* lens, int32_t type, int32_t format, void* stream) {
  DS2_REQUIRE(codes && scales && out, "cache_read: null argument");
  DS2_REQUIRE(B >= 0 && H >= 1 && C >= 0, "cache_read: bad sizes B %d H %d C %d", B, H, C);
  DS2_REQUIRE(D >= DS2_CACHE_GROUP && D <= 4096 && D % DS2_CACHE_GROUP == 0, "cache_read: head dim %d is not a multiple of 32 up to 4096", D);
  DS2_REQUIRE(type == DS2_TYPE_BF16 || type == DS2_TYPE_F16 || type == DS2_TYPE_F32, "cache_read: unknown type %d", type);
  DS2_REQUIRE(format == DS2_CACHE_MXFP8 || format == DS2_CACHE_MXFP4, "cache_read: unknown format %d", format);
  if (!B || !C) return DS2_OK;
  DS2_REQUIRE(codes->p && scales->p && out->p, "cache_read: null pointer");
  DS2_REQUIRE(aligned(*codes, 1, 16, 3) && aligned(*out, type == DS2_TYPE_F32 ? 4 : 2, 16, 3), "cache_read: rows must be 16-byte aligned");
  ReadArgs a{*codes, *scales, *out, lens, C, H, D, 0, 256 / (D / 8), 256 % (D / 8)};
  DS2_REQUIRE((int64_t)C * (D / 8) < (1ll << 31) - 1024 && (int64_t)B * H < (1ll << 24), "cache_read: too many rows for one call");
  const int64_t per = cdiv64((int64_t)C * (D / 8), 1024), blocks = per * B * H;
  DS2_REQUIRE(ds2_launch_holds(blocks, 256), "cache_read: too many rows for one call");
  a.blocks_per_head = (int)per;
  hipStream_t st = (hipStream_t)stream;
#define GO(TY, F) k_cache_read<TY, F><<<dim3((unsigned)blocks), 256, 0, st>>>(a)
#define GO2(TY) format == DS2_CACHE_MXFP8 ? (void)(GO(TY, DS2_CACHE_MXFP8)) : (void)(GO(TY, DS2_CACHE_MXFP4))
  if (type == DS2_TYPE_BF16) { GO2(DS2_TYPE_BF16); } else if (type == DS2_TYPE_F16) { GO2(DS2_TYPE_F16); } else { GO2(DS2_TYPE_F32); }
#undef GO
#undef GO2
  DS2_CHECK_LAUNCH();
  return DS2_OK;
}
