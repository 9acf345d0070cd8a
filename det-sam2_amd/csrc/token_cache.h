// Formats of the token cache (token_cache.hip, cache_attention.h) and the device helpers that its kernels share.
//
// A quantised row of D values (D a multiple of 32) is D e4m3 bytes or D / 2 bytes of e2m1 pairs (even element in the low half)
// plus one scale byte s for every 32 values: value = code * 2^(s - 127).  s is the smallest power of two (at least 2^-126) for
// which no value of the group exceeds the code's largest one, so nothing saturates and x * 2^(127 - s) is exact: the ONE rounding of
// a value is the conversion to its code (nearest, ties to even).  s = 255: the group held an infinity or a NaN, all of it reads NaN.
#pragma once
#include "common.h"
#include "../../include/detsam2_hip.h"

#define DS2_CACHE_GROUP 32
#define DS2_CAP_WIDE 256.f
// a launch holds fewer than 2^32 threads
inline bool ds2_launch_holds(int64_t blocks, int threads) { return blocks <= 0xffffffffll / threads; }

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
typedef float f32x2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));

// The weights of a row are powers of 2 relative to a running reference.  It is raised when one of them would exceed 2^DS2_LIMIT, and then set so
// that the row's largest weight is 2^DS2_SHIFT: sums and unnormalised results carry that factor, the reference that goes with them says
// so.  bf16 has the exponents of fp32 and needs none.  fp16 ends at 2^16 and loses bits below 2^-14: with weights of 2^11 to 2^15 for
// the largest, 11 bits remain down to 2^-25 of it, and below that no weight is off by more than 2^-36 of it.  (References at the largest score and a
// limit of 2^8: 11 bits down to 2^-14, nothing at all below 2^-25.  Where the largest weight falls on a value of zero and the others are e^-17.5 of
// it, rows were off by 1 to 5 %.)  Raising after 2^4 and not 2^8 costs 3 % where
// a bias lets the scores climb from key to key (4096 rows over 28736 keys, D = 64: 182 -> 187 us); elsewhere it is rare after a row's first keys.
template <bool F16>
constexpr float DS2_SHIFT = F16 ? 11.f : 0.f;
template <bool F16>
constexpr float DS2_LIMIT = F16 ? 15.f : 8.f;

#ifdef __HIPCC__
// two fp32 values -> two 16-bit values in a word (round to nearest even)
template <bool F16>
__device__ __forceinline__ unsigned ds2_pack16(float a, float b) {
  if constexpr (F16) return __builtin_bit_cast(unsigned, __builtin_convertvector((f32x2_t{a, b}), f16x2_t));
  else return __builtin_bit_cast(unsigned, __builtin_convertvector((f32x2_t{a, b}), bf16x2_t));
}
template <bool F16>
__device__ __forceinline__ float ds2_low16(unsigned w) {
  if constexpr (F16) return (float)__builtin_bit_cast(f16x2_t, w)[0];
  else return __builtin_bit_cast(float, w << 16);
}
template <bool F16>
__device__ __forceinline__ float ds2_high16(unsigned w) {
  if constexpr (F16) return (float)__builtin_bit_cast(f16x2_t, w)[1];
  else return __builtin_bit_cast(float, w & 0xffff0000u);
}

// scale byte -> the power of two it stands for; 255 -> NaN.  (0 stands for 2^-127, a subnormal: the writer never leaves it, a cache
// from elsewhere may.)
__device__ __forceinline__ float ds2_cache_scale(unsigned s) {
  const unsigned bits = s == 255u ? 0x7fc00000u : s == 0u ? 0x00400000u : s << 23;
  return __builtin_bit_cast(float, bits);
}

// Scores x scale under a cap, as exponents of 2: cap tanh(x scale / cap) log2 e.  cap - 2 cap / (1 + exp(2 u)) has no branch and saturates by
// itself, but is off by a few 2^-24 of the cap whatever u: good for caps up to DS2_CAP_WIDE (2^-14 there, an eighth of half a step of
// fp16).  Larger caps take the series of tanh below 1/4 (its next term is below 2^-26).
__device__ __forceinline__ float ds2_capped(float x, float in_cap, float cap2) {
  return __builtin_fmaf(-2.f * cap2, __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(x * in_cap)), cap2);
}
__device__ __forceinline__ float ds2_capped_wide(float x, float in_cap, float cap2, float sc) {
  const float u = x * in_cap * 0.34657359f, y = u * u;           // in_cap = 2 log2(e) scale / cap
  const float p = __builtin_fmaf(y, __builtin_fmaf(y, __builtin_fmaf(y, __builtin_fmaf(y, 62.f / 2835.f, -17.f / 315.f), 2.f / 15.f), -1.f / 3.f), 1.f);
  float near = x * sc * p, far = ds2_capped(x, in_cap, cap2);
  asm volatile("" : "+v"(near), "+v"(far));                      // (both, and a selection: no branch that splits the wave)
  return y < 0.0625f ? near : far;
}

// A kernel's arguments are a few lines of memory that no cache of the chip holds when it starts.  Asked for where they are used they
// are misses one after the other; this asks for all of them at once.
template <class Args>
__device__ __forceinline__ void ds2_ask_args(const Args& a) {
  const int* p = (const int*)&a;
  int x = 0;
#pragma unroll
  for (unsigned i = 0; i < sizeof(Args) / 4; i += 16) x ^= p[i];
  asm volatile("" ::"s"(x ^ p[sizeof(Args) / 4 - 1]));
}
#endif
