// Attention over a token cache: how the keys are split over workgroups, and the C entry points.
// The kernels that read the cache: cache_attention.h.
#include <algorithm>
#include <cmath>

#include "attention_join.h"
#include "cache_attention.h"

namespace {

struct Split {
  int own_chunk, own_parts, own_groups, pre_chunk, pre_parts, pre_groups, pre_rows;
  bool two_tiles;
  int64_t blocks, pre_blocks;
  int64_t parts() const { return (int64_t)own_parts + pre_parts; }
};

int round_up(int64_t x, int to) { return (int)((x + to - 1) / to * to); }

Split split_of(const ds2_cache_attention_args& a) {
  Split s{};
  const int64_t G = a.Hq / a.Hkv, own_rows = a.T * G, all_rows = a.B * own_rows;
  // Two tiles of 16 rows a wave where the rows of a call fill them (and a head's 128 values leave the registers for it).
  s.two_tiles = a.D <= 128 && (own_rows > 16 || (a.prefix_len && all_rows > 16));
  const int tile = s.two_tiles ? 32 : 16;
  s.own_groups = (int)cdiv64(own_rows, tile);
  const int64_t streams = (int64_t)a.B * a.Hkv * s.own_groups;
  s.own_chunk = std::min(2048, std::max(128, round_up(cdiv64(a.capacity * streams, 2048), 128)));
  s.own_parts = std::max(1, (int)cdiv64(a.capacity, s.own_chunk));
  if (a.prefix_len) {
    s.pre_rows = all_rows > tile;
    s.pre_groups = (int)cdiv64(all_rows, s.pre_rows ? 4 * tile : tile);
    const int64_t pre_streams = (int64_t)a.Hkv * s.pre_groups;
    s.pre_chunk = std::min(2048, std::max(128, round_up(cdiv64(a.prefix_len * pre_streams, 256), 32)));
    s.pre_parts = (int)cdiv64(a.prefix_len, s.pre_chunk);
    s.pre_blocks = pre_streams * s.pre_parts;
  }
  s.blocks = s.pre_blocks + streams * s.own_parts;
  return s;
}

int check(const ds2_cache_attention_args& a) {
  DS2_REQUIRE(a.B >= 0 && a.T >= 0 && a.capacity >= 0 && a.prefix_len >= 0, "cache_attention: negative size");
  DS2_REQUIRE(a.Hkv >= 1 && a.Hq >= a.Hkv && a.Hq % a.Hkv == 0, "cache_attention: %d query heads do not share %d key heads evenly", a.Hq, a.Hkv);
  DS2_REQUIRE(a.D == 32 || a.D == 64 || a.D == 96 || a.D == 128 || a.D == 256, "cache_attention: unsupported head dim %d (32, 64, 96, 128, 256)", a.D);
  DS2_REQUIRE(a.type == DS2_TYPE_BF16 || a.type == DS2_TYPE_F16, "cache_attention: queries are bf16 or fp16, got type %d", a.type);
  DS2_REQUIRE(a.format == DS2_CACHE_PLAIN || a.format == DS2_CACHE_MXFP8 || a.format == DS2_CACHE_MXFP4, "cache_attention: unknown format %d", a.format);
  DS2_REQUIRE(std::isfinite(a.scale) && std::isfinite(a.cap) && a.cap >= 0.f, "cache_attention: scale and cap must be finite, cap not negative");
  DS2_REQUIRE((int64_t)a.capacity + a.prefix_len < (1ll << 31) - 4096 && a.T < (1 << 20), "cache_attention: too many tokens");
  DS2_REQUIRE((int64_t)a.B * a.T * a.Hq < (1ll << 31) / 256, "cache_attention: too many rows (B T Hq) for one call");
  return DS2_OK;
}

// strides of a cache tensor in bytes; token stride fits 31 bits over a block of 32
int cache_rows(const ds2_strided& t, int size, int to, const char* name) {
  DS2_REQUIRE(t.p, "cache_attention: %s is missing", name);
  DS2_REQUIRE((uintptr_t)t.p % to == 0 && t.s0 * size % to == 0 && t.s1 * size % to == 0 && t.s2 * size % to == 0,
              "cache_attention: rows of %s must be %d-byte aligned", name, to);
  DS2_REQUIRE(t.s2 >= 0 && t.s2 * size < (1 << 25), "cache_attention: token stride of %s out of range", name);
  return DS2_OK;
}
#define DS2_TRY(x)        \
  do {                    \
    const int rc_ = (x);  \
    if (rc_) return rc_;  \
  } while (0)

}  // namespace

extern "C" int64_t ds2_op_cache_attention_work_bytes(const ds2_cache_attention_args* args) {
  if (!args || check(*args) || !args->B || !args->T) return 0;
  const Split s = split_of(*args);
  if (s.parts() <= 1) return 0;
  return s.parts() * args->B * args->T * args->Hq * ((int64_t)args->D + 2) * 4;
}

extern "C" int ds2_op_cache_attention(const ds2_cache_attention_args* args, void* work, int64_t work_bytes, void* stream) {
  DS2_REQUIRE(args, "cache_attention: null argument");
  const ds2_cache_attention_args& x = *args;
  DS2_TRY(check(x));
  if (!x.B || !x.T) return DS2_OK;
  DS2_REQUIRE(x.q.p && x.out && x.lens, "cache_attention: null pointer");
  const bool mx = x.format != DS2_CACHE_PLAIN;
  const int size = mx ? 1 : 2;
  CacheAttnArgs a{};
  DS2_REQUIRE((uintptr_t)x.q.p % 16 == 0 && x.q.s0 % 8 == 0 && x.q.s1 % 8 == 0 && x.q.s2 % 8 == 0 && (uintptr_t)x.out % 16 == 0,
              "cache_attention: query and output rows must be 16-byte aligned");
  a.q = (const char*)x.q.p, a.q_b = x.q.s0 * 2, a.q_t = x.q.s1 * 2, a.q_h = x.q.s2 * 2;
  a.out = (char*)x.out;
#define ROWS(src, size, to, dst)                                                                       \
  DS2_TRY(cache_rows(x.src, size, to, #src));                                                          \
  a.dst = (const uint8_t*)x.src.p, a.dst##_h = x.src.s1 * (size), a.dst##_c = (unsigned)(x.src.s2 * (size));
  if (x.capacity) {
    ROWS(k, size, 16, k) ROWS(v, size, 16, v)
    a.k_b = x.k.s0 * size, a.v_b = x.v.s0 * size;
    if (mx) {
      ROWS(k_scales, 1, 1, ks) ROWS(v_scales, 1, 1, vs)
      a.ks_b = x.k_scales.s0, a.vs_b = x.v_scales.s0;
    }
  }
  if (x.prefix_len) {
    ROWS(prefix_k, size, 16, pk) ROWS(prefix_v, size, 16, pv)
    if (mx) { ROWS(prefix_k_scales, 1, 1, pks) ROWS(prefix_v_scales, 1, 1, pvs) }
  }
#undef ROWS
  a.lens = x.lens, a.slopes = x.slopes;
  a.B = x.B, a.T = x.T, a.Hq = x.Hq, a.Hkv = x.Hkv, a.G = x.Hq / x.Hkv, a.D = x.D, a.C = x.capacity, a.P = x.prefix_len;
  a.scale = x.scale, a.cap = x.cap;
  const Split s = split_of(x);
  DS2_REQUIRE(s.blocks < (1ll << 31), "cache_attention: too many sequences for one call");
  a.own_chunk = s.own_chunk, a.own_parts = s.own_parts, a.own_groups = s.own_groups;
  a.pre_chunk = s.pre_chunk, a.pre_parts = s.pre_parts, a.pre_groups = s.pre_groups, a.pre_rows = s.pre_rows, a.pre_blocks = (int)s.pre_blocks;
  const int64_t rows = (int64_t)x.B * x.T * x.Hq;
  if (s.parts() > 1) {
    DS2_REQUIRE(work && (uintptr_t)work % 16 == 0 && work_bytes >= ds2_op_cache_attention_work_bytes(args), "cache_attention: workspace too small");
    a.part_o = (float*)work;
    a.part_ml = (f32x2_t*)(a.part_o + s.parts() * rows * x.D);
  }
  hipStream_t st = (hipStream_t)stream;
  const bool f16 = x.type == DS2_TYPE_F16;
  const unsigned blocks = (unsigned)s.blocks;
  DS2_TRY(x.format == DS2_CACHE_PLAIN ? launch_cache_attn_plain(a, f16, s.two_tiles, blocks, st)
          : x.format == DS2_CACHE_MXFP8 ? launch_cache_attn_mxfp8(a, f16, s.two_tiles, blocks, st)
                                        : launch_cache_attn_mxfp4(a, f16, s.two_tiles, blocks, st));
  if (s.parts() > 1) {
    AttnJoinArgs j{a.part_o, a.part_ml, a.out, rows, x.D, (int)s.parts(), x.lens, x.T, x.Hq, x.capacity, a.pre_parts, a.own_chunk};
    DS2_TRY(launch_attn_join(j, f16, j.parts, st));
  }
  return DS2_OK;
}
