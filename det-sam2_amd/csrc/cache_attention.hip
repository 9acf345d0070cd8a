// Attention over a token cache: how the keys are split over workgroups, and the C entry points.
// The kernels that read the cache: cache_attention.h.
#include <algorithm>
#include <cmath>

#include "attention_join.h"
#include "attention_masked.h"
#include "cache_attention.h"

namespace {

struct Split {
  int shares, own_rows, own_groups, by_rows, pre_chunk, pre_parts, pre_by_rows;
  bool tiled;                              // the prefix goes to the kernel of whole prompts
  int pre_row_tiles, pre_tiles;            // its tiles of rows, and of keys a part
  int64_t streams, blocks, pre_blocks;
  bool joined() const { return shares || pre_parts; }
  int64_t segments() const { return joined() ? shares + streams : 0; }
};

Split split_of(const ds2_cache_attention_args& a) {
  Split s{};
  const int64_t G = a.Hq / a.Hkv, rows = a.T * G, all_rows = a.B * rows;
  // The waves of a workgroup take different rows over the same keys, or every 16 rows have a workgroup whose waves split the keys.  The
  // first reads a cache once; the second leaves no wave without rows, and what it reads again are codes.  4 streams of 24 rows x 17,
  // D = 128, 4000 tokens, first / second: 16 bits 44 / 53 us, 8 bits 34 / 36, 4 bits 31 / 27; 8 heads of 64 rows, D = 128, 8000 tokens:
  // 57 / 85, 51 / 53, 45 / 38; 32 x 8 of 20 rows, 600 tokens: 28 / 29, 28 / 19, 26 / 17.
  s.by_rows = rows > (a.format == DS2_CACHE_PLAIN ? 16 : a.format == DS2_CACHE_MXFP8 ? 32 : 64);
  s.own_rows = cache_rows(a.D, s.by_rows);
  s.own_groups = (int)cdiv64(rows, s.own_rows);
  s.streams = (int64_t)a.B * a.Hkv * s.own_groups;
  // A workgroup for every stream, or equal shares of all keys, as many as the chip holds workgroups.  Streams of one unit or two are not
  // worth the join; the more streams there are, the less the longest one stands out and the longer a stream may be (uniform 8-bit
  // D = 128, a workgroup a stream against shares: 64 streams of 512 keys 13.3 / 16.5 us, of 1024 17.4 / 18.0 and ragged 17.9 / 15.9;
  // 256 streams of 1024 22.1 / 25.5; 1024 of 2048 98.5 / 114).  Waves over the same keys do not share them out: 8 streams of 497 tokens
  // and 24 rows 20 us whole, 14 in shares.  A stream has at most 128 shares, whose join is as long as their keys (one stream of 100000
  // tokens: 15 us, 24 in 1024 shares).
  const int64_t units = cdiv64(a.capacity, CACHE_UNIT);
  const bool whole = units <= std::max<int64_t>(s.by_rows ? 1 : 4, std::min<int64_t>(16, s.streams / 32));
  s.shares = whole ? 0 : (int)std::min<int64_t>(std::min<int64_t>(256 * cache_residents(a.D), 128 * s.streams), s.streams * (units + 1));
  if (a.prefix_len) {
    // A long prefix of many rows is a matrix product: the kernel of whole prompts takes it, whose key tiles in LDS serve 256 rows (16-bit
    // caches).  It costs a launch and more parts to join, so the product has to be large.
    // 8 key heads, bf16, prompt kernel / this one: D = 64, 128 rows a head behind 32768 tokens 44 / 52 us, 256 54 / 61, 512 behind 8192
    // 38 / 49; D = 128, 128 behind 32768 62 / 69, 256 86 / 114; D = 256, 256 behind 8192 70 / 80; smaller products are left here (of fp16, whose
    // weights are one operand: 39 / 44, 49 / 60, 36 / 44; 57 / 67, 76 / 109; 65 / 74).  One sequence of 64 tokens (256 rows a head, D = 128) behind 32768
    // 88 / 105, of 512 tokens 424 / 736.  (By sizes alone, whatever the queries' strides: the workspace goes by it.)
    const double product = (double)a.Hkv * all_rows * a.prefix_len * a.D;
    s.tiled = a.format == DS2_CACHE_PLAIN && product >= (a.D > 64 ? 3.0e9 : 1.8e9);
    if (s.tiled) {
      s.pre_row_tiles = (int)cdiv64(all_rows, masked_rows(a.D, 1));
      const int tiles = cdiv(a.prefix_len, masked_tile(a.D));
      // as many parts as CUs, of 4 tiles or more (8 up to 64 elements: 256 rows behind 8192 tokens 39 us, 45 in parts of 4)
      s.pre_tiles = (int)std::max<int64_t>(a.D <= 64 ? 8 : 4, cdiv64((int64_t)tiles * a.Hkv * s.pre_row_tiles, 256));
      s.pre_parts = cdiv(tiles, s.pre_tiles);
    } else {
      // Waves of one workgroup on different rows (see above) where the product is large: 8 key heads of 128, first / second: 64 rows
      // behind 8192 tokens 20.5 / 18 us, behind 32768 45 / 49; 256 behind 8192, with up to 512 own tokens each, 50 / 53; 8 bits 256 behind
      // 8000 47 / 39.  A workgroup's keys: a block of 32 for each wave, or for all of them.
      s.pre_by_rows = all_rows >= 64 && all_rows * a.prefix_len >= (a.format == DS2_CACHE_PLAIN ? 1 << 21 : 1 << 22);
      const int64_t streams = (int64_t)a.Hkv * cdiv64(all_rows, cache_rows(a.D, s.pre_by_rows));
      const int64_t least = s.pre_by_rows ? 32 : CACHE_UNIT;
      s.pre_chunk = (int)std::min<int64_t>(2048, std::max<int64_t>(least, cdiv64(cdiv64(a.prefix_len * streams, 256), least) * least));
      s.pre_parts = (int)cdiv64(a.prefix_len, s.pre_chunk);
      s.pre_blocks = streams * s.pre_parts;
    }
  }
  s.blocks = s.pre_blocks + (s.shares ? s.shares : s.streams);
  return s;
}

int64_t up16(int64_t x) { return (x + 15) / 16 * 16; }

// the workspace: segments of the sequences' own keys, where a stream's segments are, parts of the prefix
struct Work {
  int64_t seg_o, seg_ml, seg_of, pre_o, pre_ml, bytes;
};
Work work_of(const ds2_cache_attention_args& a, const Split& s) {
  Work w{};
  if (!s.joined()) return w;
  const int64_t seg = s.segments() * s.own_rows, pre = (int64_t)s.pre_parts * a.B * a.T * a.Hq;
  w.seg_ml = up16(seg * a.D * 4);
  w.seg_of = w.seg_ml + up16(seg * 8);
  w.pre_o = w.seg_of + up16(s.shares ? s.streams * 8 : 0);
  w.pre_ml = w.pre_o + up16(pre * a.D * 4);
  w.bytes = w.pre_ml + up16(pre * 8);
  return w;
}

int check(const ds2_cache_attention_args& a) {
  DS2_REQUIRE(a.B >= 0 && a.T >= 0 && a.capacity >= 0 && a.prefix_len >= 0, "cache_attention: negative size");
  DS2_REQUIRE(a.Hkv >= 1 && a.Hq >= a.Hkv && a.Hq % a.Hkv == 0, "cache_attention: %d query heads do not share %d key heads evenly", a.Hq, a.Hkv);
  DS2_REQUIRE(a.D == 32 || a.D == 64 || a.D == 96 || a.D == 128 || a.D == 256, "cache_attention: unsupported head dim %d (32, 64, 96, 128, 256)", a.D);
  DS2_REQUIRE(a.type == DS2_TYPE_BF16 || a.type == DS2_TYPE_F16, "cache_attention: queries are bf16 or fp16, got type %d", a.type);
  DS2_REQUIRE(a.format == DS2_CACHE_PLAIN || a.format == DS2_CACHE_MXFP8 || a.format == DS2_CACHE_MXFP4, "cache_attention: unknown format %d", a.format);
  DS2_REQUIRE(std::isfinite(a.scale) && std::isfinite(a.cap) && a.cap >= 0.f, "cache_attention: scale and cap must be finite, cap not negative");
  DS2_REQUIRE(a.cap == 0.f || std::fabs(a.scale) <= 1e30f * a.cap, "cache_attention: the cap is too small for the scale");      // (scale / cap is a factor)
  DS2_REQUIRE((int64_t)a.capacity + a.prefix_len < (1ll << 31) - 4096 && a.T < (1 << 20), "cache_attention: too many tokens");
  DS2_REQUIRE((int64_t)a.B * a.T * a.Hq < (1ll << 31) / 256, "cache_attention: too many rows (B T Hq) for one call");
  const Split s = split_of(a);
  DS2_REQUIRE(ds2_launch_holds(s.blocks, 256) && ds2_launch_holds((int64_t)s.pre_row_tiles * a.Hkv * s.pre_parts, 512) && s.streams * (cdiv64(a.capacity, CACHE_UNIT) + 1) < (1ll << 31) - 4096, "cache_attention: too many keys for one call");
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
  return work_of(*args, split_of(*args)).bytes;
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
  a.shares = s.shares, a.direct = !s.joined(), a.own_rows = s.own_rows, a.own_groups = s.own_groups, a.by_rows = s.by_rows;
  a.pre_chunk = s.pre_chunk, a.pre_parts = s.pre_parts, a.pre_by_rows = s.pre_by_rows, a.pre_blocks = (int)s.pre_blocks;
  if (s.joined()) {
    const Work w = work_of(x, s);
    DS2_REQUIRE(work && (uintptr_t)work % 16 == 0 && work_bytes >= w.bytes, "cache_attention: workspace too small");
    char* p = (char*)work;
    a.seg_o = (float*)p, a.seg_ml = (f32x2_t*)(p + w.seg_ml), a.seg_of = (int2*)(p + w.seg_of);
    a.pre_o = (float*)(p + w.pre_o), a.pre_ml = (f32x2_t*)(p + w.pre_ml);
  }
  hipStream_t st = (hipStream_t)stream;
  const bool f16 = x.type == DS2_TYPE_F16;
  const unsigned blocks = (unsigned)s.blocks;
  if (s.tiled) {
    MaskedArgs m{};
    m.q = a.q, m.k = (const char*)a.pk, m.v = (const char*)a.pv, m.out = a.out;
    m.q_b = a.q_b, m.q_t = a.q_t, m.q_h = a.q_h;
    m.k_t = a.pk_c, m.k_h = a.pk_h, m.v_t = a.pv_c, m.v_h = a.pv_h;
    m.slopes = a.slopes, m.row_lens = x.lens, m.row_T = x.T, m.row_C = x.capacity;
    m.B = 1, m.Lq = x.B * x.T, m.Lk = x.prefix_len, m.Hq = x.Hq, m.Hkv = x.Hkv, m.G = a.G, m.D = x.D;
    m.scale = x.scale, m.cap = x.cap;
    m.key_groups = 1, m.row_tiles = s.pre_row_tiles, m.heads = x.Hkv, m.parts = s.pre_parts, m.tiles_a_part = s.pre_tiles;
    m.part_o = a.pre_o, m.part_ml = a.pre_ml;
    const unsigned tiles = (unsigned)(s.pre_row_tiles * x.Hkv * s.pre_parts);
    // (bf16: weights of 16 bits like those over the sequences' own keys, so that a result's precision does not go by the prefix's size)
    const int mode = masked_mode(x.scale, x.cap, x.slopes);
    DS2_TRY(f16 ? launch_masked_f16(m, mode, tiles, st) : launch_masked_bf16_wide(m, mode, tiles, st));
  }
  DS2_TRY(x.format == DS2_CACHE_PLAIN ? launch_cache_attn_plain(a, f16, blocks, st)
          : x.format == DS2_CACHE_MXFP8 ? launch_cache_attn_mxfp8(a, f16, blocks, st)
                                        : launch_cache_attn_mxfp4(a, f16, blocks, st));
  if (s.joined()) {
    AttnJoinArgs j{};
    j.out = a.out, j.rows = (int64_t)x.B * x.T * x.Hq, j.D = x.D;
    j.o = a.pre_o, j.ml = a.pre_ml, j.parts = a.pre_parts;
    j.seg_o = a.seg_o, j.seg_ml = a.seg_ml, j.seg_of = a.seg_of, j.lens = x.lens;
    j.T = x.T, j.Hq = x.Hq, j.G = a.G, j.C = x.capacity, j.shares = a.shares, j.own_rows = a.own_rows, j.own_groups = a.own_groups;
    return launch_attn_join(j, f16, s.pre_parts + std::min<int64_t>(s.shares / s.streams + (s.shares ? 2 : 1), cdiv64(x.capacity, CACHE_UNIT)), st);
  }
  return DS2_OK;
}
