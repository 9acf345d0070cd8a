// Masked attention of whole prompts: how rows and keys are split over workgroups, the documents of key tiles, and the C entry
// points.  The kernels: attention_masked.h.
#include <algorithm>
#include <cmath>

#include "attention_join.h"
#include "attention_masked.h"

namespace {

template <int KT>
__global__ __launch_bounds__(64) void k_tile_docs(const int32_t* doc, int Lk, int tiles, int2* out) {
  const int b = blockIdx.x / tiles, t = blockIdx.x - b * tiles, j = t * KT + threadIdx.x % KT;
  int lo = j < Lk ? max(-1, doc[(int64_t)b * Lk + j]) : -1, hi = lo;
#pragma unroll
  for (int s = 1; s < KT; s <<= 1) {
    lo = min(lo, __shfl_xor(lo, s));
    hi = max(hi, __shfl_xor(hi, s));
  }
  if (threadIdx.x == 0) out[(int64_t)b * tiles + t] = int2{lo, hi};
}

struct Plan {
  int key_groups, row_tiles, heads, parts, tiles, tiles_a_part;
  int64_t blocks, doc_bytes, part_bytes;
};

Plan plan_of(const ds2_attention_masked_args& a) {
  Plan p{};
  const int64_t rows = (int64_t)(a.Hq / a.Hkv) * a.Lq;
  p.heads = a.B * a.Hkv;
  p.tiles = cdiv(a.Lk, masked_tile(a.D));
  // How many rows a workgroup takes (the waves of half as many split its keys) and whether the keys are split over workgroups:
  // whatever takes least time by this model.  A step of 32 keys takes a workgroup 0.8 us up to 64 elements a row (two on a CU 1.3), 1.0 up
  // to 96, 1.15 up to 128, 1.8 up to 256, and a quarter more with its keys split over waves (every step has a barrier); the call takes as
  // long as the longest workgroup or the work of a CU; parts cost a join, 7 us and what they write and read at 4 TB/s.  Measured, rows
  // whole / keys split over waves: 32 over 8 heads, D = 128, causal 1024 tokens 39 / 30 us, 2048 tokens 75 / 61, four times 2048
  // of 16 over 8 heads 98 / 123; D = 96, twice 2500 tokens of 8 over 4 heads 71 / 51.  Parts: 4 over 1 heads, D = 64, 4096 tokens over
  // 28736 in eight parts 175 us, two 332; the 1024 tokens above in one part 39, four 60.  More than 64 parts, up to as many as CUs, where each
  // keeps 1024 keys (64 / as many as CUs): 16 tokens of 4 over 1 heads, D = 64, over 2^20 keys 258 / 83 us; 64 tokens, D = 128, over 2^18
  // 94 / 65; 16 of 8 over 2 heads, D = 128, over 2^18 93 / 63.  Shorter parts gain nothing (64 tokens of 8 over 1 heads, D = 128, over 2^16
  // 38.5 / 37; 77 of 4 over 2, D = 64, over 40000 23.7 / 23.4).
  const double part_us = (double)a.B * a.Lq * a.Hq * a.D * 8 / 4e6, step_us = a.D > 128 ? 1.8 : a.D > 96 ? 1.15 : a.D > 64 ? 1.0 : 0.8;
  const double seen = a.causal && a.Lk ? 1 - 0.5 * std::min(1.0, (double)a.Lq / a.Lk) : 1;      // of all pairs
  // Tiles of a row.  How long documents are is known to the device only, which splits what a tile of rows can see; half of all keys is
  // between one document and many (6073 tokens in 7 documents, 2 heads of 64: planned for all 66 us, half 38; 4274 in 2, 4 heads: 41,
  // 36, and 61 for a quarter).
  const int reach = a.q_doc ? cdiv(p.tiles, 2) : p.tiles;
  double best = 1e300;
  p.parts = p.key_groups = 1;
  for (int kg = 1; kg <= (a.D <= 128 ? 2 : 1); ++kg) {
    const int64_t whole = cdiv64(rows, masked_rows(a.D, kg)) * p.heads;
    const int most = whole < 256 ? std::max(1, std::max(std::min(reach / 2, 64), std::min((int)cdiv64(256, whole), reach * masked_tile(a.D) / 1024))) : 1;
    for (int n = 1; n <= most; n += 1 + n / 8) {
      const double longest = (double)cdiv(reach, n) * (masked_tile(a.D) / 32) / kg;
      const double on_cu = seen < 1 ? whole * n / 256.0 : (double)cdiv64(whole * n, 256);
      const double steps = std::max(longest, longest * seen * on_cu * (a.D <= 64 && on_cu > 1 ? 0.81 : 1));
      const double us = steps * step_us * (kg > 1 ? 1.25 : 1) + (n > 1 ? 7 + n * part_us : 0);
      if (us < best) best = us, p.parts = n, p.key_groups = kg;
    }
  }
  p.row_tiles = (int)cdiv64(rows, masked_rows(a.D, p.key_groups));
  const int64_t whole = (int64_t)p.row_tiles * p.heads;
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
  DS2_REQUIRE(a.cap == 0.f || std::fabs(a.scale) <= 1e30f * a.cap, "attention_masked: the cap is too small for the scale");      // (scale / cap is a factor)
  DS2_REQUIRE((!a.q_doc) == (!a.k_doc) || !a.Lk, "attention_masked: q_doc and k_doc go together");      // (no keys: the documents of none are nowhere)
  DS2_REQUIRE(a.causal || !a.prefix, "attention_masked: a prefix goes with the causal mask");
  DS2_REQUIRE(a.Lk < (1 << 30) && a.Lq < (1 << 30) && (int64_t)(a.Hq / a.Hkv) * a.Lq < (1ll << 31) - 512, "attention_masked: sequence too long");
  DS2_REQUIRE((int64_t)a.B * a.Hkv < (1 << 24) && (int64_t)a.B * a.Lq * a.Hq < (1ll << 32), "attention_masked: too many rows for one call");
  return DS2_OK;
}

int aligned(const ds2_strided& t, const char* name) {
  DS2_REQUIRE(t.p && (uintptr_t)t.p % 16 == 0 && t.s0 % 8 == 0 && t.s1 % 8 == 0 && t.s2 % 8 == 0, "attention_masked: rows of %s must be 16-byte aligned", name);
  DS2_REQUIRE(t.s1 >= 0 && t.s1 < (1 << 23), "attention_masked: token stride of %s out of range", name);
  return DS2_OK;
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
  DS2_REQUIRE(ds2_launch_holds(p.blocks, 512), "attention_masked: too many rows for one call");
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
  a.key_groups = p.key_groups, a.row_tiles = p.row_tiles, a.heads = p.heads, a.parts = p.parts, a.tiles = p.tiles, a.tiles_a_part = p.tiles_a_part;
  a.fold = x.causal && x.D <= 64 && p.blocks <= 512;
  hipStream_t st = (hipStream_t)stream;
  if (x.q_doc && p.tiles) {
    int2* docs = (int2*)work;
    DS2_REQUIRE(ds2_launch_holds((int64_t)x.B * p.tiles, 64), "attention_masked: too many keys for one call");
    if (masked_tile(x.D) == 64) k_tile_docs<64><<<dim3((unsigned)(x.B * p.tiles)), 64, 0, st>>>(x.k_doc, x.Lk, p.tiles, docs);
    else k_tile_docs<32><<<dim3((unsigned)(x.B * p.tiles)), 64, 0, st>>>(x.k_doc, x.Lk, p.tiles, docs);
    DS2_CHECK_LAUNCH();
    a.tile_docs = docs;
  }
  const int64_t rows = (int64_t)x.B * x.Lq * x.Hq;
  if (p.parts > 1) {
    a.part_o = (float*)((char*)work + p.doc_bytes);
    a.part_ml = (f32x2_t*)(a.part_o + (int64_t)p.parts * rows * x.D);
  }
  const bool f16 = x.type == DS2_TYPE_F16;
  const int mode = masked_mode(x.scale, x.cap, x.slopes);
  if (const int rc = f16 ? launch_masked_f16(a, mode, (unsigned)p.blocks, st) : launch_masked_bf16(a, mode, (unsigned)p.blocks, st)) return rc;
  if (p.parts > 1) {
    AttnJoinArgs j{};
    j.o = a.part_o, j.ml = a.part_ml, j.out = a.out, j.rows = rows, j.D = x.D, j.parts = p.parts;
    return launch_attn_join(j, f16, p.parts, st);
  }
  return DS2_OK;
}
