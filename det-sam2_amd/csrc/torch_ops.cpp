// PyTorch-ROCm custom ops over the C-ABI: TORCH_LIBRARY(det_sam2, m).
//
// The north-star asks for the HIP stages to be "called from Python via PyTorch-ROCm custom ops"; the reference's own
// native precedent is a torch extension (sam2/csrc/connected_components.cu:284-289, pybind `get_connected_componnets`).
// This file is host-only C++ (no device code): every op checks its at::Tensor arguments (device, dtype, shape,
// contiguity), allocates its outputs with ATen on the inputs' device, takes the CURRENT HIP stream of that device from
// c10 and forwards to the extern "C" entry point of include/detsam2_hip.h - the C-ABI stays the one stable boundary, the
// ops add dispatcher visibility (torch.ops.det_sam2.*), tensor-lifetime safety (no raw data_ptr in Python) and stream
// correctness by construction.  A ds2_model travels as an int64 handle (the pointer ds2_model_create returned).
// Built into det-sam2_amd/lib/libdetsam2_torch.so by __graft_entry__.build(); loaded with torch.ops.load_library.
#include <ATen/ATen.h>
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>   // PyTorch-ROCm tensors carry DeviceType::CUDA ("HIP masquerading as
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>      // CUDA"): guard / current stream come from the masquerading forms
#include <torch/library.h>

#include <algorithm>
#include <array>
#include <cmath>
#include <tuple>
#include <vector>

#include "../../include/detsam2_hip.h"

namespace {

using at::Tensor;

ds2_model* model_of(int64_t h) {
  TORCH_CHECK(h != 0, "det_sam2: null model handle");
  return reinterpret_cast<ds2_model*>(static_cast<intptr_t>(h));
}
void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.get_device()).stream(); }
void check(int rc, const char* what) {
  TORCH_CHECK(rc == DS2_OK, "det_sam2::", what, " failed (code ", rc, "): ", ds2_last_error());   // c10::Error -> RuntimeError
}
void want(const Tensor& t, at::ScalarType dt, const char* name) {
  TORCH_CHECK(t.is_cuda(), "det_sam2: ", name, " must be a GPU tensor");
  TORCH_CHECK(t.scalar_type() == dt, "det_sam2: ", name, " must be ", toString(dt), ", got ", toString(t.scalar_type()));
  TORCH_CHECK(t.is_contiguous(), "det_sam2: ", name, " must be contiguous");
}
const float* fptr(const c10::optional<Tensor>& t) { return t.has_value() ? t->data_ptr<float>() : nullptr; }

constexpr int64_t TOK = 4096;

// A3: load_video_frames (sam2/utils/misc.py:280-284,328-342,358-359)
Tensor ingest_frames(int64_t model, const Tensor& frames_u8) {
  want(frames_u8, at::kByte, "frames_u8");
  TORCH_CHECK(frames_u8.dim() == 4 && frames_u8.size(3) == 3, "det_sam2::ingest_frames: frames_u8 must be [n,H,W,3]");
  c10::hip::HIPGuardMasqueradingAsCUDA g(frames_u8.device());
  const int64_t n = frames_u8.size(0);
  Tensor out = at::empty({n, 3, 1024, 1024}, frames_u8.options().dtype(at::kHalf));
  check(ds2_ingest_frames(model_of(model), frames_u8.data_ptr<uint8_t>(), (int32_t)n, (int32_t)frames_u8.size(1),
                          (int32_t)frames_u8.size(2), reinterpret_cast<uint16_t*>(out.data_ptr()), stream_of(frames_u8)),
        "ingest_frames");
  return out;
}

// A4 + A5: SAM2Base.forward_image (sam2_base.py:450-461), n frames per launch
std::tuple<Tensor, Tensor, Tensor> image_encoder(int64_t model, const Tensor& frames) {
  TORCH_CHECK(frames.dim() == 4 && frames.size(1) == 3, "det_sam2::image_encoder: frames must be [n,3,S,S]");
  TORCH_CHECK(frames.scalar_type() == at::kHalf || frames.scalar_type() == at::kFloat, "det_sam2::image_encoder: fp16 or fp32 frames");
  want(frames, frames.scalar_type(), "frames");
  c10::hip::HIPGuardMasqueradingAsCUDA g(frames.device());
  const int64_t n = frames.size(0);
  auto o = frames.options().dtype(at::kFloat);
  Tensor f0 = at::empty({n, 65536, 32}, o), f1 = at::empty({n, 16384, 64}, o), f2 = at::empty({n, TOK, 256}, o);
  if (frames.scalar_type() == at::kHalf)
    check(ds2_image_encoder_batch(model_of(model), reinterpret_cast<const uint16_t*>(frames.data_ptr()), (int32_t)n,
                                  f0.data_ptr<float>(), f1.data_ptr<float>(), f2.data_ptr<float>(), stream_of(frames)), "image_encoder");
  else
    check(ds2_image_encoder_f32(model_of(model), frames.data_ptr<float>(), (int32_t)n, f0.data_ptr<float>(), f1.data_ptr<float>(),
                                f2.data_ptr<float>(), stream_of(frames)), "image_encoder");
  return {f0, f1, f2};
}

// the entry tables of a bank as the C-ABI takes them (host arrays of device pointers)
struct BankTables {
  std::vector<const void*> fp;
  std::vector<int32_t> rows;
  std::vector<const float*> pp;
  std::vector<float> pos;
};
static BankTables bank_tables(int64_t B, at::TensorList feats, at::IntArrayRef tpos_rows, at::TensorList ptrs, at::ArrayRef<double> ptr_pos,
                              const char* who) {
  TORCH_CHECK(feats.size() == tpos_rows.size() && ptrs.size() == ptr_pos.size(), "det_sam2::", who, ": table lengths differ");
  TORCH_CHECK(feats.size() + ptrs.size() > 0, "det_sam2::", who, ": empty bank");
  BankTables t;
  for (size_t i = 0; i < feats.size(); ++i) {
    want(feats[i], at::kBFloat16, "feats[i]");
    TORCH_CHECK(feats[i].dim() == 3 && feats[i].size(0) == B && feats[i].size(1) == TOK && feats[i].size(2) == 64,
                "det_sam2::", who, ": feats[i] must be bf16 [B,4096,64]");
    t.fp.push_back(feats[i].data_ptr());
    t.rows.push_back((int32_t)tpos_rows[i]);
  }
  for (size_t i = 0; i < ptrs.size(); ++i) {
    want(ptrs[i], at::kFloat, "ptrs[i]");
    TORCH_CHECK(ptrs[i].dim() == 2 && ptrs[i].size(0) == B && ptrs[i].size(1) == 256, "det_sam2::", who, ": ptrs[i] must be fp32 [B,256]");
    t.pp.push_back(ptrs[i].data_ptr<float>());
    t.pos.push_back((float)ptr_pos[i]);
  }
  return t;
}

// A11: tensor part of _prepare_memory_conditioned_features (sam2_base.py:565-648)
std::tuple<Tensor, Tensor> bank_assemble(int64_t model, int64_t B, at::TensorList feats, at::IntArrayRef tpos_rows,
                                         at::TensorList ptrs, at::ArrayRef<double> ptr_pos) {
  BankTables t = bank_tables(B, feats, tpos_rows, ptrs, ptr_pos, "bank_assemble");
  const Tensor& any = feats.size() ? feats[0] : ptrs[0];
  c10::hip::HIPGuardMasqueradingAsCUDA g(any.device());
  const int64_t nk = (int64_t)feats.size() * TOK + 4 * (int64_t)ptrs.size();
  auto o = any.options().dtype(at::kFloat);
  Tensor mem = at::empty({B, nk, 64}, o), mpos = at::empty({B, nk, 64}, o);
  check(ds2_bank_assemble(model_of(model), (int32_t)B, (int32_t)t.fp.size(), t.fp.data(), t.rows.data(), (int32_t)t.pp.size(), t.pp.data(),
                          t.pos.data(), mem.data_ptr<float>(), mpos.data_ptr<float>(), stream_of(any)), "bank_assemble");
  return {mem, mpos};
}

// A11 + A12 in one call (the tracking loop): the bank's entries -> memory-conditioned features [B,4096,256]; curr [4096,256] shared
Tensor bank_memory_attention(int64_t model, int64_t B, const Tensor& curr, at::TensorList feats, at::IntArrayRef tpos_rows,
                             at::TensorList ptrs, at::ArrayRef<double> ptr_pos) {
  want(curr, at::kFloat, "curr");
  TORCH_CHECK(curr.dim() == 2 && curr.size(0) == TOK && curr.size(1) == 256, "det_sam2::bank_memory_attention: curr must be [4096,256]");
  BankTables t = bank_tables(B, feats, tpos_rows, ptrs, ptr_pos, "bank_memory_attention");
  c10::hip::HIPGuardMasqueradingAsCUDA g(curr.device());
  Tensor out = at::empty({B, TOK, 256}, curr.options());
  check(ds2_bank_memory_attention(model_of(model), (int32_t)B, curr.data_ptr<float>(), (int32_t)t.fp.size(), t.fp.data(), t.rows.data(),
                                  (int32_t)t.pp.size(), t.pp.data(), t.pos.data(), out.data_ptr<float>(), stream_of(curr)),
        "bank_memory_attention");
  return out;
}

// A12: MemoryAttention.forward (memory_attention.py:119-176).  curr [4096,256] shared by the B objects or [B,4096,256];
// curr_pos None = the model's constant position encoding, else [4096,256] / [B,4096,256].
Tensor memory_attention(int64_t model, int64_t B, const Tensor& curr, const c10::optional<Tensor>& curr_pos, const Tensor& memory,
                        const Tensor& memory_pos, int64_t num_obj_ptr_tokens) {
  want(curr, at::kFloat, "curr");
  want(memory, at::kFloat, "memory");
  want(memory_pos, at::kFloat, "memory_pos");
  TORCH_CHECK(memory.dim() == 3 && memory.size(0) == B && memory.size(2) == 64 && memory_pos.sizes() == memory.sizes(),
              "det_sam2::memory_attention: memory / memory_pos must be fp32 [B,Nk,64]");
  const bool curr_shared = curr.dim() == 2;
  TORCH_CHECK((curr_shared && curr.size(0) == TOK && curr.size(1) == 256) ||
              (curr.dim() == 3 && curr.size(0) == B && curr.size(1) == TOK && curr.size(2) == 256),
              "det_sam2::memory_attention: curr must be [4096,256] or [B,4096,256]");
  bool pos_shared = true;
  if (curr_pos.has_value()) {
    want(*curr_pos, at::kFloat, "curr_pos");
    pos_shared = curr_pos->dim() == 2;
    TORCH_CHECK(curr_pos->numel() == (pos_shared ? 1 : B) * TOK * 256, "det_sam2::memory_attention: bad curr_pos shape");
  }
  c10::hip::HIPGuardMasqueradingAsCUDA g(curr.device());
  Tensor out = at::empty({B, TOK, 256}, curr.options());
  check(ds2_memory_attention_ex(model_of(model), (int32_t)B, curr.data_ptr<float>(), curr_shared ? 1 : 0, fptr(curr_pos),
                                pos_shared ? 1 : 0, memory.data_ptr<float>(), memory_pos.data_ptr<float>(), (int32_t)memory.size(1),
                                (int32_t)num_obj_ptr_tokens, out.data_ptr<float>(), stream_of(curr)), "memory_attention");
  return out;
}

// A7 + A8: SAM2Base._forward_sam_heads (sam2_base.py:254-397) -> (low_res [B,256,256], obj_ptr [B,256], obj_logits [B], ious [B])
std::tuple<Tensor, Tensor, Tensor, Tensor> sam_heads(int64_t model, int64_t B, const Tensor& pix_feat, bool pix_bcast, bool add_no_mem_embed,
                                                     const Tensor& fpn0, const Tensor& fpn1, const c10::optional<Tensor>& point_coords,
                                                     const c10::optional<Tensor>& point_labels, const c10::optional<Tensor>& mask_inputs,
                                                     bool multimask) {
  want(pix_feat, at::kFloat, "pix_feat");
  want(fpn0, at::kFloat, "fpn0");
  want(fpn1, at::kFloat, "fpn1");
  TORCH_CHECK(pix_feat.numel() == (pix_bcast ? 1 : B) * TOK * 256, "det_sam2::sam_heads: pix_feat must be [B,4096,256] ([4096,256] with pix_bcast)");
  TORCH_CHECK(fpn0.numel() == 65536 * 32 && fpn1.numel() == 16384 * 64, "det_sam2::sam_heads: fpn0 [65536,32] / fpn1 [16384,64] expected");
  TORCH_CHECK(point_coords.has_value() == point_labels.has_value(), "det_sam2::sam_heads: point_coords and point_labels go together");
  int64_t P = 0;
  const int32_t* labels = nullptr;
  if (point_coords.has_value()) {
    want(*point_coords, at::kFloat, "point_coords");
    want(*point_labels, at::kInt, "point_labels");
    TORCH_CHECK(point_coords->dim() == 3 && point_coords->size(0) == B && point_coords->size(2) == 2 && point_labels->dim() == 2 &&
                point_labels->size(0) == B && point_labels->size(1) == point_coords->size(1),
                "det_sam2::sam_heads: point_coords [B,P,2] / point_labels [B,P] expected");
    P = point_coords->size(1);
    labels = point_labels->data_ptr<int32_t>();
  }
  if (mask_inputs.has_value()) {
    want(*mask_inputs, at::kFloat, "mask_inputs");
    TORCH_CHECK(mask_inputs->numel() == B * 256 * 256, "det_sam2::sam_heads: mask_inputs must be [B,256,256]");
  }
  c10::hip::HIPGuardMasqueradingAsCUDA g(pix_feat.device());
  auto o = pix_feat.options();
  Tensor low = at::empty({B, 256, 256}, o), ptr = at::empty({B, 256}, o), obj = at::empty({B}, o), iou = at::empty({B}, o);
  check(ds2_sam_heads_mask(model_of(model), (int32_t)B, pix_feat.data_ptr<float>(), pix_bcast ? 1 : 0, add_no_mem_embed ? 1 : 0,
                           fpn0.data_ptr<float>(), fpn1.data_ptr<float>(), P ? fptr(point_coords) : nullptr, P ? labels : nullptr, (int32_t)P,
                           fptr(mask_inputs), multimask ? 1 : 0, low.data_ptr<float>(), ptr.data_ptr<float>(), obj.data_ptr<float>(),
                           iou.data_ptr<float>(), stream_of(pix_feat)), "sam_heads");
  return {low, ptr, obj, iou};
}

// A7: PromptEncoder.forward (prompt_encoder.py:134-171) -> (sparse [B,Ns,256], dense [B,4096,256] token-major)
std::tuple<Tensor, Tensor> prompt_encoder(int64_t model, int64_t B, const c10::optional<Tensor>& point_coords,
                                          const c10::optional<Tensor>& point_labels, bool pad, const c10::optional<Tensor>& mask_inputs,
                                          const Tensor& like) {
  TORCH_CHECK(like.is_cuda() && B > 0, "det_sam2::prompt_encoder: `like` must be a device tensor");
  TORCH_CHECK(point_coords.has_value() == point_labels.has_value(), "det_sam2::prompt_encoder: point_coords and point_labels go together");
  int64_t P = 0;
  const int32_t* labels = nullptr;
  if (point_coords.has_value()) {
    want(*point_coords, at::kFloat, "point_coords");
    want(*point_labels, at::kInt, "point_labels");
    TORCH_CHECK(point_coords->dim() == 3 && point_coords->size(0) == B && point_coords->size(2) == 2 && point_labels->dim() == 2 &&
                point_labels->size(0) == B && point_labels->size(1) == point_coords->size(1),
                "det_sam2::prompt_encoder: point_coords [B,P,2] / point_labels [B,P] expected");
    P = point_coords->size(1);
    labels = point_labels->data_ptr<int32_t>();
  }
  if (mask_inputs.has_value()) {
    want(*mask_inputs, at::kFloat, "mask_inputs");
    TORCH_CHECK(mask_inputs->numel() == B * 256 * 256, "det_sam2::prompt_encoder: mask_inputs must be [B,256,256]");
  }
  c10::hip::HIPGuardMasqueradingAsCUDA g(like.device());
  auto o = like.options().dtype(at::kFloat);
  const int64_t Ns = P ? P + (pad ? 1 : 0) : 0;
  Tensor sparse = at::empty({B, Ns, 256}, o), dense = at::empty({B, TOK, 256}, o);
  check(ds2_prompt_encoder(model_of(model), (int32_t)B, P ? fptr(point_coords) : nullptr, P ? labels : nullptr, (int32_t)P, pad ? 1 : 0,
                           fptr(mask_inputs), Ns ? sparse.data_ptr<float>() : nullptr, dense.data_ptr<float>(), stream_of(like)),
        "prompt_encoder");
  return {sparse, dense};
}

// A8: MaskDecoder.predict_masks (mask_decoder.py:163-259) -> (masks [B,4,256,256], iou [B,4], mask_tokens [B,4,256], obj [B])
std::tuple<Tensor, Tensor, Tensor, Tensor> mask_decoder(int64_t model, int64_t B, const Tensor& image_embeddings, const Tensor& image_pe,
                                                        const Tensor& sparse, const Tensor& dense, const Tensor& feat_s0,
                                                        const Tensor& feat_s1) {
  want(image_embeddings, at::kFloat, "image_embeddings");
  want(image_pe, at::kFloat, "image_pe");
  want(sparse, at::kFloat, "sparse");
  want(dense, at::kFloat, "dense");
  want(feat_s0, at::kFloat, "feat_s0");
  want(feat_s1, at::kFloat, "feat_s1");
  TORCH_CHECK(image_embeddings.numel() == B * TOK * 256 && dense.numel() == B * TOK * 256 && image_pe.numel() == TOK * 256,
              "det_sam2::mask_decoder: image_embeddings / dense [B,4096,256], image_pe [4096,256] expected");
  TORCH_CHECK(sparse.dim() == 3 && sparse.size(0) == B && sparse.size(2) == 256, "det_sam2::mask_decoder: sparse [B,Ns,256] expected");
  TORCH_CHECK(feat_s0.numel() == 65536 * 32 && feat_s1.numel() == 16384 * 64, "det_sam2::mask_decoder: feat_s0 [65536,32] / feat_s1 [16384,64] expected");
  c10::hip::HIPGuardMasqueradingAsCUDA g(image_embeddings.device());
  auto o = image_embeddings.options();
  const int64_t Ns = sparse.size(1);
  Tensor masks = at::empty({B, 4, 256, 256}, o), iou = at::empty({B, 4}, o), tok = at::empty({B, 4, 256}, o), obj = at::empty({B}, o);
  check(ds2_mask_decoder(model_of(model), (int32_t)B, image_embeddings.data_ptr<float>(), image_pe.data_ptr<float>(),
                         Ns ? sparse.data_ptr<float>() : nullptr, (int32_t)Ns, dense.data_ptr<float>(), feat_s0.data_ptr<float>(),
                         feat_s1.data_ptr<float>(), masks.data_ptr<float>(), iou.data_ptr<float>(), tok.data_ptr<float>(),
                         obj.data_ptr<float>(), stream_of(image_embeddings)), "mask_decoder");
  return {masks, iou, tok, obj};
}

// A13: SAM2Base._encode_new_memory (sam2_base.py:692-743) -> maskmem bf16 [B,4096,64]
Tensor memory_encoder(int64_t model, int64_t B, const Tensor& fpn2, const Tensor& low_res, const Tensor& obj_logits, bool binarize) {
  want(fpn2, at::kFloat, "fpn2");
  want(low_res, at::kFloat, "low_res");
  want(obj_logits, at::kFloat, "obj_logits");
  TORCH_CHECK(fpn2.numel() == TOK * 256 && low_res.numel() == B * 65536 && obj_logits.numel() == B, "det_sam2::memory_encoder: bad shapes");
  c10::hip::HIPGuardMasqueradingAsCUDA g(fpn2.device());
  Tensor out = at::empty({B, TOK, 64}, fpn2.options().dtype(at::kBFloat16));
  check(ds2_memory_encoder(model_of(model), (int32_t)B, fpn2.data_ptr<float>(), low_res.data_ptr<float>(), obj_logits.data_ptr<float>(),
                           binarize ? 1 : 0, reinterpret_cast<uint16_t*>(out.data_ptr()), stream_of(fpn2)), "memory_encoder");
  return out;
}

// MemoryEncoder.forward itself (memory_encoder.py:158-181): pix_feat [B,4096,256] (or shared [4096,256]), masks fp32
// [B,1024,1024] -> vision_features fp32 [B,4096,64] (no no_obj_embed_spatial, no bf16 rounding)
Tensor memory_encoder_module(int64_t model, int64_t B, const Tensor& pix_feat, const Tensor& masks, bool skip_mask_sigmoid) {
  want(pix_feat, at::kFloat, "pix_feat");
  want(masks, at::kFloat, "masks");
  const bool shared = pix_feat.numel() == TOK * 256 && B != 1;
  TORCH_CHECK(pix_feat.numel() == (shared ? 1 : B) * TOK * 256 && masks.numel() == B * 1024 * 1024, "det_sam2::memory_encoder_module: bad shapes");
  c10::hip::HIPGuardMasqueradingAsCUDA g(pix_feat.device());
  Tensor out = at::empty({B, TOK, 64}, pix_feat.options());
  check(ds2_memory_encoder_ex(model_of(model), (int32_t)B, pix_feat.data_ptr<float>(), shared ? 1 : 0, masks.data_ptr<float>(),
                              skip_mask_sigmoid ? 1 : 0, out.data_ptr<float>(), stream_of(pix_feat)), "memory_encoder_module");
  return out;
}

// F3: F.interpolate(bilinear, antialias=True, align_corners=False) of (x*in_scale + in_bias) [B,Hin,Win] -> [B,Hout,Wout];
// threshold < inf binarises (sam2_video_predictor.py:552-561, sam2_base.py:407-415)
Tensor resize_aa(const Tensor& x, int64_t Hout, int64_t Wout, double in_scale, double in_bias, double threshold) {
  want(x, at::kFloat, "x");
  TORCH_CHECK(x.dim() == 3, "det_sam2::resize_aa: x must be [B,Hin,Win]");
  c10::hip::HIPGuardMasqueradingAsCUDA g(x.device());
  const int64_t B = x.size(0), Hin = x.size(1), Win = x.size(2);
  Tensor work = at::empty({B, Hin, Wout}, x.options()), out = at::empty({B, Hout, Wout}, x.options());
  check(ds2_resize_aa(x.data_ptr<float>(), (int32_t)B, (int32_t)Hin, (int32_t)Win, (int32_t)Hout, (int32_t)Wout, (float)in_scale,
                      (float)in_bias, std::isinf(threshold) ? INFINITY : (float)threshold, work.data_ptr<float>(), out.data_ptr<float>(),
                      stream_of(x)), "resize_aa");
  return out;
}

// F3: mask_downsample conv + any(mask > 0) (sam2_base.py:425-429,436-440) -> (mask_ds [B,256,256], obj_logits [B])
std::tuple<Tensor, Tensor> mask_prompt_prepare(int64_t model, const Tensor& mask) {
  want(mask, at::kFloat, "mask");
  TORCH_CHECK(mask.dim() == 3 && mask.size(1) == 1024 && mask.size(2) == 1024, "det_sam2::mask_prompt_prepare: mask must be [B,1024,1024]");
  c10::hip::HIPGuardMasqueradingAsCUDA g(mask.device());
  const int64_t B = mask.size(0);
  Tensor ds = at::empty({B, 256, 256}, mask.options()), obj = at::empty({B}, mask.options()), work = at::empty({B}, mask.options().dtype(at::kInt));
  check(ds2_mask_prompt_prepare(model_of(model), (int32_t)B, mask.data_ptr<float>(), ds.data_ptr<float>(), obj.data_ptr<float>(),
                                work.data_ptr<int32_t>(), stream_of(mask)), "mask_prompt_prepare");
  return {ds, obj};
}

// F3: obj_ptr = lam*obj_ptr + (1-lam)*no_obj_ptr, lam = obj_logits > 0 (sam2_base.py:441-444); functional
Tensor obj_ptr_gate(int64_t model, const Tensor& obj_ptr, const Tensor& obj_logits) {
  want(obj_ptr, at::kFloat, "obj_ptr");
  want(obj_logits, at::kFloat, "obj_logits");
  TORCH_CHECK(obj_ptr.dim() == 2 && obj_ptr.size(1) == 256 && obj_logits.numel() == obj_ptr.size(0), "det_sam2::obj_ptr_gate: bad shapes");
  c10::hip::HIPGuardMasqueradingAsCUDA g(obj_ptr.device());
  Tensor out = obj_ptr.clone();
  check(ds2_obj_ptr_gate(model_of(model), (int32_t)out.size(0), out.data_ptr<float>(), obj_logits.data_ptr<float>(), stream_of(out)), "obj_ptr_gate");
  return out;
}

// A15: _get_orig_video_res_output + `> 0` + bit-pack (sam2_video_predictor.py:618-642, det_sam2_RT.py:396-399)
std::tuple<Tensor, Tensor> mask_output(int64_t model, const Tensor& low_res, int64_t Hv, int64_t Wv, bool want_logits, bool want_packed) {
  want(low_res, at::kFloat, "low_res");
  TORCH_CHECK(low_res.dim() == 3 && low_res.size(1) == 256 && low_res.size(2) == 256, "det_sam2::mask_output: low_res must be [B,256,256]");
  TORCH_CHECK(want_logits || want_packed, "det_sam2::mask_output: nothing requested");
  c10::hip::HIPGuardMasqueradingAsCUDA g(low_res.device());
  const int64_t B = low_res.size(0);
  Tensor logits = want_logits ? at::empty({B, 1, Hv, Wv}, low_res.options()) : at::empty({0}, low_res.options());
  Tensor packed = want_packed ? at::empty({B, Hv, (Wv + 7) / 8}, low_res.options().dtype(at::kByte)) : at::empty({0}, low_res.options().dtype(at::kByte));
  check(ds2_mask_output(model_of(model), low_res.data_ptr<float>(), (int32_t)B, (int32_t)Hv, (int32_t)Wv,
                        want_logits ? logits.data_ptr<float>() : nullptr, want_packed ? packed.data_ptr<uint8_t>() : nullptr,
                        stream_of(low_res)), "mask_output");
  return {logits, packed};
}

// A14: the reference's one native op, same name (and spelling) and contract: uint8 [N,1,H,W] -> [labels int32, counts int32]
// (sam2/csrc/connected_components.cu:213-289); any H, W here.
std::vector<Tensor> get_connected_componnets(const Tensor& inputs) {
  TORCH_CHECK(inputs.is_cuda(), "inputs must be a CUDA tensor");                  // the reference's AT_ASSERTM messages (:215-227)
  TORCH_CHECK(inputs.dim() == 4, "inputs must be [N, 1, H, W] shape");
  TORCH_CHECK(inputs.scalar_type() == at::kByte, "inputs must be a uint8 type");
  TORCH_CHECK(inputs.size(1) == 1, "inputs must be [N, 1, H, W] shape");
  c10::hip::HIPGuardMasqueradingAsCUDA g(inputs.device());
  Tensor in = inputs.contiguous();
  const int64_t N = in.size(0), H = in.size(2), W = in.size(3);
  auto o = in.options().dtype(at::kInt);
  Tensor labels = at::empty({N, 1, H, W}, o), counts = at::empty({N, 1, H, W}, o), work = at::empty({2 * N * H * W}, o);
  check(ds2_connected_components(in.data_ptr<uint8_t>(), (int32_t)N, (int32_t)H, (int32_t)W, labels.data_ptr<int32_t>(),
                                 counts.data_ptr<int32_t>(), work.data_ptr<int32_t>(), stream_of(in)), "get_connected_componnets");
  return {labels, counts};
}

// A14: fill_holes_in_mask_scores (sam2/utils/misc.py:365-393), functional form
Tensor fill_holes(const Tensor& logits, int64_t max_area) {
  want(logits, at::kFloat, "logits");
  TORCH_CHECK(logits.dim() >= 2, "det_sam2::fill_holes: logits must be [..., H, W]");
  c10::hip::HIPGuardMasqueradingAsCUDA g(logits.device());
  Tensor out = logits.clone();
  const int64_t H = out.size(-2), W = out.size(-1), N = out.numel() / (H * W);
  Tensor work = at::empty({3 * N * H * W}, out.options().dtype(at::kInt));
  check(ds2_fill_holes(out.data_ptr<float>(), (int32_t)N, (int32_t)H, (int32_t)W, (int32_t)max_area, work.data_ptr<int32_t>(), stream_of(out)),
        "fill_holes");
  return out;
}

// F4 detector half: ultralytics ops.non_max_suppression + scale_boxes / clip_boxes on the raw YOLOv8 head output
// pred fp32 [nb, 4+nc, N] -> (dets fp32 [nb, max_det, 6] = xyxy, conf, cls; counts int32 [nb], -1 = candidate overflow)
std::tuple<Tensor, Tensor> yolo_postprocess(const Tensor& pred, double conf_thres, double iou_thres, int64_t max_det,
                                            const c10::optional<Tensor>& scale5) {
  want(pred, at::kFloat, "pred");
  TORCH_CHECK(pred.dim() == 3 && pred.size(1) > 4, "det_sam2::yolo_postprocess: pred must be [nb, 4+nc, N]");
  if (scale5.has_value()) {
    want(*scale5, at::kFloat, "scale5");
    TORCH_CHECK(scale5->numel() == 5, "det_sam2::yolo_postprocess: scale5 = gain, pad_x, pad_y, orig_w, orig_h");
  }
  c10::hip::HIPGuardMasqueradingAsCUDA g(pred.device());
  const int64_t nb = pred.size(0), nc = pred.size(1) - 4, N = pred.size(2);
  const int64_t wb = ds2_yolo_postprocess_work_bytes((int32_t)nb, (int32_t)N);
  Tensor work = at::empty({wb}, pred.options().dtype(at::kByte));
  Tensor dets = at::zeros({nb, max_det, 6}, pred.options()), counts = at::empty({nb}, pred.options().dtype(at::kInt));
  check(ds2_yolo_postprocess(pred.data_ptr<float>(), (int32_t)nb, (int32_t)nc, (int32_t)N, (float)conf_thres, (float)iou_thres,
                             (int32_t)max_det, fptr(scale5), dets.data_ptr<float>(), counts.data_ptr<int32_t>(), work.data_ptr(), wb,
                             stream_of(pred)), "yolo_postprocess");
  return {dets, counts};
}

// ---- token cache (include/detsam2_hip.h): quantised write / read, attention over it, masked attention of prompts
int32_t type_of(const Tensor& t, const char* name, bool f32) {
  const auto st = t.scalar_type();
  TORCH_CHECK(st == at::kBFloat16 || st == at::kHalf || (f32 && st == at::kFloat), "det_sam2: ", name, " must be bfloat16, float16",
              f32 ? " or float32" : "", ", got ", toString(st));
  return st == at::kBFloat16 ? DS2_TYPE_BF16 : st == at::kHalf ? DS2_TYPE_F16 : DS2_TYPE_F32;
}
int32_t format_of(c10::string_view f, bool plain) {
  if (f == "mxfp8") return DS2_CACHE_MXFP8;
  if (f == "mxfp4") return DS2_CACHE_MXFP4;
  TORCH_CHECK(plain && f == "plain", "det_sam2: unknown cache format \"", std::string(f.data(), f.size()), "\" (", plain ? "\"plain\", " : "", "\"mxfp8\", \"mxfp4\")");
  return DS2_CACHE_PLAIN;
}
// leading axes as strides (an axis of size 1: 0, whatever the tensor says), last axis contiguous; `lead` of the three axes, from the back
ds2_strided strided(const Tensor& t, const char* name, const at::Device& dev, int64_t dims = 4) {
  TORCH_CHECK(t.is_cuda() && t.device() == dev, "det_sam2: ", name, " must be on ", dev);
  TORCH_CHECK(t.dim() == dims, "det_sam2: ", name, " must have ", dims, " dimensions, got ", t.dim());
  TORCH_CHECK(t.size(-1) <= 1 || t.stride(-1) == 1, "det_sam2: the last dimension of ", name, " must be contiguous");
  int64_t s[3] = {0, 0, 0};
  for (int64_t i = 0; i + 1 < dims; ++i) s[3 - (dims - 1) + i] = t.size(i) == 1 ? 0 : t.stride(i);
  return ds2_strided{t.numel() ? t.data_ptr() : nullptr, s[0], s[1], s[2]};
}
int32_t int_size(int64_t n, const char* what) {
  TORCH_CHECK(n <= INT32_MAX, "det_sam2: ", what, " is too large");
  return (int32_t)n;
}
const int32_t* ints(const c10::optional<Tensor>& t, at::IntArrayRef shape, const char* name, const at::Device& dev) {
  if (!t.has_value()) return nullptr;
  want(*t, at::kInt, name);
  TORCH_CHECK(t->device() == dev, "det_sam2: ", name, " must be on ", dev);
  TORCH_CHECK(t->sizes() == shape, "det_sam2: ", name, " must be int32 ", shape, ", got ", t->sizes());
  return t->data_ptr<int32_t>();
}
void no_overlap(const Tensor& t, const char* name) {
  // every element of a written tensor has a place of its own: a broadcast axis, or strides that cross, would not
  int64_t need = 1;
  std::array<std::pair<int64_t, int64_t>, 4> ax;
  int n = 0;
  for (int64_t i = 0; i < t.dim() && n < 4; ++i)
    if (t.size(i) > 1) ax[n++] = {t.stride(i), t.size(i)};
  std::sort(ax.begin(), ax.begin() + n);
  for (int i = 0; i < n; ++i) {
    TORCH_CHECK(ax[i].first >= need, "det_sam2: elements of ", name, " overlap in memory");
    need = ax[i].first * (ax[i].second - 1) + need;
  }
}
// These ops answer only: an input that requires a gradient would get none, silently.
bool wants_gradient(const Tensor& t) { return t.requires_grad(); }
bool wants_gradient(const c10::optional<Tensor>& t) { return t.has_value() && t->requires_grad(); }
template <class... T>
void no_backward(const char* op, const T&... inputs) {
  TORCH_CHECK(!at::GradMode::is_enabled() || !(wants_gradient(inputs) || ...), "det_sam2::", op,
              " has no backward pass: detach the inputs or call it under torch.no_grad()");
}
int64_t code_bytes(int32_t format, int64_t D) { return format == DS2_CACHE_MXFP4 ? D / 2 : D; }
// lead axes and a last one
void want_rows(const Tensor& t, at::IntArrayRef lead, int64_t last, const char* what, const char* name) {
  bool same = t.dim() == (int64_t)lead.size() + 1 && t.size(-1) == last;
  for (size_t i = 0; same && i < lead.size(); ++i) same = t.size(i) == lead[i];
  TORCH_CHECK(same, "det_sam2: ", what, name, " must be ", lead, " and ", last, " in the last dimension, got ", t.sizes());
}
void want_codes(const Tensor& c, const Tensor& s, at::IntArrayRef lead, int64_t D, int32_t format, const char* name) {
  TORCH_CHECK(c.scalar_type() == at::kByte && s.scalar_type() == at::kByte, "det_sam2: codes and scales of ", name, " must be uint8");
  want_rows(c, lead, code_bytes(format, D), "codes of ", name);
  want_rows(s, lead, D / 32, "scales of ", name);
}

// new rows k (and v) [B,T,H,D] -> codes uint8 [B,H,C,D or D/2], scales uint8 [B,H,C,D/32], in place, at rows pos[b] + t
void cache_write(const Tensor& k, const c10::optional<Tensor>& v, const Tensor& pos, const c10::optional<Tensor>& count, Tensor k_codes,
                 Tensor k_scales, c10::optional<Tensor> v_codes, c10::optional<Tensor> v_scales, c10::string_view format) {
  const int32_t f = format_of(format, false), type = type_of(k, "k", true), n = v.has_value() ? 2 : 1;
  no_backward("cache_write", k, v);
  TORCH_CHECK(v_codes.has_value() == v.has_value() && v_scales.has_value() == v.has_value(), "det_sam2::cache_write: v, v_codes and v_scales go together");
  TORCH_CHECK(k.dim() == 4 && k_codes.dim() == 4, "det_sam2::cache_write: k [B,T,H,D] and k_codes [B,H,C,D or D/2] expected");
  const auto dev = k.device();
  const int64_t B = k.size(0), T = k.size(1), H = k.size(2), D = k.size(3), C = k_codes.size(2);
  const Tensor* x[2] = {&k, n > 1 ? &*v : nullptr};
  const Tensor* c[2] = {&k_codes, n > 1 ? &*v_codes : nullptr};
  const Tensor* s[2] = {&k_scales, n > 1 ? &*v_scales : nullptr};
  ds2_strided xs[2], cs[2], ss[2];
  for (int i = 0; i < n; ++i) {
    const char* name = i ? "v" : "k";
    TORCH_CHECK(x[i]->sizes() == k.sizes() && x[i]->scalar_type() == k.scalar_type(), "det_sam2::cache_write: k and v must be alike");
    want_codes(*c[i], *s[i], {B, H, C}, D, f, name);
    xs[i] = strided(*x[i], name, dev);
    cs[i] = strided(*c[i], "codes", dev);
    ss[i] = strided(*s[i], "scales", dev);
    no_overlap(*c[i], "codes");
    no_overlap(*s[i], "scales");
  }
  const int32_t* p = ints(pos, {B}, "pos", dev);
  const int32_t* ct = ints(count, {B}, "count", dev);
  c10::hip::HIPGuardMasqueradingAsCUDA g(dev);
  check(ds2_op_cache_write(n, xs, cs, ss, int_size(B, "B"), int_size(T, "T"), int_size(H, "H"), int_size(D, "D"), int_size(C, "C"), p, ct, type, f, stream_of(k)),
        "cache_write");
}

// codes / scales [B,H,C,...] -> values [B,H,C,D]; rows from lens[b] on are zero
Tensor cache_read(const Tensor& codes, const Tensor& scales, const c10::optional<Tensor>& lens, c10::string_view format, at::ScalarType dtype) {
  const int32_t f = format_of(format, false);
  TORCH_CHECK(codes.is_cuda() && codes.dim() == 4 && scales.dim() == 4, "det_sam2::cache_read: codes / scales [B,H,C,...] on the GPU expected");
  const int64_t B = codes.size(0), H = codes.size(1), C = codes.size(2), D = codes.size(3) * (f == DS2_CACHE_MXFP4 ? 2 : 1);
  want_codes(codes, scales, {B, H, C}, D, f, "the cache");
  const auto dev = codes.device();
  const ds2_strided cs = strided(codes, "codes", dev), ss = strided(scales, "scales", dev);
  const int32_t* ln = ints(lens, {B}, "lens", dev);
  c10::hip::HIPGuardMasqueradingAsCUDA g(dev);
  Tensor out = at::empty({B, H, C, D}, codes.options().dtype(dtype));
  const int32_t type = type_of(out, "dtype", true);
  const ds2_strided os = strided(out, "out", dev);
  check(ds2_op_cache_read(&cs, &ss, &os, int_size(B, "B"), int_size(H, "H"), int_size(C, "C"), int_size(D, "D"), ln, type, f, stream_of(codes)), "cache_read");
  return out;
}

Tensor scratch(int64_t bytes, const Tensor& like) { return bytes ? at::empty({bytes}, like.options().dtype(at::kByte)) : Tensor(); }

// q [B,T,Hq,D] over k, v [B,Hkv,C,...] and the shared prefix [Hkv,P,...] -> [B,T,Hq,D]
Tensor cache_attention(const Tensor& q, const Tensor& k, const Tensor& v, const c10::optional<Tensor>& k_scales,
                       const c10::optional<Tensor>& v_scales, const Tensor& lens, const c10::optional<Tensor>& prefix_k,
                       const c10::optional<Tensor>& prefix_v, const c10::optional<Tensor>& prefix_k_scales,
                       const c10::optional<Tensor>& prefix_v_scales, c10::string_view format, double scale, double cap,
                       const c10::optional<Tensor>& slopes) {
  no_backward("cache_attention", q, k, v, prefix_k, prefix_v, slopes);
  ds2_cache_attention_args a{};
  a.format = format_of(format, true);
  a.type = type_of(q, "q", false);
  const bool mx = a.format != DS2_CACHE_PLAIN;
  TORCH_CHECK(q.dim() == 4 && k.dim() == 4 && v.dim() == 4, "det_sam2::cache_attention: q [B,T,Hq,D], k / v [B,Hkv,C,...] expected");
  TORCH_CHECK(k_scales.has_value() == mx && v_scales.has_value() == mx, "det_sam2::cache_attention: scales go with the quantised formats");
  TORCH_CHECK(prefix_k.has_value() == prefix_v.has_value(), "det_sam2::cache_attention: prefix_k and prefix_v go together");
  TORCH_CHECK(prefix_k_scales.has_value() == (mx && prefix_k.has_value()) && prefix_v_scales.has_value() == (mx && prefix_k.has_value()),
              "det_sam2::cache_attention: prefix scales go with a quantised prefix");
  const auto dev = q.device();
  const int64_t B = q.size(0), T = q.size(1), Hq = q.size(2), D = q.size(3), Hkv = k.size(1), C = k.size(2);
  TORCH_CHECK(!prefix_k.has_value() || prefix_k->dim() == 3, "det_sam2::cache_attention: prefix_k must be [Hkv,P,...]");
  const int64_t P = prefix_k.has_value() ? prefix_k->size(1) : 0;
  auto rows = [&](const Tensor& t, const c10::optional<Tensor>& s, at::IntArrayRef lead, const char* name) {
    if (mx) want_codes(t, *s, lead, D, a.format, name);
    else {
      TORCH_CHECK(t.scalar_type() == q.scalar_type(), "det_sam2::cache_attention: ", name, " must be of q's type");
      want_rows(t, lead, D, "", name);
    }
  };
  rows(k, k_scales, {B, Hkv, C}, "k");
  rows(v, v_scales, {B, Hkv, C}, "v");
  a.q = strided(q, "q", dev), a.k = strided(k, "k", dev), a.v = strided(v, "v", dev);
  if (mx) a.k_scales = strided(*k_scales, "k_scales", dev), a.v_scales = strided(*v_scales, "v_scales", dev);
  if (P) {
    rows(*prefix_k, prefix_k_scales, {Hkv, P}, "prefix_k");
    rows(*prefix_v, prefix_v_scales, {Hkv, P}, "prefix_v");
    a.prefix_k = strided(*prefix_k, "prefix_k", dev, 3), a.prefix_v = strided(*prefix_v, "prefix_v", dev, 3);
    if (mx) a.prefix_k_scales = strided(*prefix_k_scales, "prefix_k_scales", dev, 3), a.prefix_v_scales = strided(*prefix_v_scales, "prefix_v_scales", dev, 3);
  }
  a.lens = ints(lens, {B}, "lens", dev);
  if (slopes.has_value()) {
    want(*slopes, at::kFloat, "slopes");
    TORCH_CHECK(slopes->device() == dev && slopes->dim() == 1 && slopes->size(0) == Hq, "det_sam2::cache_attention: slopes must be float32 [Hq] on q's device");
    a.slopes = slopes->data_ptr<float>();
  }
  a.B = int_size(B, "B"), a.T = int_size(T, "T"), a.Hq = int_size(Hq, "Hq"), a.Hkv = int_size(Hkv, "Hkv"), a.D = int_size(D, "D");
  a.capacity = int_size(C, "C"), a.prefix_len = int_size(P, "P");
  a.scale = (float)scale, a.cap = (float)cap;
  c10::hip::HIPGuardMasqueradingAsCUDA g(dev);
  Tensor out = at::empty({B, T, Hq, D}, q.options());
  if (!out.numel()) return out;
  a.out = out.data_ptr();
  const int64_t bytes = ds2_op_cache_attention_work_bytes(&a);
  const Tensor work = scratch(bytes, q);
  check(ds2_op_cache_attention(&a, bytes ? work.data_ptr() : nullptr, bytes, stream_of(q)), "cache_attention");
  return out;
}

// q [B,Lq,Hq,D], k / v [B,Lk,Hkv,D] -> [B,Lq,Hq,D]
Tensor attention_masked(const Tensor& q, const Tensor& k, const Tensor& v, double scale, bool causal, double cap,
                        const c10::optional<Tensor>& slopes, const c10::optional<Tensor>& lens, const c10::optional<Tensor>& q_start,
                        const c10::optional<Tensor>& prefix, const c10::optional<Tensor>& q_doc, const c10::optional<Tensor>& k_doc) {
  no_backward("attention_masked", q, k, v, slopes);
  ds2_attention_masked_args a{};
  a.type = type_of(q, "q", false);
  TORCH_CHECK(q.dim() == 4 && k.dim() == 4 && v.sizes() == k.sizes(), "det_sam2::attention_masked: q [B,Lq,Hq,D], k / v [B,Lk,Hkv,D] expected");
  TORCH_CHECK(k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type(), "det_sam2::attention_masked: q, k and v must be of one type");
  TORCH_CHECK(k.size(0) == q.size(0) && k.size(3) == q.size(3), "det_sam2::attention_masked: k ", k.sizes(), " does not go with q ", q.sizes());
  TORCH_CHECK(q_doc.has_value() == k_doc.has_value(), "det_sam2::attention_masked: q_doc and k_doc go together");
  TORCH_CHECK(causal || !prefix.has_value(), "det_sam2::attention_masked: a prefix goes with the causal mask");
  const auto dev = q.device();
  const int64_t B = q.size(0), Lq = q.size(1), Hq = q.size(2), D = q.size(3), Lk = k.size(1);
  a.q = strided(q, "q", dev), a.k = strided(k, "k", dev), a.v = strided(v, "v", dev);
  if (slopes.has_value()) {
    want(*slopes, at::kFloat, "slopes");
    TORCH_CHECK(slopes->device() == dev && slopes->dim() == 1 && slopes->size(0) == Hq, "det_sam2::attention_masked: slopes must be float32 [Hq] on q's device");
    a.slopes = slopes->data_ptr<float>();
  }
  a.lens = ints(lens, {B}, "lens", dev), a.q_start = ints(q_start, {B}, "q_start", dev), a.prefix = ints(prefix, {B}, "prefix", dev);
  a.q_doc = ints(q_doc, {B, Lq}, "q_doc", dev), a.k_doc = ints(k_doc, {B, Lk}, "k_doc", dev);
  a.B = int_size(B, "B"), a.Lq = int_size(Lq, "Lq"), a.Lk = int_size(Lk, "Lk"), a.Hq = int_size(Hq, "Hq"), a.Hkv = int_size(k.size(2), "Hkv");
  a.D = int_size(D, "D"), a.causal = causal ? 1 : 0;
  a.scale = (float)scale, a.cap = (float)cap;
  c10::hip::HIPGuardMasqueradingAsCUDA g(dev);
  Tensor out = at::empty({B, Lq, Hq, D}, q.options());
  if (!out.numel()) return out;
  a.out = out.data_ptr();
  const int64_t bytes = ds2_op_attention_masked_work_bytes(&a);
  const Tensor work = scratch(bytes, q);
  check(ds2_op_attention_masked(&a, bytes ? work.data_ptr() : nullptr, bytes, stream_of(q)), "attention_masked");
  return out;
}

}  // namespace

TORCH_LIBRARY(det_sam2, m) {
  m.def("ingest_frames(int model, Tensor frames_u8) -> Tensor");
  m.def("image_encoder(int model, Tensor frames) -> (Tensor, Tensor, Tensor)");
  m.def("bank_assemble(int model, int B, Tensor[] feats, int[] tpos_rows, Tensor[] ptrs, float[] ptr_pos) -> (Tensor, Tensor)");
  m.def("bank_memory_attention(int model, int B, Tensor curr, Tensor[] feats, int[] tpos_rows, Tensor[] ptrs, float[] ptr_pos) -> Tensor");
  m.def("memory_attention(int model, int B, Tensor curr, Tensor? curr_pos, Tensor memory, Tensor memory_pos, int num_obj_ptr_tokens) -> Tensor");
  m.def("sam_heads(int model, int B, Tensor pix_feat, bool pix_bcast, bool add_no_mem_embed, Tensor fpn0, Tensor fpn1, "
        "Tensor? point_coords, Tensor? point_labels, Tensor? mask_inputs, bool multimask) -> (Tensor, Tensor, Tensor, Tensor)");
  m.def("prompt_encoder(int model, int B, Tensor? point_coords, Tensor? point_labels, bool pad, Tensor? mask_inputs, Tensor like) -> (Tensor, Tensor)");
  m.def("mask_decoder(int model, int B, Tensor image_embeddings, Tensor image_pe, Tensor sparse, Tensor dense, Tensor feat_s0, Tensor feat_s1) -> (Tensor, Tensor, Tensor, Tensor)");
  m.def("memory_encoder(int model, int B, Tensor fpn2, Tensor low_res, Tensor obj_logits, bool binarize) -> Tensor");
  m.def("memory_encoder_module(int model, int B, Tensor pix_feat, Tensor masks, bool skip_mask_sigmoid) -> Tensor");
  m.def("resize_aa(Tensor x, int Hout, int Wout, float in_scale, float in_bias, float threshold) -> Tensor");
  m.def("mask_prompt_prepare(int model, Tensor mask) -> (Tensor, Tensor)");
  m.def("obj_ptr_gate(int model, Tensor obj_ptr, Tensor obj_logits) -> Tensor");
  m.def("mask_output(int model, Tensor low_res, int Hv, int Wv, bool want_logits, bool want_packed) -> (Tensor, Tensor)");
  m.def("get_connected_componnets(Tensor inputs) -> Tensor[]");
  m.def("fill_holes(Tensor logits, int max_area) -> Tensor");
  m.def("yolo_postprocess(Tensor pred, float conf_thres, float iou_thres, int max_det, Tensor? scale5) -> (Tensor, Tensor)");
  m.def("cache_write(Tensor k, Tensor? v, Tensor pos, Tensor? count, Tensor(a!) k_codes, Tensor(b!) k_scales, Tensor(c!)? v_codes, "
        "Tensor(d!)? v_scales, str format) -> ()");
  m.def("cache_read(Tensor codes, Tensor scales, Tensor? lens, str format, ScalarType dtype) -> Tensor");
  m.def("cache_attention(Tensor q, Tensor k, Tensor v, Tensor? k_scales, Tensor? v_scales, Tensor lens, Tensor? prefix_k, Tensor? prefix_v, "
        "Tensor? prefix_k_scales, Tensor? prefix_v_scales, str format, float scale, float cap, Tensor? slopes) -> Tensor");
  m.def("attention_masked(Tensor q, Tensor k, Tensor v, float scale, bool causal, float cap, Tensor? slopes, Tensor? lens, Tensor? q_start, "
        "Tensor? prefix, Tensor? q_doc, Tensor? k_doc) -> Tensor");
}

// GPU tensors on PyTorch-ROCm dispatch under the CUDA key (HIP masquerades as CUDA); a CPU tensor finds no kernel and the
// dispatcher raises NotImplementedError - there is no CPU path.
TORCH_LIBRARY_IMPL(det_sam2, CUDA, m) {
  m.impl("ingest_frames", &ingest_frames);
  m.impl("image_encoder", &image_encoder);
  m.impl("bank_assemble", &bank_assemble);
  m.impl("bank_memory_attention", &bank_memory_attention);
  m.impl("memory_attention", &memory_attention);
  m.impl("sam_heads", &sam_heads);
  m.impl("prompt_encoder", &prompt_encoder);
  m.impl("mask_decoder", &mask_decoder);
  m.impl("memory_encoder", &memory_encoder);
  m.impl("memory_encoder_module", &memory_encoder_module);
  m.impl("resize_aa", &resize_aa);
  m.impl("mask_prompt_prepare", &mask_prompt_prepare);
  m.impl("obj_ptr_gate", &obj_ptr_gate);
  m.impl("mask_output", &mask_output);
  m.impl("get_connected_componnets", &get_connected_componnets);
  m.impl("fill_holes", &fill_holes);
  m.impl("yolo_postprocess", &yolo_postprocess);
  m.impl("cache_write", &cache_write);
  m.impl("cache_read", &cache_read);
  m.impl("cache_attention", &cache_attention);
  m.impl("attention_masked", &attention_masked);
}
