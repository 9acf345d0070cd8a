// k_attn_masked for bf16 with weights as two operands: a prefix that sequences share (cache_attention.hip).
#include "attention_masked.h"

int launch_masked_bf16_wide(const MaskedArgs& a, int mode, unsigned blocks, hipStream_t st) { return launch_masked<false, true>(a, mode, blocks, st); }
