// Kernels of attention_masked.h for bf16 operands.
#include "attention_masked.h"

int launch_masked_bf16(const MaskedArgs& a, int mode, unsigned blocks, hipStream_t st) { return launch_masked<false>(a, mode, blocks, st); }
