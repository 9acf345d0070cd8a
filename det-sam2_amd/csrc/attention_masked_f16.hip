// Kernels of attention_masked.h for fp16 operands.
#include "attention_masked.h"

int launch_masked_f16(const MaskedArgs& a, int mode, unsigned blocks, hipStream_t st) { return launch_masked<true>(a, mode, blocks, st); }
