// Kernels of cache_attention.h for caches in format "mxfp4".
#include "cache_attention.h"

int launch_cache_attn_mxfp4(const CacheAttnArgs& a, bool f16, unsigned blocks, hipStream_t st) {
  return f16 ? launch_cache_attn_of<DS2_CACHE_MXFP4, true>(a, blocks, st) : launch_cache_attn_of<DS2_CACHE_MXFP4, false>(a, blocks, st);
}
