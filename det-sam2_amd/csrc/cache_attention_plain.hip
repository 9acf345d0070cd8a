// Kernels of cache_attention.h for caches in format "plain".
#include "cache_attention.h"

int launch_cache_attn_plain(const CacheAttnArgs& a, bool f16, unsigned blocks, hipStream_t st) {
  return f16 ? launch_cache_attn_of<DS2_CACHE_PLAIN, true>(a, blocks, st) : launch_cache_attn_of<DS2_CACHE_PLAIN, false>(a, blocks, st);
}
