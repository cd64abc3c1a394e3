// cache_attn_d64.hip -- instantiations of the cache attention (cache_attn_kernel.h), head_dim 64.
#include "cache_attn_kernel.h"

namespace chia {
CacheAttnFn select_cache_kernel_d64(int format, int score, int tile, int waves) {
  return pick_cache_kernel<64>(format, score, tile, waves);
}
}  // namespace chia
