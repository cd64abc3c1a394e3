// cache_attn_d128.hip -- instantiations of the cache attention (cache_attn_kernel.h), head_dim 128.
#include "cache_attn_kernel.h"

namespace chia {
CacheAttnFn select_cache_kernel_d128(int format, int score, int tile, int waves) {
  return pick_cache_kernel<128>(format, score, tile, waves);
}
}  // namespace chia
