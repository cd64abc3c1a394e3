// cache_prompt.hip -- instantiations of the cache attention for prompts (cache_prompt_kernel.h).
#include "cache_prompt_kernel.h"

namespace chia {

template <int D, int FMT>
static CacheAttnFn pick(int score) {
  switch (score) {
    case CACHE_SOFTMAX: return cache_prompt_kernel<D, FMT, CACHE_SOFTMAX>;
    case CACHE_SOFTMAX_MOD: return cache_prompt_kernel<D, FMT, CACHE_SOFTMAX_MOD>;
    case CACHE_SIGMOID: return cache_prompt_kernel<D, FMT, CACHE_SIGMOID>;
    case CACHE_RELU: return cache_prompt_kernel<D, FMT, CACHE_RELU>;
  }
  return nullptr;
}

CacheAttnFn select_cache_prompt_kernel(int head_dim, int format, int score) {
  if (head_dim == 64) return format ? pick<64, 1>(score) : pick<64, 0>(score);
  return format ? pick<128, 1>(score) : pick<128, 0>(score);
}

}  // namespace chia
