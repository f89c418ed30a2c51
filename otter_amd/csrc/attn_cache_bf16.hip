// attn_cache.hpp for __bf16 activations.
#include <type_traits>
#define OTTER_ATTN_CACHE_IMPL
#include "attn_cache.hpp"

template int otter_attn_cache_launch<__bf16>(const AttnCacheArgs&, int, int, int, unsigned, hipStream_t);
