// fp16 instances of the attention over a cache, heads of 64
#include "ee_cache_attn.cuh"

namespace ee {
EE_CACHE_ATTN(__half, 64)
}  // namespace ee
