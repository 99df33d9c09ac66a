// bf16 instances of the attention over a cache, heads of 64
#include "ee_cache_attn.cuh"

namespace ee {
EE_CACHE_ATTN(__nv_bfloat16, 64)
}  // namespace ee
