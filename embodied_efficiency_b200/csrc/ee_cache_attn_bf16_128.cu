// bf16 instances of the attention over a cache, heads of 128
#include "ee_cache_attn.cuh"

namespace ee {
EE_CACHE_ATTN(__nv_bfloat16, 128)
}  // namespace ee
