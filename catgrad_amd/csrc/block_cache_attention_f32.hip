// Attention over the 8-bit cache with f32 queries and results.
#include <algorithm>

#include "block_cache_attention.hpp"

namespace cg {
int launch_cache_attention_f32(const LaunchOn &on, const CacheAttentionPlan &p) { return launch_cache_attention_of<float>(on, p); }
int load_cache_attention_f32() { return load_cache_attention_of<float>(); }
} // namespace cg
