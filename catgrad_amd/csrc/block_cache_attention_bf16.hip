// Attention over the 8-bit cache with bf16 queries and results.
#include <algorithm>

#include "block_cache_attention.hpp"

namespace cg {
int launch_cache_attention_bf16(const LaunchOn &on, const CacheAttentionPlan &p) { return launch_cache_attention_of<__bf16>(on, p); }
int load_cache_attention_bf16() { return load_cache_attention_of<__bf16>(); }
} // namespace cg
