// Attention over the 8-bit cache: which kernel a call takes, how its keys are cut, and the sum of the parts.
#include <algorithm>

#include "block_cache_attention.hpp"

namespace cg {
namespace {

// out[row] = sum of the parts' totals over the sum of their sums, each scaled from its own maximum to the largest.  A thread takes four
// channels of a row; rows of a block of rows that was not cut are there already.
template <class T> __global__ __launch_bounds__(256) void join_parts_kernel(CacheAttentionPlan p, uint32_t lanes, uint32_t group, uint32_t all) {
    const uint32_t item = blockIdx.x * (256 / lanes) + threadIdx.x / lanes, vec = threadIdx.x % lanes;
    if (threadIdx.x / lanes >= 256 / lanes || item >= all) return;
    const uint32_t bg = item / p.rows, r = item - bg * p.rows, b = bg / p.cache.kv_heads, g = bg - b * p.cache.kv_heads;
    const uint32_t R = p.batch.count_of(b) * p.rep;
    if (r >= R) return;
    const uint32_t group0 = r / group * group;
    const KeyRange range = key_range(p, p.batch.held_by(b), group0 / p.rep, (min(group0 + group, R) - 1) / p.rep);
    if (range.parts == 1) return;
    const uint64_t row = (uint64_t)bg * p.splits * p.rows + r;
    float m = kNoMaximum;
    for (uint32_t i = 0; i < range.parts; i++) m = fmaxf(m, p.stats[row + (uint64_t)i * p.rows].x);
    float sum = 0.0f;
    float4v total = {0.0f, 0.0f, 0.0f, 0.0f};
    for (uint32_t i = 0; i < range.parts; i++) {
        const uint64_t at = row + (uint64_t)i * p.rows;
        const float2 s = p.stats[at];
        const float f = __builtin_amdgcn_exp2f(s.x - m);
        sum += s.y * f;
        total += *reinterpret_cast<const float4v *>(p.parts + at * p.cache.vdim + vec * 4) * f;
    }
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    const uint32_t s = r / p.rep, head = g * p.rep + r - s * p.rep;
    T *const dst = static_cast<T *>(p.out) + ((int64_t)b * p.batch.tokens + s) * p.out_pitch + head * p.cache.vdim + vec * 4;
    const float y[4] = {total[0] * inv, total[1] * inv, total[2] * inv, total[3] * inv};
    store_elements<T, 4>(dst, y);
}

uint32_t rows_of_group(const CacheAttentionPlan &p) {
    const uint32_t wide = std::max(p.cache.dim, p.cache.vdim);
    if (p.rows_by_wave) return wide > 128 ? 16 * kWavesOfAttention : 32 * kWavesOfAttention;
    return p.two_tiles ? 32 : 16;
}

} // namespace

size_t shape_cache_attention(cg_dtype, CacheAttentionPlan *p) {
    const uint32_t wide = std::max(p->cache.dim, p->cache.vdim);
    p->rows = p->batch.tokens * p->rep;
    p->bgs = p->batch.sequences * p->cache.kv_heads;
    p->rows_by_wave = p->rows > 32;
    p->two_tiles = !p->rows_by_wave && p->rows > 16 && wide <= 128;
    const uint32_t group = rows_of_group(*p);
    p->row_blocks = (p->rows + group - 1) / group;
    // parts: enough for two workgroups on each of the 256 compute units, none with fewer than the least tiles
    const uint64_t groups = (uint64_t)p->bgs * p->row_blocks, tiles = p->cache.capacity / kTile;
    const uint32_t least = p->rows_by_wave ? kLeastTilesRows : kLeastTilesShared;
    uint64_t splits = groups < 512 ? (512 + groups - 1) / groups : 1;
    splits = std::max<uint64_t>(1, std::min<uint64_t>({splits, tiles / least, 256}));
    p->splits = (uint32_t)splits;
    p->rep_div = make_fastdiv(p->rep);
    p->bgs_div = make_fastdiv(p->bgs);
    p->splits_div = make_fastdiv(p->splits);
    p->heads_div = make_fastdiv(p->cache.kv_heads);
    return splits == 1 ? 0 : (size_t)p->bgs * splits * p->rows * (p->cache.vdim + 2) * 4;
}

int launch_cache_attention(const LaunchOn &on, cg_dtype dtype, const CacheAttentionPlan &p) {
    if (int rc = dtype == CG_F32 ? launch_cache_attention_f32(on, p) : dtype == CG_F16 ? launch_cache_attention_f16(on, p) : launch_cache_attention_bf16(on, p)) return rc;
    if (p.splits == 1) return CG_OK;
    const uint32_t lanes = p.cache.vdim / 4, all = p.bgs * p.rows, each = 256 / lanes;
    return with_element(dtype, [&](auto e) {
        return on("cache attention join launch", join_parts_kernel<decltype(e)>, dim3((all + each - 1) / each), dim3(256), p, lanes, rows_of_group(p), all);
    });
}

int load_cache_attention_kernels() {
    hipFuncAttributes a;
    CG_HIP(hipFuncGetAttributes(&a, reinterpret_cast<const void *>(join_parts_kernel<float>)));
    if (int rc = load_cache_attention_f32()) return rc;
    if (int rc = load_cache_attention_f16()) return rc;
    return load_cache_attention_bf16();
}

} // namespace cg
