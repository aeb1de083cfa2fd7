// Attention over the 8-bit cache: which kernel a call takes, how its keys are cut, and the sum of the parts.
#include <algorithm>

#include "block_cache_attention.hpp"

namespace cg {
namespace {

// out[row] = the mean of the parts' results by their sums of weights, each scaled from its own maximum to the largest; rows of a block of
// rows that was not cut are there already.
struct RowToJoin {
    uint32_t parts, b, g, r;
    uint64_t first; // of its parts' results; they lie p.rows apart
    __device__ __forceinline__ bool find(const CacheAttentionPlan &p, uint32_t item, uint32_t group) {
        const uint32_t bg = fastdiv(item, p.rows_div);
        r = item - bg * p.rows;
        b = fastdiv(bg, p.heads_div);
        g = bg - b * p.cache.kv_heads;
        const uint32_t R = p.batch.count_of(b) * p.rep, group0 = r / group * group;
        if (r >= R) return false;
        parts = key_range(p, p.batch.held_by(b), fastdiv(group0, p.rep_div), fastdiv(min(group0 + group, R) - 1, p.rep_div)).parts;
        first = (uint64_t)bg * p.splits * p.rows + r;
        return parts > 1;
    }
    template <class T> __device__ __forceinline__ void store(const CacheAttentionPlan &p, uint32_t vec, const float4v &y4) const {
        const uint32_t s = fastdiv(r, p.rep_div), head = g * p.rep + r - s * p.rep;
        const float y[4] = {y4[0], y4[1], y4[2], y4[3]};
        store_elements<T, 4>(static_cast<T *>(p.out) + ((int64_t)b * p.batch.tokens + s) * p.out_pitch + head * p.cache.vdim + vec * 4, y);
    }
};

// A few parts: a thread takes four channels of a row, all parts asked for at once.
constexpr uint32_t kFewParts = 8;
template <class T> __global__ __launch_bounds__(256) void join_few_parts_kernel(CacheAttentionPlan p, uint32_t lanes, uint32_t each, uint32_t group, uint32_t all) {
    const uint32_t mine = threadIdx.x / lanes, item = blockIdx.x * each + mine, vec = threadIdx.x - mine * lanes;
    RowToJoin row;
    if (mine >= each || item >= all || !row.find(p, item, group)) return;
    float2 stats[kFewParts];
    float4v part[kFewParts];
#pragma unroll
    for (uint32_t i = 0; i < kFewParts; i++) { // (behind the last part: the last one again, which then counts for nothing)
        const uint64_t at = row.first + (uint64_t)min(i, row.parts - 1) * p.rows;
        stats[i] = p.stats[at];
        part[i] = *reinterpret_cast<const float4v *>(p.parts + at * p.cache.vdim + vec * 4);
    }
    float m = stats[0].x, sum = 0.0f, weight[kFewParts];
#pragma unroll
    for (uint32_t i = 1; i < kFewParts; i++) m = fmaxf(m, stats[i].x);
#pragma unroll
    for (uint32_t i = 0; i < kFewParts; i++) {
        weight[i] = i < row.parts ? stats[i].y * __builtin_amdgcn_exp2f(stats[i].x - m) : 0.0f;
        sum += weight[i];
    }
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    float4v total = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (uint32_t i = 0; i < kFewParts; i++)
        if (i < row.parts) total += part[i] * (weight[i] * inv);
    row.store<T>(p, vec, total);
}

// Many parts: a workgroup takes a row, its threads the parts' weights first, then channels of some of the parts each.
constexpr uint32_t kMostParts = 256;
template <class T> __global__ __launch_bounds__(256) void join_parts_kernel(CacheAttentionPlan p, uint32_t lanes, uint32_t each, uint32_t group) {
    __shared__ float weights[kMostParts], reduced[8];
    __shared__ float4v totals[256];
    RowToJoin row;
    if (!row.find(p, blockIdx.x, group)) return; // (the same for all threads)
    const float2 mine = threadIdx.x < row.parts ? p.stats[row.first + (uint64_t)threadIdx.x * p.rows] : make_float2(kNoMaximum, 0.0f);
    float m = mine.x;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
    if (threadIdx.x % 64 == 0) reduced[threadIdx.x / 64] = m;
    __syncthreads();
    m = fmaxf(fmaxf(reduced[0], reduced[1]), fmaxf(reduced[2], reduced[3]));
    float sum = mine.y * __builtin_amdgcn_exp2f(mine.x - m);
    weights[threadIdx.x] = sum;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
    if (threadIdx.x % 64 == 0) reduced[4 + threadIdx.x / 64] = sum;
    __syncthreads();
    sum = reduced[4] + reduced[5] + reduced[6] + reduced[7];
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    const uint32_t turn = threadIdx.x / lanes, vec = threadIdx.x - turn * lanes; // every `each`-th part
    float4v total = {0.0f, 0.0f, 0.0f, 0.0f};
    if (turn < each) {
        constexpr uint32_t kAtOnce = 8;
        for (uint32_t i0 = turn; i0 < row.parts; i0 += kAtOnce * each) {
            float4v part[kAtOnce];
#pragma unroll
            for (uint32_t k = 0; k < kAtOnce; k++) {
                const uint32_t i = min(i0 + k * each, row.parts - 1);
                part[k] = *reinterpret_cast<const float4v *>(p.parts + (row.first + (uint64_t)i * p.rows) * p.cache.vdim + vec * 4);
            }
#pragma unroll
            for (uint32_t k = 0; k < kAtOnce; k++)
                if (i0 + k * each < row.parts) total += part[k] * (weights[i0 + k * each] * inv);
        }
    }
    totals[threadIdx.x] = total;
    __syncthreads();
    if (threadIdx.x >= lanes) return;
    for (uint32_t i = 1; i < each; i++) total += totals[i * lanes + threadIdx.x];
    row.store<T>(p, vec, total);
}

uint32_t rows_of_group(const CacheAttentionPlan &p) {
    const uint32_t wide = std::max(p.cache.dim, p.cache.vdim);
    if (p.rows_by_wave) return wide > 128 ? 16 * kWavesOfAttention : 32 * kWavesOfAttention;
    return p.two_tiles ? 32 : 16;
}

} // namespace

size_t shape_cache_attention(CacheAttentionPlan *p) {
    const uint32_t wide = std::max(p->cache.dim, p->cache.vdim);
    p->rows = p->batch.tokens * p->rep;
    p->bgs = p->batch.sequences * p->cache.kv_heads;
    p->rows_by_wave = p->rows > 32;
    p->two_tiles = !p->rows_by_wave && p->rows > 16 && wide <= 128;
    const uint32_t group = rows_of_group(*p);
    p->row_blocks = (p->rows + group - 1) / group;
    // Parts: as many as end soonest.  The card holds two workgroups on each of its 256 compute units; one takes its tiles a step at a time (a tile, or one
    // for each of its waves), begins and ends in about two steps more; a join takes as long, and the time in which the parts' results are written and
    // read (a step of all units: 1.3 us, or with the waves sharing rows 5, at 4.7 TB/s).  768 workgroups for 512 places take as long as 1024:
    // a portion of 3 x 500 rows, 144 groups, took 111 us cut in three, join included, 126 in four, 109 in seven.
    const uint64_t groups = (uint64_t)p->bgs * p->row_blocks;
    const uint64_t C = p->cache.capacity; // what a block of rows sees of it, at most
    const uint64_t tiles = (p->window ? std::min(C, std::min<uint64_t>(C, p->window) + std::min(p->batch.tokens, group / p->rep + 1)) : C) / kTile;
    const uint32_t step = p->rows_by_wave ? 1 : kWavesOfAttention;
    const uint64_t joined = (uint64_t)p->bgs * p->rows * p->cache.vdim * 8 * 8 / (p->rows_by_wave ? 6000000 : 24000000); // eighths of a step, for each part
    const uint64_t most = std::max<uint64_t>(1, std::min<uint64_t>(tiles / kLeastTiles, kMostParts));
    const uint64_t by_row = (uint64_t)p->bgs * p->rows / 160; // the join of more than a few parts, a workgroup for each row: 2048 in 3 us
    uint64_t best = ~0ull;
    p->splits = 1;
    for (uint64_t s = 1; s <= most && groups * (s - 1) < 4 * 512; s++) {
        const uint64_t cost = 8 * ((groups * s + 511) / 512 * ((tiles + s * step - 1) / (s * step) + 2)) + (s > 1 ? 16 + s * joined : 0) + (s > kFewParts ? by_row : 0);
        if (cost < best) {
            best = cost;
            p->splits = (uint32_t)s;
        }
    }
    p->rep_div = make_fastdiv(p->rep);
    p->bgs_div = make_fastdiv(p->bgs);
    p->splits_div = make_fastdiv(p->splits);
    p->heads_div = make_fastdiv(p->cache.kv_heads);
    p->rows_div = make_fastdiv(p->rows);
    p->run_div = make_fastdiv((uint32_t)std::max<uint64_t>(1, 256 / ((uint64_t)p->bgs * p->splits)));
    return p->splits == 1 ? 0 : (size_t)p->bgs * p->splits * p->rows * (p->cache.vdim + 2) * 4;
}

int launch_cache_attention(const LaunchOn &on, cg_dtype dtype, const CacheAttentionPlan &p) {
    if (int rc = dtype == CG_F32 ? launch_cache_attention_f32(on, p) : dtype == CG_F16 ? launch_cache_attention_f16(on, p) : launch_cache_attention_bf16(on, p)) return rc;
    if (p.splits == 1) return CG_OK;
    const uint32_t lanes = p.cache.vdim / 4, all = p.bgs * p.rows, each = 256 / lanes, group = rows_of_group(p);
    return with_element(dtype, [&](auto e) {
        typedef decltype(e) T;
        return p.splits <= kFewParts ? on("cache attention join launch", join_few_parts_kernel<T>, dim3((all + each - 1) / each), dim3(256), p, lanes, each, group, all)
                                     : on("cache attention join launch", join_parts_kernel<T>, dim3(all), dim3(256), p, lanes, each, group);
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
