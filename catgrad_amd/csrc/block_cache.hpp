// Rotary positions and the key / value cache in 8 bits (their section of include/catgrad_hip.h): plans of the kernels in
// block_rotary.hip, block_cache_append.hip and block_cache_attention*.hip, for block_cache.cpp, which checks the arguments.
#pragma once

#include "blocks.hpp"

namespace cg {

// Where kernels go: a backend's stream (through its queue) or a caller's.
struct LaunchOn {
    LaunchQueue *queue = nullptr;
    hipStream_t stream = nullptr;
    template <class... P, class... A> int operator()(const char *what, void (*kernel)(P...), dim3 grid, dim3 block, A &&...a) const {
        return with_lds(what, kernel, grid, block, 0, std::forward<A>(a)...);
    }
    template <class... P, class... A> int with_lds(const char *what, void (*kernel)(P...), dim3 grid, dim3 block, size_t lds, A &&...a) const {
        if (queue) launch_kernel(kernel, grid, block, lds, *queue, std::forward<A>(a)...);
        else hipLaunchKernelGGL(kernel, grid, block, lds, stream, std::forward<A>(a)...);
        const hipError_t e = hipGetLastError();
        return e == hipSuccess ? CG_OK : hip_fail(e, what);
    }
};

// Sequences of up to `tokens` new tokens each, behind held[b] positions (cg_token_batch).
struct TokenBatch {
    uint32_t sequences, tokens;
    uint64_t position;
    const uint32_t *held, *counts;
#ifdef __HIPCC__
    __device__ __forceinline__ uint64_t held_by(uint32_t b) const { return held ? held[b] : position; }
    __device__ __forceinline__ uint32_t count_of(uint32_t b) const {
        const uint32_t n = counts ? counts[b] : tokens;
        return n < tokens ? n : tokens;
    }
#endif
};

struct RotaryPlan {
    TokenBatch batch;
    const void *q, *k; // k null: none
    void *q_out, *k_out;
    int64_t q_pitch, k_pitch, q_out_pitch, k_out_pitch;
    uint32_t heads, kv_heads, dim, rot;
    bool interleaved;
    float magnitude;
    const double *turns;
    // set by launch_rotary
    uint32_t group;                     // tokens of a workgroup
    FastDiv per_token, per_head, tokens; // units of a token, of a head; tokens of a sequence
};
int launch_rotary(const LaunchOn &on, cg_dtype dtype, RotaryPlan p);

constexpr int kLowestScale = -117, kHighestScale = 119; // exponents of a block's scale
struct Cache8 {
    uint8_t *k_codes, *v_codes;
    float *k_scale, *v_scale;
    uint32_t kv_heads, dim, vdim, capacity, block_log2;
};
struct CacheAppendPlan {
    TokenBatch batch;
    const void *k, *v;
    int64_t k_pitch, v_pitch;
    Cache8 cache;
};
// The launch of an append: the blocks of a head that it touches at most, and a workgroup's threads.
struct AppendShape {
    uint32_t touched, threads;
    uint64_t groups; // workgroups
};
AppendShape shape_cache_append(const CacheAppendPlan &p);
int launch_cache_append(const LaunchOn &on, cg_dtype dtype, const CacheAppendPlan &p);

struct CacheAttentionPlan {
    TokenBatch batch;
    const void *q;
    void *out;
    int64_t q_pitch, out_pitch;
    Cache8 cache;
    uint32_t heads, rep; // rep = heads / kv_heads
    uint64_t window;     // 0: all
    float scale;
    // by shape_cache_attention
    uint32_t bgs, row_blocks, splits; // (sequence, kv head) pairs; blocks of a pair's rows; parts that the keys of a block of rows are cut into
    bool rows_by_wave, two_tiles;     // which kernel: see shape_cache_attention
    uint32_t rows;                    // of a pair, at most: tokens * rep
    FastDiv rep_div, bgs_div, splits_div, heads_div, rows_div, run_div; // heads: of keys and values; run: blocks of rows for a card's units
    float *parts;                     // splits > 1: [pair][split][row][vdim] results and behind them [pair][split][row] {maximum, sum of weights}
    float2 *stats;
};
// Which kernel and cut a call takes, and the bytes of memory that it needs for the parts' results.
size_t shape_cache_attention(CacheAttentionPlan *p);
int launch_cache_attention(const LaunchOn &on, cg_dtype dtype, const CacheAttentionPlan &p);

// Loads the kernels of these files on the current device (none of them may be loaded first while a stream is captured).
int load_rotary_kernels();
int load_cache_append_kernels();
int load_cache_attention_kernels();
int launch_rotation_table(const LaunchOn &on, const double *turns, uint32_t n, double *to); // (host values as kernel arguments)

#ifdef __HIPCC__
// Elements of the three activation types as 32-bit floats and back (rounded to nearest, ties to even).
__device__ __forceinline__ float widened(float x) { return x; }
__device__ __forceinline__ float widened(_Float16 x) { return (float)x; }
__device__ __forceinline__ float widened(__bf16 x) { return (float)x; }

// N consecutive elements, in 16-byte pieces where there are as many (the hardware takes them at any element's address; a call's
// rows may lie at any).
template <class T, int N> struct Pieces {
    static constexpr int kBytes = N * (int)sizeof(T) < 16 ? N * (int)sizeof(T) : 16, kEach = kBytes / (int)sizeof(T), kCount = N / kEach;
    typedef T Piece __attribute__((ext_vector_type(kEach), aligned(sizeof(T))));
};
template <class T, int N> __device__ __forceinline__ void load_elements(const T *p, float (&x)[N]) {
    typedef Pieces<T, N> P;
    typename P::Piece v[P::kCount];
#pragma unroll
    for (int i = 0; i < P::kCount; i++) v[i] = reinterpret_cast<const typename P::Piece *>(p)[i];
#pragma unroll
    for (int i = 0; i < N; i++) x[i] = widened(v[i / P::kEach][i % P::kEach]);
}
template <class T, int N> __device__ __forceinline__ void store_elements(T *p, const float (&x)[N]) {
    typedef Pieces<T, N> P;
#pragma unroll
    for (int i = 0; i < P::kCount; i++) {
        typename P::Piece v;
#pragma unroll
        for (int j = 0; j < P::kEach; j++) v[j] = (T)x[i * P::kEach + j];
        reinterpret_cast<typename P::Piece *>(p)[i] = v;
    }
}
// A block's scale's exponent (scales are powers of two; what else a caller's memory may hold counts as the power below, within the limits).
__device__ __forceinline__ int scale_exponent(float s) {
    const int e = (int)(__float_as_uint(s) >> 23 & 255) - 127;
    return e < kLowestScale ? kLowestScale : e > kHighestScale ? kHighestScale : e;
}
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); } // e from -126 to 127
#endif

// Host: the same for one dtype's kernels, chosen by their element type.
template <class F> int with_element(cg_dtype dtype, F &&f) {
#ifdef __HIPCC__
    if (dtype == CG_F32) return f((float)0);
    if (dtype == CG_F16) return f((_Float16)0);
    if (dtype == CG_BF16) return f((__bf16)0);
#endif
    return fail(CG_ERR_DTYPE, "elements are f32, f16 or bf16");
}

} // namespace cg
