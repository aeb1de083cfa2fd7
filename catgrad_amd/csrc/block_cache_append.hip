// New tokens' keys and values into the 8-bit cache (their section of include/catgrad_hip.h).
//
// A workgroup takes one block of positions of one head, of the keys or of the values, from the first new token that falls into it to
// the last: the largest magnitude of what is new, the block's exponent e, the codes.  All new values are asked for at once and stay in
// registers between the two, so they are read once.  Keys lie token by token: a thread takes 16 channels of a token.  Values lie channel by
// channel: a thread takes 16 neighbouring positions of a channel, reads them from 16 rows (a wave's lanes take neighbouring
// channels) and stores them in one piece, together with what the piece held of older positions.  No two workgroups share a byte
// that either writes.  A block that grew has the rest of its codes rounded anew in a second sweep, which few appends need.
// Bound by memory: 4 prompts of 2048 tokens (f32, 8 heads of 128, 84 MB) 19.1 us, 4.4 TB/s.  With 16-bit elements (50 MB, and 8 MB of codes
// that are read in front of being written) 19.0 us as well: 3.1 TB/s, what bounds that is not known.  Short ragged ones are bound by latency: 7 of up to 301 tokens (f16, 6 heads of 80 / 96, 6.7 MB) 6.9 us.
#include "block_cache.hpp"
#include "device_utils.hpp"

#include <algorithm>

namespace cg {
namespace {

constexpr uint32_t kThreads = 512, kPiece = 16; // bytes (codes) of a unit of work

__device__ __forceinline__ float code_range(float x) { // within the codes' range; NaN stays
    const float c = __builtin_amdgcn_fmed3f(x, -448.0f, 448.0f);
    return x == x ? c : x;
}
__device__ __forceinline__ uint32_t codes_of(const float *x, float inv) { // the nearest codes (ties to even) to four values times inv
    int c = __builtin_amdgcn_cvt_pk_fp8_f32(code_range(x[0] * inv), code_range(x[1] * inv), 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(code_range(x[2] * inv), code_range(x[3] * inv), c, true);
}
__device__ __forceinline__ uint32_t rounded_anew(uint32_t codes, float factor) {
    const float x[4] = {__builtin_amdgcn_cvt_f32_fp8(codes, 0), __builtin_amdgcn_cvt_f32_fp8(codes, 1), __builtin_amdgcn_cvt_f32_fp8(codes, 2),
                        __builtin_amdgcn_cvt_f32_fp8(codes, 3)};
    return codes_of(x, factor);
}
__device__ __forceinline__ uint4 rounded_anew(uint4 c, float f) { return make_uint4(rounded_anew(c.x, f), rounded_anew(c.y, f), rounded_anew(c.z, f), rounded_anew(c.w, f)); }
// The bytes of `mine` where take has ones, else those of `other`.
__device__ __forceinline__ uint32_t either(uint32_t take, uint32_t mine, uint32_t other) { return (mine & take) | (other & ~take); }

// The smallest e with size <= 448 * 2^e (448 = 1.75 * 2^8), within the limits.
__device__ __forceinline__ int exponent_for(float size) {
    const uint32_t u = __float_as_uint(size);
    const int e = (int)(u >> 23) - 127 - 8 + ((u & 0x7FFFFFu) > 0x600000u ? 1 : 0);
    return e < kLowestScale ? kLowestScale : e > kHighestScale ? kHighestScale : e;
}
__device__ __forceinline__ float largest_finite(float m, float x) { return fabsf(x) < INFINITY ? fmaxf(m, fabsf(x)) : m; }

template <class T, int UNITS, bool VALUES> __device__ void append_block(const CacheAppendPlan &p, uint32_t b, uint32_t g, uint32_t nth) {
    __shared__ float sizes[kThreads / 64];
    const Cache8 &c = p.cache;
    const uint32_t n = 1u << c.block_log2, W = VALUES ? c.vdim : c.dim;
    const uint64_t held = p.batch.held_by(b), j = (held >> c.block_log2) + nth, begin = j << c.block_log2;
    if (begin >= c.capacity) return;
    const uint64_t end = held + p.batch.count_of(b);
    // new positions of the block, counted from its first
    const uint32_t t0 = held > begin ? (uint32_t)(held - begin) : 0, t1 = (uint32_t)min((uint64_t)n, end > begin ? end - begin : 0);
    if (t0 >= t1) return;
    const uint64_t bg = (uint64_t)b * c.kv_heads + g, nb = c.capacity >> c.block_log2;
    float *const scale = (VALUES ? c.v_scale : c.k_scale) + bg * nb + j;
    const int had = t0 ? scale_exponent(*scale) : kLowestScale;
    uint8_t *const codes = VALUES ? c.v_codes + (bg * nb + j) * W * n : c.k_codes + (bg * c.capacity + begin) * W;
    // row 0: position `begin` (in front of the array where that is no new token: never addressed)
    const int64_t pitch = VALUES ? p.v_pitch : p.k_pitch;
    const T *const rows = static_cast<const T *>(VALUES ? p.v : p.k) + (int64_t)g * W;
    const int64_t row0 = (int64_t)b * p.batch.tokens + (int64_t)begin - (int64_t)held;

    const uint32_t first_piece = VALUES ? t0 / kPiece : 0, pieces = VALUES ? (t1 + kPiece - 1) / kPiece - first_piece : W / kPiece;
    const uint32_t units = VALUES ? pieces * W : pieces * (t1 - t0);
    float x[UNITS][kPiece];
    uint4 old[UNITS];
    uint4 *to[UNITS];
    uint32_t piece[UNITS];
    float size = 0.0f;
#pragma unroll
    for (int i = 0; i < UNITS; i++) {
        const uint32_t id = i * blockDim.x + threadIdx.x;
        to[i] = nullptr;
        if (id >= units) continue;
        if (VALUES) {
            const uint32_t k = id / W, d = id - k * W;
            piece[i] = (first_piece + k) * kPiece;
            to[i] = reinterpret_cast<uint4 *>(codes + (uint64_t)d * n + piece[i]);
            old[i] = *to[i];
#pragma unroll
            for (uint32_t q = 0; q < kPiece; q++) { // (places that are not new: a new one's value, then zero, so that no load hangs on a branch)
                const uint32_t t = piece[i] + q;
                const float v = widened(rows[(row0 + min(max(t, t0), t1 - 1)) * pitch + d]);
                x[i][q] = t >= t0 && t < t1 ? v : 0.0f;
            }
        } else {
            const uint32_t t = id / pieces, k = id - t * pieces;
            to[i] = reinterpret_cast<uint4 *>(codes + (uint64_t)(t0 + t) * W + k * kPiece);
            load_elements<T, kPiece>(rows + (row0 + t0 + t) * pitch + k * kPiece, x[i]);
        }
    }
#pragma unroll
    for (int i = 0; i < UNITS; i++)
        if (to[i])
#pragma unroll
            for (uint32_t q = 0; q < kPiece; q++) size = largest_finite(size, x[i][q]);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) size = fmaxf(size, __shfl_xor(size, o));
    if (threadIdx.x % 64 == 0) sizes[threadIdx.x / 64] = size;
    __syncthreads();
    size = sizes[0];
    for (uint32_t i = 1; i < blockDim.x / 64; i++) size = fmaxf(size, sizes[i]);
    const int e = max(had, exponent_for(size)); // (a size of 0: the lowest)
    const bool grew = t0 && e > had;
    const float inv = power_of_two(-e), down = power_of_two(max(had - e, -64)); // (2^-64 leaves nothing of any code)
    if (threadIdx.x == 0) *scale = power_of_two(e); // (read by all in front of the barrier)
#pragma unroll
    for (int i = 0; i < UNITS; i++) {
        if (!to[i]) continue;
        uint4 r = make_uint4(codes_of(&x[i][0], inv), codes_of(&x[i][4], inv), codes_of(&x[i][8], inv), codes_of(&x[i][12], inv));
        if (VALUES && (piece[i] < t0 || piece[i] + kPiece > t1)) {
            const uint4 anew = grew ? rounded_anew(old[i], down) : old[i];
            uint32_t m[4], past[4]; // bytes that are new, that are of older positions
#pragma unroll
            for (uint32_t w = 0; w < 4; w++) {
                m[w] = past[w] = 0;
#pragma unroll
                for (uint32_t q = 0; q < 4; q++) {
                    const uint32_t t = piece[i] + 4 * w + q;
                    m[w] |= t >= t0 && t < t1 ? 255u << (8 * q) : 0;
                    past[w] |= t < t0 ? 255u << (8 * q) : 0;
                }
            }
            r = make_uint4(either(m[0], r.x, either(past[0], anew.x, old[i].x)), either(m[1], r.y, either(past[1], anew.y, old[i].y)),
                           either(m[2], r.z, either(past[2], anew.z, old[i].z)), either(m[3], r.w, either(past[3], anew.w, old[i].w)));
        }
        *to[i] = r;
    }
    if (!grew) return;
    // pieces that hold older positions alone
    const uint32_t rest = VALUES ? t0 / kPiece * W : t0 * pieces;
    for (uint32_t id = threadIdx.x; id < rest; id += blockDim.x) {
        uint4 *at;
        if (VALUES) {
            const uint32_t k = id / W, d = id - k * W;
            at = reinterpret_cast<uint4 *>(codes + (uint64_t)d * n + k * kPiece);
        } else {
            at = reinterpret_cast<uint4 *>(codes) + id;
        }
        *at = rounded_anew(*at, down);
    }
}

// One token a sequence, as in every step of a decoder: a wave takes a head's keys or values, a lane four channels of them.  Nothing of
// the block is read but its scale, unless that grows: then every lane rounds anew what lies in its own channels' (values) or
// places' (keys) bytes, and no lane touches another's.  64 sequences of 8 heads of 128 bf16
// channels: 4.3 us, all of it latency (a launch, the positions held, the scale and the token), where the workgroups above take 6.4 for their barrier, their
// four times as many waves and the pieces of the block that a value is put into.
template <class T, bool VALUES> __device__ void append_token(const CacheAppendPlan &p, uint32_t b, uint32_t g, uint32_t lane) {
    const Cache8 &c = p.cache;
    const uint32_t n = 1u << c.block_log2, W = VALUES ? c.vdim : c.dim, d = lane * 4;
    const bool mine = d < W;
    const uint64_t held = p.batch.held_by(b), j = held >> c.block_log2;
    if (held >= c.capacity || !p.batch.count_of(b)) return;
    float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (mine) load_elements<T, 4>(static_cast<const T *>(VALUES ? p.v : p.k) + (int64_t)b * (VALUES ? p.v_pitch : p.k_pitch) + g * W + d, x);
    const uint32_t t = (uint32_t)held & (n - 1);
    const uint64_t bg = (uint64_t)b * c.kv_heads + g, nb = c.capacity >> c.block_log2;
    float *const scale = (VALUES ? c.v_scale : c.k_scale) + bg * nb + j;
    const int had = t ? scale_exponent(*scale) : kLowestScale;
    uint8_t *const codes = VALUES ? c.v_codes + ((bg * nb + j) * W + d) * n : c.k_codes + (bg * c.capacity + (j << c.block_log2)) * W;
    float size = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; i++) size = largest_finite(size, x[i]);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) size = fmaxf(size, __shfl_xor(size, o));
    const int e = max(had, exponent_for(size));
    const uint32_t made = codes_of(x, power_of_two(-e));
    if (lane == 0) *scale = power_of_two(e); // (every lane's own read of it stands in front of the exchange above)
    if (t && e > had) {
        const float down = power_of_two(max(had - e, -64)); // (2^-64 leaves nothing of any code)
        if (VALUES) {
            for (uint32_t i = 0; mine && i < 4; i++)
                for (uint32_t k = 0; k * kPiece < t; k++) {
                    uint4 *const at = reinterpret_cast<uint4 *>(codes + (uint64_t)i * n + k * kPiece);
                    const uint4 old = *at, anew = rounded_anew(old, down);
                    uint32_t past[4];
#pragma unroll
                    for (uint32_t w = 0; w < 4; w++) {
                        const uint32_t first = k * kPiece + 4 * w;
                        past[w] = t >= first + 4 ? ~0u : t > first ? (1u << (8 * (t - first))) - 1 : 0;
                    }
                    *at = make_uint4(either(past[0], anew.x, old.x), either(past[1], anew.y, old.y), either(past[2], anew.z, old.z), either(past[3], anew.w, old.w));
                }
        } else {
            for (uint32_t i = lane; i < t * (W / kPiece); i += 64) {
                uint4 *const at = reinterpret_cast<uint4 *>(codes) + i;
                *at = rounded_anew(*at, down);
            }
        }
    }
    if (!mine) return;
    if (VALUES) {
#pragma unroll
        for (uint32_t i = 0; i < 4; i++) codes[(uint64_t)i * n + t] = (uint8_t)(made >> (8 * i));
    } else {
        *reinterpret_cast<uint32_t *>(codes + (uint64_t)t * W + d) = made;
    }
}
template <class T> __global__ __launch_bounds__(64) void cache_append_token_kernel(CacheAppendPlan p) {
    const uint32_t id = blockIdx.x >> 1, g = id % p.cache.kv_heads, b = id / p.cache.kv_heads;
    if (blockIdx.x & 1) append_token<T, true>(p, b, g, threadIdx.x);
    else append_token<T, false>(p, b, g, threadIdx.x);
}

template <class T, int UNITS> __global__ __launch_bounds__(kThreads) void cache_append_kernel(CacheAppendPlan p, uint32_t touched) {
    uint32_t id = blockIdx.x;
    const uint32_t nth = id % touched;
    id /= touched;
    const bool values = id & 1;
    id >>= 1;
    const uint32_t g = id % p.cache.kv_heads, b = id / p.cache.kv_heads;
    if (values) append_block<T, UNITS, true>(p, b, g, nth);
    else append_block<T, UNITS, false>(p, b, g, nth);
}

} // namespace

AppendShape shape_cache_append(const CacheAppendPlan &p) {
    const uint32_t n = 1u << p.cache.block_log2, heads = p.cache.kv_heads * 2;
    if (p.batch.tokens == 1) return {1, 64, (uint64_t)p.batch.sequences * heads};
    const uint32_t touched = std::min(p.cache.capacity / n, (p.batch.tokens + n - 2) / n + 1);
    // a thread for a piece of a block, up to 512, then up to four of the largest blocks' pieces a thread (2 x 500 tokens, f32, heads of 256 in blocks of 128: 12.0 us;
    // with half as many threads and twice as many pieces each 15.4)
    const uint32_t pieces = n * std::max(p.cache.dim, p.cache.vdim) / kPiece;
    return {touched, std::min(kThreads, (pieces + 63) / 64 * 64), (uint64_t)touched * p.batch.sequences * heads};
}

int launch_cache_append(const LaunchOn &on, cg_dtype dtype, const CacheAppendPlan &p) {
    const AppendShape s = shape_cache_append(p);
    return with_element(dtype, [&](auto e) {
        typedef decltype(e) T;
        const dim3 grid((uint32_t)s.groups), block(s.threads);
        if (p.batch.tokens == 1) return on("cache append launch", cache_append_token_kernel<T>, grid, block, p);
        const uint32_t pieces = (std::max(p.cache.dim, p.cache.vdim) << p.cache.block_log2) / kPiece;
        return pieces <= kThreads ? on("cache append launch", cache_append_kernel<T, 1>, grid, block, p, s.touched)
                                  : on("cache append launch", cache_append_kernel<T, 4>, grid, block, p, s.touched);
    });
}

int load_cache_append_kernels() {
    hipFuncAttributes a;
    CG_HIP(hipFuncGetAttributes(&a, reinterpret_cast<const void *>(cache_append_kernel<float, 1>)));
    return CG_OK;
}

} // namespace cg
