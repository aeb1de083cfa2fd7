// Rotary positions of query and key heads (their section of include/catgrad_hip.h).
//
//   x' = m (x cos a - y sin a),  y' = m (y cos a + x sin a),  a = 2 pi position * turns[i]
//
// for the pairs (x, y) of every head.  Bound by memory: every value is read and written once, in 16-byte pieces.  A workgroup
// takes up to `group` tokens.  It asks for its first values, works out its tokens' cosines and sines meanwhile, once for all heads,
// into LDS, and turns what has arrived.  The product of a position and a frequency is taken in 64 bits and reduced to a fraction of
// a turn there (in 32 bits the angle at position 2^17 would be off by 2^-7); the fraction in 32 bits is off by 2^-25 of a turn.
// Four prompts of 2048 tokens (200 MB in and out) 39 us, 5.2 TB/s (a large copy reaches 4.7); one token 2.5 us, a launch's latency.
#include "block_cache.hpp"
#include "device_utils.hpp"

#include <algorithm>

namespace cg {
namespace {

constexpr uint32_t kThreads = 256, kUnits = 4; // units of a thread, all of them asked for at once
constexpr uint32_t kMostPairs = 1024;          // cosines and sines of a workgroup

// A unit is VEC pairs of a head, or VEC values behind the turned ones.  VEC 1: pairs that are no whole 16 bytes.
template <class T, int VEC, bool INTERLEAVED> __global__ __launch_bounds__(kThreads) void rotary_kernel(RotaryPlan p) {
    __shared__ float2 turn[kMostPairs];
    const uint32_t pairs = p.rot / 2, all = p.batch.sequences * p.batch.tokens, first = blockIdx.x * p.group;
    const uint32_t n = min(p.group, all - first), units = n * p.per_token.d, pair_units = pairs / VEC;
    float x[kUnits][VEC], y[kUnits][VEC];
    T *to[kUnits];
    uint32_t at[kUnits]; // the unit's pairs in `turn`; ~0: values that go along; to null: nothing
#pragma unroll
    for (uint32_t i = 0; i < kUnits; i++) {
        const uint32_t id = (blockIdx.y * kUnits + i) * kThreads + threadIdx.x;
        to[i] = nullptr;
        at[i] = ~0u;
        if (id >= units) continue;
        const uint32_t t = fastdiv(id, p.per_token), in_token = id - t * p.per_token.d, h = fastdiv(in_token, p.per_head), u = in_token - h * p.per_head.d;
        const uint32_t token = first + t, b = fastdiv(token, p.tokens), s = token - b * p.tokens.d;
        if (s >= p.batch.count_of(b)) continue;
        const bool is_q = h < p.heads;
        const uint32_t head = is_q ? h : h - p.heads;
        const bool pair = u < pair_units;
        const uint32_t d = pair ? (INTERLEAVED ? 2 * VEC * u : VEC * u) : p.rot + VEC * (u - pair_units);
        const T *src = static_cast<const T *>(is_q ? p.q : p.k) + token * (is_q ? p.q_pitch : p.k_pitch) + head * p.dim + d;
        to[i] = static_cast<T *>(is_q ? p.q_out : p.k_out) + token * (is_q ? p.q_out_pitch : p.k_out_pitch) + head * p.dim + d;
        if (pair && INTERLEAVED) {
            float z[2 * VEC];
            load_elements<T, 2 * VEC>(src, z);
#pragma unroll
            for (int j = 0; j < VEC; j++) {
                x[i][j] = z[2 * j];
                y[i][j] = z[2 * j + 1];
            }
        } else {
            load_elements<T, VEC>(src, x[i]);
            if (pair) load_elements<T, VEC>(src + pairs, y[i]);
        }
        if (pair) at[i] = t * pairs + VEC * u;
    }
    for (uint32_t i = threadIdx.x; i < n * pairs; i += kThreads) {
        const uint32_t t = i / pairs, token = first + t, b = fastdiv(token, p.tokens), s = token - b * p.tokens.d;
        const double turns = (double)(p.batch.held_by(b) + s) * p.turns[i - t * pairs];
        float si, co;
        sincospif(2.0f * (float)(turns - rint(turns)), &si, &co);
        turn[i] = make_float2(co * p.magnitude, si * p.magnitude);
    }
    __syncthreads();
#pragma unroll
    for (uint32_t i = 0; i < kUnits; i++) {
        if (!to[i]) continue;
        if (at[i] == ~0u) {
            store_elements<T, VEC>(to[i], x[i]);
            continue;
        }
        float z[2 * VEC];
#pragma unroll
        for (int j = 0; j < VEC; j++) {
            const float2 c = turn[at[i] + j];
            const float a = fmaf(x[i][j], c.x, -y[i][j] * c.y), o = fmaf(y[i][j], c.x, x[i][j] * c.y);
            z[INTERLEAVED ? 2 * j : j] = a;
            z[INTERLEAVED ? 2 * j + 1 : VEC + j] = o;
        }
        if (INTERLEAVED) {
            store_elements<T, 2 * VEC>(to[i], z);
        } else {
            float lo[VEC], hi[VEC];
#pragma unroll
            for (int j = 0; j < VEC; j++) {
                lo[j] = z[j];
                hi[j] = z[VEC + j];
            }
            store_elements<T, VEC>(to[i], lo);
            store_elements<T, VEC>(to[i] + pairs, hi);
        }
    }
}

constexpr uint32_t kMostTurns = 256;
struct Turns {
    double f[kMostTurns];
};
__global__ void rotation_turns_kernel(Turns t, uint32_t n, double *to) {
    if (threadIdx.x < n) to[threadIdx.x] = t.f[threadIdx.x];
}

template <class T, int VEC> int launch_vec(const LaunchOn &on, RotaryPlan p) {
    const uint32_t pairs = p.rot / 2, units = (pairs + p.dim - p.rot) / VEC, per_token = units * (p.heads + (p.k ? p.kv_heads : 0));
    const uint32_t all = p.batch.sequences * p.batch.tokens;
    // as many tokens as a workgroup's threads take units of, but so many workgroups that the card is full, and within LDS
    p.group = std::max(1u, std::min({kThreads * kUnits / per_token, kMostPairs / pairs, all / 1024}));
    p.per_head = make_fastdiv(units);
    p.per_token = make_fastdiv(per_token);
    p.tokens = make_fastdiv(p.batch.tokens);
    const dim3 grid((all + p.group - 1) / p.group, (p.group * per_token + kThreads * kUnits - 1) / (kThreads * kUnits));
    return p.interleaved ? on("rotary launch", rotary_kernel<T, VEC, true>, grid, dim3(kThreads), p) : on("rotary launch", rotary_kernel<T, VEC, false>, grid, dim3(kThreads), p);
}

} // namespace

int launch_rotary(const LaunchOn &on, cg_dtype dtype, RotaryPlan p) {
    return with_element(dtype, [&](auto e) {
        typedef decltype(e) T;
        constexpr int kVec = 16 / (int)sizeof(T);
        const bool whole = p.rot / 2 % kVec == 0 && p.dim % kVec == 0;
        return whole ? launch_vec<T, kVec>(on, p) : launch_vec<T, 1>(on, p);
    });
}

int launch_rotation_table(const LaunchOn &on, const double *turns, uint32_t n, double *to) {
    Turns t{};
    std::copy(turns, turns + std::min(n, kMostTurns), t.f);
    return on("rotation table launch", rotation_turns_kernel, dim3(1), dim3(kMostTurns), t, n, to);
}

int load_rotary_kernels() {
    hipFuncAttributes a;
    CG_HIP(hipFuncGetAttributes(&a, reinterpret_cast<const void *>(rotary_kernel<float, 1, false>)));
    return CG_OK;
}

} // namespace cg
