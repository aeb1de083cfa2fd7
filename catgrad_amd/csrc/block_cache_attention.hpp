// Attention over the 8-bit cache (their section of include/catgrad_hip.h): the kernel, instantiated by element type in
// block_cache_attention_{f32,f16,bf16}.hip and launched from block_cache_attention.hip.
//
// One pass over the codes with the running maximum and sum of the soft-max, on v_mfma_f32_16x16x32_f16.  A wave takes tiles of 64
// positions and up to 32 rows (a row: one query head of one token; the heads that share a key / value head lie together), all in
// registers.  The products are taken transposed, scores^T = K q^T and out^T = V^T P^T, with the positions of a tile dealt out so
// that nothing has to change lanes between the two: the instruction leaves a lane four scores of one row (its column), at rows
// 4 quad + i of the left operand, and wants eight neighbouring values of k of one column from it.  So row 4 a + i of the kt-th left
// operand (kt = 0 .. 3) is position 16 a + 4 kt + i: a lane's 16 scores are the positions 16 quad .. 16 quad + 15 of its row, the
// weights of the second product as they come, and its codes of a value channel for them are 16 neighbouring bytes (values lie
// channel by channel within a block).  Channels of K are dealt out the same way, 16 neighbouring bytes of a position's key to a lane.  So all
// codes come by 16-byte loads straight into the registers from which the instruction takes them, without LDS or barriers.
//
// Numbers.  E4M3 codes are exact in 16-bit floats.  A row of q is scaled by a power of two so that its largest magnitude lies
// in [2^7, 2^8), and is one 16-bit float a value, or with 32-bit inputs the sum of two (2^-23 of the row's largest; 16-bit inputs are
// exact but where they lie 2^22 below it).  Bfloat16 queries of more than 64 channels are two codes instead, the nearest and the nearest to what is left, together exact but
// where they lie 2^14 below the row's largest (there to 2^-22 of it): then the instruction takes the keys' codes as they are (v_mfma_scale_f32_16x16x128_f8f6f4, at twice the rate, so that the two cost
// what one 16-bit float does, without the widening of keys: four prompts of 2048 tokens of 16 heads of 128, 84 us against 89).  A block's scale multiplies the scores in 32 bits.  Weights are exp2(score - m) <= 2^15
// with m the running maximum less 8, which moves only where a score is 15 or more above it (most tiles move none: then nothing is
// rescaled).  A score is a product whose difference from m is rounded once; behind a maximum beyond 2^20 the product is rounded first, as the maximum is, so that no score seems to lie above
// its own maximum; where 8 is less than half a step of the scores, m is the maximum itself.  Weights are held
// as one 16-bit float (2^-12) or two (2^-23), and so is their sum, by the same instruction from ones.  Either way a weight is off by up to
// 2^-33 of its row's largest, and may be zero below that.
// Totals are in units of a scale 2^unit.  Where many rows have 16-bit results and all value blocks that a workgroup's rows see have scales within
// 2^15 of each other (they are looked over in front: ScaleRange), the unit is the largest of them, codes are widened times their scale in it, which is exact, and
// the instruction adds to the totals itself.  It cuts its sums off a little below their last bit: results of 16-bit floats measured 2^-13.6 too small behind 4 million positions in
// one part, 2^-12 behind 16 million, where half a step is 2^-11; so it does up to kMostTiles tiles.
// Else the products of a tile start from zero, in units of the tile's largest scale, and a vector instruction adds them to totals whose unit is the largest scale
// so far, times the one in units of the other: the unit only rises, so that no total grows beyond its sum of weights times codes, and a block of zeros, whose scale is
// the smallest, adds zeros.  (Scales lie within 2^236 of each other: where a row sees nothing but values 2^126 below those of another row of its wave, its total runs
// out of the normal numbers, to 2^-157 of the wave's largest scale.)  A tile whose blocks of 16 or 32 positions lie farther than 2^15 apart is taken a block at a time.  (Prompts of 4 x 2048 tokens, bf16, 16 heads of 128:
// 87 us, the second way 96.)
//
// Positions that a row does not see: their weights are set to zero, and since zero times NaN is NaN, a tile that not all rows
// see whole has its NaN codes of values taken out, and put back into the totals of the rows that do see them.
#pragma once

#include <type_traits>

#include "block_cache.hpp"
#include "device_utils.hpp"

namespace cg {

typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef _Float16 half8v __attribute__((ext_vector_type(8)));
typedef float float4v __attribute__((ext_vector_type(4)));
typedef float float2v __attribute__((ext_vector_type(2)));
typedef int int8v __attribute__((ext_vector_type(8)));
typedef short short2v __attribute__((ext_vector_type(2)));

constexpr uint32_t kTile = 64;           // positions of a wave's tile
constexpr uint32_t kWavesOfAttention = 4;
constexpr float kNoMaximum = -3.0e38f;   // of a row that has seen nothing
constexpr float kFar = 0x1p20f;          // scores below are rounded by less than 2^-4
constexpr uint32_t kMostTiles = 65536;   // that the instruction adds to totals itself
constexpr int kExact = 15; // a code times 2^-15 is exact as a 16-bit float (whole multiples of 2^-9, 2^-24)
// The fewest tiles worth a part of their own: of a token behind 8000 12.9 us, with eight 14.4; a prompt of 1024 tokens of nine heads 23 us, with eight 34.
constexpr uint32_t kLeastTiles = 4;

// The positions that rows of the tokens s0 .. s1 of a sequence see, cut into at most `splits` parts of whole tiles.
struct KeyRange {
    uint32_t end, first_tile, end_tile, parts, each;
};
__device__ __forceinline__ KeyRange key_range(const CacheAttentionPlan &p, uint64_t held, uint32_t s0, uint32_t s1) {
    const uint64_t C = p.cache.capacity, end = min(held + s1 + 1, C), q0 = held + s0 + 1;
    const uint64_t lo = p.window && q0 > p.window ? min(q0 - p.window, end) : 0;
    KeyRange r;
    r.end = (uint32_t)end;
    r.first_tile = (uint32_t)(lo / kTile);
    r.end_tile = (uint32_t)((end + kTile - 1) / kTile);
    const uint32_t n = r.end_tile - r.first_tile;
    r.parts = max(1u, min(p.splits, n / kLeastTiles));
    r.each = (n + r.parts - 1) / r.parts;
    return r;
}

#ifdef __HIPCC__
// codes 2 i, 2 i + 1 of a word, times a power of two, as 16-bit floats (exact with 1)
template <bool HIGH> __device__ __forceinline__ half2v two_of(uint32_t codes, float scale) { return __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)codes, scale, HIGH); }
__device__ __forceinline__ half8v eight_of(uint32_t lo, uint32_t hi, float scale) {
    const half2v a = two_of<false>(lo, scale), b = two_of<true>(lo, scale), c = two_of<false>(hi, scale), d = two_of<true>(hi, scale);
    return half8v{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
__device__ __forceinline__ uint32_t word_of(const uint4 &v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }
// the k-th eight codes of sixteen
__device__ __forceinline__ half8v eight_of(const uint4 &v, int k, float scale = 1.0f) { return eight_of(word_of(v, 2 * k), word_of(v, 2 * k + 1), scale); }
__device__ __forceinline__ uint32_t nan_bytes(uint32_t c) { return ((c & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u; } // bit 7 of the bytes that are NaN
__device__ __forceinline__ uint4 without_nan(const uint4 &c) {
    return make_uint4(c.x & ~((nan_bytes(c.x) >> 7) * 255), c.y & ~((nan_bytes(c.y) >> 7) * 255), c.z & ~((nan_bytes(c.z) >> 7) * 255), c.w & ~((nan_bytes(c.w) >> 7) * 255));
}
// over the four lanes that share a row
__device__ __forceinline__ float quads_max(float x) {
    x = fmaxf(x, __shfl_xor(x, 16));
    return fmaxf(x, __shfl_xor(x, 32));
}
__device__ __forceinline__ int quads_max(int x) {
    x = max(x, __shfl_xor(x, 16));
    return max(x, __shfl_xor(x, 32));
}
__device__ __forceinline__ uint32_t quads_max(uint32_t x) {
    x = max(x, (uint32_t)__shfl_xor((int)x, 16));
    return max(x, (uint32_t)__shfl_xor((int)x, 32));
}

// What a wave knows of its rows, and does with a tile.  RT: 16-row groups; NL: 64-channel pieces of a head.  CUT: heads of at most 96
// channels, whose second 64 are two pieces of 16 (in 16-bit floats one step of the products, of which the quads take eight channels each) and whose values
// are six groups of 16, not eight (only where rows are many: few are bound by memory).  Portions of 3 x 500 tokens behind texts, f32 heads of 96 / 80: 86 us where it was 102.
template <class T, int NL, int RT, bool CUT = false> struct AttentionWave {
    static_assert(!CUT || NL == 2, "");
    static constexpr int kPieces = sizeof(T) == 4 ? 2 : 1, NV = CUT ? 6 : 4 * NL, kSteps = CUT ? 3 : 2 * NL;

    // Queries as codes, for the instructions that take both operands as such.
    static constexpr bool kCodes = std::is_same<T, __bf16>::value && NL >= 2;
    static constexpr int kQueryPieces = kCodes ? 2 : kPieces, kQuerySteps = kCodes ? NL / 2 : kSteps;
    static constexpr bool kHalves = CUT && !kCodes; // quads 2 and 3 take the second eight channels of what 0 and 1 take
    static constexpr int kLower = 5; // the second codes are in units of 2^-5

    const CacheAttentionPlan &p;
    const uint32_t lane = threadIdx.x & 63, col = lane & 15, quad = lane >> 4;
    uint32_t b, g, row0, R;
    typename std::conditional<kCodes, int8v, half8v>::type q[RT][kQueryPieces][kQuerySteps];
    float row_factor[RT];
    uint32_t begin[RT], seen_by[RT]; // the lane's rows see seen_by positions from begin on
    int all_from, all_to, any_from, any_to; // positions that all of the wave's rows see, that any does
    // Totals: sums of weight * value in units of 2^unit.  sums: of the weights, by the same instruction from ones; the first counts.
    float4v total[RT][NV];
    float4v sums[RT];
    float maximum[RT];    // less 8: see the top
    bool rounded = false; // scores are rounded in front of their difference from it
    int unit = kLowestScale;
    // of the tile at hand
    float4v score[RT][4];
    int mine;    // the lane's first position
    bool masked; // not all rows see all of it

    __device__ __forceinline__ AttentionWave(const CacheAttentionPlan &plan) : p(plan) {}
    __device__ __forceinline__ int64_t token_of(int rt) const { return (int64_t)b * p.batch.tokens + fastdiv(min(row0 + rt * 16 + col, R - 1), p.rep_div); }

    // The queries of rows row0 .. of a pair's R rows: asked for, and made ready.
    typedef float Queries[RT][NL][16];
    __device__ __forceinline__ void ask_rows(Queries &x) const {
        const Cache8 &c = p.cache;
        const T *src[RT];
#pragma unroll
        for (int rt = 0; rt < RT; rt++) {
            const uint32_t rr = min(row0 + rt * 16 + col, R - 1), s = fastdiv(rr, p.rep_div);
            src[rt] = static_cast<const T *>(p.q) + ((int64_t)b * p.batch.tokens + s) * p.q_pitch + (g * p.rep + rr - s * p.rep) * c.dim;
        }
#pragma unroll
        for (int rt = 0; rt < RT; rt++)
#pragma unroll
            for (int l = 0; l < NL; l++) load_elements<T, 16>(src[rt] + min(channel(l), c.dim - 16), x[rt][l]); // (behind dim: the last channels again, below zeros)
    }
    __device__ __forceinline__ void begin_rows(Queries &x, uint64_t held) {
        const Cache8 &c = p.cache;
        all_from = 0, all_to = 0x7FFFFFFF, any_from = 0x7FFFFFFF, any_to = -1;
#pragma unroll
        for (int rt = 0; rt < RT; rt++) {
            const uint32_t r = row0 + rt * 16 + col;
            const uint64_t at = held + fastdiv(min(r, R - 1), p.rep_div); // its position
            const int last = r < R ? (int)min(at, (uint64_t)c.capacity - 1) : -1;
            begin[rt] = last >= 0 && p.window && at + 1 > p.window ? (uint32_t)min(at + 1 - p.window, (uint64_t)c.capacity) : 0;
            seen_by[rt] = (uint32_t)(last + 1) - begin[rt];
            uint32_t largest = 0; // magnitude, by its bits
#pragma unroll
            for (int l = 0; l < NL; l++)
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    largest = max(largest, __float_as_uint(x[rt][l][i]) & 0x7FFFFFFFu);
                }
            largest = quads_max(largest);
            const bool finite = largest < 0x7F800000u; // (else the row's scores are NaN)
            const int e = finite && largest ? __builtin_amdgcn_frexp_expf(__uint_as_float(largest)) : 0;
            row_factor[rt] = finite ? ldexpf(fabsf(p.scale) * 1.44269504088896341f, e - 8) : NAN;
            // times 2^(8 - e), the sign of the scale and, behind dim, zero (a row that is not finite: its factor makes its scores NaN)
            const int up = 8 - e;
            if (__any(up > 126)) { // (2^(8 - e) would be no float)
#pragma unroll
                for (int l = 0; l < NL; l++)
#pragma unroll
                    for (int i = 0; i < 16; i++) x[rt][l][i] = __builtin_amdgcn_ldexpf(x[rt][l][i], max(up - 126, 0));
            }
            const float by = copysignf(power_of_two(min(up, 126)), p.scale);
#pragma unroll
            for (int l = 0; l < NL; l++) {
                const float f = channel(l) < c.dim ? by : 0.0f;
                if constexpr (kCodes) {
#pragma unroll
                    for (int w = 0; w < 4; w++) {
                        float y[4];
#pragma unroll
                        for (int i = 0; i < 4; i++) y[i] = x[rt][l][w * 4 + i] * f;
                        int codes = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
                        codes = __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], codes, true);
                        const float2v a = __builtin_amdgcn_cvt_pk_f32_fp8(codes, false), b = __builtin_amdgcn_cvt_pk_f32_fp8(codes, true);
                        constexpr float unit_of_lower = 1.0f / (1 << kLower);
                        short2v lower = {};
                        lower = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(lower, y[0] - a[0], y[1] - a[1], unit_of_lower, false);
                        lower = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(lower, y[2] - b[0], y[3] - b[1], unit_of_lower, true);
                        q[rt][0][l / 2][l % 2 * 4 + w] = codes;
                        q[rt][1][l / 2][l % 2 * 4 + w] = __builtin_bit_cast(int, lower);
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < (kHalves && l == 1 ? 8 : 16); i++) {
                        const float y = (kHalves && l == 1 && quad >= 2 ? x[rt][l][(8 + i) % 16] : x[rt][l][i]) * f;
                        const _Float16 h = (_Float16)y;
                        q[rt][0][2 * l + i / 8][i % 8] = h;
                        if (kPieces == 2) q[rt][kPieces - 1][2 * l + i / 8][i % 8] = (_Float16)(y - (float)h);
                    }
                }
            }
            if (last >= 0) {
                all_from = max(all_from, (int)begin[rt]);
                all_to = min(all_to, last);
                any_from = min(any_from, (int)begin[rt]);
                any_to = max(any_to, last);
            }
            maximum[rt] = kNoMaximum;
            sums[rt] = {};
#pragma unroll
            for (int v = 0; v < NV; v++) total[rt][v] = float4v{0.0f, 0.0f, 0.0f, 0.0f};
        }
#pragma unroll
        for (int o = 1; o < 16; o <<= 1) {
            all_from = max(all_from, __shfl_xor(all_from, o));
            all_to = min(all_to, __shfl_xor(all_to, o));
            any_from = min(any_from, __shfl_xor(any_from, o));
            any_to = max(any_to, __shfl_xor(any_to, o));
        }
        all_from = __builtin_amdgcn_readfirstlane(all_from);
        all_to = __builtin_amdgcn_readfirstlane(all_to);
        any_from = __builtin_amdgcn_readfirstlane(any_from);
        any_to = __builtin_amdgcn_readfirstlane(any_to);
    }

    // The first of the lane's 16 channels of a piece.
    __device__ __forceinline__ uint32_t channel(int l) const { return l * 64 + (kHalves && l == 1 ? quad & 1 : quad) * 16; }
    // Where a tile's codes lie, from an address that is the same for all lanes (tile t, position row kt or channel group v) and one of the lane's
    // (behind dim the query is zero: any code of the same key will do).
    __device__ __forceinline__ uint32_t key_lane(int l) const {
        const uint32_t d = channel(l);
        return ((col >> 2) * 16 + (col & 3)) * p.cache.dim + (d < p.cache.dim ? d : 0);
    }
    __device__ __forceinline__ uint64_t key_tile(uint32_t t, int kt) const { return ((uint64_t)t * kTile + kt * 4) * p.cache.dim; }
    __device__ __forceinline__ uint32_t value_lane() const {
        const uint32_t n = p.cache.block_log2, at = quad * 16;
        return (((at >> n) * p.cache.vdim + col) << n) + (at & ((1u << n) - 1));
    }
    __device__ __forceinline__ uint64_t value_tile(uint32_t t, int v) const { // (behind vdim: the last channels again; nothing is made of their totals)
        const uint32_t n = p.cache.block_log2, at = t * kTile;
        return (((uint64_t)(at >> n) * p.cache.vdim + min(v * 16u, p.cache.vdim - 16)) << n) + (at & ((1u << n) - 1));
    }
    // A tile that reaches behind the capacity, where no row sees anything: lanes there take the cache's last position or block.
    __device__ __forceinline__ bool reaches_beyond(uint32_t t) const { return (t + 1) * kTile > p.cache.capacity; }
    __device__ __forceinline__ uint64_t key_at_end(uint32_t t, int kt, int l) const {
        const uint32_t at = min(t * kTile + (col >> 2) * 16 + kt * 4 + (col & 3), p.cache.capacity - 1), d = channel(l);
        return (uint64_t)at * p.cache.dim + (d < p.cache.dim ? d : 0);
    }
    __device__ __forceinline__ uint64_t value_at_end(uint32_t t, int v) const {
        const uint32_t n = p.cache.block_log2, at = (t * kTile + quad * 16) & ((1u << n) - 1);
        return (((uint64_t)block_of(t) * p.cache.vdim + min(v * 16u, p.cache.vdim - 16) + col) << n) + at;
    }
    __device__ __forceinline__ uint32_t block_of(uint32_t t) const { return min((t * kTile + quad * 16) >> p.cache.block_log2, (p.cache.capacity >> p.cache.block_log2) - 1); }

    __device__ __forceinline__ bool sees(int rt, int i) const { return (uint32_t)mine - begin[rt] + (uint32_t)i < seen_by[rt]; } // i: of the lane's 16 positions

    // scores^T; keys(kt, l): the codes
    template <class K> __device__ __forceinline__ void scores(uint32_t t, K &&keys) {
        const int at = (int)(t * kTile);
        mine = at + (int)quad * 16;
        masked = at < all_from || at + (int)kTile - 1 > all_to;
        uint4 codes[4][NL]; // (asked for one row of positions ahead)
#pragma unroll
        for (int l = 0; l < NL; l++) codes[0][l] = keys(0, l);
#pragma unroll
        for (int kt = 0; kt < 4; kt++) {
#pragma unroll
            for (int l = 0; l < NL && kt < 3; l++) codes[kt + 1][l] = keys(kt + 1, l);
            __builtin_amdgcn_sched_barrier(0);
            if constexpr (kCodes) {
                int8v a[kQuerySteps];
#pragma unroll
                for (int l = 0; l < NL; l++)
#pragma unroll
                    for (int w = 0; w < 4; w++) a[l / 2][l % 2 * 4 + w] = (int)word_of(codes[kt][l], w);
#pragma unroll
                for (int rt = 0; rt < RT; rt++) {
                    float4v s = {0.0f, 0.0f, 0.0f, 0.0f};
                    constexpr int one = 0x7F7F7F7F, lower = one - 0x01010101 * kLower; // scales: 2^(byte - 127)
#pragma unroll
                    for (int piece = 1; piece >= 0; piece--)
#pragma unroll
                        for (int st = 0; st < kQuerySteps; st++) s = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a[st], q[rt][piece][st], s, 0, 0, 0, one, 0, piece ? lower : one);
                    score[rt][kt] = s;
                }
            } else {
                half8v a[kSteps];
#pragma unroll
                for (int l = 0; l < NL; l++) {
                    const uint4 &k = codes[kt][l];
                    if (kHalves && l == 1) {
                        a[2] = eight_of(quad < 2 ? k.x : k.z, quad < 2 ? k.y : k.w, 1.0f);
                        continue;
                    }
                    a[2 * l] = eight_of(k, 0);
                    a[2 * l + 1] = eight_of(k, 1);
                }
#pragma unroll
                for (int rt = 0; rt < RT; rt++) {
                    float4v s = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int piece = kPieces - 1; piece >= 0; piece--)
#pragma unroll
                        for (int st = 0; st < kSteps; st++) s = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[st], q[rt][piece][st], s, 0, 0, 0);
                    score[rt][kt] = s;
                }
            }
        }
    }

    // The scores become weights; ks: the scale of the lane's block.
    __device__ __forceinline__ void weigh(float ks) {
        float factor[RT], largest[RT];
        bool moves = false;
#pragma unroll
        for (int rt = 0; rt < RT; rt++) {
            factor[rt] = row_factor[rt] * ks;
            float m = -INFINITY;
            if (masked) {
#pragma unroll
                for (int i = 0; i < 16; i++) m = fmaxf(m, sees(rt, i) ? score[rt][i / 4][i % 4] : -INFINITY);
            } else {
#pragma unroll
                for (int i = 0; i < 16; i++) m = fmaxf(m, score[rt][i / 4][i % 4]);
            }
            largest[rt] = m == -INFINITY ? m : m * factor[rt]; // (a block that nobody has begun may have any scale: a negative one would make this infinite)
            moves = moves || largest[rt] - maximum[rt] > 15.0f;
        }
        if (__any(moves)) {
            bool far = false;
#pragma unroll
            for (int rt = 0; rt < RT; rt++) {
                const float top = quads_max(largest[rt]), below = top - 8.0f, m = fmaxf(maximum[rt], top - below > 8.0f ? top : below);
                const float down = __builtin_amdgcn_exp2f(maximum[rt] - m);
                maximum[rt] = m;
                far = far || (fabsf(m) > kFar && m > kNoMaximum);
                sums[rt][0] *= down;
#pragma unroll
                for (int v = 0; v < NV; v++) total[rt][v] *= down;
            }
            rounded = __any(far) || rounded;
        }
        if (rounded) {
#pragma unroll
            for (int rt = 0; rt < RT; rt++) {
#pragma unroll
                for (int i = 0; i < 16; i++) score[rt][i / 4][i % 4] *= factor[rt];
                factor[rt] = 1.0f;
            }
        }
#pragma unroll
        for (int rt = 0; rt < RT; rt++) {
#pragma unroll
            for (int i = 0; i < 16; i++) score[rt][i / 4][i % 4] = __builtin_amdgcn_exp2f(fmaf(score[rt][i / 4][i % 4], factor[rt], -maximum[rt]));
            if (masked) {
#pragma unroll
                for (int i = 0; i < 16; i++) score[rt][i / 4][i % 4] = sees(rt, i) ? score[rt][i / 4][i % 4] : 0.0f;
            }
        }
    }

    // out^T += V^T weights^T; values(v): the codes, without NaN from the call of clean() on; vs: the scale of the lane's block.  DIRECT: the
    // instruction adds to the totals, in whose unit all of the tile's codes are exact.
    template <bool DIRECT, class V, class C> __device__ __forceinline__ void products(float vs, V &&values, C &&clean) {
        // NaN among the values of a tile that not every row sees whole
        if (masked) {
            uint32_t found = 0;
#pragma unroll
            for (int v = 0; v < NV; v++) {
                const uint4 codes = values(v);
                found |= nan_bytes(codes.x) | nan_bytes(codes.y) | nan_bytes(codes.z) | nan_bytes(codes.w);
            }
            asm volatile("" ::: "memory"); // (codes in LDS are read where they are used, not all of them in front)
            if (__any(found != 0)) {
#pragma unroll
                for (int rt = 0; rt < RT; rt++) {
                    half8v seen[2];
#pragma unroll
                    for (int i = 0; i < 16; i++) seen[i / 8][i % 8] = sees(rt, i) ? (_Float16)1.0f : (_Float16)0.0f;
#pragma unroll
                    for (int v = 0; v < NV; v++) {
                        const uint4 codes = values(v);
                        float4v n = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                        for (int st = 0; st < 2; st++) { // from the code of 1 where a NaN is
                            const uint32_t lo = (nan_bytes(word_of(codes, 2 * st)) >> 7) * 0x38, hi = (nan_bytes(word_of(codes, 2 * st + 1)) >> 7) * 0x38;
                            n = __builtin_amdgcn_mfma_f32_16x16x32_f16(eight_of(lo, hi, 1.0f), seen[st], n, 0, 0, 0);
                        }
#pragma unroll
                        for (int i = 0; i < 4; i++) total[rt][v][i] = n[i] > 0.0f ? NAN : total[rt][v][i];
                        __builtin_amdgcn_sched_barrier(0); // (few do this: in few registers)
                    }
                }
                clean();
            }
        }
        int e = scale_exponent(vs), largest_e = 0, smallest_e = 0; // of the lane's value block; of the tile
        if constexpr (!DIRECT) {
            if (p.cache.block_log2 < 6) {
                const bool seen = mine + 15 >= any_from && mine <= any_to; // (a block that no row sees counts for nothing: its scale may be anything)
                const int none = -1000;
                largest_e = quads_max(seen ? e : none);
                smallest_e = -quads_max(seen ? -e : none);
                if (largest_e == none) largest_e = smallest_e = kLowestScale;
                e = seen ? e : largest_e;
            } else {
                largest_e = smallest_e = e;
            }
            largest_e = __builtin_amdgcn_readfirstlane(largest_e);
            smallest_e = __builtin_amdgcn_readfirstlane(smallest_e);
        }
        half8v w[RT][kPieces][2];
        const half8v ones = {1, 1, 1, 1, 1, 1, 1, 1};
#pragma unroll
        for (int rt = 0; rt < RT; rt++) {
#pragma unroll
            for (int i = 0; i < 16; i++) {
                const float x = score[rt][i / 4][i % 4];
                const _Float16 h = (_Float16)x;
                w[rt][0][i / 8][i % 8] = h;
                if (kPieces == 2) w[rt][kPieces - 1][i / 8][i % 8] = (_Float16)(x - (float)h);
            }
            float4v s = DIRECT ? sums[rt] : float4v{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int piece = kPieces - 1; piece >= 0; piece--)
#pragma unroll
                for (int st = 0; st < 2; st++) s = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, w[rt][piece][st], s, 0, 0, 0);
            if (DIRECT) sums[rt] = s;
            else sums[rt][0] += s[0];
        }
        // a pass over the tile's values, their codes times the lane's `scale`; by: a unit of its sums in units of the totals
        auto add = [&](float scale, float by) {
            constexpr int kAhead = 2;
            uint4 codes[NV];
#pragma unroll
            for (int v = 0; v < kAhead; v++) codes[v] = values(v);
#pragma unroll
            for (int v = 0; v < NV; v++) {
                half8v a[2];
                if (v + kAhead < NV) codes[v + kAhead] = values(v + kAhead);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int st = 0; st < 2; st++) a[st] = eight_of(codes[v], st, scale);
#pragma unroll
                for (int rt = 0; rt < RT; rt++) {
                    float4v s = DIRECT ? total[rt][v] : float4v{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int piece = kPieces - 1; piece >= 0; piece--)
#pragma unroll
                        for (int st = 0; st < 2; st++) s = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[st], w[rt][piece][st], s, 0, 0, 0);
#pragma unroll
                    for (int i = 0; i < 4; i++) total[rt][v][i] = DIRECT ? s[i] : fmaf(s[i], by, total[rt][v][i]);
                }
            }
        };
        if constexpr (DIRECT) {
            asm volatile("" ::: "memory");
            add(power_of_two(min(max(e - unit, -kExact), 0)), 1.0f); // (a block that no row sees may have any scale: its weights are zero)
        } else {
            const int passes = largest_e - smallest_e > kExact ? 4 : 1; // (the same for all lanes of a wave)
            for (int pass = 0; pass < passes; pass++) {
                asm volatile("" ::: "memory");
                const int wanted = passes > 1 ? __builtin_amdgcn_readlane(e, pass * 16) : largest_e; // the sums' unit
                if (wanted > unit) { // the totals in the same
                    const int down = unit - wanted;
                    unit = wanted;
#pragma unroll
                    for (int rt = 0; rt < RT; rt++)
#pragma unroll
                        for (int v = 0; v < NV; v++)
#pragma unroll
                            for (int i = 0; i < 4; i++) total[rt][v][i] = __builtin_amdgcn_ldexpf(total[rt][v][i], down);
                }
                add(passes == 1 || (int)quad == pass ? power_of_two(max(e - wanted, -kExact)) : 0.0f, __builtin_amdgcn_ldexpf(1.0f, wanted - unit));
            }
        }
    }
    // Totals become results: divided first (sums of weights of 2^8 and more, times a value of 2^119, are no 32-bit floats; their quotient is).
    __device__ __forceinline__ void end_tiles() {
#pragma unroll
        for (int rt = 0; rt < RT; rt++) {
            const float sum = sums[rt][0], inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
            for (int v = 0; v < NV; v++)
#pragma unroll
                for (int i = 0; i < 4; i++) total[rt][v][i] = total[rt][v][i] * inv * power_of_two(unit);
        }
    }

    // The rows' results, or those of one of their parts.
    __device__ __forceinline__ void store(uint32_t parts, uint32_t split) const {
        const Cache8 &c = p.cache;
#pragma unroll
        for (int rt = 0; rt < RT; rt++) {
            const uint32_t r = row0 + rt * 16 + col;
            if (r >= R) continue;
            if (parts == 1) {
                const uint32_t head = g * p.rep + r - fastdiv(r, p.rep_div) * p.rep;
                T *const dst = static_cast<T *>(p.out) + token_of(rt) * p.out_pitch + head * c.vdim + quad * 4;
#pragma unroll
                for (int v = 0; v < NV; v++) {
                    if (v * 16 >= (int)c.vdim) continue;
                    const float y[4] = {total[rt][v][0], total[rt][v][1], total[rt][v][2], total[rt][v][3]};
                    store_elements<T, 4>(dst + v * 16, y);
                }
            } else {
                const uint64_t at = ((uint64_t)(b * c.kv_heads + g) * p.splits + split) * p.rows + r;
                if (quad == 0) p.stats[at] = make_float2(maximum[rt], sums[rt][0]);
                float *const dst = p.parts + at * c.vdim + quad * 4;
#pragma unroll
                for (int v = 0; v < NV; v++)
                    if (v * 16 < (int)c.vdim) *reinterpret_cast<float4v *>(dst + v * 16) = total[rt][v];
            }
        }
    }
};

// Which rows and tiles a workgroup takes: `group` rows of a pair from group0 on, the tiles of part `split`.
struct AttentionShare {
    uint32_t bg, b, g, split, group0, R;
    uint64_t held;
    KeyRange range;
    uint32_t tile, end_tile;
    __device__ __forceinline__ bool find(const CacheAttentionPlan &p, uint32_t group) {
        const uint32_t id = fastdiv(blockIdx.x, p.bgs_div), block = fastdiv(id, p.splits_div);
        bg = blockIdx.x - id * p.bgs;
        split = id - block * p.splits;
        // The longest rows first, but every other run of as many as there are compute units the other way round: a unit takes one of each run, and what it
        // takes of two adds up to as much as any other's.
        const uint32_t run = fastdiv(block, p.run_div), begin = run * p.run_div.d;
        group0 = (p.row_blocks - 1 - (run & 1 ? begin + min(begin + p.run_div.d, p.row_blocks) - 1 - block : block)) * group;
        b = fastdiv(bg, p.heads_div);
        g = bg - b * p.cache.kv_heads;
        held = p.batch.held_by(b);
        R = p.batch.count_of(b) * p.rep;
        if (group0 >= R) return false;
        range = key_range(p, held, fastdiv(group0, p.rep_div), fastdiv(min(group0 + group, R) - 1, p.rep_div));
        if (split >= range.parts) return false;
        tile = range.first_tile + split * range.each;
        end_tile = min(tile + range.each, range.end_tile);
        return true;
    }
};

// The exponents of the value blocks of a workgroup's tiles that its rows see, looked over by each of its waves.
struct ScaleRange {
    int largest = kLowestScale, smallest = kHighestScale;
    __device__ __forceinline__ void look(const CacheAttentionPlan &p, const float *v_scale, const AttentionShare &my) {
        const uint32_t n = p.cache.block_log2, end = min(my.end_tile * kTile, my.range.end); // (blocks behind range.end may have any scale)
        for (uint32_t j = (my.tile * kTile >> n) + (threadIdx.x & 63); j << n < end; j += 64) {
            const int e = scale_exponent(v_scale[j]);
            largest = max(largest, e);
            smallest = min(smallest, e);
        }
    }
    // Whether codes are exact in units of the largest.
    __device__ __forceinline__ bool near(int *unit) {
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) {
            largest = max(largest, __shfl_xor(largest, o));
            smallest = min(smallest, __shfl_xor(smallest, o));
        }
        const int l = __builtin_amdgcn_readfirstlane(largest);
        if (l - __builtin_amdgcn_readfirstlane(smallest) > kExact) return false;
        *unit = l;
        return true;
    }
};

// Few rows: the waves of a workgroup have the same rows, take their tiles in turns, codes straight to registers, and add their results up
// in LDS.  Bound by memory: a token each of 32 sequences behind 16300 (bf16, 32 heads of 128 on 8, 1.07 GB, of which two passes find a sixth in the card's cache) 162 us, 6.6 TB/s; one behind 131000
// (f32, 268 MB) 51 us, 5.2 TB/s.
template <class T, int NL, int RT> __global__ __launch_bounds__(64 * kWavesOfAttention, NL * RT > 2 ? 1 : 2) void cache_attention_kernel(CacheAttentionPlan p) {
    typedef AttentionWave<T, NL, RT> Wave;
    constexpr int NV = Wave::NV;
    AttentionShare my;
    if (!my.find(p, 16 * RT)) return;
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    Wave w(p);
    w.b = my.b;
    w.g = my.g;
    w.R = my.R;
    w.row0 = my.group0;
    const Cache8 &c = p.cache;
    const uint32_t nb = c.capacity >> c.block_log2;
    const uint8_t *const keys = c.k_codes + (uint64_t)my.bg * c.capacity * c.dim, *const values = c.v_codes + (uint64_t)my.bg * c.capacity * c.vdim;
    const float *const k_scale = c.k_scale + (uint64_t)my.bg * nb, *const v_scale = c.v_scale + (uint64_t)my.bg * nb;
    uint4 k_now[4][NL], v_now[NV];
    float ks_now = 0.0f, vs_now = 0.0f;
    uint32_t key_lane[NL];
#pragma unroll
    for (int l = 0; l < NL; l++) key_lane[l] = w.key_lane(l);
    const uint32_t value_lane = w.value_lane();
    auto ask_keys = [&](uint32_t t) {
        ks_now = k_scale[w.block_of(t)];
        if (w.reaches_beyond(t)) {
#pragma unroll
            for (int kt = 0; kt < 4; kt++)
#pragma unroll
                for (int l = 0; l < NL; l++) k_now[kt][l] = *reinterpret_cast<const uint4 *>(keys + w.key_at_end(t, kt, l));
        } else {
#pragma unroll
            for (int kt = 0; kt < 4; kt++)
#pragma unroll
                for (int l = 0; l < NL; l++) k_now[kt][l] = *reinterpret_cast<const uint4 *>(keys + w.key_tile(t, kt) + key_lane[l]);
        }
    };
    auto ask_values = [&](uint32_t t) {
        vs_now = v_scale[w.block_of(t)];
        if (w.reaches_beyond(t)) {
#pragma unroll
            for (int v = 0; v < NV; v++) v_now[v] = *reinterpret_cast<const uint4 *>(values + w.value_at_end(t, v));
        } else {
#pragma unroll
            for (int v = 0; v < NV; v++) v_now[v] = *reinterpret_cast<const uint4 *>(values + w.value_tile(t, v) + value_lane);
        }
    };
    uint32_t tile = my.tile + wave;
    if (tile < my.end_tile) {
        ask_keys(tile);
        ask_values(tile);
    }
    typename Wave::Queries x;
    w.ask_rows(x);
    w.begin_rows(x, my.held);
    for (; tile < my.end_tile; tile += kWavesOfAttention) {
        const bool more = tile + kWavesOfAttention < my.end_tile;
        w.scores(tile, [&](int kt, int l) { return k_now[kt][l]; });
        const float ks = ks_now;
        if (more) ask_keys(tile + kWavesOfAttention); // (into the registers that the products have read)
        w.weigh(ks);
        w.template products<false>(vs_now, [&](int v) { return v_now[v]; },
                                   [&] {
#pragma unroll
                                       for (int v = 0; v < NV; v++) v_now[v] = without_nan(v_now[v]);
                                   });
        if (more) ask_values(tile + kWavesOfAttention);
    }
    // the waves' totals: of two and two, then of the last two
    __shared__ float4v shared_total[2][RT * NV][64];
    __shared__ float2 shared_stats[2][RT][64];
    __shared__ int shared_unit[2];
#pragma unroll
    for (uint32_t half = 2; half >= 1; half /= 2) {
        if (wave >= half && wave < 2 * half) {
            shared_unit[wave - half] = w.unit;
#pragma unroll
            for (int rt = 0; rt < RT; rt++) {
                shared_stats[wave - half][rt][lane] = make_float2(w.maximum[rt], w.sums[rt][0]);
#pragma unroll
                for (int v = 0; v < NV; v++) shared_total[wave - half][rt * NV + v][lane] = w.total[rt][v];
            }
        }
        __syncthreads();
        if (wave < half) {
            const int its_unit = shared_unit[wave], unit = max(w.unit, its_unit);
#pragma unroll
            for (int rt = 0; rt < RT; rt++) {
                const float2 other = shared_stats[wave][rt][lane];
                const float m = fmaxf(w.maximum[rt], other.x), mine = __builtin_amdgcn_exp2f(w.maximum[rt] - m), its = __builtin_amdgcn_exp2f(other.x - m);
                w.maximum[rt] = m;
                w.sums[rt][0] = w.sums[rt][0] * mine + other.y * its;
                const float my_part = __builtin_amdgcn_ldexpf(mine, w.unit - unit), its_part = __builtin_amdgcn_ldexpf(its, its_unit - unit);
#pragma unroll
                for (int v = 0; v < NV; v++) w.total[rt][v] = w.total[rt][v] * my_part + shared_total[wave][rt * NV + v][lane] * its_part;
            }
            w.unit = unit;
        }
        __syncthreads();
    }
    if (wave > 0) return;
    w.end_tiles();
    w.store(my.range.parts, my.split);
}

// Many rows: every wave of a workgroup has rows of its own, and all walk the same tiles, whose codes come straight into LDS, a tile ahead, in
// the order in which the lanes take them.  Bound by what waits for what: scores, their maximum, exponentials and products follow each other in each wave, and the two waves of a
// SIMD cover that in part.  Four prompts of 2048 tokens (bf16,
// 16 heads of 128 on 8, 69 GFLOP) 82 to 84 us in a run of calls, matrix pipes busy for 29 % of the cycles, vector instructions for 42 %; of the 31 us of a workgroup of 9 to 16
// tiles 6 to 8 are its beginning and end.  128 rows share what a tile costs to fetch; with 16 a wave the widening would be done twice as often.
template <class T, int NL, int RT, bool CUT = false> __global__ __launch_bounds__(64 * kWavesOfAttention, 2) void cache_attention_rows_kernel(CacheAttentionPlan p) {
    typedef AttentionWave<T, NL, RT, CUT> Wave;
    typedef __attribute__((address_space(3))) char lds_char;
    constexpr int NV = Wave::NV;
    constexpr int kKeys = 4 * NL, kCodes = kKeys + NV; // 1 KB pieces of a tile, of which each wave asks for some
    constexpr bool kOwnCopy = NL <= 2; // (LDS for two workgroups on a compute unit)
    constexpr bool kMayAdd = sizeof(T) == 2; // the instruction may add to the totals
    extern __shared__ float lds_dyn[];
    lds_char *const lds = (lds_char *)lds_dyn;
    AttentionShare my;
    if (!my.find(p, kWavesOfAttention * 16 * RT)) return;
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    Wave w(p);
    w.b = my.b;
    w.g = my.g;
    w.R = my.R;
    w.row0 = my.group0 + wave * 16 * RT;
    const Cache8 &c = p.cache;
    const uint32_t nb = c.capacity >> c.block_log2;
    const uint8_t *const keys = c.k_codes + (uint64_t)my.bg * c.capacity * c.dim, *const values = c.v_codes + (uint64_t)my.bg * c.capacity * c.vdim;
    const float *const k_scale = c.k_scale + (uint64_t)my.bg * nb, *const v_scale = c.v_scale + (uint64_t)my.bg * nb;
    float ks_next = 0.0f, vs_next = 0.0f;
    uint32_t key_lane[NL];
#pragma unroll
    for (int l = 0; l < NL; l++) key_lane[l] = w.key_lane(l);
    const uint32_t value_lane = w.value_lane();
    auto ask = [&](uint32_t t, uint32_t place) __attribute__((always_inline)) { // the first two waves ask for keys, the others for values
        auto into = [&](uint32_t i, const uint8_t *from) {
            __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)from,
                                             (__attribute__((address_space(3))) void *)(lds + (place * kCodes + i) * 1024), 16, 0, 0);
        };
        const uint32_t n = wave & 1; // (its half of them)
        constexpr int kHalfKeys = kKeys / 2, kHalfValues = NV / 2;
        const uint32_t k0 = n * kHalfKeys, v0 = n * kHalfValues;
        if (w.reaches_beyond(t)) {
#pragma unroll
            for (int i = 0; i < kHalfKeys; i++)
                if (wave < 2) into(k0 + i, keys + w.key_at_end(t, n * 2 + i / NL, i % NL));
#pragma unroll
            for (int i = 0; i < kHalfValues; i++)
                if (wave >= 2) into(kKeys + v0 + i, values + w.value_at_end(t, v0 + i));
        } else if (wave < 2) {
#pragma unroll
            for (int i = 0; i < kHalfKeys; i++) into(k0 + i, keys + w.key_tile(t, n * 2 + i / NL) + key_lane[i % NL]);
        } else {
#pragma unroll
            for (int i = 0; i < kHalfValues; i++) into(kKeys + v0 + i, values + w.value_tile(t, v0 + i) + value_lane);
        }
        ks_next = k_scale[w.block_of(t)];
        vs_next = v_scale[w.block_of(t)];
    };
    ScaleRange scales;
    const bool few_tiles = kMayAdd && my.end_tile <= my.tile + kMostTiles;
    if (few_tiles) scales.look(p, v_scale, my);
    uint32_t from = 0, to = 0; // tiles that the wave's rows see
    typename Wave::Queries x;
    if (w.row0 < my.R) w.ask_rows(x); // (in front of the tile: they are wanted first)
    ask(my.tile, 0);
    if (w.row0 < my.R) {
        w.begin_rows(x, my.held);
        from = (uint32_t)max(w.any_from, 0) / kTile;
        to = w.any_to < 0 ? 0 : (uint32_t)w.any_to / kTile + 1;
    }
    const bool near = few_tiles && scales.near(&w.unit);
    auto walk = [&](auto direct) {
        for (uint32_t t = my.tile; t < my.end_tile; t++) {
            const uint32_t place = (t - my.tile) & 1;
            asm volatile("" ::: "memory");
            __builtin_amdgcn_s_waitcnt(0x0070); // vmcnt(0) lgkmcnt(0): this wave's part of the tile is in LDS, and it has read the one before
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
            const float ks = ks_next, vs = vs_next;
            if (t + 1 < my.end_tile) ask(t + 1, place ^ 1);
            if (t < from || t >= to) continue;
            const lds_char *const codes = lds + place * kCodes * 1024 + lane * 16;
            auto piece = [&](int n) {
                typedef uint32_t u4 __attribute__((ext_vector_type(4)));
                const u4 v = *reinterpret_cast<const __attribute__((address_space(3))) u4 *>(codes + n * 1024);
                return make_uint4(v[0], v[1], v[2], v[3]);
            };
            w.scores(t, [&](int kt, int l) { return piece(kt * NL + l); });
            w.weigh(ks);
            // codes without NaN go to memory of the wave's own (each lane reads what it wrote), so that what the products read is one address
            // either way: a choice at every piece would keep them from being asked for ahead
            const lds_char *values_at = codes + kKeys * 1024;
            bool clean = false;
            auto value = [&](int v) {
                typedef uint32_t u4 __attribute__((ext_vector_type(4)));
                const u4 x = *reinterpret_cast<const __attribute__((address_space(3))) u4 *>(values_at + v * 1024);
                return make_uint4(x[0], x[1], x[2], x[3]);
            };
            w.template products<decltype(direct)::value>(vs, [&](int v) { return !kOwnCopy && clean ? without_nan(value(v)) : value(v); },
                       [&] {
                           clean = true;
                           if (!kOwnCopy) return;
                           lds_char *const own = lds + (2 * kCodes + wave * NV) * 1024 + lane * 16;
#pragma unroll
                           for (int v = 0; v < NV; v++) {
                               typedef uint32_t u4 __attribute__((ext_vector_type(4)));
                               const uint4 x = without_nan(value(v));
                               *reinterpret_cast<__attribute__((address_space(3))) u4 *>(own + v * 1024) = u4{x.x, x.y, x.z, x.w};
                           }
                           values_at = own;
                       });
        }
    };
    if constexpr (kMayAdd) {
        if (near) walk(std::true_type{});
        else walk(std::false_type{});
    } else {
        walk(std::false_type{});
    }
    __builtin_amdgcn_s_waitcnt(0x0070); // no load may write LDS that another workgroup gets
    if (w.row0 >= my.R) return;
    w.end_tiles();
    w.store(my.range.parts, my.split);
}

template <class T> int launch_cache_attention_of(const LaunchOn &on, const CacheAttentionPlan &p) {
    const dim3 grid(p.bgs * p.splits * p.row_blocks), block(64 * kWavesOfAttention);
    const uint32_t nl = (std::max(p.cache.dim, p.cache.vdim) + 63) / 64;
    auto launch = [&](auto kernel, size_t lds = 0) { return on.with_lds("cache attention launch", kernel, grid, block, lds, p); };
    if (p.rows_by_wave) { // LDS: two tiles, and the waves' copies
        if (nl == 1) return launch(cache_attention_rows_kernel<T, 1, 2>, (2 * 8 + kWavesOfAttention * 4) * 1024);
        if (nl == 2 && std::max(p.cache.dim, p.cache.vdim) <= 96) return launch(cache_attention_rows_kernel<T, 2, 2, true>, (2 * 14 + kWavesOfAttention * 6) * 1024);
        return nl == 2 ? launch(cache_attention_rows_kernel<T, 2, 2>, (2 * 16 + kWavesOfAttention * 8) * 1024) : launch(cache_attention_rows_kernel<T, 4, 1>, 2 * 32 * 1024);
    }
    if (nl == 1) return p.two_tiles ? launch(cache_attention_kernel<T, 1, 2>) : launch(cache_attention_kernel<T, 1, 1>);
    if (nl == 2) return p.two_tiles ? launch(cache_attention_kernel<T, 2, 2>) : launch(cache_attention_kernel<T, 2, 1>);
    return launch(cache_attention_kernel<T, 4, 1>);
}
template <class T> int load_cache_attention_of() {
    hipFuncAttributes a;
    CG_HIP(hipFuncGetAttributes(&a, reinterpret_cast<const void *>(cache_attention_kernel<T, 1, 1>)));
    return CG_OK;
}
#endif

int launch_cache_attention_f32(const LaunchOn &on, const CacheAttentionPlan &p);
int launch_cache_attention_f16(const LaunchOn &on, const CacheAttentionPlan &p);
int launch_cache_attention_bf16(const LaunchOn &on, const CacheAttentionPlan &p);
int load_cache_attention_f32();
int load_cache_attention_f16();
int load_cache_attention_bf16();

} // namespace cg
