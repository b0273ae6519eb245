// Group-wise 4-bit quantiser: per group of a row, scale = max |w| times the fp32 value of 1/7 (rounded to the scales' type) and
// code = w / scale, the exact quotient rounded to the nearest integer, ties to even.
//
// Every element is read once and leaves as half a byte, so memory should bound it, as it does for fp32.  With 16-bit elements
// there are twice as many to convert per byte, and a warp's loads and conversions take turns: 11008 x 4096 bf16 keeps DRAM at 38 % and
// the SM at 66 % of their peaks.  A lane
// takes sixteen consecutive elements (two or four 16-byte loads) and writes their eight bytes; 2, 4, 8 or 16 neighbouring lanes
// share a group, whose maximum is a few shuffles.  A warp has kUnroll such pieces of 512 elements in flight.
//
// Measured: 22016 x 4096 fp32 in groups of 32 64 us = 6.5 TB/s (0.99 of a copy); bf16 in groups of 128 14.4 us for 4096 x 4096 = 2.9
// TB/s, 30 us for 11008 x 4096 = 3.8.  Any alignment: 11008 x 4094 bf16 109 us.
#include <type_traits>

#include "qm_w4.cuh"

namespace qm {

using namespace w4;

namespace {

constexpr int kThreads = 256, kUnroll = 2;

// Scale and reciprocal for a group with largest value a, ready for code_of: both sides of the quotient are multiplied by `up`, 2^64
// for scales near or below the smallest normal number, which have no reciprocal.  some = false: the codes are 0.
struct Quotient {
    float s, inv, up;
    bool some;
};

template <typename S>
__device__ __forceinline__ Quotient quotient_for(S stored)
{
    Quotient q;
    q.s = to_float(stored);
    q.some = q.s > 0.0f && q.s < INFINITY;
    q.up = q.s < 0x1p-100f ? 0x1p64f : 1.0f;
    q.s *= q.up;
    q.inv = q.some ? __frcp_rn(q.s) : 0.0f;
    return q;
}

// The code of w.  q = w * (1 / s) rounded is off by at most one; the remainder w - q s is exact in one fma (w and q s are multiples
// of the smaller of their last places and the result has at most 24 bits: for |q| >= 2 it is at most s and a multiple of s's last
// place, for |q| = 1 it is a difference of numbers within a factor of two), so comparing it with s / 2 finds the nearest
// integer and the ties.
__device__ __forceinline__ int code_of(float w, const Quotient &z)
{
    w *= z.up;
    const float q = rintf(w * z.inv);
    const float r = fmaf(-q, z.s, w), half = 0.5f * z.s;
    int n = (int)q;  // |w| is at most a few scales, or the group has no codes
    const bool odd = (n & 1) != 0;
    if (r > half || (r == half && odd)) n += 1;
    if (r < -half || (r == -half && odd)) n -= 1;
    return min(max(n, -8), 7);
}

// Eight elements from 16-byte loads.
template <typename T>
struct Eight {
    uint4 v[sizeof(T) / 2];
    __device__ __forceinline__ void load(const T *p)
    {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) v[i] = __ldcs(reinterpret_cast<const uint4 *>(p) + i);
    }
    __device__ __forceinline__ void zero()
    {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) v[i] = make_uint4(0, 0, 0, 0);
    }
    __device__ __forceinline__ float at(int i) const
    {
        if constexpr (std::is_same<T, __nv_bfloat16>::value) {
            const uint32_t w = reinterpret_cast<const uint32_t *>(v)[i >> 1];
            return __uint_as_float((i & 1) ? w & 0xFFFF0000u : w << 16);
        } else {
            return to_float(reinterpret_cast<const T *>(v)[i]);
        }
    }
    // The largest magnitude as the bits of T (two of them for 16-bit types, in both halves of the word): magnitudes order like
    // unsigned integers, and an infinity or a NaN is above every number.
    __device__ __forceinline__ uint32_t magnitude() const
    {
        const uint32_t *w = reinterpret_cast<const uint32_t *>(v);
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 2 * (int)sizeof(T); ++i) {
            if constexpr (sizeof(T) == 4) m = max(m, w[i] & 0x7FFFFFFFu);
            else m = __vmaxu2(m, w[i] & 0x7FFF7FFFu);
        }
        return m;
    }
};

template <typename T>
__device__ __forceinline__ uint32_t larger_magnitude(uint32_t a, uint32_t b)
{
    if constexpr (sizeof(T) == 4) return max(a, b);
    else return __vmaxu2(a, b);
}

template <typename T>
__device__ __forceinline__ float magnitude_value(uint32_t m)
{
    if constexpr (sizeof(T) == 4) {
        return __uint_as_float(m);
    } else {
        const unsigned short h = (unsigned short)max(m & 0xFFFFu, m >> 16);
        if constexpr (std::is_same<T, __half>::value) return __half2float(__ushort_as_half(h));
        else return __uint_as_float((uint32_t)h << 16);
    }
}

// The codes of eight elements, whose group has a scale.
template <typename T, typename S>
__device__ __forceinline__ uint32_t eight_codes(const Eight<T> &w, const Quotient &z)
{
    // t = w (1 / s), corrected once with its exact remainder, is the quotient to its last place and the quotient itself where fp32 can
    // hold that; adding and taking away 1.5 x 2^23 rounds it, ties to even.  With a 16-bit w and a 16-bit s that is the
    // rounding of w / s: a middle k + 1/2 is either met exactly or missed by 2^-16 of it.  With a 32-bit s (or w) the quotient can
    // be closer: where one is, the eight are rounded by their remainders.  (|t| is at most 7.1 unless the scale lost digits, as a
    // subnormal fp16 does.)
    constexpr bool kSixteen = sizeof(T) == 2 && sizeof(S) == 2;
    constexpr float kRound = 12582912.0f;
    float r[8], edge = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float v = w.at(j);
        float t = v * z.inv;
        if constexpr (kSixteen) t = fmaf(fmaf(-t, z.s, v), z.inv, t);
        r[j] = __fadd_rn(__fadd_rn(t, kRound), -kRound);
        if constexpr (!kSixteen) edge = fmaxf(edge, fabsf(t - r[j]));
    }
    // codes + 8 as base-16 digits, four in one fp32 whole number; the digits' high bits are then turned round
    const float low = fmaf(r[3], 4096.0f, fmaf(r[2], 256.0f, fmaf(r[1], 16.0f, r[0]))) + (8388608.0f + 34952.0f);
    const float high = fmaf(r[7], 4096.0f, fmaf(r[6], 256.0f, fmaf(r[5], 16.0f, r[4]))) + (8388608.0f + 34952.0f);
    uint32_t word = __byte_perm(__float_as_uint(low), __float_as_uint(high), 0x5410) ^ 0x88888888u;
    const bool small = z.up != 1.0f || (std::is_same<S, __half>::value && z.s < 0x1p-14f);
    if (small || (!kSixteen && !(edge < 0.4999f))) {
        word = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) word |= (uint32_t)(code_of(w.at(j), z) & 15) << (4 * j);
    }
    return word;
}

// k % 16 == 0 and rows on 16-byte boundaries.  Pieces of 512 elements are dealt to the warps.
template <typename T, typename S>
__global__ void __launch_bounds__(kThreads, 4) quantize_w4_kernel(const T *__restrict__ W, int64_t ldw, uint8_t *__restrict__ packed, S *__restrict__ scales,
                                                               int rows, int k, int group_shift)
{
    const int lane = threadIdx.x & 31;
    const int lanes = 1 << (group_shift - 4);  // lanes that share a group
    const int per_row = (k + 511) / 512, groups = (k + (1 << group_shift) - 1) >> group_shift;
    // from one piece of a warp to its next: so many rows and pieces on (a division per piece costs as much as its codes)
    const int warps = gridDim.x * (kThreads / 32), first = blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
    const int step_r = warps / per_row, step_p = warps - step_r * per_row;
    int r = first / per_row, piece = first - r * per_row;
    while (r < rows) {
        Eight<T> w[kUnroll][2];
        int row[kUnroll], at[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            row[u] = r, at[u] = r < rows ? piece * 512 + lane * 16 : k;
            if (at[u] < k) {
                const T *src = W + (int64_t)r * ldw + at[u];
                w[u][0].load(src);
                w[u][1].load(src + 8);
            } else {
                w[u][0].zero();
                w[u][1].zero();
            }
            r += step_r, piece += step_p;
            if (piece >= per_row) piece -= per_row, ++r;
        }
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            uint32_t m = larger_magnitude<T>(w[u][0].magnitude(), w[u][1].magnitude());
            for (int d = 1; d < lanes; d <<= 1) m = larger_magnitude<T>(m, __shfl_xor_sync(0xFFFFFFFFu, m, d));
            if (at[u] >= k) continue;
            const S stored = from_float<S>(__fmul_rn(magnitude_value<T>(m), 1.0f / 7.0f));
            const Quotient z = quotient_for(stored);
            uint2 codes = make_uint2(0, 0);
            if (z.some) codes = make_uint2(eight_codes<T, S>(w[u][0], z), eight_codes<T, S>(w[u][1], z));
            __stcs(reinterpret_cast<uint2 *>(packed + (int64_t)row[u] * (k / 2) + at[u] / 2), codes);
            if ((lane & (lanes - 1)) == 0) scales[(int64_t)row[u] * groups + (at[u] >> group_shift)] = stored;
        }
    }
}

// Any even k and any alignment: one warp per group.
template <typename T, typename S>
__global__ void __launch_bounds__(kThreads) quantize_w4_any_kernel(const T *__restrict__ W, int64_t ldw, uint8_t *__restrict__ packed,
                                                                   S *__restrict__ scales, int64_t rows, int64_t k, int group)
{
    const int lane = threadIdx.x & 31;
    const int64_t groups = (k + group - 1) / group, all = rows * groups;
    for (int64_t i = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5); i < all; i += (int64_t)gridDim.x * (kThreads / 32)) {
        const int64_t row = all <= 0xFFFFFFFFll ? (int64_t)((uint32_t)i / (uint32_t)groups) : i / groups;
        const int64_t first = (i - row * groups) * group, last = min(k, first + group);
        const T *w = W + row * ldw;
        // a lane has elements (2 lane, 2 lane + 1) of every 64 of the group
        float low[4], high[4], a = 0.0f;
        bool nan = false;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int64_t j = first + 64 * u + 2 * lane;
            low[u] = high[u] = 0.0f;
            if (j < last) low[u] = to_float(w[j]), high[u] = to_float(w[j + 1]);  // k is even, and so is every group's end
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            nan |= low[u] != low[u] || high[u] != high[u];
            a = fmaxf(a, fmaxf(fabsf(low[u]), fabsf(high[u])));
        }
        for (int d = 16; d; d >>= 1) a = fmaxf(a, __shfl_xor_sync(0xFFFFFFFFu, a, d));
        if (__any_sync(0xFFFFFFFFu, nan)) a = __int_as_float(0x7FC00000);
        const S stored = from_float<S>(__fmul_rn(a, 1.0f / 7.0f));
        if (lane == 0) scales[i] = stored;
        const Quotient z = quotient_for(stored);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int64_t j = first + 64 * u + 2 * lane;
            if (j >= last) continue;
            const int l = z.some ? code_of(low[u], z) : 0, h = z.some ? code_of(high[u], z) : 0;
            packed[row * (k / 2) + j / 2] = (uint8_t)((l & 15) | (h << 4));
        }
    }
}

}  // namespace

int quantize_w4_launch(const void *W, int type, int64_t ldw, uint8_t *packed, void *scales, int scale_type, int64_t rows, int64_t k, int group,
                       cudaStream_t stream)
{
    return with_type(type, [&](auto t) {
        using T = typename decltype(t)::type;
        return with_same_or_float<T>(scale_type, [&](auto u) {
            using S = typename decltype(u)::type;
            const T *w = static_cast<const T *>(W);
            S *s = static_cast<S *>(scales);
            const bool vec = k % 16 == 0 && k < (1 << 30) && rows < (1 << 30) && (reinterpret_cast<uintptr_t>(W) & 15u) == 0 &&
                             (ldw * (int64_t)sizeof(T)) % 16 == 0 && (reinterpret_cast<uintptr_t>(packed) & 7u) == 0;
            if (vec) {
                const int64_t pieces = rows * ((k + 511) / 512), blocks = (pieces + 8 * kUnroll - 1) / (8 * kUnroll);
                return launch_in_turn("quantize_w4_kernel launch", quantize_w4_kernel<T, S>, (unsigned)(blocks < 148 * 4 ? blocks : 148 * 4), kThreads, 0,
                                      stream, w, ldw, packed, s, (int)rows, (int)k, group == 32 ? 5 : group == 64 ? 6 : group == 128 ? 7 : 8);
            }
            const int64_t blocks = (rows * ((k + group - 1) / group) + 7) / 8;
            return launch_in_turn("quantize_w4_any_kernel launch", quantize_w4_any_kernel<T, S>, (unsigned)(blocks < 148 * 32 ? blocks : 148 * 32), kThreads,
                                  0, stream, w, ldw, packed, s, rows, k, group);
        });
    });
}

}  // namespace qm
