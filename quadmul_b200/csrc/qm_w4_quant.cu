// Group-wise 4-bit quantiser: per group of a row, scale = max |w| times the fp32 value of 1/7 (rounded to the scales' type) and
// code = w / scale, the exact quotient rounded to the nearest integer, ties to even.
#include "qm_w4.cuh"

namespace qm {

using namespace w4;

// The code of w for scale s.  q = w * (1 / s) rounded is off by at most one; the remainder w - q s is exact in one fma (w and q s
// are multiples of the smaller of their last places and the result has at most 24 bits: for |q| >= 2 it is at most s and a
// multiple of s's last place, for |q| = 1 it is a difference of numbers within a factor of two), so comparing it with s / 2
// finds the nearest integer and the ties.
__device__ __forceinline__ int code_of(float w, float s, float inv)
{
    float q = rintf(w * inv);
    const float r = fmaf(-q, s, w), half = 0.5f * s;
    if (r > half || (r == half && ((int)q & 1))) q += 1.0f;
    else if (r < -half || (r == -half && ((int)q & 1))) q -= 1.0f;
    return (int)fminf(fmaxf(q, -8.0f), 7.0f);
}

// One warp per group, whatever the group's width.
template <typename T, typename S>
__global__ void __launch_bounds__(256) quantize_w4_kernel(const T *__restrict__ W, int64_t ldw, uint8_t *__restrict__ packed, S *__restrict__ scales,
                                                          int64_t rows, int64_t k, int group)
{
    const int lane = threadIdx.x & 31;
    const int64_t groups = (k + group - 1) / group;
    for (int64_t i = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); i < rows * groups; i += (int64_t)gridDim.x * 8) {
        const int64_t row = i / groups, g = i - row * groups;
        const int64_t first = g * group, last = min(k, first + group);
        const T *w = W + row * ldw;
        float a = 0.0f;
        bool nan = false;
        for (int64_t j = first + lane; j < last; j += 32) {
            const float v = to_float(w[j]);
            nan |= v != v;
            a = fmaxf(a, fabsf(v));
        }
        for (int d = 16; d; d >>= 1) a = fmaxf(a, __shfl_xor_sync(0xFFFFFFFFu, a, d));
        if (__any_sync(0xFFFFFFFFu, nan)) a = __int_as_float(0x7FC00000);
        const S stored = from_float<S>(__fmul_rn(a, 1.0f / 7.0f));
        if (lane == 0) scales[i] = stored;
        float s = to_float(stored);
        const bool some = s > 0.0f && s < INFINITY;
        // a scale near or below the smallest normal number has no reciprocal: both sides of the quotient times 2^64, exactly
        const float up = s < 0x1p-100f ? 0x1p64f : 1.0f;
        s *= up;
        for (int64_t j = first + 2 * lane; j < last; j += 64) {
            int low = 0, high = 0;
            if (some) {
                low = code_of(to_float(w[j]) * up, s, 1.0f / s);
                high = code_of(to_float(w[j + 1]) * up, s, 1.0f / s);
            }
            packed[row * (k / 2) + j / 2] = (uint8_t)((low & 15) | (high << 4));
        }
    }
}

int quantize_w4_launch(const void *W, int type, int64_t ldw, uint8_t *packed, void *scales, int scale_type, int64_t rows, int64_t k, int group,
                       cudaStream_t stream)
{
    return with_type(type, [&](auto t) {
        using T = typename decltype(t)::type;
        return with_same_or_float<T>(scale_type, [&](auto u) {
            using S = typename decltype(u)::type;
            const int64_t blocks = (rows * ((k + group - 1) / group) + 7) / 8;
            quantize_w4_kernel<T, S><<<(unsigned)(blocks < 148 * 32 ? blocks : 148 * 32), 256, 0, stream>>>(static_cast<const T *>(W), ldw, packed,
                                                                                                        static_cast<S *>(scales), rows, k, group);
            return launched("quantize_w4_kernel launch");
        });
    });
}

}  // namespace qm
