// 4-bit weights with group scales, general form: one thread per output, any k and any alignment.
#include "qm_w4.cuh"

namespace qm {

using namespace w4;

template <typename T, typename S>
__global__ void __launch_bounds__(256) w4_simt_kernel(const T *__restrict__ X, int64_t ldx, const uint8_t *__restrict__ B, const S *__restrict__ scales,
                                                      int group, const int *__restrict__ offsets, int experts, T *__restrict__ out, int64_t ldo, int rows,
                                                      int n, int k)
{
    const int64_t row = (int64_t)blockIdx.y * 16 + threadIdx.y;
    const int col = blockIdx.x * 16 + threadIdx.x;
    if (row >= rows || col >= n) return;
    int e = 0;
    if (offsets) {
        // clamped as documented; the row's expert is the first whose segment holds it
        int begin = 0;
        for (e = 0; e < experts; ++e) {
            const int first = max(begin, min(offsets[e], rows)), last = max(first, min(offsets[e + 1], rows));
            if (row >= first && row < last) break;
            begin = last;
        }
        if (e == experts) return;
    }
    const int groups = (k + group - 1) / group;
    const uint8_t *b = B + ((int64_t)e * n + col) * (k / 2);
    const S *s = scales + ((int64_t)e * n + col) * groups;
    const T *x = X + row * ldx;
    float sum = 0.0f;
    for (int g = 0; g < groups; ++g) {
        float part = 0.0f;
        for (int i = g * group; i < min(k, (g + 1) * group); i += 2) {
            const int byte = (int8_t)b[i / 2];
            const int low = (int)((uint32_t)byte << 28) >> 28, high = byte >> 4;
            part = fmaf(to_float(x[i]), (float)low, part);
            part = fmaf(to_float(x[i + 1]), (float)high, part);
        }
        sum = fmaf(to_float(s[g]), part, sum);
    }
    out[row * ldo + col] = from_float<T>(sum);
}

int w4_simt_launch(const W4Args &a)
{
    return with_type(a.type, [&](auto t) {
        using T = typename decltype(t)::type;
        return with_same_or_float<T>(a.scale_type, [&](auto u) {
            using S = typename decltype(u)::type;
            const dim3 grid((unsigned)((a.n + 15) / 16), (unsigned)((a.rows + 15) / 16));
            w4_simt_kernel<T, S><<<grid, dim3(16, 16), 0, a.stream>>>(static_cast<const T *>(a.X), a.ldx, a.B, static_cast<const S *>(a.scales), a.group,
                                                                      a.offsets, a.experts, static_cast<T *>(a.out), a.ldo, a.rows, a.n, a.k);
            return launched("w4_simt_kernel launch");
        });
    });
}

}  // namespace qm
