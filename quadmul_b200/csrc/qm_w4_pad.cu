// What the 4-bit-weight kernels need beside their own work: operands that TMA and 16-byte loads cannot address (k no multiple of 32,
// rows of X or B off 16-byte boundaries) are copied once into a workspace with k rounded up to 32 and zeros behind it; an empty
// sum (k == 0) is written as such.  The copies are bound by memory; next to a product of many rows they are small, and with few
// rows a call costs about three passes over the weights instead of one.
#include "qm_ptx.cuh"
#include "qm_w4.cuh"

namespace qm {

using namespace w4;

namespace {

constexpr int kThreads = 256;

// rows x row_bytes from `src` (pitch src_pitch, any alignment) to rows of dst_pitch bytes (a multiple of 16) on 16-byte boundaries;
// zeros behind row_bytes.  A thread makes 16 bytes out of aligned words, shifted into place; where a word of the shift would lie
// outside the matrix (its first and last bytes) it takes single bytes.
__global__ void __launch_bounds__(kThreads) w4_pad_kernel(const uint8_t *src, int64_t src_pitch, int64_t row_bytes, uint8_t *dst,
                                                          int dst_pitch, int64_t rows)
{
    ptx::grid_dependency_wait();
    ptx::grid_launch_dependents();
    const int pieces = dst_pitch / 16;
    const uintptr_t begin = reinterpret_cast<uintptr_t>(src), end = begin + (rows - 1) * src_pitch + row_bytes;
    for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < rows * pieces; i += (int64_t)gridDim.x * kThreads) {
        const int64_t row = rows * pieces <= 0xFFFFFFFFll ? (int64_t)((uint32_t)i / (uint32_t)pieces) : i / pieces;
        const int at = (int)(i - row * pieces) * 16;
        const uintptr_t from = begin + row * src_pitch + at, words = from & ~(uintptr_t)3;
        const int here = (int)min((int64_t)16, row_bytes - at);  // bytes of this piece that the row has (a piece with none reads nothing)
        uint32_t o[4] = {0, 0, 0, 0};
        if (here == 16 && words >= begin && words + 20 <= end) {
            uint32_t w[5];
#pragma unroll
            for (int j = 0; j < 5; ++j) w[j] = ptx::ld_behind_wait(reinterpret_cast<const uint32_t *>(words) + j);
#pragma unroll
            for (int j = 0; j < 4; ++j) o[j] = __funnelshift_r(w[j], w[j + 1], 8 * (int)(from & 3));
        } else {
#pragma unroll
            for (int j = 0; j < 16; ++j)
                if (j < here) o[j >> 2] |= ptx::ld_behind_wait(reinterpret_cast<const uint8_t *>(from) + j) << (8 * (j & 3));
        }
        *reinterpret_cast<uint4 *>(dst + row * dst_pitch + at) = make_uint4(o[0], o[1], o[2], o[3]);
    }
}

// zeros in the rows of out that some expert has (all rows without offsets): a block per row
__global__ void __launch_bounds__(kThreads) w4_zero_kernel(unsigned short *out, int64_t ldo, const int *offsets, int experts, int rows,
                                                           int n)
{
    ptx::grid_dependency_wait();
    ptx::grid_launch_dependents();
    if (offsets) {
        // the experts' segments cover what lies between the first offset and the largest, both clamped
        const int row = (int)blockIdx.x;
        bool before = false, behind = false;
        for (int e = threadIdx.x; e <= experts; e += kThreads) {
            const int o = max(0, min(ptx::ld_behind_wait(offsets + e), rows));
            before |= e == 0 && row < o;
            behind |= row < o;
        }
        if (__syncthreads_or(before) || !__syncthreads_or(behind)) return;
    }
    for (int c = threadIdx.x; c < n; c += kThreads) out[(int64_t)blockIdx.x * ldo + c] = 0;
}

int64_t padded_k(int k) { return ((int64_t)k + 31) / 32 * 32; }

bool pad_x(const W4Args &a) { return a.k % 32 != 0 || a.ldx % 8 != 0 || (reinterpret_cast<uintptr_t>(a.X) & 15u) != 0; }
bool pad_b(const W4Args &a) { return a.k % 32 != 0 || (reinterpret_cast<uintptr_t>(a.B) & 15u) != 0; }

int pad(const void *src, int64_t src_pitch, int64_t row_bytes, uint8_t *dst, int64_t dst_pitch, int64_t rows, cudaStream_t s)
{
    const int64_t blocks = (rows * (dst_pitch / 16) + kThreads - 1) / kThreads;
    return launch_chained("w4_pad_kernel launch", w4_pad_kernel, (unsigned)(blocks < 148 * 16 ? blocks : 148 * 16), kThreads, 0, s,
                          static_cast<const uint8_t *>(src), src_pitch, row_bytes, dst, (int)dst_pitch, rows);
}

}  // namespace

size_t w4_workspace(const W4Args &a)
{
    if (a.k <= 0 || a.rows <= 0 || a.n <= 0 || a.experts <= 0) return 0;
    const size_t x = pad_x(a) ? ((size_t)a.rows * padded_k(a.k) * 2 + 15) / 16 * 16 : 0;
    return x + (pad_b(a) ? (size_t)a.experts * a.n * (padded_k(a.k) / 2) : 0);
}

int w4_pad_launch(W4Args *a, void *workspace)
{
    W4Args g = *a;
    uint8_t *at = static_cast<uint8_t *>(workspace);
    const int64_t kp = padded_k(a->k);
    if (pad_x(*a)) {
        int st = pad(a->X, a->ldx * 2, (int64_t)a->k * 2, at, kp * 2, a->rows, a->stream);
        if (st != QM_OK) return st;
        g.X = at, g.ldx = kp;
        at += ((size_t)a->rows * kp * 2 + 15) / 16 * 16;
    }
    if (pad_b(*a)) {
        int st = pad(a->B, a->k / 2, a->k / 2, at, kp / 2, (int64_t)a->experts * a->n, a->stream);
        if (st != QM_OK) return st;
        g.B = at;
    }
    g.k = (int)kp;
    *a = g;
    return QM_OK;
}

int w4_zero_launch(const W4Args &a)
{
    return launch_chained("w4_zero_kernel launch", w4_zero_kernel, (unsigned)a.rows, kThreads, 0, a.stream, static_cast<unsigned short *>(a.out), a.ldo,
                          a.offsets, a.experts, a.rows, a.n);
}

}  // namespace qm
