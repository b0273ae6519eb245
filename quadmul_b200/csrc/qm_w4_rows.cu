// 4-bit weights with group scales, few rows of X: weight streaming.
//
// out[r][c] = sum over groups g of scale[c][g] * sum over i in g of x[r][i] q[c][i].  With up to 16 rows of X the product reads
// every weight once and is bound by memory; what a kernel has to do is keep loads in flight and convert codes fast enough.
//
//  * A CTA (16 warps) takes blocks of 8 RG rows of B, WK of its warps split K between them in steps of 128 elements.  A lane
//    (g, q) = (lane / 4, lane % 4) loads 16 bytes, 32 codes, of row g of each 8-row group, straight into registers; three
//    steps are in flight per warp (96 KB per SM with RG = 4), across the end of a block, so the stream does not stop there.
//  * The product runs on mma.sync.m16n8k16: 16 rows of B x 8 rows of X.  The codes become 16-bit floats in registers, exactly
//    (codes_to_pairs), and the sums of a group are exact products added in fp32; the group's scale is applied to the fp32 sum, so
//    no weight is ever rounded.  The order of K inside an instruction is free as long as both operands use the same one: a word of
//    eight codes unpacks into pairs (e0, e4) .. (e3, e7), and the rows of X are put into that order once, when they are staged.
//  * One instruction adds up over the four lanes of a row, so these must hold codes of one group: with groups of 128 and more
//    every lane uses its own 32 codes; for groups of 64 and 32 the lanes of a row trade words (4 or 8 shuffles a step).
//  * The rows of X that a warp needs (its share of K) sit in shared memory in the order of the lanes that read them: staged by
//    the lane that uses them, so without a barrier, once for all blocks of an expert.
//  * The warps' partial tiles meet in shared memory (two buffers, one barrier a block) and are added in a fixed order.
//
// With experts a unit of work is (expert, tile of its rows, block of B); every CTA takes a contiguous range of units, so the rows
// of X change rarely.
#include <atomic>
#include <cstdlib>
#include <type_traits>

#include "qm_ptx.cuh"
#include "qm_w4.cuh"

namespace qm {

using namespace w4;

namespace {

constexpr int kWarps = 16, kThreads = kWarps * 32;
constexpr int kDepth = 3;        // steps in flight per warp
constexpr int kStep = 128;       // elements of K per step
constexpr int kMaxSmem = 232448 - 1024;

struct RowsParams {
    const void *X;
    int64_t ldx;
    const uint8_t *B;
    const void *scales;
    const int *offsets;
    void *out;
    int64_t ldo;
    int rows, n, k, experts;
    int group_shift, groups;
    int tile;      // rows of X per unit, at most 16
    int warps_k;   // warps that split K; the others take further rows of B
    int vec_scales;  // a step's scales can be loaded as one vector
};

template <typename T>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, const float (&c)[4])
{
    if constexpr (std::is_same<T, __half>::value)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
                     : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
                     : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}

// GPS scales of one step as they lie in memory
template <typename S, int GPS>
struct RawScales {
    static constexpr int kWords = GPS * (int)sizeof(S) >= 4 ? GPS * (int)sizeof(S) / 4 : 1;
    uint32_t w[kWords];
};

template <typename S, int GPS>
__device__ __forceinline__ float scale_at(const RawScales<S, GPS> &r, int j, int src_lane)
{
    if constexpr (sizeof(S) == 4) {
        return __uint_as_float(__shfl_sync(0xFFFFFFFFu, r.w[j], src_lane));
    } else {
        const uint32_t v = __shfl_sync(0xFFFFFFFFu, r.w[j >> 1], src_lane);
        const unsigned short h = (unsigned short)((j & 1) ? v >> 16 : v);
        if constexpr (std::is_same<S, __half>::value) return __half2float(__ushort_as_half(h));
        else return __bfloat162float(__ushort_as_bfloat16(h));
    }
}

// GPS = groups per step of 128 elements (4, 2 or 1 for groups of 32, 64, and 128 or more), RG = 8-row groups of B per warp,
// TT = 8-row tiles of X.
template <typename T, typename S, int GPS, int RG, int TT>
__global__ void __launch_bounds__(kThreads, 1) w4_rows_kernel(const RowsParams p)
{
    constexpr int kTiles = RG / 2;  // 16-row tiles of B per warp
    extern __shared__ uint4 smem_u4[];
    const T *__restrict__ X = static_cast<const T *>(p.X);
    const S *__restrict__ scales = static_cast<const S *>(p.scales);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
    const int wk = warp % p.warps_k, wr = warp / p.warps_k;
    const int block_rows = 8 * RG * (kWarps / p.warps_k);
    const int blocks = (p.n + block_rows - 1) / block_rows;
    const int steps = (p.k + kStep - 1) / kStep, chunks = p.k / 32;
    const int slots = p.tile;                                     // staged rows of X
    const int staged = (steps + p.warps_k - 1) / p.warps_k;       // steps a warp has room for
    const int mine = max(1, (steps - wk + p.warps_k - 1) / p.warps_k);
    const int64_t row_bytes = p.k / 2;

    // [warp][step][set][row of X][q] 16 bytes
    uint4 *xs = smem_u4 + (size_t)warp * staged * 4 * slots * 4;
    float *red = reinterpret_cast<float *>(smem_u4 + (size_t)kWarps * staged * 4 * slots * 4);
    const int red_floats = kWarps * kTiles * TT * 128;  // one of two buffers
    int *seg = reinterpret_cast<int *>(red + 2 * red_floats), *tiles = seg + p.experts + 1;

    ptx::grid_launch_dependents();
    if (!p.offsets) {
        // L2 prefetch of this CTA's first block: returns no data, changes nothing the program can observe
        const int row = (int)((int64_t)blockIdx.x * blocks / gridDim.x) * block_rows + (int)threadIdx.x;
        if ((int)threadIdx.x < block_rows && row < p.n)
            asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(p.B + (int64_t)row * row_bytes), "r"((int)row_bytes) : "memory");
    }
    ptx::grid_dependency_wait();  // nothing above read or wrote global memory

    int pairs;  // (expert, tile of rows)
    if (p.offsets) {
        if (warp == 0) scan_segments(p.offsets, p.experts, p.rows, p.tile, seg, tiles, lane);
        __syncthreads();
        pairs = tiles[p.experts];
    } else {
        pairs = (p.rows + p.tile - 1) / p.tile;
    }
    const int64_t units = (int64_t)pairs * blocks;  // the host has seen to it that they fit an int
    const int u_begin = (int)(units * blockIdx.x / gridDim.x), u_end = (int)(units * (blockIdx.x + 1) / gridDim.x);
    if (u_begin >= u_end) return;

    auto expert_of = [&](int pair) { return p.offsets ? expert_of_tile(tiles, p.experts, pair) : 0; };

    // ---- loads run kDepth steps ahead of the products
    struct Step {
        uint4 w[RG];
        RawScales<S, GPS> s;
    };
    int lu = u_begin;  // unit and step that are loaded next
    int li = 0;
    int lpair = -1, lexpert = 0;
    const uint8_t *lb = nullptr;  // this lane's 16 bytes of row group 0 at step wk
    const S *ls = nullptr;        // the scales of the row whose scales this lane fetches, at step wk
    int lrows = 0;                // rows of B from this lane's first one on
    bool ls_ok = false;
    const int srow = (q % RG) * 8 + g;  // lane (g, q) fetches the scales of row q * 8 + g and hands them to the lanes that need them
    auto load = [&](Step &b) {
#pragma unroll
        for (int r = 0; r < RG; ++r) b.w[r] = make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int j = 0; j < RawScales<S, GPS>::kWords; ++j) b.s.w[j] = 0;
        if (lu >= u_end) return;
        if (li == 0) {
            const int pair = lu / blocks, rb = lu - pair * blocks;
            if (pair != lpair) lpair = pair, lexpert = expert_of(pair);
            const int first = rb * block_rows + wr * 8 * RG;
            lb = p.B + ((int64_t)lexpert * p.n + first + g) * row_bytes + q * 16 + (int64_t)wk * 64;
            ls = scales + ((int64_t)lexpert * p.n + first + srow) * p.groups;
            lrows = p.n - first - g;
            ls_ok = first + srow < p.n;
        }
        const int t = wk + li * p.warps_k;
        if (4 * t + q < chunks) {
            const uint8_t *src = lb + (int64_t)li * p.warps_k * 64;
#pragma unroll
            for (int r = 0; r < RG; ++r)
                if (8 * r < lrows) b.w[r] = __ldcs(reinterpret_cast<const uint4 *>(src + 8 * r * row_bytes));
        }
        if (ls_ok && t < steps) {
            const int first = GPS > 1 ? t * GPS : (t * kStep) >> p.group_shift;
            if constexpr (GPS == 1) {
                if constexpr (sizeof(S) == 4) b.s.w[0] = __float_as_uint(to_float(__ldg(ls + first)));
                else b.s.w[0] = __ldg(reinterpret_cast<const unsigned short *>(ls + first));
            } else if (p.vec_scales) {
                if constexpr (RawScales<S, GPS>::kWords == 1) b.s.w[0] = __ldg(reinterpret_cast<const uint32_t *>(ls + first));
                else if constexpr (RawScales<S, GPS>::kWords == 2) {
                    const uint2 v = __ldg(reinterpret_cast<const uint2 *>(ls + first));
                    b.s.w[0] = v.x, b.s.w[1] = v.y;
                } else {
                    const uint4 v = __ldg(reinterpret_cast<const uint4 *>(ls + first));
                    b.s.w[0] = v.x, b.s.w[1] = v.y, b.s.w[2] = v.z, b.s.w[3] = v.w;
                }
            } else {
#pragma unroll
                for (int j = 0; j < GPS; ++j) {
                    if (first + j >= p.groups) continue;
                    if constexpr (sizeof(S) == 4) b.s.w[j] = __float_as_uint(to_float(__ldg(ls + first + j)));
                    else b.s.w[j >> 1] |= (uint32_t)__ldg(reinterpret_cast<const unsigned short *>(ls + first + j)) << (16 * (j & 1));
                }
            }
        }
        if (++li == mine) li = 0, ++lu;
    };

    // Element of a step's 128 at which the eight codes begin that lane (g, q) multiplies in set s (see the trade below).
    auto set_begin = [&](int s) {
        if constexpr (GPS == 1) return 32 * q + 8 * s;
        else if constexpr (GPS == 2) return 32 * (2 * (s >> 1) + (q & 1)) + 8 * (2 * (q >> 1) + (s & 1));
        else return 32 * s + 8 * q;
    };

    Step buf[kDepth];
#pragma unroll
    for (int d = 0; d < kDepth; ++d) load(buf[d]);

    int cu = u_begin;
    int ci = 0, cpair = -1, parity = 0;
    int first_row = 0, tokens = 0, rb = 0;
    float acc[kTiles][TT][4];

    auto stage_x = [&]() {
        // every lane stores what it will read: the eight elements of each set, in the order of the unpacked codes
        for (int tt = 0; tt < TT; ++tt) {
            const int slot = 8 * tt + g;
            if (slot >= slots) continue;
            const T *row = X + (int64_t)(first_row + slot) * p.ldx;
            for (int i = 0; i < mine; ++i) {
#pragma unroll
                for (int s = 0; s < 4; ++s) {
                    const int at = (wk + i * p.warps_k) * kStep + set_begin(s);
                    uint4 v = make_uint4(0, 0, 0, 0);
                    if (slot < tokens && at < p.k) v = __ldg(reinterpret_cast<const uint4 *>(row + at));
                    const uint4 o = make_uint4(__byte_perm(v.x, v.z, 0x5410), __byte_perm(v.x, v.z, 0x7632), __byte_perm(v.y, v.w, 0x5410),
                                               __byte_perm(v.y, v.w, 0x7632));  // (0, 4), (1, 5), (2, 6), (3, 7)
                    if (i < staged) xs[((i * 4 + s) * slots + slot) * 4 + q] = o;
                }
            }
        }
    };

    auto product = [&](Step &b) {
        if constexpr (GPS > 1) {
            // lanes q and q ^ 2 trade: afterwards sets 0, 1 hold codes of the first 64 elements of the step and sets 2, 3 of the last
#pragma unroll
            for (int r = 0; r < RG; ++r) {
                uint4 &w = b.w[r];
                const bool low = q < 2;
                const uint32_t s0 = low ? w.z : w.x, s1 = low ? w.w : w.y;
                const uint32_t r0 = __shfl_xor_sync(0xFFFFFFFFu, s0, 2), r1 = __shfl_xor_sync(0xFFFFFFFFu, s1, 2);
                if (low) w.z = r0, w.w = r1;
                else w.x = r0, w.y = r1;
                if constexpr (GPS == 4) {
                    // lanes q and q ^ 1 trade: afterwards set s holds codes of elements 32 s .. 32 s + 31
                    const bool even = (q & 1) == 0;
                    const uint32_t t0 = even ? w.y : w.x, t1 = even ? w.w : w.z;
                    const uint32_t v0 = __shfl_xor_sync(0xFFFFFFFFu, t0, 1), v1 = __shfl_xor_sync(0xFFFFFFFFu, t1, 1);
                    if (even) w.y = v0, w.w = v1;
                    else w.x = v0, w.z = v1;
                }
            }
        }
        const bool two = TT == 2 && tokens > 8;
        const bool has0 = g < slots, has1 = 8 + g < slots;
        float part[kTiles][TT][4];
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            uint4 x0 = make_uint4(0, 0, 0, 0), x1 = x0;
            const uint4 *src = xs + (ci * 4 + s) * slots * 4 + lane;
            if (has0) x0 = src[0];
            if (two && has1) x1 = src[32];
            constexpr float kZero[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            const bool fresh = s % (4 / GPS) == 0;  // a group begins
#pragma unroll
            for (int tl = 0; tl < kTiles; ++tl) {
                uint32_t lo[4], hi[4];
                const uint4 &w0 = b.w[2 * tl], &w1 = b.w[2 * tl + 1];
                codes_to_pairs(s == 0 ? w0.x : s == 1 ? w0.y : s == 2 ? w0.z : w0.w, lo, Tag<T>());
                codes_to_pairs(s == 0 ? w1.x : s == 1 ? w1.y : s == 2 ? w1.z : w1.w, hi, Tag<T>());
                const uint32_t a0[4] = {lo[0], hi[0], lo[1], hi[1]}, a1[4] = {lo[2], hi[2], lo[3], hi[3]};
                if (fresh) mma16816<T>(part[tl][0], a0, x0.x, x0.y, kZero);
                else mma16816<T>(part[tl][0], a0, x0.x, x0.y, part[tl][0]);
                mma16816<T>(part[tl][0], a1, x0.z, x0.w, part[tl][0]);
                if constexpr (TT == 2) {
                    if (two) {
                        if (fresh) mma16816<T>(part[tl][1], a0, x1.x, x1.y, kZero);
                        else mma16816<T>(part[tl][1], a0, x1.x, x1.y, part[tl][1]);
                        mma16816<T>(part[tl][1], a1, x1.z, x1.w, part[tl][1]);
                    }
                }
            }
            if ((s + 1) % (4 / GPS) == 0) {  // a group ends: its fp32 sums times its scale
                const int j = s / (4 / GPS);
#pragma unroll
                for (int tl = 0; tl < kTiles; ++tl) {
                    const float s0 = scale_at<S, GPS>(b.s, j, (lane & 28) | (2 * tl)), s1 = scale_at<S, GPS>(b.s, j, (lane & 28) | (2 * tl + 1));
#pragma unroll
                    for (int c = 0; c < 4; ++c) acc[tl][0][c] = fmaf(c < 2 ? s0 : s1, part[tl][0][c], acc[tl][0][c]);
                    if constexpr (TT == 2) {
                        if (two) {
#pragma unroll
                            for (int c = 0; c < 4; ++c) acc[tl][1][c] = fmaf(c < 2 ? s0 : s1, part[tl][1][c], acc[tl][1][c]);
                        }
                    }
                }
            }
        }
    };

    auto reduce_store = [&]() {
        // register c of lane l of tile tl at position (l + 2 tl + (c >> 1)) % 32: writes and reads hit 32 different banks
        float *buffer = red + parity * red_floats;
        parity ^= 1;
#pragma unroll
        for (int tl = 0; tl < kTiles; ++tl) {
#pragma unroll
            for (int tt = 0; tt < TT; ++tt) {
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    buffer[(((warp * kTiles + tl) * TT + tt) * 4 + c) * 32 + ((lane + 2 * tl + (c >> 1)) & 31)] = acc[tl][tt][c];
            }
        }
        __syncthreads();  // the other buffer may be written after the next one of these: every reader of it is then done
        T *out = static_cast<T *>(p.out);
        for (int o = threadIdx.x; o < block_rows * tokens; o += kThreads) {
            const int tok = o / block_rows, row = o - tok * block_rows;
            const int col = rb * block_rows + row;
            if (col >= p.n) continue;
            const int ww = row / (8 * RG), r = row - ww * 8 * RG, tl = r >> 4, half = (r >> 3) & 1;
            const int c = 2 * half + (tok & 1), l = (r & 7) * 4 + ((tok & 7) >> 1);
            float sum = 0.0f;
            for (int w = 0; w < p.warps_k; ++w)
                sum += buffer[((((ww * p.warps_k + w) * kTiles + tl) * TT + (tok >> 3)) * 4 + c) * 32 + ((l + 2 * tl + half) & 31)];
            out[(int64_t)(first_row + tok) * p.ldo + col] = from_float<T>(sum);
        }
    };

    for (;;) {
#pragma unroll
        for (int d = 0; d < kDepth; ++d) {
            if (ci == 0) {
                if (cu >= u_end) return;
                const int pair = cu / blocks;
                rb = cu - pair * blocks;
                if (pair != cpair) {
                    cpair = pair;
                    if (p.offsets) {
                        const int e = expert_of(pair);
                        first_row = seg[e] + (pair - tiles[e]) * p.tile;
                        tokens = min(p.tile, seg[e + 1] - first_row);
                    } else {
                        first_row = pair * p.tile;
                        tokens = min(p.tile, p.rows - first_row);
                    }
                    stage_x();
                }
#pragma unroll
                for (int tl = 0; tl < kTiles; ++tl)
#pragma unroll
                    for (int tt = 0; tt < TT; ++tt)
#pragma unroll
                        for (int c = 0; c < 4; ++c) acc[tl][tt][c] = 0.0f;
            }
            product(buf[d]);
            load(buf[d]);
            if (++ci == mine) {
                ci = 0, ++cu;
                reduce_store();
            }
        }
    }
}

int log2_of(int v)
{
    int s = 0;
    while ((1 << s) < v) ++s;
    return s;
}

struct RowsPlan {
    int tile, warps_k, rg;
    size_t smem;
};

size_t rows_smem(int k, int tile, int warps_k, int rg, int experts)
{
    const int steps = (k + kStep - 1) / kStep, staged = (steps + warps_k - 1) / warps_k;
    return (size_t)kWarps * staged * 4 * tile * 64 + 2 * (size_t)kWarps * (rg / 2) * (tile > 8 ? 2 : 1) * 512 + (size_t)(experts + 1) * 8;
}

// false: the staged rows of X do not fit
bool rows_plan(const W4Args &a, int sms, RowsPlan *plan)
{
    RowsPlan p;
    const int steps = (a.k + kStep - 1) / kStep;
    // warps beyond the steps of K would idle: they take further rows of B instead
    p.warps_k = steps >= 12 ? 16 : steps >= 6 ? 8 : 4;
    p.tile = a.offsets ? 16 : (a.rows < 16 ? a.rows : 16);
    p.rg = 4;
    (void)sms;
    while (p.tile > 8 && rows_smem(a.k, p.tile, p.warps_k, p.rg, a.experts) > (size_t)kMaxSmem) p.tile = 8;
    p.smem = rows_smem(a.k, p.tile, p.warps_k, p.rg, a.experts);
    *plan = p;
    return p.smem <= (size_t)kMaxSmem;
}

template <typename T, typename S, int GPS, int RG, int TT>
int rows_launch_variant(const W4Args &a, const RowsPlan &plan, const DeviceCtx &ctx)
{
    auto kernel = w4_rows_kernel<T, S, GPS, RG, TT>;
    static std::atomic<bool> configured[64];  // set once per device; a repeated cudaFuncSetAttribute is harmless
    if (!configured[ctx.device & 63].load(std::memory_order_acquire)) {
        cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmem);
        if (e != cudaSuccess) return record_cuda_error(e, "cudaFuncSetAttribute(w4_rows_kernel)");
        configured[ctx.device & 63].store(true, std::memory_order_release);
    }
    RowsParams p;
    p.X = a.X, p.ldx = a.ldx, p.B = a.B, p.scales = a.scales, p.offsets = a.offsets, p.out = a.out, p.ldo = a.ldo;
    p.rows = a.rows, p.n = a.n, p.k = a.k, p.experts = a.experts;
    p.group_shift = log2_of(a.group), p.groups = (a.k + a.group - 1) / a.group;
    p.tile = plan.tile, p.warps_k = plan.warps_k;
    // a step's scales lie on a boundary of their own size when a row has a multiple of GPS of them
    p.vec_scales = p.groups % GPS == 0 && (reinterpret_cast<uintptr_t>(a.scales) & (GPS * sizeof(S) - 1)) == 0;
    const int block_rows = 8 * RG * (kWarps / plan.warps_k);
    const int64_t blocks = (a.n + block_rows - 1) / block_rows;
    // with experts the units are known on the device only: at most one tile more than whole ones per expert that can have rows
    const int64_t pairs = a.offsets ? a.rows / plan.tile + (a.experts < a.rows ? a.experts : a.rows) : (a.rows + plan.tile - 1) / plan.tile;
    const int64_t units = pairs * blocks;
    if (units > 0x7FFFFFFF) return QM_ERR_SHAPE;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(units < ctx.num_sms ? units : ctx.num_sms), 1, 1);
    cfg.blockDim = dim3(kThreads, 1, 1);
    cfg.dynamicSmemBytes = plan.smem;
    cfg.stream = a.stream;
    cudaLaunchAttribute attr[1];
    static const bool allow_pdl = !std::getenv("QM_NO_PDL");
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = allow_pdl ? 1 : 0;
    cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, p);
    return e == cudaSuccess ? QM_OK : record_cuda_error(e, "w4_rows_kernel launch");
}

}  // namespace

bool w4_rows_eligible(const W4Args &a, const DeviceCtx &ctx)
{
    RowsPlan plan;
    return a.k > 0 && a.k % 32 == 0 && a.ldx % 8 == 0 && ((reinterpret_cast<uintptr_t>(a.X) | reinterpret_cast<uintptr_t>(a.B)) & 15u) == 0 &&
           rows_plan(a, ctx.num_sms, &plan);
}

int w4_rows_launch(const W4Args &a, const DeviceCtx &ctx)
{
    RowsPlan plan;
    if (!rows_plan(a, ctx.num_sms, &plan)) return QM_ERR_ARG;
    auto by_type = [&](auto t) {
        using T = typename decltype(t)::type;
        return with_same_or_float<T>(a.scale_type, [&](auto u) {
            using S = typename decltype(u)::type;
            auto by_group = [&](auto tt) {
                constexpr int TT = decltype(tt)::value;
                if (a.group == 32) return rows_launch_variant<T, S, 4, 4, TT>(a, plan, ctx);
                if (a.group == 64) return rows_launch_variant<T, S, 2, 4, TT>(a, plan, ctx);
                return rows_launch_variant<T, S, 1, 4, TT>(a, plan, ctx);
            };
            return plan.tile > 8 ? by_group(std::integral_constant<int, 2>()) : by_group(std::integral_constant<int, 1>());
        });
    };
    return a.type == QM_TYPE_F16 ? by_type(Tag<__half>()) : by_type(Tag<__nv_bfloat16>());
}

}  // namespace qm
