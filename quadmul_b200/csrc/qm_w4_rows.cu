// 4-bit weights with group scales, few rows of X: weight streaming.
//
// out[r][c] = sum over groups g of scale[c][g] * sum over i in g of x[r][i] q[c][i].  With up to 16 rows of X the product reads
// every weight once and is bound by memory; what a kernel has to do is keep loads in flight and convert codes fast enough.
//
//  * A CTA (16 warps) takes blocks of 8 RG rows of B, WK of its warps split K between them in steps of 128 elements.  Every
//    warp has a ring of p.depth boxes (8 RG rows x 64 bytes) of its own, filled by TMA loads that its first lane issues as soon
//    as a box has been read: no other warp takes part, the loads run on across the end of a block, and up to 128 KB are on the
//    way per SM.  Lane (g, q) = (lane / 4, lane % 4) reads 16 bytes, 32 codes, of row g of each 8-row group.
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
#include "qm_tc_common.cuh"
#include "qm_w4.cuh"

namespace qm {

using namespace w4;

namespace {

constexpr int kWarps = 16, kThreads = kWarps * 32;
constexpr int kMaxDepth = 4;     // boxes in flight per warp
constexpr int kStep = 128;       // elements of K per step
constexpr int kMaxSmem = 232448 - 1024;

struct RowsParams {
    const void *X;
    int64_t ldx;
    const void *scales;
    const int *offsets;
    void *out;
    int64_t ldo;
    int rows, n, k, experts;
    int group_shift, groups;
    int tile;      // rows of X per unit, at most 16
    int depth;     // boxes in a warp's ring
    int *status;
    int warps_k;   // warps that split K; the others take further rows of B
    int vec_scales;  // a step's scales can be loaded as one vector
};

// d = a b, or d += a b: 16 rows of B x 16 elements of K x 8 rows of X
template <typename T, bool FRESH>
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1)
{
    if constexpr (std::is_same<T, __half>::value) {
        if constexpr (FRESH)
            asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
        else
            asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    } else {
        if constexpr (FRESH)
            asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
        else
            asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    }
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
__global__ void __launch_bounds__(kThreads, 1) w4_rows_kernel(const __grid_constant__ CUtensorMap tmapB, const RowsParams p)
{
    constexpr int kTiles = RG / 2;            // 16-row tiles of B per warp
    constexpr int kBoxBytes = 8 * RG * 64;
    extern __shared__ __align__(128) uint4 smem_u4[];
    const T *__restrict__ X = static_cast<const T *>(p.X);
    const S *__restrict__ scales = static_cast<const S *>(p.scales);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
    const int wk = warp % p.warps_k, wr = warp / p.warps_k;
    const int block_rows = 8 * RG * (kWarps / p.warps_k);
    const int blocks = (p.n + block_rows - 1) / block_rows;
    const int steps = (p.k + kStep - 1) / kStep;
    const int slots = p.tile;                                     // staged rows of X
    const int staged = (steps + p.warps_k - 1) / p.warps_k;       // steps a warp has room for
    const int mine = max(1, (steps - wk + p.warps_k - 1) / p.warps_k);

    // ring [warp][box], X [warp][step][set][row][q] 16 bytes, partial tiles, barriers, segments
    const uint32_t ring = ptx::smem_u32(smem_u4) + (uint32_t)(warp * p.depth * kBoxBytes);
    uint4 *xs = smem_u4 + (kWarps * p.depth * kBoxBytes) / 16 + (size_t)warp * staged * 4 * slots * 4;
    float *red = reinterpret_cast<float *>(smem_u4 + (kWarps * p.depth * kBoxBytes) / 16 + (size_t)kWarps * staged * 4 * slots * 4);
    constexpr int kRedFloats = kWarps * kTiles * TT * 128;  // one of two buffers
    uint64_t *bars = reinterpret_cast<uint64_t *>(red + 2 * kRedFloats);
    const uint32_t bar0 = ptx::smem_u32(bars + warp * kMaxDepth);
    int *abort_word = reinterpret_cast<int *>(bars + kWarps * kMaxDepth);
    int *seg = abort_word + 2, *tiles = seg + p.experts + 1;

    ptx::grid_launch_dependents();
    if (threadIdx.x == 0) *abort_word = 0;
    if (lane == 0) {
        for (int s = 0; s < p.depth; ++s) ptx::mbar_init(bar0 + 8u * s, 1);
        ptx::fence_mbar_init();
        ptx::fence_proxy_async_smem();
        ptx::prefetch_tmap(&tmapB);
        if (!p.offsets) {
            // L2 prefetch of this warp's first boxes: returns no data, changes nothing the program can observe
            const int row = (int)((int64_t)((p.rows + p.tile - 1) / p.tile) * blocks * blockIdx.x / gridDim.x) % blocks * block_rows + wr * 8 * RG;
            for (int i = 0; i < min(mine, p.depth); ++i)
                asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global.tile [%0, {%1, %2}];" ::"l"(&tmapB), "r"((wk + i * p.warps_k) * 64), "r"(row) : "memory");
        }
    }
    ptx::grid_dependency_wait();  // nothing above read or wrote global memory

    int pairs;  // (expert, tile of rows)
    if (p.offsets) {
        if (warp == 0) scan_segments(p.offsets, p.experts, p.rows, p.tile, seg, tiles, lane);
        __syncthreads();
        pairs = tiles[p.experts];
    } else {
        __syncthreads();
        pairs = (p.rows + p.tile - 1) / p.tile;
    }
    const int64_t units = (int64_t)pairs * blocks;  // the host has seen to it that they fit an int
    const int u_begin = (int)(units * blockIdx.x / gridDim.x), u_end = (int)(units * (blockIdx.x + 1) / gridDim.x);
    if (u_begin >= u_end) return;

    auto expert_of = [&](int pair) { return p.offsets ? expert_of_tile(tiles, p.experts, pair) : 0; };

    // ---- boxes of codes run p.depth steps ahead of the products
    int lu = u_begin, li = 0, lslot = 0, lrow = 0;
    auto load_box = [&]() {
        if (lu >= u_end) return;
        if (li == 0) {
            const int pair = lu / blocks;
            lrow = expert_of(pair) * p.n + (lu - pair * blocks) * block_rows + wr * 8 * RG;
        }
        if (lane == 0) {
            ptx::mbar_arrive_expect_tx(bar0 + 8u * lslot, kBoxBytes);
            ptx::tma_load_2d(ring + lslot * kBoxBytes, &tmapB, (wk + li * p.warps_k) * 64, lrow, bar0 + 8u * lslot);
        }
        if (++lslot == p.depth) lslot = 0;
        if (++li == mine) li = 0, ++lu;
    };
    // ---- scales two steps ahead: lane (g, q) fetches those of row q * 8 + g and hands them to the lanes that need them
    using Raw = RawScales<S, GPS>;
    int su = u_begin, si = 0;
    const S *sp = nullptr;
    bool s_ok = false;
    const int srow = (q % RG) * 8 + g;
    auto load_scales = [&](Raw &s) {
#pragma unroll
        for (int j = 0; j < Raw::kWords; ++j) s.w[j] = 0;
        if (su >= u_end) return;
        if (si == 0) {
            const int pair = su / blocks, row = (su - pair * blocks) * block_rows + wr * 8 * RG + srow;
            sp = scales + ((int64_t)expert_of(pair) * p.n + row) * p.groups;
            s_ok = row < p.n;
        }
        const int t = wk + si * p.warps_k;
        if (s_ok && t < steps) {
            const int first = GPS > 1 ? t * GPS : (t * kStep) >> p.group_shift;
            if constexpr (GPS == 1) {
                if constexpr (sizeof(S) == 4) s.w[0] = __float_as_uint(to_float(__ldg(sp + first)));
                else s.w[0] = __ldg(reinterpret_cast<const unsigned short *>(sp + first));
            } else if (p.vec_scales) {
                if constexpr (Raw::kWords == 1) s.w[0] = __ldg(reinterpret_cast<const uint32_t *>(sp + first));
                else if constexpr (Raw::kWords == 2) {
                    const uint2 v = __ldg(reinterpret_cast<const uint2 *>(sp + first));
                    s.w[0] = v.x, s.w[1] = v.y;
                } else {
                    const uint4 v = __ldg(reinterpret_cast<const uint4 *>(sp + first));
                    s.w[0] = v.x, s.w[1] = v.y, s.w[2] = v.z, s.w[3] = v.w;
                }
            } else {
#pragma unroll
                for (int j = 0; j < GPS; ++j) {
                    if (first + j >= p.groups) continue;
                    if constexpr (sizeof(S) == 4) s.w[j] = __float_as_uint(to_float(__ldg(sp + first + j)));
                    else s.w[j >> 1] |= (uint32_t)__ldg(reinterpret_cast<const unsigned short *>(sp + first + j)) << (16 * (j & 1));
                }
            }
        }
        if (++si == mine) si = 0, ++su;
    };

    // Element of a step's 128 at which the eight codes begin that lane (g, q) multiplies in set s (see the trade below).
    auto set_begin = [&](int s) {
        if constexpr (GPS == 1) return 32 * q + 8 * s;
        else if constexpr (GPS == 2) return 32 * (2 * (s >> 1) + (q & 1)) + 8 * (2 * (q >> 1) + (s & 1));
        else return 32 * s + 8 * q;
    };

    for (int d = 0; d < p.depth; ++d) load_box();
    Raw raw[2];
    load_scales(raw[0]);
    load_scales(raw[1]);

    int cu = u_begin, ci = 0, cslot = 0, cpair = -1, parity = 0;
    uint32_t phase = 0;
    bool dead = false;  // a wait gave up: run on without data, so that the block's barriers still meet
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

    auto product = [&](const Raw &raw_scales) {
        if (!dead && !ptx::warp_wait<false>(bar0 + 8u * cslot, phase, abort_word, lane)) {
            dead = true;
            if (lane == 0) tc::report_timeout(p.status, kWaitConvertPacked), *abort_word = 1;
        }
        uint4 wv[RG];
#pragma unroll
        for (int r = 0; r < RG; ++r) wv[r] = ptx::lds128(ring + cslot * kBoxBytes + r * 512 + lane * 16);
        if (++cslot == p.depth) cslot = 0, phase ^= 1u;
        __syncwarp();  // the box is in registers
        if (!dead) load_box();
        if constexpr (GPS > 1) {
            // lanes q and q ^ 2 trade: afterwards sets 0, 1 hold codes of the first 64 elements of the step and sets 2, 3 of the last
#pragma unroll
            for (int r = 0; r < RG; ++r) {
                uint4 &w = wv[r];
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
            const bool fresh = s % (4 / GPS) == 0;  // a group begins
#pragma unroll
            for (int tl = 0; tl < kTiles; ++tl) {
                uint32_t lo[4], hi[4];
                const uint4 &w0 = wv[2 * tl], &w1 = wv[2 * tl + 1];
                codes_to_pairs(s == 0 ? w0.x : s == 1 ? w0.y : s == 2 ? w0.z : w0.w, lo, Tag<T>());
                codes_to_pairs(s == 0 ? w1.x : s == 1 ? w1.y : s == 2 ? w1.z : w1.w, hi, Tag<T>());
                if (fresh) mma16816<T, true>(part[tl][0], lo[0], hi[0], lo[1], hi[1], x0.x, x0.y);
                else mma16816<T, false>(part[tl][0], lo[0], hi[0], lo[1], hi[1], x0.x, x0.y);
                mma16816<T, false>(part[tl][0], lo[2], hi[2], lo[3], hi[3], x0.z, x0.w);
                if constexpr (TT == 2) {
                    if (two) {
                        if (fresh) mma16816<T, true>(part[tl][1], lo[0], hi[0], lo[1], hi[1], x1.x, x1.y);
                        else mma16816<T, false>(part[tl][1], lo[0], hi[0], lo[1], hi[1], x1.x, x1.y);
                        mma16816<T, false>(part[tl][1], lo[2], hi[2], lo[3], hi[3], x1.z, x1.w);
                    }
                }
            }
            if ((s + 1) % (4 / GPS) == 0) {  // a group ends: its fp32 sums times its scale
                const int j = s / (4 / GPS);
#pragma unroll
                for (int tl = 0; tl < kTiles; ++tl) {
                    const float s0 = scale_at<S, GPS>(raw_scales, j, (lane & 28) | (2 * tl)), s1 = scale_at<S, GPS>(raw_scales, j, (lane & 28) | (2 * tl + 1));
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
        float *buffer = red + parity * kRedFloats;
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
            out[(int64_t)(first_row + tok) * p.ldo + col] = from_float<T>(sum * kCodeUnit<T>);
        }
    };

    for (;;) {
#pragma unroll
        for (int d = 0; d < 2; ++d) {
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
            product(raw[d]);
            load_scales(raw[d]);
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
    int tile, warps_k, rg, depth;
    size_t smem;
};

size_t rows_smem(int k, const RowsPlan &p, int experts)
{
    const int steps = (k + kStep - 1) / kStep, staged = (steps + p.warps_k - 1) / p.warps_k;
    return (size_t)kWarps * p.depth * 512 * p.rg + (size_t)kWarps * staged * 4 * p.tile * 64 + 2 * (size_t)kWarps * (p.rg / 2) * (p.tile > 8 ? 2 : 1) * 512 +
           kWarps * kMaxDepth * 8 + 8 + (size_t)(experts + 1) * 8;
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
    // the deepest ring that leaves room for X; two boxes a warp are the least that keeps the stream going
    auto fit = [&]() {
        for (p.depth = kMaxDepth; p.depth >= 2; --p.depth)
            if (rows_smem(a.k, p, a.experts) <= (size_t)kMaxSmem) return true;
        return false;
    };
    bool ok = fit();
    if (!ok && p.tile > 8) {
        p.tile = 8;
        ok = fit();
    }
    if (ok) p.smem = rows_smem(a.k, p, a.experts);
    *plan = p;
    return ok;
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
    CUtensorMap tmB;
    int st = tc::make_packed_tmap(&tmB, a.B, a.experts * a.n, a.k / 2, 8 * RG, CU_TENSOR_MAP_SWIZZLE_NONE);
    if (st != QM_OK) return st;
    RowsParams p;
    p.depth = plan.depth, p.status = ctx.status;
    p.X = a.X, p.ldx = a.ldx, p.scales = a.scales, p.offsets = a.offsets, p.out = a.out, p.ldo = a.ldo;
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
    cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, tmB, p);
    return e == cudaSuccess ? QM_OK : record_cuda_error(e, "w4_rows_kernel launch");
}

}  // namespace

bool w4_rows_eligible(const W4Args &a, const DeviceCtx &ctx)
{
    RowsPlan plan;
    return a.k > 0 && a.k % 32 == 0 && a.ldx % 8 == 0 && (int64_t)a.experts * a.n <= 0x7FFFFFFF - 512 && ((reinterpret_cast<uintptr_t>(a.X) | reinterpret_cast<uintptr_t>(a.B)) & 15u) == 0 &&
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
