// 4-bit weights with group scales on the 5th-generation tensor cores: many rows of X, and a few rows where the weights are not.
//
// out[r][c] = sum over i of x[r][i] w[c][i], w[c][i] = scale[c][i / group] q[c][i].  128 rows of B (a CTA's) lie on the UMMA M axis,
// rows of X on the N axis, so the converted weights are the operand that tcgen05.mma takes from TMEM: they never go through
// shared memory as 16-bit values, and X is used as TMA brings it.  A stage is 128 elements of K.
//
//   warp 0       TMA producer of B: packed rows (64-byte swizzle) into a ring of kRingW stages of 8 KB
//   warp 2       TMA producer of X: two 64-element sub-blocks (128-byte swizzle) of up to 128 rows into a ring of kRingX stages
//   warp 3       relay of X's arrival to the MMA issuer
//   warps 12-    converters, kSets sets of four that take the stages in turn; a thread owns a row of B: 64 bytes of codes become 128
//                scaled 16-bit values in 64 TMEM columns (tcgen05.st)
//   warp 1       MMA issuer (of the pair's leader): eight tcgen05.mma.kind::f16 a stage, fp32 accumulators in 256 TMEM columns
//   warps 4-11   epilogue: two warps per lane quarter; lanes hold consecutive columns of out
//
// code * scale is rounded to X's type (half a step of the type, as the result is): scaling the fp32 sums of every group instead, as
// the kernel for few rows does, would need an accumulator pass per group.  fp16 has no room for scales far from one, so a
// row's scales are first divided by the power of two below the largest, and its sums are multiplied by it again: a group whose
// scale is less than 2^-14 of its row's largest loses digits, nothing overflows.
//
// PAIR form (G = 2, persistent): two CTAs share a 256 x N tile, N <= 256; each converts its own 128 rows of B and loads half
// of the rows of X, so a stage brings 24 KB into each SM for 1024 tensor clocks (a 128-row tile would need twice X's part).
// N follows the rows that are left, in steps of 16: with experts a short segment costs its own width.
// SPLIT form (G = 1): where there are few tiles, a cluster of up to 8 CTAs shares one 128 x N tile, N <= 128, each taking a
// part of K; the partial tiles meet in the CTAs' shared memory and are added in a fixed order.
// All waits are bounded as in gemm_tc_kernel.
//
// Measured (groups of 128, bf16, a few calls in a row; a long run meets the power cap): 2048 x 12288 x 4096 138-142 us = 1.45-1.49
// PFLOP/s, tensor pipe 82 % active (fp16 144-149 us; the library's 16-bit product of that size 136); 8192 rows over 8 experts of 11008 x
// 4096 505 us = 1.46 PFLOP/s (fp16 529).  Few columns per item are bound by the stages' turn-round, about 700 clocks each: 512 rows
// over 32 experts of 4096 x 4096 95 us = 2.9 TB/s; a quarter of the MMAs, no tcgen05.st, longer rings or wider loads change that by
// 3 % at most, no conversion by 14 %.  SPLIT is a chain of latencies: 16 x 4096 x 4096 10.2 us, 128 x 4096 x 4096 13.2.
#include <cuda.h>

#include <atomic>
#include <cstdlib>

#include "qm_ptx.cuh"
#include "qm_tc_common.cuh"
#include "qm_w4.cuh"

namespace qm {

using namespace w4;

namespace {

using namespace ptx;
using namespace tc;

constexpr int kRowsB = 128;     // rows of B per CTA
constexpr int kStageK = 128;    // elements of K per stage
constexpr int kRingW = 7, kRingX = 4;
constexpr int kBytesW = kRowsB * kStageK / 2;  // 8 KB
constexpr int kRowsX = 128;                    // rows of X a CTA holds
constexpr int kSubX = kRowsX * 128;            // 64 elements of K: 16 KB
constexpr int kBytesX = 2 * kSubX;
constexpr int kBoxRows = 32;
constexpr int kAccCols = 256, kStageCols = 64, kTmemCols = 512;
constexpr int kEpiWarp = 4, kNumEpiWarps = 8, kConvWarp = 12, kSets = 3, kNumConvWarps = 4 * kSets;
constexpr int kNumWarps = kConvWarp + kNumConvWarps, kNumThreads = kNumWarps * 32;
constexpr int kNumBarriers = 2 * kRingW + 3 * kRingX + 2;
constexpr int kMaxParts = 8;    // of K: a cluster
constexpr int kEpiBytes = 16 * 32 * 2;  // per epilogue warp: 16 rows of out x 32 columns
constexpr int kSmemFixed = 1024 + kRingW * kBytesW + kRingX * kBytesX + kNumEpiWarps * kEpiBytes + kNumBarriers * 8 + 16 + kRowsB * 4;
static_assert(kAccCols + kRingX * kStageCols <= kTmemCols, "TMEM budget");
static_assert(kSmemFixed + 8 * 4097 <= 232448, "shared memory");

struct TcParams {
    const void *scales;
    const int *offsets;
    void *out;
    int64_t ldo;
    int rows, n, k, experts;
    int group_shift, groups;
    int tile;        // rows of X per tile: a multiple of 16
    int vec_scales;  // the four scales of a stage (groups of 32), or two (64), can be loaded as one vector
    int vec_out;     // out's rows begin on 16-byte boundaries
    int *status;
};

// D[tmem] (+)= A[tmem] * B[smem desc], 16-bit floats -> fp32.  One thread issues it.
template <int G>
__device__ __forceinline__ void umma_f16_ta(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc, uint32_t accumulate)
{
    if constexpr (G == 1)
        asm volatile(
            "{\n"
            " .reg .pred p;\n"
            " setp.ne.b32 p, %4, 0;\n"
            " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n"
            "}\n" ::"r"(tmem_d),
            "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate)
            : "memory");
    else
        asm volatile(
            "{\n"
            " .reg .pred p;\n"
            " setp.ne.b32 p, %4, 0;\n"
            " tcgen05.mma.cta_group::2.kind::f16 [%0], [%1], %2, %3, p;\n"
            "}\n" ::"r"(tmem_d),
            "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate)
            : "memory");
}

// One arrival on the barrier (in BOTH CTAs of a pair) once every MMA issued so far has finished.
template <int G>
__device__ __forceinline__ void commit_all(uint32_t bar)
{
    if constexpr (G == 1)
        umma_commit<1>(bar);
    else
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
                     "h"((uint16_t)3)
                     : "memory");
}

__device__ __forceinline__ void tmem_st_x32(uint32_t taddr, const uint32_t (&v)[32])
{
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
        "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
        "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]),
        "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]),
        "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
        : "memory");
}

__device__ __forceinline__ void tmem_st_wait()
{
    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

__device__ __forceinline__ float2 lds_cluster_f2(uint32_t addr)
{
    float2 v;
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
    return v;
}

__device__ __forceinline__ uint32_t cluster_nctarank()
{
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
    return r;
}

// The power of two below a row's largest scale (1 for a row of zeros or with a scale that is not finite); bf16 has fp32's range
// and needs none.
template <typename T, typename S>
__device__ __forceinline__ float row_unit(const S *s, int groups)
{
    if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        return 1.0f;
    } else {
        // Magnitudes order like unsigned integers, an infinity or a NaN above every number.  The loads go out many at a time: the
        // row comes from DRAM, and a few in turn held 37 x 1100 x 2208 up for 9,000 clocks.  (Those behind the end repeat the last.)
        uint32_t most = 0;
        constexpr int kVec = 16 / (int)sizeof(S), kAhead = 4;
        if ((reinterpret_cast<uintptr_t>(s) & 15u) == 0 && groups % kVec == 0) {
            const uint4 *v = reinterpret_cast<const uint4 *>(s);
            const int last = groups / kVec - 1;
            for (int j = 0; j <= last; j += kAhead) {
                uint4 u[kAhead];
#pragma unroll
                for (int i = 0; i < kAhead; ++i) u[i] = ld_behind_wait(v + min(j + i, last));
#pragma unroll
                for (int i = 0; i < kAhead; ++i) {
                    const uint32_t w[4] = {u[i].x, u[i].y, u[i].z, u[i].w};
#pragma unroll
                    for (int o = 0; o < 4; ++o) {
                        if constexpr (sizeof(S) == 4) most = max(most, w[o] & 0x7FFFFFFFu);
                        else most = __vmaxu2(most, w[o] & 0x7FFF7FFFu);
                    }
                }
            }
            if constexpr (sizeof(S) == 2) most = max(most & 0xFFFFu, most >> 16);
        } else {
            using Bits = typename std::conditional<sizeof(S) == 4, uint32_t, unsigned short>::type;
            const Bits *v = reinterpret_cast<const Bits *>(s);
            for (int j = 0; j < groups; j += 4 * kAhead) {
                uint32_t u[4 * kAhead];
#pragma unroll
                for (int i = 0; i < 4 * kAhead; ++i) u[i] = ld_behind_wait(v + min(j + i, groups - 1));
#pragma unroll
                for (int i = 0; i < 4 * kAhead; ++i) most = max(most, u[i] & (sizeof(S) == 4 ? 0x7FFFFFFFu : 0x7FFFu));
            }
        }
        float top;
        if constexpr (sizeof(S) == 4) top = __uint_as_float(most);
        else top = __half2float(__ushort_as_half((unsigned short)most));
        if (!(top > 0.0f) || !(top < INFINITY)) return 1.0f;
        // exponent bits alone; the smallest normal number for a subnormal one, and no larger than leaves a finite reciprocal
        const uint32_t e = min(max(__float_as_uint(top) >> 23, 1u), 253u);
        return __uint_as_float(e << 23);
    }
}

template <int G, typename T, typename S>
__global__ void __launch_bounds__(kNumThreads, 1)
w4_tc_kernel(const __grid_constant__ CUtensorMap tmapW, const __grid_constant__ CUtensorMap tmapX, const __grid_constant__ CUtensorMap tmapX128,
             const TcParams p)
{
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw_u32 = smem_u32(smem_raw);
    const uint32_t x0 = (raw_u32 + 1023u) & ~1023u;   // X ring: [stage][sub-block][row][128 B]
    const uint32_t w0 = x0 + kRingX * kBytesX;        // B ring: [stage][row][64 B]
    const uint32_t epi0 = w0 + kRingW * kBytesW;      // epilogue: [warp][row of X][32 columns]
    const uint32_t bar0 = epi0 + kNumEpiWarps * kEpiBytes;
    auto w_full = [&](int s) { return bar0 + 8u * s; };
    auto w_empty = [&](int s) { return bar0 + 8u * (kRingW + s); };
    auto x_full = [&](int s) { return bar0 + 8u * (2 * kRingW + s); };
    auto a_full = [&](int s) { return bar0 + 8u * (2 * kRingW + kRingX + s); };       // converted stage; the leader's copy is waited on
    auto ax_empty = [&](int s) { return bar0 + 8u * (2 * kRingW + 2 * kRingX + s); };  // converted stage and its X stage are free
    const uint32_t acc_full = bar0 + 8u * (2 * kRingW + 3 * kRingX), acc_empty = acc_full + 8u;
    const uint32_t tmem_slot = bar0 + 8u * kNumBarriers;
    uint8_t *generic0 = smem_raw + (bar0 - raw_u32);
    uint32_t *tmem_slot_ptr = reinterpret_cast<uint32_t *>(generic0 + 8 * kNumBarriers);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(generic0 + 8 * kNumBarriers + 4);
    float *unit_of_row = reinterpret_cast<float *>(generic0 + 8 * kNumBarriers + 16);
    int *seg = reinterpret_cast<int *>(unit_of_row + kRowsB), *tiles = seg + p.experts + 1;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = (int)cluster_ctarank();                  // half of the pair, or part of K
    const int parts = G == 1 ? (int)cluster_nctarank() : 1;   // parts of K
    const int cluster = G == 1 ? (int)blockIdx.x / parts : (int)blockIdx.x / 2;
    const int clusters = G == 1 ? (int)gridDim.x / parts : (int)gridDim.x / 2;
    const int tilesP = (p.n + kRowsB * G - 1) / (kRowsB * G);
    const int num_kb = (p.k + kStageK - 1) / kStageK;
    const int kb0 = G == 1 ? (int)((int64_t)rank * num_kb / parts) : 0, kb1 = G == 1 ? (int)((int64_t)(rank + 1) * num_kb / parts) : num_kb;

    if (threadIdx.x == 0) {
        for (int s = 0; s < kRingW; ++s) mbar_init(w_full(s), 1), mbar_init(w_empty(s), 4);
        for (int s = 0; s < kRingX; ++s) mbar_init(x_full(s), 1), mbar_init(a_full(s), 5 * G), mbar_init(ax_empty(s), 1);
        mbar_init(acc_full, 1);
        mbar_init(acc_empty, G * kNumEpiWarps);
        *abort_flag = 0;
        fence_mbar_init();
        fence_proxy_async_smem();
    }
    if (warp == 0 && lane == 0) prefetch_tmap(&tmapW);
    if (warp == 2 && lane == 0) prefetch_tmap(&tmapX), prefetch_tmap(&tmapX128);
    if (warp == 1) {
        tmem_alloc<G>(tmem_slot, kTmemCols);
        tmem_relinquish<G>();
    }
    grid_dependency_wait();  // nothing above read or wrote global memory
    if (p.offsets && warp == 3) scan_segments(p.offsets, p.experts, p.rows, p.tile, seg, tiles, lane);
    tc_fence_before_sync();
    __syncthreads();
    grid_launch_dependents();  // (the TMEM is taken by now: a successor that wants some waits for this kernel, not the other way round)
    if (G == 2) {  // the pair's barriers are there (in the SPLIT form a CTA keeps to itself until the parts are added up)
        cluster_arrive();
        cluster_wait();
    }
    tc_fence_after_sync();
    const uint32_t tmem_base = *tmem_slot_ptr;
    const uint32_t tmem_a0 = tmem_base + kAccCols;
    const int num_items = (p.offsets ? tiles[p.experts] : (p.rows + p.tile - 1) / p.tile) * tilesP;

    // Item t: rows [row, row + count) of X times rows [col, col + 128 G) of expert e's matrix; width = count rounded up for the
    // MMA.  Items of an expert are consecutive, in an order that shares operand rows in L2.
    struct Item {
        int e, row, count, width, col;
    };
    auto item = [&](int t) {
        Item it;
        int first = 0, last = p.rows, local = t;
        it.e = 0;
        if (p.offsets) {
            it.e = expert_of_tile(tiles, p.experts, t / tilesP);
            first = seg[it.e], last = seg[it.e + 1];
            local = t - tiles[it.e] * tilesP;
        }
        int tp, tq;
        tile_coords(local, tilesP, (last - first + p.tile - 1) / p.tile, tp, tq);
        it.row = first + tq * p.tile;
        it.count = min(p.tile, last - it.row);
        it.width = (it.count + 15) & ~15;
        it.col = tp * kRowsB * G;
        return it;
    };
    auto give_up = [&](int site) {
        report_timeout(p.status, site);
        *abort_flag = 1;
    };

    if (warp == 0) {
        // ------------------------------ producer of B ------------------------------
        const bool elected = elect_one();
        uint32_t it = 0;
        bool ok = true;
        for (int t = cluster; t < num_items && ok; t += clusters) {
            const Item m = item(t);
            const int y = m.e * p.n + m.col + (G == 2 ? rank * kRowsB : 0);
            for (int kb = kb0; kb < kb1; ++kb, ++it) {
                const int s = it % kRingW;
                if (!warp_wait<false>(w_empty(s), ((it / kRingW) & 1u) ^ 1u, abort_flag, lane)) {
                    if (lane == 0) give_up(kWaitProducerSlot);
                    ok = false;
                    break;
                }
                if (elected) {
                    mbar_arrive_expect_tx(w_full(s), kBytesW);
                    tma_load_2d(w0 + s * kBytesW, &tmapW, kb * (kStageK / 2), y, w_full(s));
                }
                __syncwarp();
            }
        }
    } else if (warp == 2) {
        // ------------------------------ producer of X ------------------------------
        const bool elected = elect_one();
        uint32_t it = 0;
        bool ok = true;
        for (int t = cluster; t < num_items && ok; t += clusters) {
            const Item m = item(t);
            const int share = m.width / G, boxes = (share + kBoxRows - 1) / kBoxRows;
            const bool whole = boxes == kRowsX / kBoxRows;  // one box per sub-block
            const int y = m.row + (G == 2 ? rank * share : 0);
            for (int kb = kb0; kb < kb1; ++kb, ++it) {
                const int s = it % kRingX;
                if (!warp_wait<false>(ax_empty(s), ((it / kRingX) & 1u) ^ 1u, abort_flag, lane)) {
                    if (lane == 0) give_up(kWaitProducerSlot);
                    ok = false;
                    break;
                }
                if (elected) {
                    const uint32_t dst = x0 + s * kBytesX;
                    mbar_arrive_expect_tx(x_full(s), (uint32_t)boxes * 2 * kBoxRows * 128);
                    if (whole) {
                        tma_load_2d(dst, &tmapX128, kb * kStageK, y, x_full(s));
                        tma_load_2d(dst + kSubX, &tmapX128, kb * kStageK + 64, y, x_full(s));
                    } else {
                        for (int b = 0; b < boxes; ++b) {
                            tma_load_2d(dst + b * kBoxRows * 128, &tmapX, kb * kStageK, y + b * kBoxRows, x_full(s));
                            tma_load_2d(dst + kSubX + b * kBoxRows * 128, &tmapX, kb * kStageK + 64, y + b * kBoxRows, x_full(s));
                        }
                    }
                }
                __syncwarp();
            }
        }
    } else if (warp == 3) {
        // ------------------------------ relay: this CTA's rows of X have arrived ------------------------------
        // The MMA issuer waits for one signal per stage that covers both operands of both CTAs.
        uint32_t it = 0;
        bool ok = true;
        for (int t = cluster; t < num_items && ok; t += clusters) {
            for (int kb = kb0; kb < kb1; ++kb, ++it) {
                const int s = it % kRingX;
                if (!warp_wait<false>(x_full(s), (it / kRingX) & 1u, abort_flag, lane)) {
                    if (lane == 0) give_up(kWaitMmaOperands);
                    ok = false;
                    break;
                }
                if (lane == 0) {
                    if constexpr (G == 2) mbar_arrive_cluster(a_full(s), 0);
                    else mbar_arrive(a_full(s));
                }
                __syncwarp();
            }
        }
    } else if (warp == 1) {
        // ------------------------------ MMA issuer ------------------------------
        if (G == 1 || rank == 0) {  // uniform over the warp, as is everything below but the elected lane
            constexpr uint32_t kFormat = std::is_same<T, __half>::value ? 0u : 1u;  // of both operands
            const bool elected = elect_one();
            uint32_t it = 0, lt = 0;
            bool ok = true;
            for (int t = cluster; t < num_items && ok; t += clusters, ++lt) {
                const Item m = item(t);
                const uint32_t idesc = (1u << 4) | (kFormat << 7) | (kFormat << 10) | ((uint32_t)(m.width >> 3) << 17) | ((uint32_t)(128 * G >> 4) << 24);
                if (!warp_wait<false>(acc_empty, (lt & 1u) ^ 1u, abort_flag, lane)) {
                    if (lane == 0) give_up(kWaitMmaAcc);
                    break;
                }
                tc_fence_after_sync();
                for (int kb = kb0; kb < kb1; ++kb, ++it) {
                    const int s = it % kRingX;
                    if (!warp_wait<false>(a_full(s), (it / kRingX) & 1u, abort_flag, lane)) {
                        if (lane == 0) give_up(kWaitMmaOperands);
                        ok = false;
                        break;
                    }
                    tc_fence_after_sync();
                    const uint64_t dX = make_smem_desc(x0 + s * kBytesX);
                    const uint32_t ta = tmem_a0 + (uint32_t)(s * kStageCols);
                    if (elected) {
#pragma unroll
                        for (int h = 0; h < 2; ++h)
#pragma unroll
                            for (int k4 = 0; k4 < 4; ++k4)
                                umma_f16_ta<G>(tmem_base, ta + 32u * h + 8u * k4, dX + (uint64_t)(h * (kSubX >> 4) + 2 * k4), idesc,
                                               (h | k4) != 0 ? 1u : (kb != kb0 ? 1u : 0u));
                        commit_all<G>(ax_empty(s));
                    }
                    __syncwarp();
                }
                if (ok && elected) commit_all<G>(acc_full);
                __syncwarp();
            }
        }
    } else if (warp >= kConvWarp) {
        // ------------------------------ converters ------------------------------
        const int set = (warp - kConvWarp) >> 2, quarter = warp & 3;
        const int r = quarter * 32 + lane;              // row of this CTA's part of B = TMEM lane
        const uint32_t swz = (uint32_t)((r >> 1) & 3);  // 64-byte TMA swizzle: chunk ^= (row / 2) % 4
        const S *scales = static_cast<const S *>(p.scales);
        uint32_t it = 0;
        bool ok = true;
        for (int t = cluster; t < num_items && ok; t += clusters) {
            const Item m = item(t);
            const int c = m.col + (G == 2 ? rank * kRowsB : 0) + r;
            const bool live = c < p.n;
            const S *sp = scales + ((int64_t)m.e * p.n + (live ? c : 0)) * p.groups;
            float inv = 1.0f;
            if constexpr (std::is_same<T, __half>::value) inv = 1.0f / row_unit<T, S>(sp, p.groups);  // exact: a power of two
            // the scales of the four 32-element pieces of stage kb
            auto load_scales = [&](int kb, float(&v)[4]) {
                const int first = (kb * kStageK) >> p.group_shift;
                if (p.group_shift >= 7) {
                    v[0] = v[1] = v[2] = v[3] = load_float(sp + first);
                } else if (p.vec_scales) {
                    if (p.group_shift == 6) {
                        const S *a = sp + first;
                        if constexpr (sizeof(S) == 4) {
                            const uint2 u = ld_behind_wait(reinterpret_cast<const uint2 *>(a));
                            v[0] = v[1] = __uint_as_float(u.x), v[2] = v[3] = __uint_as_float(u.y);
                        } else {
                            const float2 u = unpack2(ld_behind_wait(reinterpret_cast<const uint32_t *>(a)), Tag<T>());
                            v[0] = v[1] = u.x, v[2] = v[3] = u.y;
                        }
                    } else {
                        const S *a = sp + first;
                        if constexpr (sizeof(S) == 4) {
                            const uint4 u = ld_behind_wait(reinterpret_cast<const uint4 *>(a));
                            v[0] = __uint_as_float(u.x), v[1] = __uint_as_float(u.y), v[2] = __uint_as_float(u.z), v[3] = __uint_as_float(u.w);
                        } else {
                            const uint2 u = ld_behind_wait(reinterpret_cast<const uint2 *>(a));
                            const float2 lo = unpack2(u.x, Tag<T>()), hi = unpack2(u.y, Tag<T>());
                            v[0] = lo.x, v[1] = lo.y, v[2] = hi.x, v[3] = hi.y;
                        }
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int g = (kb * kStageK + 32 * j) >> p.group_shift;
                        v[j] = g < p.groups ? load_float(sp + g) : 0.0f;
                    }
                }
            };
            // this set's stages of the item are those with (it + kb - kb0) % kSets == set
            const int first_kb = kb0 + (int)(((uint32_t)(set + kSets) - it % kSets) % kSets);
            float next[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            if (live && first_kb < kb1) load_scales(first_kb, next);
            for (int kb = first_kb; kb < kb1; kb += kSets) {
                const uint32_t i = it + (uint32_t)(kb - kb0);
                const int ws = i % kRingW, s = i % kRingX;
                float sc[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) sc[j] = next[j] * (inv * kCodeUnit<T>);
                if (live && kb + kSets < kb1) load_scales(kb + kSets, next);
                if (!warp_wait<false>(w_full(ws), (i / kRingW) & 1u, abort_flag, lane)) {
                    if (lane == 0) give_up(kWaitConvertPacked);
                    ok = false;
                    break;
                }
                uint4 w[4];
                const uint32_t src = w0 + ws * kBytesW + (uint32_t)r * 64;
#pragma unroll
                for (int j = 0; j < 4; ++j) w[j] = lds128(src + (((uint32_t)j ^ swz) << 4));
                if (!warp_wait<false>(ax_empty(s), ((i / kRingX) & 1u) ^ 1u, abort_flag, lane)) {
                    if (lane == 0) give_up(kWaitConvertSlot);
                    ok = false;
                    break;
                }
                tc_fence_after_sync();
                const uint32_t ta = tmem_a0 + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(s * kStageCols);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    uint32_t v[32];
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const uint4 u = w[2 * h + j];
                        const float f = sc[2 * h + j];
                        const uint32_t f2 = pack2(f, f, Tag<T>());
                        const uint32_t word[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
                        for (int o = 0; o < 4; ++o) {
                            uint32_t pair[4];
                            codes_in_order(word[o], pair, Tag<T>());
#pragma unroll
                            for (int i2 = 0; i2 < 4; ++i2) {
                                if constexpr (sizeof(S) == 4) {  // the product is rounded once, from fp32
                                    const float2 q = unpack2(pair[i2], Tag<T>());
                                    v[16 * j + 4 * o + i2] = pack2(q.x * f, q.y * f, Tag<T>());
                                } else {
                                    v[16 * j + 4 * o + i2] = fma2(pair[i2], f2, 0x80008000u, Tag<T>());
                                }
                            }
                        }
                    }
                    tmem_st_x32(ta + h * 32, v);
                }
                tmem_st_wait();
                tc_fence_before_sync();
                __syncwarp();
                if (lane == 0) {
                    // The codes' slot is handed back only here, where they have been used.  Handed back behind the loads, with the
                    // wait for the stage in between, it was filled again before they had returned: an arrive does not wait for
                    // loads on their way, and the next copy comes through another proxy.
                    mbar_arrive(w_empty(ws));
                    if constexpr (G == 2) mbar_arrive_cluster(a_full(s), 0);
                    else mbar_arrive(a_full(s));
                }
            }
            it += (uint32_t)(kb1 - kb0);
        }
    } else if (warp >= kEpiWarp) {
        // ------------------------------ epilogue ------------------------------
        const int quarter = warp & 3, half = (warp - kEpiWarp) >> 2;
        const int r = quarter * 32 + lane;
        const S *scales = static_cast<const S *>(p.scales);
        T *out = static_cast<T *>(p.out);
        uint32_t lt = 0;
        for (int t = cluster; t < num_items; t += clusters, ++lt) {
            const Item m = item(t);
            const int c = m.col + (G == 2 ? rank * kRowsB : 0) + r;  // column of out
            float unit = 1.0f;
            if constexpr (std::is_same<T, __half>::value) {
                if (c < p.n) unit = row_unit<T, S>(scales + ((int64_t)m.e * p.n + c) * p.groups, p.groups);
            }
            if (!warp_wait<false>(acc_full, lt & 1u, abort_flag, lane)) {
                if (lane == 0) give_up(kWaitEpilogueAcc);
                break;
            }
            tc_fence_after_sync();
            const uint32_t taddr = tmem_base + ((uint32_t)(quarter * 32) << 16);
            const uint32_t buf = epi0 + (uint32_t)((warp - kEpiWarp) * kEpiBytes);
            const int col0 = c - lane;  // the warp's first column
            const int chunks = m.width / 16;
            for (int ch = half; ch < chunks; ch += 2) {
                uint32_t v[16];
                tmem_ld_x16(taddr + (uint32_t)(ch * 16), v);
                tmem_ld_wait();
                if (G == 2 && ch + 2 >= chunks) {
                    // this warp's last columns are in registers: the accumulator may be overwritten once all warps say so
                    tc_fence_before_sync();
                    __syncwarp();
                    if (lane == 0) mbar_arrive_cluster(acc_empty, 0);
                }
                if (G == 1 && parts > 1) {
                    // partial tile -> shared memory [row of X][row of B] (the X ring, which is empty by now)
                    float *part = reinterpret_cast<float *>(smem_raw + (x0 - raw_u32));
#pragma unroll
                    for (int j = 0; j < 16; ++j) part[(ch * 16 + j) * kRowsB + r] = __uint_as_float(v[j]);
                    continue;
                }
                // through the warp's buffer, so that a store writes 64 contiguous bytes of eight rows.  (Straight from the
                // registers, two bytes a lane and one row at a time behind bounds checks, the epilogue took 11,800 clocks of a
                // tile whose MMAs take 32,700.)
#pragma unroll
                for (int j = 0; j < 16; j += 2) {
                    const uint32_t two = pack2(__uint_as_float(v[j]) * unit, __uint_as_float(v[j + 1]) * unit, Tag<T>());
                    asm volatile("st.shared.u16 [%0], %1;" ::"r"(buf + j * 64 + lane * 2), "h"((unsigned short)two) : "memory");
                    asm volatile("st.shared.u16 [%0], %1;" ::"r"(buf + j * 64 + 64 + lane * 2), "h"((unsigned short)(two >> 16)) : "memory");
                }
                __syncwarp();
                const int row0 = ch * 16, sub = lane >> 2, piece = (lane & 3) * 8;
                T *dst = out + (int64_t)(m.row + row0 + sub) * p.ldo + col0 + piece;
                const uint4 a0 = lds128(buf + lane * 16), a1 = lds128(buf + 512 + lane * 16);
                if (p.vec_out && row0 + 16 <= m.count && col0 + 32 <= p.n) {
                    *reinterpret_cast<uint4 *>(dst) = a0;
                    *reinterpret_cast<uint4 *>(dst + 8 * p.ldo) = a1;
                } else {
#pragma unroll 1
                    for (int o = 0; o < 2; ++o, dst += 8 * p.ldo) {
                        if (row0 + sub + 8 * o >= m.count) continue;
                        const uint4 a = o ? a1 : a0;
                        const uint32_t word[4] = {a.x, a.y, a.z, a.w};
                        unsigned short *d16 = reinterpret_cast<unsigned short *>(dst);
#pragma unroll
                        for (int j = 0; j < 8; ++j)
                            if (col0 + piece + j < p.n) d16[j] = (unsigned short)(word[j >> 1] >> (16 * (j & 1)));
                    }
                }
                __syncwarp();  // the buffer is rewritten next
            }
            // a warp whose half has no columns hands the accumulator back as well
            if (G == 2 && half >= chunks) {
                tc_fence_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive_cluster(acc_empty, 0);
            }
            if (G == 1 && parts > 1 && half == 0) unit_of_row[r] = unit;
        }
    }

    // ------------------------------ sum of the K parts ------------------------------
    if constexpr (G == 1) {
        if (parts > 1) {
            tc_fence_before_sync();
            __syncthreads();
            cluster_arrive();
            cluster_wait();
            if (cluster < num_items) {
                // this CTA finishes every parts-th row of the tile; a thread two neighbouring columns of a row at a time
                const Item m = item(cluster);
                T *out = static_cast<T *>(p.out);
                const int todo = (m.count - rank + parts - 1) / parts;
                for (int i = threadIdx.x; i < todo * (kRowsB / 2); i += kNumThreads) {
                    const int row = rank + (i / (kRowsB / 2)) * parts, pos = (i % (kRowsB / 2)) * 2, col = m.col + pos;
                    if (col >= p.n) continue;
                    float2 v[kMaxParts];
#pragma unroll
                    for (int o = 0; o < kMaxParts; ++o)
                        if (o < parts) v[o] = lds_cluster_f2(mapa_cluster(x0 + (uint32_t)(row * kRowsB + pos) * 4u, (uint32_t)o));
                    float a = 0.0f, b = 0.0f;
#pragma unroll
                    for (int o = 0; o < kMaxParts; ++o)
                        if (o < parts) a += v[o].x, b += v[o].y;
                    const uint32_t two = pack2(a * unit_of_row[pos], b * unit_of_row[pos + 1], Tag<T>());
                    unsigned short *dst = reinterpret_cast<unsigned short *>(out + (int64_t)(m.row + row) * p.ldo + col);
                    if (p.vec_out && col + 1 < p.n) {
                        *reinterpret_cast<uint32_t *>(dst) = two;
                    } else {
                        dst[0] = (unsigned short)two;
                        if (col + 1 < p.n) dst[1] = (unsigned short)(two >> 16);
                    }
                }
            }
        }
    }

    // ------------------------------ teardown ------------------------------
    tc_fence_before_sync();
    __syncthreads();
    cluster_arrive();
    cluster_wait();
    if (warp == 1) {
        tc_fence_after_sync();
        tmem_dealloc<G>(tmem_base, kTmemCols);
    }
}

int make_x_tmap(CUtensorMap *map, const W4Args &a, int box_rows)
{
    EncodeTiledFn fn = encode_fn();
    if (!fn) return record_cuda_error(cudaErrorUnknown, "cuTensorMapEncodeTiled entry point");
    cuuint64_t dims[2] = {(cuuint64_t)a.k, (cuuint64_t)a.rows};
    cuuint64_t strides[1] = {(cuuint64_t)a.ldx * 2};
    cuuint32_t box[2] = {64, (cuuint32_t)box_rows};
    cuuint32_t estr[2] = {1, 1};
    CUresult r = fn(map, a.type == QM_TYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void *>(a.X), dims,
                    strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                    CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? QM_OK : record_cuda_error(cudaErrorInvalidValue, "cuTensorMapEncodeTiled(X)");
}

struct TcPlanW4 {
    int pair;   // 1: the PAIR form
    int tile;   // rows of X per tile
    int parts;  // SPLIT form: parts of K
};

template <int G, typename T, typename S>
int configure(int device)
{
    static std::atomic<bool> configured[64];  // set once per device; a repeated cudaFuncSetAttribute is harmless
    if (configured[device & 63].load(std::memory_order_acquire)) return QM_OK;
    cudaError_t e = cudaFuncSetAttribute(w4_tc_kernel<G, T, S>, cudaFuncAttributeMaxDynamicSharedMemorySize, 232448);
    if (e != cudaSuccess) return record_cuda_error(e, "cudaFuncSetAttribute(w4_tc_kernel)");
    configured[device & 63].store(true, std::memory_order_release);
    return QM_OK;
}

// Clusters of `size` CTAs that the device holds at once, asked once per device and size (after configure).
template <int G, typename T, typename S>
int max_clusters(int device, int size)
{
    static std::atomic<int> known[64][9];
    std::atomic<int> &slot = known[device & 63][size];
    int n = slot.load(std::memory_order_relaxed);
    if (n) return n;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)size * 64, 1, 1);
    cfg.blockDim = dim3(kNumThreads, 1, 1);
    cfg.dynamicSmemBytes = kSmemFixed + 16;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)size;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cudaOccupancyMaxActiveClusters(&n, w4_tc_kernel<G, T, S>, &cfg) != cudaSuccess || n < 1) {
        (void)cudaGetLastError();
        return 1;  // right, if slow, and asked again next time
    }
    slot.store(n, std::memory_order_relaxed);
    return n;
}

template <int G, typename T, typename S>
int tc_launch_variant(const W4Args &a, const TcPlanW4 &plan, const DeviceCtx &ctx)
{
    auto kernel = w4_tc_kernel<G, T, S>;
    const size_t smem = kSmemFixed + (size_t)(a.experts + 1) * 8;
    CUtensorMap tmW, tmX, tmX128;
    int st = make_packed_tmap(&tmW, a.B, a.experts * a.n, a.k / 2, kRowsB, CU_TENSOR_MAP_SWIZZLE_64B);
    if (st == QM_OK) st = make_x_tmap(&tmX, a, kBoxRows);
    if (st == QM_OK) st = make_x_tmap(&tmX128, a, kRowsX);
    if (st != QM_OK) return st;
    TcParams p;
    p.scales = a.scales, p.offsets = a.offsets, p.out = a.out, p.ldo = a.ldo;
    p.rows = a.rows, p.n = a.n, p.k = a.k, p.experts = a.experts;
    p.group_shift = a.group == 32 ? 5 : a.group == 64 ? 6 : a.group == 128 ? 7 : 8;
    p.groups = (a.k + a.group - 1) / a.group;
    p.tile = plan.tile;
    const int gps = a.group >= 128 ? 1 : 128 / a.group;
    p.vec_scales = p.groups % gps == 0 && (reinterpret_cast<uintptr_t>(a.scales) & (gps * sizeof(S) - 1)) == 0;
    p.vec_out = (reinterpret_cast<uintptr_t>(a.out) & 15u) == 0 && (a.ldo & 7) == 0;
    p.status = ctx.status;

    const int64_t tilesP = (a.n + kRowsB * G - 1) / (kRowsB * G);
    // with experts: at most one tile more than whole ones per expert that can have rows
    const int64_t tilesQ = a.offsets ? a.rows / plan.tile + (a.experts < a.rows ? a.experts : a.rows) : (a.rows + plan.tile - 1) / plan.tile;
    if (tilesP * tilesQ > 0x7FFFFFFF / 8) return QM_ERR_SHAPE;
    const int size = G == 2 ? 2 : plan.parts;
    int64_t clusters = tilesP * tilesQ;
    if (G == 2) {
        const int units = max_clusters<G, T, S>(ctx.device, 2);
        if (clusters > units) clusters = units;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(clusters * size), 1, 1);
    cfg.blockDim = dim3(kNumThreads, 1, 1);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = a.stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)size;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    static const bool allow_pdl = !std::getenv("QM_NO_PDL");
    cfg.numAttrs = allow_pdl ? 2 : 1;
    cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, tmW, tmX, tmX128, p);
    return e == cudaSuccess ? QM_OK : record_cuda_error(e, "w4_tc_kernel launch");
}

// How the product is cut.
TcPlanW4 tc_plan(const W4Args &a, const DeviceCtx &ctx)
{
    TcPlanW4 plan = {1, 256, 1};
    const int num_kb = (a.k + kStageK - 1) / kStageK;
    const int pairs = ctx.num_sms / 2;
    if (a.offsets) {
        // Tiles of 256 rows at any segment length: an item's MMAs are as wide as its rows anyway, and a segment cut in two converts
        // its weights twice.  (n = k = 4096, 32 experts: 4,096 rows 122 us, with tiles of 128 rows 155; 512 rows 95.4 us, with tiles
        // of 64 96.0.)
        return plan;
    }
    const int64_t pair_tiles = (int64_t)((a.n + 255) / 256) * ((a.rows + 255) / 256);
    const int64_t single = (int64_t)((a.n + 127) / 128) * ((a.rows + 127) / 128);
    if (single <= ctx.num_sms && pair_tiles < ctx.num_sms / 4) {
        plan.pair = 0;
        plan.tile = 128;
        int parts = (int)(ctx.num_sms / single);
        if (parts > kMaxParts) parts = kMaxParts;
        if (parts > num_kb) parts = num_kb;
        plan.parts = parts < 1 ? 1 : parts;
        return plan;
    }
    // PAIR form: tiles go round over the pairs, and a tile costs its width plus the epilogue and the refill of the pipeline, which
    // take about as long as 12 columns of an average main loop.  The width with the fewest rounds' cost: 2048 x 12288 has 384 tiles
    // of 256 rows, six rounds of 74 pairs, but 432 of 240, six rounds of 0.94 of the length.  (Below 192 the converters and
    // the loads of B no longer hide behind the MMAs.)
    double best = 0.0;
    for (int width = 256; width >= 192; width -= 16) {
        const int64_t tiles = (int64_t)((a.n + 255) / 256) * ((a.rows + width - 1) / width);
        const double cost = (double)((tiles + pairs - 1) / pairs) * (width + 12);
        if (best == 0.0 || cost < best) best = cost, plan.tile = width;
    }
    return plan;
}

}  // namespace

int w4_tc_launch(const W4Args &a, const DeviceCtx &ctx)
{
    const TcPlanW4 base = tc_plan(a, ctx);
    auto by_type = [&](auto t) {
        using T = typename decltype(t)::type;
        return with_same_or_float<T>(a.scale_type, [&](auto u) {
            using S = typename decltype(u)::type;
            int st = base.pair ? configure<2, T, S>(ctx.device) : configure<1, T, S>(ctx.device);
            if (st != QM_OK) return st;
            if (base.pair) return tc_launch_variant<2, T, S>(a, base, ctx);
            // clusters of the wanted size that the device cannot all hold at once would run in turns
            TcPlanW4 plan = base;
            const int64_t single = (int64_t)((a.n + 127) / 128) * ((a.rows + plan.tile - 1) / plan.tile);
            while (plan.parts > 1 && single > max_clusters<1, T, S>(ctx.device, plan.parts)) --plan.parts;
            return tc_launch_variant<1, T, S>(a, plan, ctx);
        });
    };
    return a.type == QM_TYPE_F16 ? by_type(Tag<__half>()) : by_type(Tag<__nv_bfloat16>());
}

}  // namespace qm
