// 4-bit weights with group scales, few rows of X: weight streaming.
//
// out[r][c] = sum over groups g of scale[c][g] * sum over i in g of x[r][i] q[c][i].  With a few rows of X the product reads every
// weight once and should be bound by memory; what costs is making operands of the codes.  As 16-bit floats they take nine
// instructions per eight codes, and a kernel built that way stood at half of the HBM rate with its issue slots full.  As int8 (times
// 16, nibble in the high half of the byte) they take three.  So X becomes whole numbers instead, once per launch and CTA:
//
//   In every stretch of K that shares a weight scale (at most 128 elements) the row of X is divided by a power of two above its
//   largest value and rounded to 22 bits, v = d1 2^16 + d2 2^8 + d3 with signed bytes d.  The three dot products of a stretch
//   are exact in int32 (mma.sync.m16n8k32), and scale * (d1 . q, d2 . q, d3 . q) is added in fp32, one rounding per stretch, as
//   an fp32 sum of products would have one per product.  The only loss is that of elements below 2^-13 of their stretch's largest
//   (bf16; 2^-10 for fp16): their last bits are rounded at 2^-22 of it, four times fp32's own last place.
//   That is nothing beside the other elements' products, but a weight of zero can take the largest one out of a sum.  So where more
//   than a quarter of a stretch's elements lose digits (an element hundreds, fp16, or thousands of times its neighbours), or one is an
//   infinity or a NaN, the row's outputs are computed from their definition instead, element by element: 1 x 4096 x 4096 14 us,
//   8 x 4096 x 4096 58 us with all rows so.  Finding out costs a vote per 256 elements of X, and a count where one of them is small
//   enough to lose digits: 8 x 4096 x 4096 of normal numbers 7.8 -> 8.3 us (fp16, whose digits reach further down, 8.9; 10.2 where every
//   piece is counted).
//
//  * A CTA (16 warps) takes blocks of 32 rows of B per warp group; WK of its warps split K between them in steps of 128 elements.
//    Lane (g, q) = (lane / 4, lane % 4) loads 16 bytes, 32 codes, of row g of each 8-row group straight into registers; kDepth steps
//    are on the way per warp (64 KB per SM; a third costs registers that are not there), across the end of a block, so the stream
//    does not stop there.  (TMA rings in their place, one per warp or one per CTA with a loading warp, were slower: a small box
//    costs its thread about 400 clocks, and 1 x 4096 x 4096 has time for four.)
//  * A word's even and odd elements are the two halves of an operand fragment; which K an instruction's columns stand for is free
//    as long as X is laid out alike.  But an instruction adds up over the four lanes of a row, so these must hold codes of
//    one group: with groups of 128 and more every lane uses its own 32 codes; for 64 and 32 the lanes of a row trade words.
//  * With many blocks of B fewer warps split K (WK) and there are more warp groups, which share the rows of X and nothing else: a
//    group meets at a named barrier of its own at the end of its 32 rows, so that one adds up while another multiplies.
//  * Rows of X sit in the eight columns of an instruction.  WIDE (3 to 8 rows): a column per row, an instruction per byte d.
//    Otherwise (1 or 2 rows) the three bytes of both rows take six columns of one instruction.
//  * The warps' partial tiles meet in shared memory (two buffers, one barrier a block) and are added in a fixed order.
//
// Measured (groups of 128, bf16): 1 x 57344 x 8192 53.4 us = 4.5 TB/s, 8 rows of it 90 us; 1 x 4096 x 4096 4.9 us, of which a launch
// in a dependent chain is 2.4; 128 rows over 32 experts of 4096 x 4096 73-77 us = 3.6-3.8 TB/s, DRAM at 45 % and the SM at 43 % of
// their peaks.  Groups of 32 cost 1.2 us more at 1 x 4096 x 4096: the lanes trade words.
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
constexpr int kDepth = 2;                          // steps on the way per warp
constexpr int kStep = 128;                         // elements of K per step
constexpr int kRG = 4, kTiles = 2, kRows = 8 * kRG;  // 8-row groups, 16-row tiles and rows of B per warp
constexpr int kRedFloats = kWarps * kTiles * 128;  // one of two buffers
constexpr int kMaxSmem = 232448;  // eight rows of 8192 elements just fit
constexpr int kNarrowRows = 2, kWideRows = 8;

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
    int warps_k;     // warps that split K; the others take further rows of B
    int vec_scales;  // a step's scales can be loaded as one vector
};

// d (+)= a b: 16 rows of B x 32 elements of K x 8 columns
template <bool FRESH>
__device__ __forceinline__ void mma16832(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1)
{
    // a fresh sum starts at the bits of 1.5 x 2^23, so that what comes out reads as that number plus the sum (below 2^22)
    if constexpr (FRESH)
        asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
            : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "r"(0x4B400000));
    else
        asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ float sum_value(int d) { return __fadd_rn(__int_as_float(d), -12582912.0f); }

// The GPS scales of one step as they lie in memory
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
        if constexpr (std::is_same<S, __half>::value) return __half2float(__ushort_as_half((unsigned short)((j & 1) ? v >> 16 : v)));
        else return __uint_as_float((j & 1) ? v & 0xFFFF0000u : v << 16);
    }
}

// Barrier of `threads` threads; true for all of them if `any` is for one.
__device__ __forceinline__ bool barrier_or(int id, int threads, bool any)
{
    uint32_t r;
    asm volatile(
        "{\n"
        " .reg .pred p, q;\n"
        " setp.ne.u32 p, %3, 0;\n"
        " barrier.cta.red.or.pred q, %1, %2, p;\n"
        " selp.u32 %0, 1, 0, q;\n"
        "}\n"
        : "=r"(r)
        : "r"(id), "r"(threads), "r"((uint32_t)any)
        : "memory");
    return r != 0;
}

// Element j of eight 16-bit floats
template <typename T>
__device__ __forceinline__ float element(const uint4 &v, int j)
{
    const uint32_t w = j < 2 ? v.x : j < 4 ? v.y : j < 6 ? v.z : v.w;
    if constexpr (std::is_same<T, __half>::value) return __half2float(__ushort_as_half((unsigned short)((j & 1) ? w >> 16 : w)));
    else return __uint_as_float((j & 1) ? w & 0xFFFF0000u : w << 16);
}

// The eight codes of a word as fp32: nibble n is (n ^ 8) - 8, and n ^ 8 in the last bits of 2^23 reads as 2^23 + (n ^ 8).
__device__ __forceinline__ float code_as_float(uint32_t w, int j) { return __fadd_rn(__uint_as_float(and_xor(w >> (4 * j), 0xFu, 0x4B000008u)), -8388616.0f); }

// A thread's share of one output from its definition: pieces `part`, `part` + `parts`, ... of 32 elements of K (X and B are such that these
// are aligned, and no group ends inside one).  It takes few registers: what the caller has on the way stays in its own.
template <typename T, typename S>
__device__ __noinline__ float plain_part(const T *x, const uint8_t *b, const S *s, int k, int group_shift, int part, int parts)
{
    float sum = 0.0f;
    for (int i = part * 32; i < k; i += parts * 32) {
        uint4 w = ptx::ld_behind_wait(reinterpret_cast<const uint4 *>(b + i / 2));
        const float scale = load_float(s + (i >> group_shift));
        float even = 0.0f, odd = 0.0f;
#pragma unroll 1
        for (int o = 0; o < 4; ++o) {
            const uint4 e = ptx::ld_behind_wait(reinterpret_cast<const uint4 *>(x + i) + o);
            const uint32_t codes = w.x;
            w.x = w.y, w.y = w.z, w.z = w.w;
#pragma unroll
            for (int j = 0; j < 8; j += 2) {
                even = fmaf(element<T>(e, j), code_as_float(codes, j), even);
                odd = fmaf(element<T>(e, j + 1), code_as_float(codes, j + 1), odd);
            }
        }
        sum = fmaf(scale, even + odd, sum);
    }
    return sum;
}

// The largest magnitudes of the even and the odd ones of eight elements, as the bits of T: these order like numbers.
__device__ __forceinline__ uint32_t magnitudes(const uint4 &v)
{
    return __vmaxu2(__vmaxu2(v.x & 0x7FFF7FFFu, v.y & 0x7FFF7FFFu), __vmaxu2(v.z & 0x7FFF7FFFu, v.w & 0x7FFF7FFFu));
}

// How a stretch is scaled, from the bits of its largest magnitude.
struct Stretch {
    uint32_t e, ec;  // biased exponent: the largest is below 2^(e - 126); as it is used (below 2^-101 the bits run out early)
    __device__ __forceinline__ float up() const { return __uint_as_float((274u - ec) << 23); }  // 2^21 over the power of two above the largest
    __device__ __forceinline__ float down() const { return __uint_as_float((ec - 20u) << 23); }  // one over that
};
template <typename T>
__device__ __forceinline__ Stretch stretch_of(uint32_t m)
{
    float top;
    if constexpr (std::is_same<T, __half>::value) top = __half2float(__ushort_as_half((unsigned short)m));
    else top = __uint_as_float(m << 16);
    Stretch s;
    s.e = __float_as_uint(top) >> 23;
    s.ec = min(max(s.e, 25u), 254u);
    return s;
}

// One less than the smallest magnitude of eight elements that is not zero, as the bits of T (0xFFFF: all are zero): with the sign bit
// set and one taken away a zero is the largest signed number, the others keep their order.
__device__ __forceinline__ uint32_t smallest_less_one(const uint4 &v)
{
    auto key = [](uint32_t w) { return (w | 0x80008000u) - 0x00010001u; };
    const uint32_t k = __vmins2(__vmins2(key(v.x), key(v.y)), __vmins2(key(v.z), key(v.w))) ^ 0x80008000u;
    return min(k & 0xFFFFu, k >> 16);
}

// Whether the stretch that LANES neighbouring lanes have eight elements of each cannot be written as bytes: one is not finite, or more
// than a quarter of those that are not zero lose digits.  The whole warp.  These are counted only where some lane of it has one that
// is so much smaller than its stretch's largest (m) that it can lose some: T's digits end where the 21 bits below m's power of two do.
template <typename T, int LANES>
__device__ __forceinline__ bool loses_digits(const uint4 &v, uint32_t m, const Stretch &s)
{
    constexpr bool kHalf = std::is_same<T, __half>::value;
    constexpr int kMantissa = kHalf ? 10 : 7, kExponent = kHalf ? 0x7C00 : 0x7F80;
    bool bad = s.e == 255u;
    const int exact_from = s.e < 25u ? kExponent : (int)(m & kExponent) - ((20 - kMantissa) << kMantissa);
    if (__any_sync(0xFFFFFFFFu, (int)smallest_less_one(v) + 1 < exact_from)) {
        int count = 0;  // elements that are not zero, and in the upper half those that lose digits
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float x = element<T>(v, j);
            count += (x != 0.0f ? 1 : 0) + (__fmul_rn(rintf(x * s.up()), s.down()) != x ? 1 << 16 : 0);
        }
#pragma unroll
        for (int d = 1; d < LANES; d <<= 1) count += __shfl_xor_sync(0xFFFFFFFFu, count, d);
        bad |= 4 * (count >> 16) > (count & 0xFFFF);
    }
    return bad;
}

// GPS = groups per step of 128 elements (4, 2 or 1 for groups of 32, 64, and 128 or more).
template <typename T, typename S, int GPS, bool WIDE>
__global__ void __launch_bounds__(kThreads, 1) w4_rows_kernel(const RowsParams p)
{
    constexpr int TT = WIDE ? 3 : 1;               // instructions per 16 rows of B and 32 elements of K
    constexpr int kTile = WIDE ? kWideRows : kNarrowRows;  // rows of X per unit
    constexpr int kColumns = 8;
    constexpr int kPlace = 2 * TT * 32;            // 16-byte pieces of X per step
    extern __shared__ uint4 smem_u4[];
    const T *X = static_cast<const T *>(p.X);
    const S *scales = static_cast<const S *>(p.scales);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
    const int groups_of_rows = kWarps / p.warps_k;
    const int wk = warp % p.warps_k, wr = warp / p.warps_k;
    const int block_rows = kRows * groups_of_rows;
    const int blocks = (p.n + block_rows - 1) / block_rows;
    const int steps = (p.k + kStep - 1) / kStep, chunks = p.k / 32;
    const uint32_t row_bytes = (uint32_t)p.k / 2;
    // a warp has `mine` steps, WK apart (one without a step works on a place of zeros); X has a place for each, for all warp groups
    const int mine = max(1, (steps - wk + p.warps_k - 1) / p.warps_k);
    const int places = max(steps, p.warps_k);

    // X [place][pair of sets][instruction][lane] 16 bytes, X's units [place][group][column], partial tiles, rows of X that
    // bytes do not hold, segments
    uint4 *xs = smem_u4;
    float *unit = reinterpret_cast<float *>(smem_u4 + (size_t)places * kPlace);
    float *red = unit + (size_t)places * GPS * kColumns;
    unsigned *odd_rows = reinterpret_cast<unsigned *>(red + 2 * kRedFloats);  // [pair's parity][kWarps]
    int *seg = reinterpret_cast<int *>(odd_rows + 2 * kWarps), *tiles = seg + p.experts + 1;

    // CTA c takes the units from first_unit(c) up to first_unit(c + 1); the host has seen to it that their number fits an int
    auto first_unit = [&](int units, unsigned c) {
        const unsigned each = (unsigned)units / gridDim.x, more = (unsigned)units % gridDim.x;
        return c * each + min(c, more);
    };
    const int row_tiles = (p.rows + kTile - 1) / kTile;
    if (!p.offsets && (int)threadIdx.x < block_rows) {
        // L2 prefetch of this CTA's first block: returns no data, changes nothing the program can observe
        const int row = (int)(first_unit(row_tiles * blocks, blockIdx.x) % blocks) * block_rows + (int)threadIdx.x;
        if (row < p.n) asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(p.B + (int64_t)row * row_bytes), "r"(row_bytes) : "memory");
    }
    ptx::grid_dependency_wait();  // nothing above read or wrote global memory
    ptx::grid_launch_dependents();

    int pairs = row_tiles;  // (expert, tile of rows)
    if (p.offsets) {
        if (warp == 0) scan_segments(p.offsets, p.experts, p.rows, kTile, seg, tiles, lane);
        __syncthreads();
        pairs = tiles[p.experts];
    }
    const int u_begin = (int)first_unit(pairs * blocks, blockIdx.x), u_end = (int)first_unit(pairs * blocks, blockIdx.x + 1);
    if (u_begin >= u_end) return;
    auto expert_of = [&](int pair) { return p.offsets ? expert_of_tile(tiles, p.experts, pair) : 0; };

    // Two walks over (unit, step): loads, and products kDepth steps behind.
    struct Walk {
        int left, pair, block, step, expert;
    };
    auto advance = [&](Walk &w) {
        if (++w.step < mine) return;
        w.step = 0;
        --w.left;
        if (++w.block < blocks) return;
        w.block = 0;
        ++w.pair;
        if (p.offsets && w.left > 0) w.expert = expert_of_tile(tiles, p.experts, w.pair);
    };
    Walk cw;
    cw.left = u_end - u_begin, cw.pair = u_begin / blocks, cw.block = u_begin - cw.pair * blocks, cw.step = 0;
    cw.expert = expert_of(cw.pair);
    Walk lw = cw;

    struct Step {
        uint4 w[kRG];
        RawScales<S, GPS> s;
    };
    const uint8_t *lb = nullptr;  // the expert's matrix
    uint32_t lrow[kRG];           // this lane's rows in it (rows beyond n repeat the last one: nobody reads their sums)
    const S *sp = nullptr;        // lane (g, q) fetches the scales of row q * 8 + g and hands them to the lanes that need them
    auto load = [&](Step &b) {
        if (lw.left <= 0) return;
        if (lw.step == 0) {
            const int first = lw.block * block_rows + wr * kRows;
            lb = p.B + (int64_t)lw.expert * p.n * row_bytes;
#pragma unroll
            for (int r = 0; r < kRG; ++r) lrow[r] = (uint32_t)min(first + 8 * r + g, p.n - 1) * row_bytes;
            sp = scales + ((int64_t)lw.expert * p.n + min(first + q * 8 + g, p.n - 1)) * p.groups;
        }
        const int t = wk + lw.step * p.warps_k;
        const uint8_t *src = lb + (4 * t + q < chunks ? t * 64 + q * 16 : 0);  // beyond K the codes meet zeros
#pragma unroll
        for (int r = 0; r < kRG; ++r) b.w[r] = ptx::ldcs_behind_wait(reinterpret_cast<const uint4 *>(src + lrow[r]));
        using Raw = RawScales<S, GPS>;
        const int first = GPS > 1 ? t * GPS : (t * kStep) >> p.group_shift;
        if (t >= steps) {
#pragma unroll
            for (int j = 0; j < Raw::kWords; ++j) b.s.w[j] = 0;
        } else if constexpr (GPS == 1) {
            if constexpr (sizeof(S) == 4) b.s.w[0] = __float_as_uint(load_float(sp + first));
            else b.s.w[0] = ptx::ld_behind_wait(reinterpret_cast<const unsigned short *>(sp + first));
        } else if (p.vec_scales) {
            if constexpr (Raw::kWords == 1) b.s.w[0] = ptx::ld_behind_wait(reinterpret_cast<const uint32_t *>(sp + first));
            else if constexpr (Raw::kWords == 2) {
                const uint2 v = ptx::ld_behind_wait(reinterpret_cast<const uint2 *>(sp + first));
                b.s.w[0] = v.x, b.s.w[1] = v.y;
            } else {
                const uint4 v = ptx::ld_behind_wait(reinterpret_cast<const uint4 *>(sp + first));
                b.s.w[0] = v.x, b.s.w[1] = v.y, b.s.w[2] = v.z, b.s.w[3] = v.w;
            }
        } else {
#pragma unroll
            for (int j = 0; j < Raw::kWords; ++j) b.s.w[j] = 0;
#pragma unroll
            for (int j = 0; j < GPS; ++j) {
                if (first + j >= p.groups) continue;
                if constexpr (sizeof(S) == 4) b.s.w[j] = __float_as_uint(load_float(sp + first + j));
                else b.s.w[j >> 1] |= (uint32_t)ptx::ld_behind_wait(reinterpret_cast<const unsigned short *>(sp + first + j)) << (16 * (j & 1));
            }
        }
        advance(lw);
    };
    Step buf[kDepth];
#pragma unroll
    for (int d = 0; d < kDepth; ++d) load(buf[d]);

    unsigned bad_rows = 0;  // rows of X that bytes do not hold, as far as this warp has seen
    bool staged_bad = false, cpair_seen = false;
    int parity = 0, pair_parity = 0, first_row = 0, tokens = 0, cpair = -1;
    float acc[kTiles][4];

    // This warp's share of the rows of X as bytes d1, d2, d3.  A lane takes eight elements of a row (side = which row of a pair,
    // word = which of the step's sixteen eights): the word of codes they will meet is lane (g, q)'s in set s.
    auto stage_x = [&]() {
        const int side = lane >> 4, word = lane & 15;
        const int s = GPS == 1 ? word & 3 : GPS == 2 ? 2 * (word >> 3) + (word & 1) : word >> 2;
        const int qq = GPS == 1 ? word >> 2 : GPS == 2 ? 2 * ((word >> 1) & 1) + ((word >> 2) & 1) : word & 3;
        if (groups_of_rows > 1 && cpair_seen) __syncthreads();  // another group may still read the rows before
        cpair_seen = true;
        unsigned bad = 0;
        uint4 v[kTile / 2], ahead[kTile / 2];
        auto fetch = [&](int i) {
            const int at = (wk + i * p.warps_k) * kStep + word * 8;
#pragma unroll
            for (int r = 0; r < kTile / 2; ++r) {
                ahead[r] = make_uint4(0, 0, 0, 0);
                if (i < mine && 2 * r + side < tokens && at < p.k)
                    ahead[r] = ptx::ld_behind_wait(reinterpret_cast<const uint4 *>(X + (int64_t)(first_row + 2 * r + side) * p.ldx + at));
            }
        };
        fetch(wr);
        for (int i = wr; i < mine; i += groups_of_rows) {  // the warp groups share their common steps
            const int t = wk + i * p.warps_k;
#pragma unroll
            for (int r = 0; r < kTile / 2; ++r) v[r] = ahead[r];
            fetch(i + groups_of_rows);
#pragma unroll
            for (int r = 0; r < kTile / 2; ++r) {
                const int row = 2 * r + side;
                if (2 * r >= tokens) continue;  // (columns without a row hold anything: nobody reads their sums)
                uint32_t m = magnitudes(v[r]);
#pragma unroll
                for (int d = 1; d < 16 / GPS; d <<= 1) m = __vmaxu2(m, __shfl_xor_sync(0xFFFFFFFFu, m, d));
                m = max(m & 0xFFFFu, m >> 16);
                const Stretch st = stretch_of<T>(m);
                if (loses_digits<T, 16 / GPS>(v[r], m, st)) bad |= 1u << row;
                uint32_t z[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    // 1.5 x 2^23 rounds to a whole number; 128 more in the two low digits makes their bytes unsigned
                    z[j] = __float_as_uint(fmaf(element<T>(v[r], j), st.up(), 12582912.0f + 32896.0f));
                }
                // even elements 0, 2, 4, 6 and odd elements 1, 3, 5, 7: their bytes 0 (d3 + 128), 1 (d2 + 128) and 2 (d1 + 64)
                uint32_t d[3][2];
#pragma unroll
                for (int o = 0; o < 2; ++o) {
                    const uint32_t a = __byte_perm(z[o], z[2 + o], 0x5140), b = __byte_perm(z[4 + o], z[6 + o], 0x5140);
                    d[2][o] = __byte_perm(a, b, 0x5410) ^ 0x80808080u;
                    d[1][o] = __byte_perm(a, b, 0x7632) ^ 0x80808080u;
                    const uint32_t c = __byte_perm(__byte_perm(z[o], z[2 + o], 0x0062), __byte_perm(z[4 + o], z[6 + o], 0x0062), 0x5410);
                    d[0][o] = ((c | 0x80808080u) - 0x40404040u) ^ 0x80808080u;
                }
                const float f = __uint_as_float((st.ec - 24u) << 23);  // one over up, and over the codes' factor of 16
                const bool lead = (word & (16 / GPS - 1)) == 0;
                const int j = GPS == 1 ? 0 : GPS == 2 ? word >> 3 : word >> 2;
                uint2 *dst = reinterpret_cast<uint2 *>(xs + t * kPlace + (s >> 1) * TT * 32) + (s & 1);
                float *uf = unit + (t * GPS + j) * kColumns;
                if constexpr (WIDE) {
#pragma unroll
                    for (int b = 0; b < 3; ++b) dst[2 * (b * 32 + row * 4 + qq)] = make_uint2(d[b][0], d[b][1]);
                    if (lead) uf[row] = f;
                } else {
#pragma unroll
                    for (int b = 0; b < 3; ++b) dst[2 * ((2 * b + row) * 4 + qq)] = make_uint2(d[b][0], d[b][1]);
                    if (lead) uf[row] = f * 65536.0f, uf[2 + row] = f * 256.0f, uf[4 + row] = f, uf[6 + row] = 0.0f;
                }
            }
        }
        bad_rows = __reduce_or_sync(0xFFFFFFFFu, bad);
        pair_parity ^= 1;
        if (lane == 0) odd_rows[pair_parity * kWarps + warp] = bad_rows;
        if (groups_of_rows > 1) staged_bad = __syncthreads_or(bad_rows != 0);
        else __syncwarp();
    };

    auto product = [&](Step &b) {
        if constexpr (GPS > 1) {
            // lanes q and q ^ 2 trade: afterwards sets 0, 1 hold codes of the first 64 elements and sets 2, 3 of the last
#pragma unroll
            for (int r = 0; r < kRG; ++r) {
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
        const int t = wk + cw.step * p.warps_k;
        const uint4 *xp = xs + t * kPlace + lane;
        const float *uf = unit + t * GPS * kColumns + 2 * q;
        int sum[kTiles][TT][4];
        uint4 xv[TT];
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            if (s % 2 == 0) {
#pragma unroll
                for (int i = 0; i < TT; ++i) xv[i] = xp[((s / 2) * TT + i) * 32];
            }
            const bool fresh = s % (4 / GPS) == 0;  // a group begins
#pragma unroll
            for (int tl = 0; tl < kTiles; ++tl) {
                const uint4 &u0 = b.w[2 * tl], &u1 = b.w[2 * tl + 1];
                const uint32_t w0 = s == 0 ? u0.x : s == 1 ? u0.y : s == 2 ? u0.z : u0.w, w1 = s == 0 ? u1.x : s == 1 ? u1.y : s == 2 ? u1.z : u1.w;
                // even elements x 16 and odd elements x 16 of rows g and g + 8
                const uint32_t a0 = (w0 << 4) & 0xF0F0F0F0u, a1 = (w1 << 4) & 0xF0F0F0F0u, a2 = w0 & 0xF0F0F0F0u, a3 = w1 & 0xF0F0F0F0u;
#pragma unroll
                for (int i = 0; i < TT; ++i) {
                    const uint32_t b0 = s % 2 == 0 ? xv[i].x : xv[i].z, b1 = s % 2 == 0 ? xv[i].y : xv[i].w;
                    if (fresh) mma16832<true>(sum[tl][i], a0, a1, a2, a3, b0, b1);
                    else mma16832<false>(sum[tl][i], a0, a1, a2, a3, b0, b1);
                }
            }
            if ((s + 1) % (4 / GPS) == 0) {  // a group ends
                const int j = s / (4 / GPS);
                const float2 f = *reinterpret_cast<const float2 *>(uf + j * kColumns);
#pragma unroll
                for (int tl = 0; tl < kTiles; ++tl) {
                    const float s0 = scale_at<S, GPS>(b.s, j, (lane & 28) | (2 * tl)), s1 = scale_at<S, GPS>(b.s, j, (lane & 28) | (2 * tl + 1));
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        float v = sum_value(sum[tl][0][c]);
                        if constexpr (WIDE) v = fmaf(fmaf(v, 256.0f, sum_value(sum[tl][1][c])), 256.0f, sum_value(sum[tl][2][c]));
                        acc[tl][c] = fmaf(c < 2 ? s0 : s1, v * ((c & 1) ? f.y : f.x), acc[tl][c]);
                    }
                }
            }
        }
    };

    // the group's 32 x tokens outputs are shared out so that a thread adds up to eight partial sums at a time
    const int share_bits = (WIDE ? 0 : 2) + (p.warps_k == 16 ? 1 : 0);  // threads per output: the bytes of X (and an idle one), halves of WK
    const int group_threads = p.warps_k * 32;
    auto reduce_store = [&]() {
        // register c of lane l of tile tl at position (l + 2 tl + (c >> 1)) % 32: writes and reads hit 32 different banks
        float *buffer = red + parity * kRedFloats;
        parity ^= 1;
#pragma unroll
        for (int tl = 0; tl < kTiles; ++tl)
#pragma unroll
            for (int c = 0; c < 4; ++c) buffer[((warp * kTiles + tl) * 4 + c) * 32 + ((lane + 2 * tl + (c >> 1)) & 31)] = acc[tl][c];
        // the other buffer may be written after the next of these barriers: every reader of it is then done
        const bool any_bad = barrier_or(1 + wr, group_threads, bad_rows != 0) || staged_bad;
        T *out = static_cast<T *>(p.out);
        const int todo = tokens << (5 + share_bits);
        for (int o = (int)threadIdx.x - wr * group_threads; (o & ~31) < todo; o += group_threads) {  // whole warps, for the shuffles
            const int index = o >> share_bits, part = WIDE ? o : o >> 2, b = o & 3;
            const int tok = min(index >> 5, kTile - 1), r = index & 31, tl = r >> 4, half = (r >> 3) & 1;
            const int c = 2 * half + (tok & 1), l = (r & 7) * 4 + (WIDE ? tok >> 1 : b);
            const float *src = buffer + (((wr * p.warps_k + (p.warps_k == 16 ? (part & 1) * 8 : 0)) * kTiles + tl) * 4 + c) * 32 + ((l + 2 * tl + half) & 31);
            float sum = 0.0f;
#pragma unroll
            for (int w = 0; w < 8; ++w)
                if (w < p.warps_k) sum += src[w * kTiles * 128];
            if (!WIDE && b == 3) sum = 0.0f;
            const int col = cw.block * block_rows + wr * kRows + r;
            if (any_bad && o < todo && col < p.n) {
                unsigned bad = 0;
                for (int w = 0; w < kWarps; ++w) bad |= odd_rows[pair_parity * kWarps + w];
                if (bad >> tok & 1) {  // the threads that share the output share K instead
                    const int64_t brow = (int64_t)cw.expert * p.n + col;
                    sum = plain_part(X + (int64_t)(first_row + tok) * p.ldx, p.B + brow * (p.k / 2), scales + brow * p.groups, p.k, p.group_shift,
                                     o & ((1 << share_bits) - 1), 1 << share_bits);
                }
            }
            if constexpr (!WIDE) {
                sum += __shfl_xor_sync(0xFFFFFFFFu, sum, 2);
                sum += __shfl_xor_sync(0xFFFFFFFFu, sum, 1);
            }
            if (p.warps_k == 16) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, WIDE ? 1 : 4);
            if (o >= todo || (o & ((1 << share_bits) - 1)) != 0 || col >= p.n) continue;
            out[(int64_t)(first_row + tok) * p.ldo + col] = from_float<T>(sum);
        }
    };

    for (;;) {
#pragma unroll
        for (int d = 0; d < kDepth; ++d) {
            if (cw.step == 0) {
                if (cw.left <= 0) return;
                if (cw.pair != cpair) {
                    cpair = cw.pair;
                    if (p.offsets) {
                        first_row = seg[cw.expert] + (cw.pair - tiles[cw.expert]) * kTile;
                        tokens = min(kTile, seg[cw.expert + 1] - first_row);
                    } else {
                        first_row = cw.pair * kTile;
                        tokens = min(kTile, p.rows - first_row);
                    }
                    stage_x();
                }
#pragma unroll
                for (int tl = 0; tl < kTiles; ++tl)
#pragma unroll
                    for (int c = 0; c < 4; ++c) acc[tl][c] = 0.0f;
            }
            product(buf[d]);
            load(buf[d]);
            if (cw.step == mine - 1) reduce_store();
            advance(cw);
        }
    }
}

struct RowsPlan {
    bool wide;
    int warps_k;
    size_t smem;
};

// false: X does not fit
bool rows_plan(const W4Args &a, int sms, RowsPlan *plan)
{
    RowsPlan p;
    const int steps = (a.k + kStep - 1) / kStep;
    p.wide = a.offsets ? a.rows > (a.experts < a.rows ? a.experts : a.rows) : a.rows > kNarrowRows;
    // Warps that split K: all, or as many as there are steps.  Only where a CTA has many blocks to do, and the block's end is long (WIDE),
    // warp groups that take turns at it pay (us with WK = 16, 8 and 4): 128 rows over 32 experts of 4096 x 4096, at most 28 units a CTA,
    // 84, 78 and 78; 8 x 57344 x 8192, 12 units, 90, 88 and 112; 8 x 28672 x 4096, 6 units, 24.2, 25.1 and 25.4; one row of
    // 57344 x 8192 53.7, 55.0 and 59.0.  (8 is within 4 % of the better of the two on either side.)
    const int tile = p.wide ? kWideRows : kNarrowRows;
    const int64_t pairs = a.offsets ? (a.experts < a.rows ? a.experts : a.rows) : (a.rows + tile - 1) / tile;  // (with experts: at most)
    const int64_t units = pairs * ((a.n + kRows - 1) / kRows);
    p.warps_k = (p.wide && units >= 16 * (int64_t)sms) || steps <= 4 ? 4 : steps <= 8 ? 8 : 16;
    const int places = steps > p.warps_k ? steps : p.warps_k, gps = a.group >= kStep ? 1 : kStep / a.group;
    p.smem = (size_t)places * ((p.wide ? 3 : 1) * 1024 + gps * 32) + 2 * (size_t)kRedFloats * 4 + 2 * kWarps * 4 + (size_t)(a.experts + 1) * 8;
    *plan = p;
    return p.smem <= (size_t)kMaxSmem;
}

template <typename T, typename S, int GPS, bool WIDE>
int rows_launch_variant(const W4Args &a, const RowsPlan &plan, const DeviceCtx &ctx)
{
    auto kernel = w4_rows_kernel<T, S, GPS, WIDE>;
    static std::atomic<bool> configured[64];  // set once per device; a repeated cudaFuncSetAttribute is harmless
    if (!configured[ctx.device & 63].load(std::memory_order_acquire)) {
        cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmem);
        if (e != cudaSuccess) return record_cuda_error(e, "cudaFuncSetAttribute(w4_rows_kernel)");
        configured[ctx.device & 63].store(true, std::memory_order_release);
    }
    RowsParams p;
    p.X = a.X, p.ldx = a.ldx, p.B = a.B, p.scales = a.scales, p.offsets = a.offsets, p.out = a.out, p.ldo = a.ldo;
    p.rows = a.rows, p.n = a.n, p.k = a.k, p.experts = a.experts;
    p.group_shift = a.group == 32 ? 5 : a.group == 64 ? 6 : a.group == 128 ? 7 : 8;
    p.groups = (a.k + a.group - 1) / a.group;
    p.warps_k = plan.warps_k;
    // a step's scales lie on a boundary of their own size when a row has a multiple of GPS of them
    p.vec_scales = p.groups % GPS == 0 && (reinterpret_cast<uintptr_t>(a.scales) & 15u) == 0;
    const int block_rows = kRows * (kWarps / plan.warps_k), tile = WIDE ? kWideRows : kNarrowRows;
    const int64_t blocks = (a.n + block_rows - 1) / block_rows;
    // with experts the units are known on the device only: at most one tile more than whole ones per expert that can have rows
    const int64_t pairs = a.offsets ? a.rows / tile + (a.experts < a.rows ? a.experts : a.rows) : (a.rows + tile - 1) / tile;
    const int64_t units = pairs * blocks;
    if (units > 0x7FFFFFFF) return QM_ERR_SHAPE;
    return launch_chained("w4_rows_kernel launch", kernel, (unsigned)(units < ctx.num_sms ? units : ctx.num_sms), kThreads, plan.smem, a.stream, p);
}

}  // namespace

bool w4_rows_eligible(const W4Args &a, const DeviceCtx &ctx)
{
    RowsPlan plan;
    const int sms = ctx.num_sms;
    return a.k > 0 && a.k % 32 == 0 && a.ldx % 8 == 0 && (int64_t)a.n * (a.k / 2) < (1ll << 32) &&
           ((reinterpret_cast<uintptr_t>(a.X) | reinterpret_cast<uintptr_t>(a.B)) & 15u) == 0 && rows_plan(a, sms, &plan);
}

int w4_rows_launch(const W4Args &a, const DeviceCtx &ctx)
{
    RowsPlan plan;
    if (!rows_plan(a, ctx.num_sms, &plan)) return QM_ERR_ARG;
    auto by_type = [&](auto t) {
        using T = typename decltype(t)::type;
        return with_same_or_float<T>(a.scale_type, [&](auto u) {
            using S = typename decltype(u)::type;
            auto by_group = [&](auto wide) {
                constexpr bool WIDE = decltype(wide)::value;
                if (a.group == 32) return rows_launch_variant<T, S, 4, WIDE>(a, plan, ctx);
                if (a.group == 64) return rows_launch_variant<T, S, 2, WIDE>(a, plan, ctx);
                return rows_launch_variant<T, S, 1, WIDE>(a, plan, ctx);
            };
            return plan.wide ? by_group(std::true_type()) : by_group(std::false_type());
        });
    };
    return a.type == QM_TYPE_F16 ? by_type(Tag<__half>()) : by_type(Tag<__nv_bfloat16>());
}

}  // namespace qm
