// Tokens to experts and back: a stable counting sort of the assignments with the copy of their rows, the weighted sum that
// brings the experts' rows back, and the gradients of both.  All of it is bound by memory: rows move in 16-byte pieces with
// several in flight per thread, and nothing is read twice but indices (and dy, for every four of top_k).
//
// Sorting.  slot(t, j) = (assignments to lower experts) + (earlier assignments to the same expert): a counting sort, stable, without
// atomics on anything that decides an order.  Up to kFewIds assignments take ONE launch: every block counts all ids itself
// (they are L2 hits), which saves two launches and a workspace.  More take three: counts per block of assignments, a scan of
// the counts over the blocks, and the placing.  With up to 64 experts ids are counted without atomics: a lane has the counts of
// one or two experts in registers, and finds who of 32 ids names them from a ballot per bit of the id.
//
// The launches take their turn in the stream: these kernels read indices that the kernel before may have written, and addresses come
// from them, so none starts before that one has ended.
//
// Measured (bf16): sort of 16 x 8 by 64 experts 8.2 us, of 8192 x 2 rows of 4096 48.6 us = 4.1 TB/s; combine of 4096 x 8 rows of
// 4096 49 us = 6.1 TB/s, its gradients 93 us = 6.1 TB/s (0.93 of a copy).  Single elements (rows off 16-byte boundaries, 3000 x 4 of
// 5119): sort 66 us = 2.3 TB/s, combine 49 us = 3.1.
#include <atomic>

#include "qm_w4.cuh"

namespace qm {

using namespace w4;

namespace {

constexpr int kThreads = 256;       // of the sums and their gradients
constexpr int kSortThreads = 1024;
constexpr int kFewIds = 16384;
constexpr int kFewBlocks = 148, kManyBlocks = 148 * 2;  // blocks that share the assignments

// VEC elements of T that move together: 16 bytes, or one element where rows are not on 16-byte boundaries.
template <typename T, int VEC>
struct Piece {
    static_assert(VEC == 1 || VEC * sizeof(T) == 16, "piece");
    T v[VEC];
    __device__ __forceinline__ void load(const T *p)
    {
        if constexpr (VEC == 1) v[0] = __ldcs(p);
        else *reinterpret_cast<uint4 *>(v) = __ldcs(reinterpret_cast<const uint4 *>(p));
    }
    __device__ __forceinline__ void store(T *p) const
    {
        if constexpr (VEC == 1) __stcs(p, v[0]);
        else __stcs(reinterpret_cast<uint4 *>(p), *reinterpret_cast<const uint4 *>(v));
    }
};

__device__ __forceinline__ int expert_id(int64_t id, int experts) { return id >= 0 && id < experts ? (int)id : -1; }

// Ids [first, last) -> how many go to each expert, added to counts[0 .. experts) in shared memory; the whole block.
template <typename I>
__device__ __forceinline__ void count_range(const I *__restrict__ ids, int64_t first, int64_t last, int experts, int *counts)
{
    constexpr int kAhead = 8;  // loads in flight
    const int lane = threadIdx.x & 31;
    int mine[2] = {0, 0};  // of experts lane and lane + 32
    unsigned flip[5];      // bit b of a lane's expert: who has another one
#pragma unroll
    for (int b = 0; b < 5; ++b) flip[b] = (lane >> b) & 1 ? 0u : 0xFFFFFFFFu;
    for (int64_t base = first + (threadIdx.x & ~31); base < last; base += kAhead * (int64_t)blockDim.x) {
        int e[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int64_t i = base + u * (int64_t)blockDim.x + lane;
            e[u] = i < last ? expert_id((int64_t)__ldg(ids + i), experts) : -1;
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            if (base + u * (int64_t)blockDim.x >= last) break;  // uniform over the warp
            if (experts <= 64) {
                unsigned same = __ballot_sync(0xFFFFFFFFu, e[u] >= 0);
#pragma unroll
                for (int b = 0; b < 5; ++b) same &= __ballot_sync(0xFFFFFFFFu, (e[u] >> b) & 1) ^ flip[b];
                const unsigned high = __ballot_sync(0xFFFFFFFFu, e[u] & 32);
                mine[0] += __popc(same & ~high);
                mine[1] += __popc(same & high);
            } else if (e[u] >= 0) {
                atomicAdd(counts + e[u], 1);
            }
        }
    }
    if (experts <= 64) {
        if (lane < experts && mine[0]) atomicAdd(counts + lane, mine[0]);
        if (lane + 32 < experts && mine[1]) atomicAdd(counts + lane + 32, mine[1]);
    }
}

// counts[block][expert] of the block's assignments
template <typename I>
__global__ void __launch_bounds__(kSortThreads) moe_count_kernel(const I *__restrict__ ids, int experts, int count, int per_block, int *__restrict__ counts)
{
    extern __shared__ int mine[];
    for (int e = threadIdx.x; e < experts; e += kSortThreads) mine[e] = 0;
    __syncthreads();
    const int64_t first = (int64_t)blockIdx.x * per_block;
    count_range(ids, first, min((int64_t)count, first + per_block), experts, mine);
    __syncthreads();
    for (int e = threadIdx.x; e < experts; e += kSortThreads) counts[(int64_t)blockIdx.x * experts + e] = mine[e];
}

// counts[block][expert] -> how many earlier blocks have, totals[expert]; one warp per expert
__global__ void __launch_bounds__(kThreads) moe_scan_kernel(int *__restrict__ counts, int *__restrict__ totals, int experts, int blocks)
{
    const int e = (int)(blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5)), lane = threadIdx.x & 31;
    if (e >= experts) return;
    int sum = 0;
    for (int base = 0; base < blocks; base += 32) {
        const int b = base + lane;
        const int v = b < blocks ? counts[(int64_t)b * experts + e] : 0;
        int s = v;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int o = __shfl_up_sync(0xFFFFFFFFu, s, d);
            if (lane >= d) s += o;
        }
        if (b < blocks) counts[(int64_t)b * experts + e] = sum + s - v;
        sum += __shfl_sync(0xFFFFFFFFu, s, 31);
    }
    if (lane == 0) totals[e] = sum;
}

// Slots of the block's tokens and the copy of their rows.  counts == NULL: the block counts all ids itself.
template <typename T, typename I, int VEC>
__global__ void __launch_bounds__(kSortThreads) moe_place_kernel(const T *__restrict__ X, int64_t ldx, const I *__restrict__ ids, int experts, int tokens,
                                                             int top_k, int hidden, int per_block, const int *__restrict__ counts,
                                                             const int *__restrict__ totals, T *__restrict__ xs, int64_t ldxs, int *__restrict__ offsets,
                                                             int *__restrict__ slots)
{
    extern __shared__ int smem[];
    int *next = smem, *total = smem + experts, *at = total + experts;  // at: the experts, then the slots of the block's assignments
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t first = (int64_t)blockIdx.x * per_block * top_k;
    const int64_t last = min((int64_t)tokens * top_k, first + (int64_t)per_block * top_k);
    for (int e = threadIdx.x; e < experts; e += kSortThreads) {
        next[e] = counts ? counts[(int64_t)blockIdx.x * experts + e] : 0;
        total[e] = counts ? totals[e] : 0;
    }
    for (int i = threadIdx.x; i < (int)(last - first); i += kSortThreads) at[i] = expert_id((int64_t)__ldg(ids + first + i), experts);
    __syncthreads();
    if (!counts) {
        count_range(ids, 0, first, experts, next);
        count_range(ids, first, (int64_t)tokens * top_k, experts, total);
        __syncthreads();
    }
    if (warp == 0) {
        // offsets: an exclusive scan of the totals; next[e] becomes the slot of the block's first assignment to e
        int sum = 0;
        for (int base = 0; base < experts; base += 32) {
            const int e = base + lane;
            const int v = e < experts ? total[e] + (counts ? 0 : next[e]) : 0;
            int s = v;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const int o = __shfl_up_sync(0xFFFFFFFFu, s, d);
                if (lane >= d) s += o;
            }
            if (e < experts) {
                next[e] += sum + s - v;
                if (blockIdx.x == 0) offsets[e] = sum + s - v;
            }
            sum += __shfl_sync(0xFFFFFFFFu, s, 31);
        }
        if (blockIdx.x == 0 && lane == 0) offsets[experts] = sum;
        __syncwarp();
        // the block's assignments in order, 32 at a time; lanes with the same expert are ranked by a match
        for (int base = 0; base < (int)(last - first); base += 32) {
            const int i = base + lane;
            const int e = i < (int)(last - first) ? at[i] : -1;
            const unsigned same = __match_any_sync(0xFFFFFFFFu, e);
            const int rank = __popc(same & ((1u << lane) - 1u));
            // (a slot is below all assignments unless the ids were changed under way: nothing is written outside xs then either)
            const int place = e >= 0 ? next[e] + rank : -1, slot = place < tokens * top_k ? place : -1;
            __syncwarp();
            if (e >= 0 && rank == 0) next[e] += __popc(same);
            __syncwarp();
            if (i < (int)(last - first)) {
                slots[first + i] = slot;
                at[i] = slot;
            }
        }
    }
    __syncthreads();
    if (hidden == 0) return;
    const int pieces = hidden / VEC;
    const int block_tokens = top_k > 0 ? (int)((last - first) / top_k) : 0;
    // the block's (token, piece) pairs are dealt to its threads
    constexpr int kAhead = VEC == 1 ? 8 : 4;
    const int step_t = kSortThreads / pieces, step_c = kSortThreads - step_t * pieces;  // (a division per piece costs more than the copy)
    int t = (int)threadIdx.x / pieces, c = (int)threadIdx.x - t * pieces;
    while (t < block_tokens) {
        Piece<T, VEC> v[kAhead];
        int tt[kAhead], cc[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            tt[u] = t, cc[u] = c * VEC;
            if (t < block_tokens) v[u].load(X + ((int64_t)blockIdx.x * per_block + t) * ldx + cc[u]);
            t += step_t, c += step_c;
            if (c >= pieces) c -= pieces, ++t;
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            if (tt[u] >= block_tokens) continue;
            T *dst = xs + cc[u];
            for (int j = 0; j < top_k; ++j) {
                const int slot = at[tt[u] * top_k + j];
                if (slot >= 0) v[u].store(dst + (int64_t)slot * ldxs);
            }
        }
    }
}

// y[t] = sum of weight * row; a block takes one token and a stretch of `hidden`
template <typename T, typename S, int VEC>
__global__ void __launch_bounds__(kThreads) moe_combine_kernel(const T *__restrict__ ys, int64_t ldys, int rows, const int *__restrict__ slots,
                                                               const S *__restrict__ weights, T *__restrict__ y, int64_t ldy, int top_k, int hidden,
                                                               int parts)
{
    constexpr int kAhead = 8;                // rows in flight per thread
    constexpr int kCols = VEC == 1 ? 4 : 1;  // pieces of a row per thread and turn: single elements need more of them in flight
    const int64_t t = blockIdx.x / parts;
    const int part = (int)(blockIdx.x % parts);
    // (unsigned: from the last piece of a long row one step goes beyond 2^31)
    const unsigned width = (unsigned)hidden;
    for (unsigned c0 = (part * kThreads * kCols + threadIdx.x) * VEC; c0 < width; c0 += (unsigned)parts * (kThreads * kCols * VEC)) {
        float sum[kCols][VEC];
#pragma unroll
        for (int o = 0; o < kCols; ++o)
#pragma unroll
            for (int i = 0; i < VEC; ++i) sum[o][i] = 0.0f;
        for (int j0 = 0; j0 < top_k; j0 += kAhead) {
            Piece<T, VEC> v[kAhead][kCols];
            float w[kAhead];
            bool live[kAhead];
#pragma unroll
            for (int j = 0; j < kAhead; ++j) {
                live[j] = false;
                if (j0 + j >= top_k) continue;
                const int at = __ldg(slots + t * top_k + j0 + j);
                live[j] = at >= 0 && at < rows;
                if (!live[j]) continue;
                w[j] = weights ? to_float(__ldg(weights + t * top_k + j0 + j)) : 1.0f;
#pragma unroll
                for (int o = 0; o < kCols; ++o)
                    if (c0 + o * kThreads * VEC < width) v[j][o].load(ys + (int64_t)at * ldys + c0 + o * kThreads * VEC);
            }
#pragma unroll
            for (int j = 0; j < kAhead; ++j) {
                if (!live[j]) continue;
#pragma unroll
                for (int o = 0; o < kCols; ++o)
#pragma unroll
                    for (int i = 0; i < VEC; ++i) sum[o][i] = fmaf(w[j], to_float(v[j][o].v[i]), sum[o][i]);
            }
        }
#pragma unroll
        for (int o = 0; o < kCols; ++o) {
            if (c0 + o * kThreads * VEC >= width) continue;
            Piece<T, VEC> r;
#pragma unroll
            for (int i = 0; i < VEC; ++i) r.v[i] = from_float<T>(sum[o][i]);
            r.store(y + t * ldy + c0 + o * kThreads * VEC);
        }
    }
}

// Both gradients of one token: dy is read once for every four of its experts, every row of ys once, every row of dys is written once;
// the products with the rows are summed over the block in a fixed order.
template <typename T, typename S, int VEC>
__global__ void __launch_bounds__(kThreads) moe_combine_grad_kernel(const T *__restrict__ dy, int64_t lddy, const T *__restrict__ ys, int64_t ldys, int rows,
                                                                    const int *__restrict__ slots, const S *__restrict__ weights, T *__restrict__ dys,
                                                                    int64_t lddys, S *__restrict__ dweights, int top_k, int hidden)
{
    constexpr int kAhead = 4;
    __shared__ float part[kThreads / 32][kAhead];
    const int64_t t = blockIdx.x;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int j0 = 0; j0 < top_k; j0 += kAhead) {
        int at[kAhead];
        float w[kAhead], dot[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            at[j] = j0 + j < top_k ? __ldg(slots + t * top_k + j0 + j) : -1;
            if (at[j] >= rows) at[j] = -1;
            w[j] = at[j] >= 0 ? to_float(__ldg(weights + t * top_k + j0 + j)) : 0.0f;
            dot[j] = 0.0f;
        }
#pragma unroll(VEC == 1 ? 4 : 1)
        for (int c = (int)threadIdx.x * VEC; c < hidden; c += kThreads * VEC) {
            Piece<T, VEC> d, v[kAhead];
            d.load(dy + t * lddy + c);
#pragma unroll
            for (int j = 0; j < kAhead; ++j)
                if (at[j] >= 0) v[j].load(ys + (int64_t)at[j] * ldys + c);
#pragma unroll
            for (int j = 0; j < kAhead; ++j) {
                if (at[j] < 0) continue;
                Piece<T, VEC> o;
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    const float g = to_float(d.v[i]);
                    dot[j] = fmaf(g, to_float(v[j].v[i]), dot[j]);
                    o.v[i] = from_float<T>(w[j] * g);
                }
                o.store(dys + (int64_t)at[j] * lddys + c);
            }
        }
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
#pragma unroll
            for (int s = 16; s; s >>= 1) dot[j] += __shfl_xor_sync(0xFFFFFFFFu, dot[j], s);
            if (lane == 0) part[warp][j] = dot[j];
        }
        __syncthreads();
        if (threadIdx.x < kAhead && j0 + (int)threadIdx.x < top_k) {
            float sum = 0.0f;
#pragma unroll
            for (int k = 0; k < kThreads / 32; ++k) sum += part[k][threadIdx.x];
            dweights[t * top_k + j0 + threadIdx.x] = from_float<S>(sum);
        }
        __syncthreads();
    }
}

bool on16(const void *p, int64_t pitch, int size) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && (pitch * size) % 16 == 0; }

// f gets the piece width: 16 bytes where `vec`, else one element
template <typename T, typename F>
int with_pieces(bool vec, F f)
{
    return vec ? f(std::integral_constant<int, 16 / (int)sizeof(T)>()) : f(std::integral_constant<int, 1>());
}

constexpr int kMaxSlots = 8192;  // slots a block keeps in shared memory; top_k is at most half of it

constexpr size_t kMaxSmem = (2 * (size_t)kMaxExperts + kMaxSlots) * sizeof(int);

int block_count(int tokens, int per) { return (int)(((int64_t)tokens + per - 1) / per); }

int tokens_per_block(int tokens, int top_k)
{
    const int blocks = (int64_t)tokens * top_k <= kFewIds ? kFewBlocks : kManyBlocks;
    const int per = (int)(((int64_t)tokens + blocks - 1) / blocks), most = kMaxSlots / (top_k > 0 ? top_k : 1);
    return per < 1 ? 1 : per < most ? per : most;
}

}  // namespace

size_t moe_sort_workspace(int tokens, int top_k, int experts)
{
    if ((int64_t)tokens * top_k <= kFewIds) return 0;
    const int blocks = block_count(tokens, tokens_per_block(tokens, top_k));
    return ((size_t)blocks + 1) * experts * sizeof(int);
}

int moe_sort_launch(const MoeSortArgs &a)
{
    const int per = tokens_per_block(a.tokens, a.top_k), blocks = a.tokens > 0 ? block_count(a.tokens, per) : 1;
    const int count = a.tokens * a.top_k;
    const size_t smem = ((size_t)2 * a.experts + (size_t)per * a.top_k) * sizeof(int);
    int *counts = nullptr, *totals = nullptr;
    auto by_id = [&](auto id) {
        using I = typename decltype(id)::type;
        const I *ids = static_cast<const I *>(a.ids);
        if (count > kFewIds && a.experts > 0) {  // (without experts there is nothing to count)
            totals = a.workspace;
            counts = a.workspace + a.experts;
            int st = launch_in_turn("moe_count_kernel launch", moe_count_kernel<I>, (unsigned)blocks, kSortThreads, (size_t)a.experts * sizeof(int), a.stream, ids,
                                    a.experts, count, per * a.top_k, counts);
            if (st != QM_OK) return st;
            st = launch_in_turn("moe_scan_kernel launch", moe_scan_kernel, (unsigned)((a.experts + 7) / 8), kThreads, 0, a.stream, counts, totals, a.experts,
                                blocks);
            if (st != QM_OK) return st;
        }
        return with_type(a.type, [&](auto t) {
            using T = typename decltype(t)::type;
            const bool vec = on16(a.X, a.ldx, sizeof(T)) && on16(a.xs, a.ldxs, sizeof(T)) && a.hidden % (16 / (int)sizeof(T)) == 0;
            return with_pieces<T>(vec, [&](auto v) {
                constexpr int VEC = decltype(v)::value;
                auto kernel = moe_place_kernel<T, I, VEC>;
                if (smem > 48 * 1024) {
                    // The limit belongs to the kernel, not to the launch: the largest one, set once per device, so that no call can lower
                    // it between another thread's setting and its launch (a repeated cudaFuncSetAttribute is harmless).
                    static std::atomic<bool> configured[64];
                    int device = 0;
                    cudaError_t e = cudaGetDevice(&device);
                    if (e != cudaSuccess) return record_cuda_error(e, "cudaGetDevice");
                    if (!configured[device & 63].load(std::memory_order_acquire)) {
                        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kMaxSmem);
                        if (e != cudaSuccess) return record_cuda_error(e, "cudaFuncSetAttribute(moe_place_kernel)");
                        configured[device & 63].store(true, std::memory_order_release);
                    }
                }
                return launch_in_turn("moe_place_kernel launch", kernel, (unsigned)blocks, kSortThreads, smem, a.stream, static_cast<const T *>(a.X), a.ldx, ids,
                                      a.experts, a.tokens, a.top_k, a.hidden, per, (const int *)counts, (const int *)totals, static_cast<T *>(a.xs), a.ldxs,
                                      a.offsets, a.slots);
            });
        });
    };
    return a.id_bytes == 8 ? by_id(Tag<int64_t>()) : by_id(Tag<int32_t>());
}

int moe_combine_launch(const MoeCombineArgs &a)
{
    return with_type(a.type, [&](auto t) {
        using T = typename decltype(t)::type;
        return with_same_or_float<T>(a.weight_type, [&](auto u) {
            using S = typename decltype(u)::type;
            const bool vec = on16(a.ys, a.ldys, sizeof(T)) && on16(a.out, a.ldo, sizeof(T)) && a.hidden % (16 / (int)sizeof(T)) == 0;
            return with_pieces<T>(vec, [&](auto v) {
                constexpr int VEC = decltype(v)::value;
                // a thread per piece while the grid allows it
                constexpr int kStretch = kThreads * (VEC == 1 ? 4 : VEC);
                int64_t parts = (a.hidden + kStretch - 1) / kStretch;
                if (parts * a.tokens > 0x7FFFFFFF) parts = 1;
                return launch_in_turn("moe_combine_kernel launch", moe_combine_kernel<T, S, VEC>, (unsigned)(parts * a.tokens), kThreads, 0, a.stream,
                                      static_cast<const T *>(a.ys), a.ldys, a.rows, a.slots, static_cast<const S *>(a.weights), static_cast<T *>(a.out), a.ldo,
                                      a.top_k, a.hidden, (int)parts);
            });
        });
    });
}

int moe_combine_grad_launch(const MoeCombineArgs &a)
{
    return with_type(a.type, [&](auto t) {
        using T = typename decltype(t)::type;
        return with_same_or_float<T>(a.weight_type, [&](auto u) {
            using S = typename decltype(u)::type;
            const bool vec = on16(a.dy, a.lddy, sizeof(T)) && on16(a.ys, a.ldys, sizeof(T)) && on16(a.out, a.ldo, sizeof(T)) &&
                             a.hidden % (16 / (int)sizeof(T)) == 0;
            return with_pieces<T>(vec, [&](auto v) {
                constexpr int VEC = decltype(v)::value;
                return launch_in_turn("moe_combine_grad_kernel launch", moe_combine_grad_kernel<T, S, VEC>, (unsigned)a.tokens, kThreads, 0, a.stream,
                                      static_cast<const T *>(a.dy), a.lddy, static_cast<const T *>(a.ys), a.ldys, a.rows, a.slots,
                                      static_cast<const S *>(a.weights), static_cast<T *>(a.out), a.ldo, static_cast<S *>(a.dweights), a.top_k, a.hidden);
            });
        });
    });
}

}  // namespace qm
