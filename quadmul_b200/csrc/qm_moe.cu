// Tokens to experts and back: a stable counting sort of the assignments with the copy of their rows, the weighted sum that
// brings the experts' rows back, and the gradients of both.  All of it is bound by memory.
#include "qm_w4.cuh"

namespace qm {

using namespace w4;

// Offsets and slots.  One warp walks the assignments in order; lanes with the same expert are ranked by a match, so the
// order within an expert is the order of the assignments.
template <typename I>
__global__ void __launch_bounds__(1024) moe_slots_kernel(const I *__restrict__ ids, int experts, int count, int *__restrict__ offsets,
                                                         int *__restrict__ slots)
{
    extern __shared__ int next[];  // experts + 1
    for (int e = threadIdx.x; e <= experts; e += blockDim.x) next[e] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < count; i += blockDim.x) {
        const I id = ids[i];
        if (id >= 0 && id < (I)experts) atomicAdd(&next[(int)id + 1], 1);
    }
    __syncthreads();
    if (threadIdx.x == 0)
        for (int e = 0; e < experts; ++e) next[e + 1] += next[e];
    __syncthreads();
    for (int e = threadIdx.x; e <= experts; e += blockDim.x) offsets[e] = next[e];
    __syncthreads();
    if (threadIdx.x >= 32) return;
    const int lane = threadIdx.x;
    for (int base = 0; base < count; base += 32) {
        const int i = base + lane;
        const I id = i < count ? ids[i] : (I)-1;
        const bool live = id >= 0 && id < (I)experts;
        const int e = live ? (int)id : -1;
        const unsigned same = __match_any_sync(0xFFFFFFFFu, e);
        const int rank = __popc(same & ((1u << lane) - 1u));
        const int at = live ? next[e] + rank : -1;
        __syncwarp();
        if (live && rank == 0) next[e] += __popc(same);
        __syncwarp();
        if (i < count) slots[i] = at;
    }
}

template <typename T>
__global__ void __launch_bounds__(256) moe_copy_kernel(const T *__restrict__ X, int64_t ldx, const int *__restrict__ slots, T *__restrict__ xs,
                                                       int64_t ldxs, int top_k, int hidden)
{
    const int t = blockIdx.x;
    for (int i = threadIdx.x; i < hidden; i += blockDim.x) {
        const T v = X[(int64_t)t * ldx + i];
        for (int j = 0; j < top_k; ++j) {
            const int at = slots[(int64_t)t * top_k + j];
            if (at >= 0) xs[(int64_t)at * ldxs + i] = v;
        }
    }
}

int moe_sort_launch(const MoeSortArgs &a)
{
    const int count = a.tokens * a.top_k;
    const size_t smem = ((size_t)a.experts + 1) * sizeof(int);
    if (a.id_bytes == 8)
        moe_slots_kernel<int64_t><<<1, 1024, smem, a.stream>>>(static_cast<const int64_t *>(a.ids), a.experts, count, a.offsets, a.slots);
    else
        moe_slots_kernel<int32_t><<<1, 1024, smem, a.stream>>>(static_cast<const int32_t *>(a.ids), a.experts, count, a.offsets, a.slots);
    int st = launched("moe_slots_kernel launch");
    if (st != QM_OK || count == 0 || a.hidden == 0) return st;
    return with_type(a.type, [&](auto t) {
        using T = typename decltype(t)::type;
        moe_copy_kernel<T><<<(unsigned)a.tokens, 256, 0, a.stream>>>(static_cast<const T *>(a.X), a.ldx, a.slots, static_cast<T *>(a.xs), a.ldxs, a.top_k,
                                                                     a.hidden);
        return launched("moe_copy_kernel launch");
    });
}

template <typename T, typename S>
__global__ void __launch_bounds__(256) moe_combine_kernel(const T *__restrict__ ys, int64_t ldys, int rows, const int *__restrict__ slots,
                                                          const S *__restrict__ weights, T *__restrict__ y, int64_t ldy, int top_k, int hidden)
{
    const int64_t t = blockIdx.x;
    for (int i = threadIdx.x; i < hidden; i += blockDim.x) {
        float sum = 0.0f;
        for (int j = 0; j < top_k; ++j) {
            const int at = slots[t * top_k + j];
            if (at < 0 || at >= rows) continue;
            sum = fmaf(weights ? to_float(weights[t * top_k + j]) : 1.0f, to_float(ys[(int64_t)at * ldys + i]), sum);
        }
        y[t * ldy + i] = from_float<T>(sum);
    }
}

template <typename T, typename S>
__global__ void __launch_bounds__(256) moe_combine_grad_kernel(const T *__restrict__ dy, int64_t lddy, const T *__restrict__ ys, int64_t ldys, int rows,
                                                               const int *__restrict__ slots, const S *__restrict__ weights, T *__restrict__ dys,
                                                               int64_t lddys, S *__restrict__ dweights, int top_k, int hidden)
{
    __shared__ float part[8];
    const int64_t i = blockIdx.x, t = i / top_k;  // one assignment per block
    const int at = slots[i];
    if (at < 0 || at >= rows) {
        if (threadIdx.x == 0) dweights[i] = from_float<S>(0.0f);
        return;
    }
    const float w = to_float(weights[i]);
    float dot = 0.0f;
    for (int c = threadIdx.x; c < hidden; c += blockDim.x) {
        const float d = to_float(dy[t * lddy + c]);
        dot = fmaf(d, to_float(ys[(int64_t)at * ldys + c]), dot);
        dys[(int64_t)at * lddys + c] = from_float<T>(w * d);
    }
    for (int d = 16; d; d >>= 1) dot += __shfl_xor_sync(0xFFFFFFFFu, dot, d);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = dot;
    __syncthreads();
    if (threadIdx.x == 0) {
        float sum = 0.0f;
        for (int k = 0; k < 8; ++k) sum += part[k];
        dweights[i] = from_float<S>(sum);
    }
}

int moe_combine_launch(const MoeCombineArgs &a)
{
    return with_type(a.type, [&](auto t) {
        using T = typename decltype(t)::type;
        return with_same_or_float<T>(a.weight_type, [&](auto u) {
            using S = typename decltype(u)::type;
            moe_combine_kernel<T, S><<<(unsigned)a.tokens, 256, 0, a.stream>>>(static_cast<const T *>(a.ys), a.ldys, a.rows, a.slots,
                                                                               static_cast<const S *>(a.weights), static_cast<T *>(a.out), a.ldo, a.top_k,
                                                                               a.hidden);
            return launched("moe_combine_kernel launch");
        });
    });
}

int moe_combine_grad_launch(const MoeCombineArgs &a)
{
    return with_type(a.type, [&](auto t) {
        using T = typename decltype(t)::type;
        return with_same_or_float<T>(a.weight_type, [&](auto u) {
            using S = typename decltype(u)::type;
            moe_combine_grad_kernel<T, S><<<(unsigned)(a.tokens * a.top_k), 256, 0, a.stream>>>(
                static_cast<const T *>(a.dy), a.lddy, static_cast<const T *>(a.ys), a.ldys, a.rows, a.slots, static_cast<const S *>(a.weights),
                static_cast<T *>(a.out), a.ldo, static_cast<S *>(a.dweights), a.top_k, a.hidden);
            return launched("moe_combine_grad_kernel launch");
        });
    });
}

}  // namespace qm
