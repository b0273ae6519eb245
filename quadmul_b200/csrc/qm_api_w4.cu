// C ABI of the 4-bit-weight products, their quantiser and the expert routing (include/quadmul_b200.h): argument checks and
// dispatch.  The reference has no counterpart of these entry points.
#include <climits>

#include "qm_w4.cuh"

using namespace qm;

namespace {

constexpr int kMaxK = (1 << 30) - 32;  // a row of X is below 2^31 bytes, rounded up to 32 elements or not

constexpr int kMaxRows = INT_MAX - 512;     // rounded up to whole tiles, and a tile further, it is an int
constexpr int kMaxHidden = INT_MAX - 4096;  // as is a place in a row, one turn of a block further

bool known_group(int g) { return g == 32 || g == 64 || g == 128 || g == 256; }

bool aligned_to(const void *p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & (uintptr_t)(bytes - 1)) == 0; }

int check_w4(const W4Args &a)
{
    if (a.rows < 0 || a.rows > kMaxRows || a.n < 0 || a.k < 0 || (a.k & 1) || a.k > kMaxK || a.experts < 0 || a.experts > kMaxExperts) return QM_ERR_SHAPE;
    if (a.type != QM_TYPE_F16 && a.type != QM_TYPE_BF16) return QM_ERR_ARG;
    if (a.scale_type != QM_TYPE_F32 && a.scale_type != a.type) return QM_ERR_ARG;
    if (!known_group(a.group)) return QM_ERR_ARG;
    if (a.rows == 0 || a.n == 0) return QM_OK;
    if (!a.out || (a.k > 0 && (!a.X || (a.experts > 0 && (!a.B || !a.scales))))) return QM_ERR_NULL;
    if (a.ldo < a.n || a.ldx < a.k || (int64_t)a.experts * a.n > INT_MAX - 512) return QM_ERR_SHAPE;
    if (!aligned_to(a.X, 2) || !aligned_to(a.out, 2) || !aligned_to(a.scales, w4::type_bytes(a.scale_type))) return QM_ERR_ALIGN;
    return QM_OK;
}

int w4_dispatch(W4Args a, void *workspace, size_t workspace_bytes)
{
    int st = check_w4(a);
    if (st != QM_OK || a.rows == 0 || a.n == 0 || a.experts == 0) return st;
    const size_t need = w4_workspace(a);
    if (need && (!workspace || workspace_bytes < need)) return QM_ERR_WORKSPACE;
    if (need && !aligned_to(workspace, 16)) return QM_ERR_ALIGN;
    DeviceCtx *ctx = nullptr;
    st = device_ctx(&ctx);
    if (st != QM_OK) return st;
    if (a.k == 0) return w4_zero_launch(a);
    if (need && (st = w4_pad_launch(&a, workspace)) != QM_OK) return st;
    const int average = a.rows / (a.experts < a.rows ? a.experts : a.rows);
    // The kernel for few rows up to a whole pass over the weights.  One matrix, rows against tcgen05 kernel: 8 x 4096 x 4096 8.2 and 10.3
    // us, 9 rows (two passes) 10.9 and 10.3; 8 x 11008 x 4096 13.8 and 17.2, 9 rows 20.2 and 17.5.  With experts some have more rows
    // than the average, and theirs are two passes: 32 experts of 4096 x 4096 with 6 rows on average 81 and 92 us, with 8 100 and 92;
    // 8 of 11008 x 4096 60 and 67, 70 and 67; 64 of 1024 x 2048 36 and 35, 43 and 35.
    if (average <= (a.offsets ? 6 : 8) && w4_rows_eligible(a, *ctx)) return w4_rows_launch(a, *ctx);
    return w4_tc_launch(a, *ctx);
}

int check_moe(int type, int tokens, int top_k, int hidden)
{
    if (tokens < 0 || top_k < 0 || top_k > kMaxExperts || hidden < 0 || hidden > kMaxHidden || (int64_t)tokens * top_k > INT_MAX) return QM_ERR_SHAPE;
    return w4::known_type(type) ? QM_OK : QM_ERR_ARG;
}

}  // namespace

extern "C" {

int qm_gemm_w4(const void *X, int type, int64_t ldx, const void *B, const void *scales, int scale_type, int group, void *out, int64_t ldo, int m,
               int n, int k, void *workspace, size_t workspace_bytes, void *stream)
{
    return w4_dispatch({X, type, ldx, static_cast<const uint8_t *>(B), scales, scale_type, group, nullptr, 1, out, ldo, m, n, k,
                        static_cast<cudaStream_t>(stream)},
                       workspace, workspace_bytes);
}

int qm_moe_gemm_w4(const void *X, int type, int64_t ldx, const void *B, const void *scales, int scale_type, int group, const int *offsets,
                   int experts, void *out, int64_t ldo, int rows, int n, int k, void *workspace, size_t workspace_bytes, void *stream)
{
    if (!offsets) return QM_ERR_NULL;
    if (!aligned_to(offsets, 4)) return QM_ERR_ALIGN;
    return w4_dispatch({X, type, ldx, static_cast<const uint8_t *>(B), scales, scale_type, group, offsets, experts, out, ldo, rows, n, k,
                        static_cast<cudaStream_t>(stream)},
                       workspace, workspace_bytes);
}

size_t qm_gemm_w4_workspace_bytes(const void *X, int64_t ldx, const void *B, int experts, int rows, int n, int k)
{
    W4Args a = {};
    a.X = X, a.ldx = ldx, a.B = static_cast<const uint8_t *>(B), a.experts = experts, a.rows = rows, a.n = n, a.k = k;
    return w4_workspace(a);
}

int qm_quantize_w4(const void *W, int type, int64_t ldw, void *packed, void *scales, int scale_type, int64_t rows, int64_t k, int group, void *stream)
{
    if (rows < 0 || k < 0 || (k & 1)) return QM_ERR_SHAPE;
    if (!w4::known_type(type) || (scale_type != QM_TYPE_F32 && scale_type != type) || !known_group(group)) return QM_ERR_ARG;
    if (rows == 0 || k == 0) return QM_OK;
    if (!W || !packed || !scales) return QM_ERR_NULL;
    if (ldw < k) return QM_ERR_SHAPE;
    if (!aligned_to(W, w4::type_bytes(type)) || !aligned_to(scales, w4::type_bytes(scale_type))) return QM_ERR_ALIGN;
    return quantize_w4_launch(W, type, ldw, static_cast<uint8_t *>(packed), scales, scale_type, rows, k, group, static_cast<cudaStream_t>(stream));
}

int qm_moe_sort(const void *X, int type, int64_t ldx, const void *ids, int id_bytes, int experts, void *xs, int64_t ldxs, int *offsets, int *slots,
                int tokens, int top_k, int hidden, void *workspace, size_t workspace_bytes, void *stream)
{
    int st = check_moe(type, tokens, top_k, hidden);
    if (st != QM_OK) return st;
    if (id_bytes != 4 && id_bytes != 8) return QM_ERR_ARG;
    if (experts < 0 || experts > kMaxExperts) return QM_ERR_SHAPE;
    if (!offsets) return QM_ERR_NULL;
    const bool some = tokens > 0 && top_k > 0;
    if (some && (!ids || !slots || (hidden > 0 && (!X || !xs)))) return QM_ERR_NULL;
    if (some && (ldx < hidden || ldxs < hidden)) return QM_ERR_SHAPE;
    if (!aligned_to(offsets, 4) || !aligned_to(slots, 4) || !aligned_to(ids, id_bytes) || !aligned_to(X, w4::type_bytes(type)) ||
        !aligned_to(xs, w4::type_bytes(type)))
        return QM_ERR_ALIGN;
    const size_t need = moe_sort_workspace(tokens, top_k, experts);
    if (need && (!workspace || workspace_bytes < need)) return QM_ERR_WORKSPACE;
    if (need && !aligned_to(workspace, 4)) return QM_ERR_ALIGN;
    return moe_sort_launch({X, type, ldx, ids, id_bytes, experts, xs, ldxs, offsets, slots, tokens, top_k, hidden, static_cast<int *>(workspace),
                            static_cast<cudaStream_t>(stream)});
}

size_t qm_moe_sort_workspace_bytes(int tokens, int top_k, int experts)
{
    if (tokens < 0 || top_k < 0 || experts < 0) return 0;
    return moe_sort_workspace(tokens, top_k, experts);
}

int qm_moe_combine(const void *ys, int type, int64_t ldys, int rows, const int *slots, const void *weights, int weight_type, void *y, int64_t ldy,
                   int tokens, int top_k, int hidden, void *stream)
{
    int st = check_moe(type, tokens, top_k, hidden);
    if (st != QM_OK) return st;
    if (weight_type != QM_TYPE_F32 && weight_type != type) return QM_ERR_ARG;
    if (rows < 0) return QM_ERR_SHAPE;
    if (tokens == 0 || hidden == 0) return QM_OK;
    if (!y || (top_k > 0 && (!slots || (rows > 0 && !ys)))) return QM_ERR_NULL;
    if (ldy < hidden || ldys < hidden) return QM_ERR_SHAPE;
    const int size = w4::type_bytes(type);
    if (!aligned_to(ys, size) || !aligned_to(y, size) || !aligned_to(slots, 4) || !aligned_to(weights, w4::type_bytes(weight_type))) return QM_ERR_ALIGN;
    return moe_combine_launch({nullptr, 0, ys, ldys, type, rows, slots, weights, weight_type, y, ldy, nullptr, tokens, top_k, hidden,
                               static_cast<cudaStream_t>(stream)});
}

int qm_moe_combine_grad(const void *dy, int64_t lddy, const void *ys, int64_t ldys, int type, int rows, const int *slots, const void *weights,
                        int weight_type, void *dys, int64_t lddys, void *dweights, int tokens, int top_k, int hidden, void *stream)
{
    int st = check_moe(type, tokens, top_k, hidden);
    if (st != QM_OK) return st;
    if (weight_type != QM_TYPE_F32 && weight_type != type) return QM_ERR_ARG;
    if (rows < 0) return QM_ERR_SHAPE;
    if (tokens == 0 || top_k == 0) return QM_OK;
    if (!slots || !weights || !dweights || (hidden > 0 && (!dy || (rows > 0 && (!ys || !dys))))) return QM_ERR_NULL;
    if (lddy < hidden || ldys < hidden || lddys < hidden) return QM_ERR_SHAPE;
    const int size = w4::type_bytes(type), wsize = w4::type_bytes(weight_type);
    if (!aligned_to(dy, size) || !aligned_to(ys, size) || !aligned_to(dys, size) || !aligned_to(slots, 4) || !aligned_to(weights, wsize) ||
        !aligned_to(dweights, wsize))
        return QM_ERR_ALIGN;
    return moe_combine_grad_launch({dy, lddy, ys, ldys, type, rows, slots, weights, weight_type, dys, lddys, dweights, tokens, top_k, hidden,
                                    static_cast<cudaStream_t>(stream)});
}

}  // extern "C"
