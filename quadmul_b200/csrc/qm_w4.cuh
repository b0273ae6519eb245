// Element types and small device helpers shared by the 4-bit-weight kernels and the expert-routing kernels.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "qm_internal.h"

namespace qm {
namespace w4 {

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T>
__device__ __forceinline__ T from_float(float v);  // one rounding, to nearest even
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

inline bool known_type(int t) { return t == QM_TYPE_F32 || t == QM_TYPE_F16 || t == QM_TYPE_BF16; }
inline int type_bytes(int t) { return t == QM_TYPE_F32 ? 4 : 2; }

template <typename T>
struct Tag {
    using type = T;
};

// Calls f with a Tag of the element type `t` names; an unknown value does not get past the argument checks.
template <typename F>
int with_type(int t, F f)
{
    switch (t) {
        case QM_TYPE_F32: return f(Tag<float>());
        case QM_TYPE_F16: return f(Tag<__half>());
        case QM_TYPE_BF16: return f(Tag<__nv_bfloat16>());
        default: return QM_ERR_ARG;
    }
}

// `other` is fp32 or has the type T that the call's main operand has.
template <typename T, typename F>
int with_same_or_float(int other, F f)
{
    return other == QM_TYPE_F32 ? f(Tag<float>()) : f(Tag<T>());
}

inline int launched(const char *what)
{
    cudaError_t e = cudaPeekAtLastError();
    return e == cudaSuccess ? QM_OK : record_cuda_error(e, what);
}

}  // namespace w4
}  // namespace qm
