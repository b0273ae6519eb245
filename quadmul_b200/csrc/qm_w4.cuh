// Element types and small device helpers shared by the 4-bit-weight kernels and the expert-routing kernels.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdlib>

#include "qm_internal.h"
#include "qm_ptx.cuh"

namespace qm {
namespace w4 {

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }

// *p as fp32, by a load that stays behind the wait for the kernel before
__device__ __forceinline__ float load_float(const float *p) { return ptx::ld_behind_wait(p); }
__device__ __forceinline__ float load_float(const __half *p) { return __half2float(__ushort_as_half(ptx::ld_behind_wait(reinterpret_cast<const unsigned short *>(p)))); }
__device__ __forceinline__ float load_float(const __nv_bfloat16 *p)
{
    return __uint_as_float((uint32_t)ptx::ld_behind_wait(reinterpret_cast<const unsigned short *>(p)) << 16);
}

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

// Launch that may begin while the previous kernel of the stream still runs: the kernel waits (griddepcontrol.wait) before it
// touches global memory, reads it with loads that stay behind the wait (ptx::ld_behind_wait), and lets its own successor begin
// only then, so that no kernel is resident while the last but one before it still runs.  QM_NO_PDL=1 turns that off.
template <typename... P, typename... A>
int launch_chained(const char *what, void (*kernel)(P...), unsigned blocks, unsigned threads, size_t smem, cudaStream_t stream, A... args)
{
    static const bool allow = !std::getenv("QM_NO_PDL");
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(blocks, 1, 1);
    cfg.blockDim = dim3(threads, 1, 1);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = allow ? 1 : 0;
    cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
    return e == cudaSuccess ? QM_OK : record_cuda_error(e, what);
}

// Launch behind everything the stream has before it.
template <typename... P, typename... A>
int launch_in_turn(const char *what, void (*kernel)(P...), unsigned blocks, unsigned threads, size_t smem, cudaStream_t stream, A... args)
{
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(blocks, 1, 1);
    cfg.blockDim = dim3(threads, 1, 1);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
    return e == cudaSuccess ? QM_OK : record_cuda_error(e, what);
}

// One lane of the (converged) warp, always the same one.  The code around it stays uniform over the warp, so that the compiler
// keeps descriptors and addresses in uniform registers, which is where tcgen05.mma and TMA instructions take them: issued from a
// divergent branch an MMA cost 85 clocks, most of them moves, and 28 from uniform code.
__device__ __forceinline__ bool elect_one()
{
    uint32_t r;
    asm volatile(
        "{\n"
        " .reg .pred p;\n"
        " elect.sync _|p, 0xFFFFFFFF;\n"
        " selp.u32 %0, 1, 0, p;\n"
        "}\n"
        : "=r"(r));
    return r != 0;
}

// The experts' segments, from offsets that may be anything: seg[e] (e = 0 .. experts) is the running maximum of the offsets
// clamped to [0, rows], so expert e has the rows [seg[e], seg[e + 1]); tiles[e] is how many tiles of `tile` rows the experts
// below e have.  Run by one warp; seg and tiles are shared memory, to be read after a barrier.
__device__ __forceinline__ void scan_segments(const int *offsets, int experts, int rows, int tile, int *seg, int *tiles, int lane)
{
    int top = 0, sum = 0;  // running maximum and sum of what came before
    for (int base = 0; base <= experts; base += 32) {
        const int e = base + lane;
        int v = e <= experts ? max(0, min(ptx::ld_behind_wait(offsets + e), rows)) : 0;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int o = __shfl_up_sync(0xFFFFFFFFu, v, d);
            if (lane >= d) v = max(v, o);
        }
        v = max(v, top);
        int before = __shfl_up_sync(0xFFFFFFFFu, v, 1);  // seg[e - 1]
        if (lane == 0) before = base == 0 ? v : top;
        int t = (v - before + tile - 1) / tile;  // tiles of expert e - 1 (none before expert 0)
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int o = __shfl_up_sync(0xFFFFFFFFu, t, d);
            if (lane >= d) t += o;
        }
        t += sum;
        if (e <= experts) seg[e] = v, tiles[e] = t;
        top = __shfl_sync(0xFFFFFFFFu, v, 31);
        sum = __shfl_sync(0xFFFFFFFFu, t, 31);
    }
}

// The expert that has tile p: the last e with tiles[e] <= p (p < tiles[experts]).
__device__ __forceinline__ int expert_of_tile(const int *tiles, int experts, int p)
{
    int lo = 0, hi = experts;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (tiles[mid] <= p) lo = mid;
        else hi = mid;
    }
    return lo;
}

// (a & mask) ^ flip in one instruction
__device__ __forceinline__ uint32_t and_xor(uint32_t a, uint32_t mask, uint32_t flip)
{
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0x6A;" : "=r"(r) : "r"(a), "r"(mask), "r"(flip));
    return r;
}

__device__ __forceinline__ uint32_t fma2(uint32_t a, uint32_t b, uint32_t c, Tag<__nv_bfloat16>)
{
    uint32_t r;
    asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
    return r;
}
__device__ __forceinline__ uint32_t fma2(uint32_t a, uint32_t b, uint32_t c, Tag<__half>)
{
    uint32_t r;
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
    return r;
}

// Eight codes e0 .. e7 of one word -> four pairs (e0, e1), (e2, e3), (e4, e5), (e6, e7) of 16-bit floats, exactly: q for fp16, q / 4
// for bf16 (kCodeUnit).  A nibble n is the code q = (n ^ 8) - 8; u = n ^ 8 is made to read as a float and one fma takes the 8 away.
//   A byte permute puts a byte into both halves of a word; one half keeps the low nibble, the other the high one.
//   In the last mantissa bits of a power of two whose last place is 1 (bf16 128, fp16 1024) u reads as that power plus u.
//   fp16 has room for a nibble four bits up, whose last place then counts 1/16.
//   bf16 has not, but there bits 4 .. 7 with nothing above them are a (sub)normal number u 2^-129: the lowest exponent bit goes
//   on where the mantissa ends.  fma.bf16x2 keeps subnormal numbers, and 2^127 is the largest factor, hence the quarter.
// So a pair costs a permute, a lop3 and an fma.
template <typename T>
constexpr float kCodeUnit = 1.0f;
template <>
constexpr float kCodeUnit<__nv_bfloat16> = 4.0f;

__device__ __forceinline__ void codes_in_order(uint32_t w, uint32_t (&c)[4], Tag<__nv_bfloat16> tag)
{
#pragma unroll
    for (int j = 0; j < 4; ++j) c[j] = fma2(and_xor(__byte_perm(w, 0u, 0x1111 * j), 0x00F0000Fu, 0x00804308u), 0x7F003E80u, 0xC000C208u, tag);
}
__device__ __forceinline__ void codes_in_order(uint32_t w, uint32_t (&c)[4], Tag<__half> tag)
{
#pragma unroll
    for (int j = 0; j < 4; ++j)
        c[j] = fma2(and_xor(__byte_perm(w, 0u, 0x1111 * j), 0x00F0000Fu, 0x64806408u), 0x2C003C00u, 0xD480E408u, tag);
}

__device__ __forceinline__ uint32_t pack2(float lo, float hi, Tag<__nv_bfloat16>)
{
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi, Tag<__half>)
{
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ float2 unpack2(uint32_t v, Tag<__nv_bfloat16>) { return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xFFFF0000u)); }
__device__ __forceinline__ float2 unpack2(uint32_t v, Tag<__half>)
{
    return make_float2(__half2float(__ushort_as_half((unsigned short)v)), __half2float(__ushort_as_half((unsigned short)(v >> 16))));
}

}  // namespace w4
}  // namespace qm
