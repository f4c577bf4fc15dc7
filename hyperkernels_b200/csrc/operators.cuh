// operators.cuh -- what the operators round the attention (qk_rotary.cu, shared_prefix.cu) share: element types and the checks of
// their views.
#pragma once

#include <algorithm>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "attn_common.cuh"

namespace hk {

// two 16-bit elements in a word; rounded to nearest, ties to even
template <class T>
__device__ __forceinline__ float2 unpack(uint32_t v);
template <>
__device__ __forceinline__ float2 unpack<__nv_bfloat16>(uint32_t v) {
    return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
}
template <>
__device__ __forceinline__ float2 unpack<__half>(uint32_t v) {
    return __half22float2(reinterpret_cast<const __half2&>(v));
}
template <class T>
__device__ __forceinline__ uint32_t pack(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack<__nv_bfloat16>(float a, float b) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return reinterpret_cast<const uint32_t&>(v);
}
template <>
__device__ __forceinline__ uint32_t pack<__half>(float a, float b) {
    const __half2 v = __floats2half2_rn(a, b);
    return reinterpret_cast<const uint32_t&>(v);
}

inline int esize(int dtype) { return dtype == HK_F32 ? 4 : 2; }

// Whether stretches of `row` elements at all places of these dimensions lie apart: from the smallest stride on, each step goes past
// all that the dimensions before it reach.  (Dimensions that interleave without meeting are not recognised; no slice or transposition
// of a tensor has such.)
struct Dim {
    int64_t n, stride;
};
template <int N>
bool lie_apart(Dim (&d)[N], int64_t row) {
    std::sort(d, d + N, [](const Dim& a, const Dim& b) { return a.stride < b.stride; });
    __int128 reach = row;
    for (const Dim& x : d) {
        if (x.n <= 1) continue;
        if (x.stride < reach) return false;
        reach += (__int128)(x.n - 1) * x.stride;
    }
    return true;
}

// A view of `n` heads whose rows the kernels read or write in pieces of up to 16 bytes.
inline int check_view(const hk_view& v, int64_t B, int64_t n, int64_t T, int dtype, bool written) {
    if (!v.ptr) return HK_ERR_NULL_POINTER;
    if (reinterpret_cast<uintptr_t>(v.ptr) & 15u) return HK_ERR_MISALIGNED;
    Dim d[] = {{B, v.strideB}, {T, v.strideM}, {n, v.strideH}};
    for (const Dim& x : d)
        if (x.n > 1 && (x.stride < 0 || x.stride % (16 / esize(dtype)))) return HK_ERR_MISALIGNED;
    return written && !lie_apart(d, HEAD_DIM) ? HK_ERR_UNSUPPORTED : HK_OK;  // rows on top of each other
}

}  // namespace hk
