// tile_math.cuh -- pieces of the kernels that take 128 rows against tiles of keys on tcgen05 (shared_prefix_sm100.cu,
// serving_sm100.cu): products of 16-bit operands, the low parts of fp32 ones, exponentials beside the special function unit.
#pragma once

#include <type_traits>

#include "operators.cuh"

namespace hk {

// tcgen05.mma of 16-bit operands (K = 16), one CTA
__host__ __device__ constexpr uint32_t make_idesc_16(int M, int N, bool bf16, bool b_mn_major) {
    const uint32_t fmt = bf16 ? 1u : 0u;
    return (1u << 4) | (fmt << 7) | (fmt << 10) | ((b_mn_major ? 1u : 0u) << 16) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}
constexpr uint32_t IDESC_NEGATE_A = 1u << 13;
__device__ __forceinline__ void umma_ss_16(uint32_t leader, uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n"
        ".reg .pred p, q;\n"
        "setp.ne.b32 p, %4, 0;\n"
        "setp.ne.b32 q, %5, 0;\n"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n"
        "}\n"
        ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc), "r"(leader)
        : "memory");
}
__device__ __forceinline__ void umma_ts_16(uint32_t leader, uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n"
        ".reg .pred p, q;\n"
        "setp.ne.b32 p, %4, 0;\n"
        "setp.ne.b32 q, %5, 0;\n"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n"
        "}\n"
        ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(acc), "r"(leader)
        : "memory");
}

// What the tensor core leaves of an fp32 word when it cuts it off to TF32, rounded to nearest, since it is cut off too: always
// towards zero, every product would be a little too small.
__device__ __forceinline__ uint32_t tf32_rest(uint32_t x) { return __float_as_uint(__uint_as_float(x) - __uint_as_float(x & 0xffffe000u)) + 0x1000u; }

// 2^x of two numbers, for x >= -126, without the special function unit, which is what the softmax of 16-bit types is bound by: x is
// split into the nearest whole number, which goes to the exponent, and the rest, of whose power a polynomial (least relative error on
// [-1/2, 1/2], found by reweighted least squares) is 2.7e-6 off.
__device__ __forceinline__ float2 ex2_poly(float2 x) {
    const float2 big = make_float2(12582912.f, 12582912.f), minus = make_float2(-12582912.f, -12582912.f);  // 1.5 * 2^23
    x = make_float2(fmaxf(x.x, -126.f), fmaxf(x.y, -126.f));
    const float2 t = __fadd2_rn(x, big), n = __fadd2_rn(t, minus), f = __ffma2_rn(n, make_float2(-1.f, -1.f), x);
    float2 p = __ffma2_rn(f, make_float2(9.5701022e-3f, 9.5701022e-3f), make_float2(5.5917859e-2f, 5.5917859e-2f));
    p = __ffma2_rn(p, f, make_float2(0.24024744f, 0.24024744f));
    p = __ffma2_rn(p, f, make_float2(0.69312179f, 0.69312179f));
    p = __ffma2_rn(p, f, make_float2(0.99999928f, 0.99999928f));
    return make_float2(__uint_as_float(__float_as_uint(p.x) + (__float_as_uint(t.x) << 23)), __uint_as_float(__float_as_uint(p.y) + (__float_as_uint(t.y) << 23)));
}

// The largest of three, or NaN if one is.
__device__ __forceinline__ float max3_or_nan(float a, float b, float c) {
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// The 2^ of what a softmax's reference lies below the row's largest score.  A weight takes the type of the values, and fp16 has none below
// 2^-24: with the largest at 2^7 (2^15 where a stale maximum may lie 2^8 lower), those down to 2^-31 of it are kept, where many of
// them would be lost beside one that is large.  The sums and the LSE take it back by themselves.
template <class X>
__host__ __device__ constexpr float lift() { return std::is_same<X, __half>::value ? 7.f : 0.f; }

// Tiles of `rows` rows of a view of keys or values, all heads and batches (tma_load_tile): 128 bytes of each row side by side,
// swizzled; fp32 rows are two such pieces.  mn_major: the values as an MN-major operand of fp32 products.
// lines: 128 bytes are brought into the L2, not 256; for rows of 16-bit types whose neighbours are asked for by others, at other times.
int prefix_tile_map(CUtensorMap* map, const hk_view& v, int dtype, int64_t B, int H, int64_t T, int rows, bool mn_major, bool lines = false);

}  // namespace hk
