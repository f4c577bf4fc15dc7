// qk_rotary.cu -- what stands between the projections and the attention: rotary positions with several axes and RMS norms of
// every query and key row with the rotation in the same pass, and their backward passes.  include/hk_attention.h has the
// formulas.
//
// Every call is bound by HBM: each row is read and written once, and the arithmetic of a row (about 10 operations an element
// backward) is a fraction of what an SM can do meanwhile.  A warp takes a token and goes through its heads: the 32 lanes
// compute the 32 pairs' sines and cosines once, and all heads use them.  Eight lanes share a row, each with elements
// 4 s .. 4 s + 3 and 32 + 4 s .. 32 + 4 s + 3, so both halves of a pair are in one lane whether pairs are neighbours or half a
// row apart, and a load instruction of a warp takes whole 128-byte lines of four rows.
#include <cmath>

#include "operators.cuh"

namespace hk {
namespace {

enum QkMode { QK_ROTATE = 0, QK_NORM = 1, QK_NORM_BACK = 2 };
constexpr int QK_WARPS = 8;
constexpr int QK_BACK_CTAS = 4;  // per SM at most: room in the workspace

struct RowView {
    char* ptr;
    int64_t sB, sM, sH;  // bytes
};

struct QkArgs {
    RowView x[2], y[2], dx[2];  // [queries, keys]; y: results forward, their gradients backward
    const void* w[2];
    const void* positions;
    int64_t pA, pB, pT;
    float* partial;
    int nh, rows;  // query heads, heads of both
    uint32_t T, units;
    int per_unit, units_per_token;  // heads a warp takes with one set of angles
    int pos64, w_dtype, back;
    float eps;
    hk_rotary_plan plan;
};

__device__ __forceinline__ float4 load4(const float* p) { return __ldcs(reinterpret_cast<const float4*>(p)); }
template <class T>
__device__ __forceinline__ float4 load4(const T* p) {
    const uint2 v = __ldcs(reinterpret_cast<const uint2*>(p));
    const float2 a = unpack<T>(v.x), b = unpack<T>(v.y);
    return make_float4(a.x, a.y, b.x, b.y);
}
__device__ __forceinline__ void store4(float* p, float4 v) { *reinterpret_cast<float4*>(p) = v; }
template <class T>
__device__ __forceinline__ void store4(T* p, float4 v) {
    *reinterpret_cast<uint2*>(p) = make_uint2(pack<T>(v.x, v.y), pack<T>(v.z, v.w));
}

struct Row8 {
    float v[8];  // elements 4 s .. 4 s + 3, then 32 + 4 s ..
};
template <class T>
__device__ __forceinline__ Row8 load_row(const char* p, int sub) {
    const float4 a = load4(reinterpret_cast<const T*>(p) + 4 * sub), b = load4(reinterpret_cast<const T*>(p) + 32 + 4 * sub);
    return Row8{{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w}};
}
// The same row as 16-bit words, kept for the elements that do not change: their way through fp32 gives a NaN other bits.
struct Words {
    uint32_t w[4];
};
template <class T>
__device__ __forceinline__ Row8 load_row(const char* p, int sub, Words& raw) {
    const uint2 a = __ldcs(reinterpret_cast<const uint2*>(p) + sub), b = __ldcs(reinterpret_cast<const uint2*>(p + 64) + sub);
    raw = {{a.x, a.y, b.x, b.y}};
    Row8 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = unpack<T>(raw.w[i]);
        r.v[2 * i] = f.x;
        r.v[2 * i + 1] = f.y;
    }
    return r;
}
template <class T>
__device__ __forceinline__ void store_row(char* p, int sub, const Row8& r, const Words& raw, const Words& keep) {
    uint32_t o[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = (pack<T>(r.v[2 * i], r.v[2 * i + 1]) & ~keep.w[i]) | (raw.w[i] & keep.w[i]);
    reinterpret_cast<uint2*>(p)[sub] = make_uint2(o[0], o[1]);
    reinterpret_cast<uint2*>(p + 64)[sub] = make_uint2(o[2], o[3]);
}
template <class T>
__device__ __forceinline__ void store_row(char* p, int sub, const Row8& r) {
    store4(reinterpret_cast<T*>(p) + 4 * sub, make_float4(r.v[0], r.v[1], r.v[2], r.v[3]));
    store4(reinterpret_cast<T*>(p) + 32 + 4 * sub, make_float4(r.v[4], r.v[5], r.v[6], r.v[7]));
}
__device__ __forceinline__ float weight_at(const void* w, int dtype, int i) {
    return !w ? 1.f
           : dtype == HK_BF16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(w)[i])
           : dtype == HK_F16  ? __half2float(static_cast<const __half*>(w)[i])
                              : static_cast<const float*>(w)[i];
}

// A pair that does not turn (a still one, position 0) keeps its elements whatever the other one holds: 0 times an infinity
// would be NaN, and a NaN would come out as another one.
__device__ __forceinline__ bool is_still(float c, float s) { return c == 1.f && s == 0.f; }
__device__ __forceinline__ void turn(float& a, float& b, float c, float s) {
    const float p = fmaf(-b, s, a * c), q = fmaf(a, s, b * c);
    a = is_still(c, s) ? a : p;
    b = is_still(c, s) ? b : q;
}
__device__ __forceinline__ void rotate(Row8& r, const float (&c)[4], const float (&s)[4], bool interleaved) {
    if (interleaved) {
#pragma unroll
        for (int i = 0; i < 4; ++i) turn(r.v[2 * i], r.v[2 * i + 1], c[i], s[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) turn(r.v[i], r.v[i + 4], c[i], s[i]);
    }
}
__device__ __forceinline__ float sum8(float x) {  // over the eight lanes of a row
#pragma unroll
    for (int off = 4; off > 0; off >>= 1) x += __shfl_xor_sync(0xffffffffu, x, off);
    return x;
}
__device__ __forceinline__ float rms_inverse(const Row8& x, float eps) {
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) ss = fmaf(x.v[i], x.v[i], ss);
    return rsqrtf(fmaf(sum8(ss), 1.f / 64.f, eps));
}

// U rows of each of the warp's four groups of lanes are loaded before the first is used.
template <class X, class Y, int MODE, int U>
__global__ void __launch_bounds__(QK_WARPS * 32) qk_rotary_kernel(const __grid_constant__ QkArgs a) {
    constexpr bool KEEPS = MODE == QK_ROTATE && sizeof(X) == 2 && sizeof(Y) == 2;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, grp = lane >> 3, sub = lane & 7;
    const uint64_t my_turn = a.plan.turn[lane];
    const int my_axis = a.plan.axis[lane];
    const bool interleaved = a.plan.interleaved != 0;
    pdl_wait();
    pdl_trigger();
    float w[2][MODE == QK_ROTATE ? 1 : 8], dw[2][MODE == QK_NORM_BACK ? 8 : 1];
    if (MODE != QK_ROTATE)
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int i = 0; i < 8; ++i) w[k][i] = weight_at(a.w[k], a.w_dtype, (i < 4 ? 0 : 28) + 4 * sub + i);
    if (MODE == QK_NORM_BACK)
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int i = 0; i < 8; ++i) dw[k][i] = 0.f;

    for (uint32_t u = blockIdx.x * QK_WARPS + warp; u < a.units; u += gridDim.x * QK_WARPS) {
        const uint32_t token = u / a.units_per_token, b = token / a.T, t = token - b * a.T;
        const int first = (int)(u - token * a.units_per_token) * a.per_unit, end = min(first + a.per_unit, a.rows);
        float c[4], s[4];
        {
            uint64_t angle = 0;
            if (my_axis != HK_ROTARY_STILL) {
                const int64_t at = my_axis * a.pA + b * a.pB + t * a.pT;
                angle = my_turn * (uint64_t)(a.pos64 ? static_cast<const int64_t*>(a.positions)[at] : (int64_t)static_cast<const int32_t*>(a.positions)[at]);
            }
            float mc, ms;
            sincospif((float)(int32_t)(angle >> 32) * 0x1p-31f, &ms, &mc);
            if (a.back) ms = -ms;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int pair = interleaved ? (i < 2 ? 2 * sub + i : 16 + 2 * sub + i - 2) : 4 * sub + i;
                c[i] = __shfl_sync(0xffffffffu, mc, pair);
                s[i] = __shfl_sync(0xffffffffu, ms, pair);
            }
        }
        Words keep;  // which of a row's 16-bit elements stay as they are
        if (KEEPS) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int lo = (2 * i) & 3, hi = lo + 1;
                keep.w[i] = interleaved ? (is_still(c[i], s[i]) ? 0xffffffffu : 0u)
                                        : (is_still(c[lo], s[lo]) ? 0xffffu : 0u) | (is_still(c[hi], s[hi]) ? 0xffff0000u : 0u);
            }
        }
        auto row = [&](const RowView* v, int r) {
            const int k = r >= a.nh;
            return v[k].ptr + b * v[k].sB + t * v[k].sM + (r - (k ? a.nh : 0)) * v[k].sH;
        };
        for (int r0 = first; r0 < end; r0 += 4 * U) {
            Row8 x[U], g[MODE == QK_NORM_BACK ? U : 1];
            Words raw[KEEPS ? U : 1];
#pragma unroll
            for (int i = 0; i < U; ++i) {
                const int r = min(r0 + 4 * i + grp, end - 1);  // behind the end: computed and not used
                if constexpr (KEEPS) x[i] = load_row<X>(row(a.x, r), sub, raw[i]);
                else x[i] = load_row<X>(row(a.x, r), sub);
                if (MODE == QK_NORM_BACK) g[i] = load_row<Y>(row(a.y, r), sub);
            }
#pragma unroll
            for (int i = 0; i < U; ++i) {
                const int r = r0 + 4 * i + grp;
                const bool k = r >= a.nh, valid = r < end;
                if (MODE == QK_ROTATE) {
                    rotate(x[i], c, s, interleaved);
                    if constexpr (KEEPS) {
                        if (valid) store_row<Y>(row(a.y, r), sub, x[i], raw[i], keep);
                    } else if (valid) {
                        store_row<Y>(row(a.y, r), sub, x[i]);
                    }
                } else if (MODE == QK_NORM) {
                    const float inv = rms_inverse(x[i], a.eps);
#pragma unroll
                    for (int e = 0; e < 8; ++e) x[i].v[e] *= inv * (k ? w[1][e] : w[0][e]);
                    rotate(x[i], c, s, interleaved);
                    if (valid) store_row<Y>(row(a.y, r), sub, x[i]);
                } else {
                    const float inv = rms_inverse(x[i], a.eps);
                    rotate(g[i], c, s, interleaved);
                    float dot = 0.f;
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        x[i].v[e] *= inv;
                        const float gx = g[i].v[e] * x[i].v[e];
                        dw[0][e] += valid && !k ? gx : 0.f;
                        dw[1][e] += valid && k ? gx : 0.f;
                        g[i].v[e] *= k ? w[1][e] : w[0][e];
                        dot = fmaf(g[i].v[e], x[i].v[e], dot);
                    }
                    dot = sum8(dot) * (1.f / 64.f);
#pragma unroll
                    for (int e = 0; e < 8; ++e) g[i].v[e] = inv * fmaf(-x[i].v[e], dot, g[i].v[e]);
                    if (valid) store_row<X>(row(a.dx, r), sub, g[i]);
                }
            }
        }
    }
    if (MODE == QK_NORM_BACK) {  // sums of the CTA's rows: [queries, keys][64]
        __shared__ float sums[QK_WARPS * 4][2][64];
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int e = 0; e < 8; ++e) sums[threadIdx.x >> 3][k][(e < 4 ? 0 : 28) + 4 * sub + e] = dw[k][e];
        __syncthreads();
        if (threadIdx.x < 128) {
            float x = 0.f;
#pragma unroll
            for (int i = 0; i < QK_WARPS * 4; ++i) x += sums[i][threadIdx.x >> 6][threadIdx.x & 63];
            a.partial[blockIdx.x * 128 + threadIdx.x] = x;
        }
    }
}

// The CTAs' sums, 16 columns a CTA, 16 threads a column; always in the same order.
__global__ void __launch_bounds__(256) qk_weight_sum_kernel(const float* partial, int n, float* dq, float* dk) {
    __shared__ float sums[16][17];
    const int col = threadIdx.x & 15, part = threadIdx.x >> 4, at = blockIdx.x * 16 + col;
    pdl_wait();
    pdl_trigger();
    float x = 0.f;
#pragma unroll 4
    for (int i = part; i < n; i += 16) x += partial[i * 128 + at];
    sums[part][col] = x;
    __syncthreads();
    if (part == 0) {
#pragma unroll
        for (int i = 1; i < 16; ++i) x += sums[i][col];
        float* to = at < 64 ? dq : dk;
        if (to) to[at & 63] = x;
    }
}

RowView row_view(const hk_view& v, int dtype) {
    const int64_t e = esize(dtype);
    return {static_cast<char*>(v.ptr), v.strideB * e, v.strideM * e, v.strideH * e};
}

template <int MODE, int U>
using QkKernel = void (*)(QkArgs);

template <int MODE, int U>
QkKernel<MODE, U> pick(int x, int y) {
    typedef __nv_bfloat16 bf16;
    if (x == HK_F32 && y == HK_F32) return qk_rotary_kernel<float, float, MODE, U>;
    if (x == HK_BF16 && y == HK_BF16) return qk_rotary_kernel<bf16, bf16, MODE, U>;
    if (x == HK_F16 && y == HK_F16) return qk_rotary_kernel<__half, __half, MODE, U>;
    if (x == HK_BF16 && y == HK_F32) return qk_rotary_kernel<bf16, float, MODE, U>;
    if (x == HK_F16 && y == HK_F32) return qk_rotary_kernel<__half, float, MODE, U>;
    if constexpr (MODE == QK_ROTATE) {  // gradients from the attention back to the projection's type
        if (x == HK_F32 && y == HK_BF16) return qk_rotary_kernel<float, bf16, MODE, U>;
        if (x == HK_F32 && y == HK_F16) return qk_rotary_kernel<float, __half, MODE, U>;
    }
    return nullptr;
}

int qk_run(const hk_qk_params* p, int mode, bool back, cudaStream_t stream) {
    if (!p) return HK_ERR_NULL_POINTER;
    if (p->B <= 0 || p->nh <= 0 || p->nh_k < 0 || p->T <= 0 || p->T > (1 << 30)) return HK_ERR_BAD_SHAPE;
    if ((int64_t)p->nh + p->nh_k > (1 << 20) || (int64_t)p->B * p->T >= (1LL << 31)) return HK_ERR_BAD_SHAPE;
    for (int d : {p->dtype, p->out_dtype})
        if (d < HK_F32 || d > HK_F16) return HK_ERR_UNSUPPORTED;
    if (p->dtype != p->out_dtype && p->dtype != HK_F32 && p->out_dtype != HK_F32) return HK_ERR_UNSUPPORTED;
    if (mode != QK_ROTATE) {
        if (p->out_dtype != p->dtype && p->out_dtype != HK_F32) return HK_ERR_UNSUPPORTED;
        if ((p->q_weight || p->k_weight) && p->weight_dtype != HK_F32 && p->weight_dtype != p->dtype) return HK_ERR_UNSUPPORTED;
        if (!(p->eps >= 0.f) || !std::isfinite(p->eps)) return HK_ERR_BAD_SHAPE;
    }
    if (p->pos_bits != 32 && p->pos_bits != 64) return HK_ERR_UNSUPPORTED;
    int axes = 0;  // 1 + the last axis that a pair asks for
    for (int i = 0; i < 32; ++i)
        if (p->plan.axis[i] != HK_ROTARY_STILL) axes = p->plan.axis[i] >= axes ? p->plan.axis[i] + 1 : axes;
    if (p->plan.n_axes < axes) return HK_ERR_BAD_SHAPE;
    if (axes > 0 && !p->positions) return HK_ERR_NULL_POINTER;
    if (reinterpret_cast<uintptr_t>(p->positions) & (p->pos_bits / 8 - 1)) return HK_ERR_MISALIGNED;

    QkArgs a{};
    const int n[2] = {p->nh, p->nh_k};
    // [read, written, read beside it]: the rotation reads the gradients when it goes backward
    const hk_view* src[2] = {back && mode == QK_ROTATE ? &p->dq_out : &p->q, back && mode == QK_ROTATE ? &p->dk_out : &p->k};
    const hk_view* dst[2] = {back ? &p->dq : &p->q_out, back ? &p->dk : &p->k_out};
    const hk_view* grad[2] = {&p->dq_out, &p->dk_out};
    const int src_t = back && mode == QK_ROTATE ? p->out_dtype : p->dtype, dst_t = back ? p->dtype : p->out_dtype;
    for (int k = 0; k < 2; ++k) {
        if (n[k] == 0) continue;
        int rc;
        if ((rc = check_view(*src[k], p->B, n[k], p->T, src_t, false)) || (rc = check_view(*dst[k], p->B, n[k], p->T, dst_t, true))) return rc;
        if (mode == QK_NORM_BACK && (rc = check_view(*grad[k], p->B, n[k], p->T, p->out_dtype, false))) return rc;
        a.x[k] = row_view(*src[k], src_t);
        if (mode == QK_NORM_BACK) {
            a.y[k] = row_view(*grad[k], p->out_dtype);
            a.dx[k] = row_view(*dst[k], dst_t);
        } else {
            a.y[k] = row_view(*dst[k], dst_t);
        }
        if (mode != QK_ROTATE) {
            a.w[k] = k ? p->k_weight : p->q_weight;
            if (reinterpret_cast<uintptr_t>(a.w[k]) & (esize(p->weight_dtype) - 1)) return HK_ERR_MISALIGNED;
        }
    }
    if (mode == QK_NORM_BACK) {
        if (!p->workspace || p->workspace_bytes < hk_qk_norm_rotary_workspace_bytes(p) || (reinterpret_cast<uintptr_t>(p->workspace) & 15u))
            return HK_ERR_WORKSPACE;
        if ((reinterpret_cast<uintptr_t>(p->dq_weight) | reinterpret_cast<uintptr_t>(p->dk_weight)) & 3u) return HK_ERR_MISALIGNED;
        a.partial = static_cast<float*>(p->workspace);
    }
    a.positions = p->positions;
    a.pA = p->pos_strideA; a.pB = p->pos_strideB; a.pT = p->pos_strideT;
    a.nh = p->nh; a.rows = p->nh + p->nh_k;
    a.T = (uint32_t)p->T;
    a.pos64 = p->pos_bits == 64;
    a.w_dtype = p->weight_dtype;
    a.back = back;
    a.eps = p->eps;
    a.plan = p->plan;

    constexpr int U_FWD = 4, U_BACK = 2;
    const int step = 4 * (mode == QK_NORM_BACK ? U_BACK : U_FWD);
    const uint32_t tokens = (uint32_t)(p->B * p->T);
    // Few tokens: a warp takes as few heads as keep its loads in flight, so that more SMs take part.
    a.per_unit = a.rows;
    if (tokens < (uint32_t)sm_count() * 16) a.per_unit = tokens * ((a.rows + step - 1) / step) < (uint32_t)sm_count() * QK_WARPS ? 4 : step;
    a.units_per_token = (a.rows + a.per_unit - 1) / a.per_unit;
    a.units = tokens * a.units_per_token;
    uint32_t blocks = (a.units + QK_WARPS - 1) / QK_WARPS;
    QkKernel<0, 0> kernel = mode == QK_ROTATE ? pick<QK_ROTATE, U_FWD>(src_t, dst_t)
                            : mode == QK_NORM ? pick<QK_NORM, U_FWD>(src_t, dst_t)
                                              : pick<QK_NORM_BACK, U_BACK>(src_t, p->out_dtype);
    if (!kernel) return HK_ERR_UNSUPPORTED;
    if (mode == QK_NORM_BACK) blocks = std::min(blocks, (uint32_t)sm_count() * 2);
    LaunchConfig lc(blocks, QK_WARPS * 32, 0, stream, 1, true);
    if (cudaLaunchKernelEx(&lc.cfg, kernel, a) != cudaSuccess) return check_launch();
    count_launch();
    if (mode == QK_NORM_BACK && (p->dq_weight || p->dk_weight)) {
        LaunchConfig sum(8, 256, 0, stream, 1, true);
        if (cudaLaunchKernelEx(&sum.cfg, qk_weight_sum_kernel, (const float*)a.partial, (int)blocks, p->dq_weight, p->dk_weight) != cudaSuccess)
            return check_launch();
        count_launch();
    }
    return check_launch();
}

}  // namespace
}  // namespace hk

using namespace hk;

extern "C" {

int hk_rotary_plan_fill(hk_rotary_plan* plan, int n_axes, const int* sections, double base, const double* frequency, int interleaved) {
    if (!plan || !sections) return HK_ERR_NULL_POINTER;
    if (n_axes < 1 || n_axes > 32 || (!frequency && !(base > 0.0 && std::isfinite(base)))) return HK_ERR_BAD_SHAPE;
    hk_rotary_plan r{};
    int n = 0;
    for (int a = 0; a < n_axes; ++a) {
        if (sections[a] < 0 || sections[a] > 32 - n) return HK_ERR_BAD_SHAPE;
        for (int i = 0; i < sections[a]; ++i, ++n) {
            const double f = frequency ? frequency[n] : std::pow(base, -n / 32.0);
            if (!std::isfinite(f)) return HK_ERR_BAD_SHAPE;
            // turns per position without whole ones, which an integer position turns into whole turns again
            const long double turns = (long double)f / 6.283185307179586476925286766559005768L;
            const long double part = turns - std::floor(turns);
            const long double scaled = std::nearbyint(std::ldexp(part, 64));
            r.turn[n] = scaled >= 18446744073709551616.0L ? 0u : (uint64_t)scaled;
            r.axis[n] = (uint8_t)a;
        }
    }
    for (; n < 32; ++n) r.axis[n] = HK_ROTARY_STILL;
    r.n_axes = n_axes;
    r.interleaved = interleaved != 0;
    *plan = r;
    return HK_OK;
}

int hk_rotary_forward(const hk_qk_params* p, void* stream) { return qk_run(p, QK_ROTATE, false, static_cast<cudaStream_t>(stream)); }
int hk_rotary_backward(const hk_qk_params* p, void* stream) { return qk_run(p, QK_ROTATE, true, static_cast<cudaStream_t>(stream)); }
int hk_qk_norm_rotary_forward(const hk_qk_params* p, void* stream) { return qk_run(p, QK_NORM, false, static_cast<cudaStream_t>(stream)); }
int hk_qk_norm_rotary_backward(const hk_qk_params* p, void* stream) { return qk_run(p, QK_NORM_BACK, true, static_cast<cudaStream_t>(stream)); }

size_t hk_qk_norm_rotary_workspace_bytes(const hk_qk_params*) { return (size_t)sm_count() * QK_BACK_CTAS * 128 * sizeof(float); }

}  // extern "C"
