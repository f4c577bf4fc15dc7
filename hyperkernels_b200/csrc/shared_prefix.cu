// shared_prefix.cu -- attention of a batch whose requests share a prefix (include/hk_attention.h: hk_shared_prefix_attention).
#include <cmath>

#include "operators.cuh"

namespace hk {
namespace {

struct PrefixArgs {
    hk_view Q, Kp, Vp, K, V, O;
    float* LSE;
    int64_t lse_sB, lse_sH;
    const int32_t* lengths;
    int B, H, group, T, P, S;  // query heads, query heads of a key head, new tokens, prefix keys, rows of the requests' caches
    float scale_log2e;
    int causal;
};

__device__ __forceinline__ float2 load2(const float* p) { return *reinterpret_cast<const float2*>(p); }
__device__ __forceinline__ float2 load2(const __nv_bfloat16* p) { return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(p)); }
__device__ __forceinline__ float2 load2(const __half* p) { return __half22float2(*reinterpret_cast<const __half2*>(p)); }
__device__ __forceinline__ void store2(float* p, float2 v) { *reinterpret_cast<float2*>(p) = v; }
__device__ __forceinline__ void store2(__nv_bfloat16* p, float2 v) { *reinterpret_cast<__nv_bfloat162*>(p) = __floats2bfloat162_rn(v.x, v.y); }
__device__ __forceinline__ void store2(__half* p, float2 v) { *reinterpret_cast<__half2*>(p) = __floats2half2_rn(v.x, v.y); }

template <class X>
__device__ __forceinline__ const X* row_of(const hk_view& v, int64_t b, int64_t h, int64_t m) {
    return static_cast<const X*>(v.ptr) + b * v.strideB + h * v.strideH + m * v.strideM;
}

// A warp per row: two elements a lane, one key after the other.
template <class X>
__global__ void __launch_bounds__(256) prefix_rows_kernel(const __grid_constant__ PrefixArgs a) {
    const int lane = threadIdx.x & 31;
    const int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (row >= (int64_t)a.B * a.H * a.T) return;
    const int i = (int)(row % a.T), h = (int)(row / a.T % a.H), b = (int)(row / a.T / a.H), hk = h / a.group;
    const int len = a.lengths ? min(max(a.lengths[b], 0), a.S) : a.S;
    const int seen = a.causal ? min(len, max(0, len - a.T + i + 1)) : len;
    float2 q = load2(row_of<X>(a.Q, b, h, i) + 2 * lane), o = make_float2(0.f, 0.f);
    q.x *= a.scale_log2e;
    q.y *= a.scale_log2e;
    float m = -INFINITY, l = 0.f;
    auto take = [&](const X* k, const X* v) {
        const float2 kk = load2(k + 2 * lane), vv = load2(v + 2 * lane);
        float s = q.x * kk.x + q.y * kk.y;
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
        const float mn = fmaxf(m, s), alpha = ex2_approx(m - mn), p = ex2_approx(s - mn);
        m = mn;
        l = l * alpha + p;
        o.x = o.x * alpha + p * vv.x;
        o.y = o.y * alpha + p * vv.y;
    };
    for (int j = 0; j < a.P; ++j) take(row_of<X>(a.Kp, 0, hk, j), row_of<X>(a.Vp, 0, hk, j));
    for (int j = 0; j < seen; ++j) take(row_of<X>(a.K, b, hk, j), row_of<X>(a.V, b, hk, j));
    const float f = l > 0.f ? 1.f / l : 0.f;
    store2(const_cast<X*>(row_of<X>(a.O, b, h, i)) + 2 * lane, make_float2(o.x * f, o.y * f));
    if (lane == 0) a.LSE[b * a.lse_sB + h * a.lse_sH + i] = l > 0.f ? (m + log2f(l)) * LN2 : -INFINITY;
}

int check(const hk_shared_prefix_params* p) {
    if (!p) return HK_ERR_NULL_POINTER;
    if (p->dtype < HK_F32 || p->dtype > HK_F16) return HK_ERR_UNSUPPORTED;
    if (p->B <= 0 || p->nh <= 0 || p->nh_kv <= 0 || p->T <= 0 || p->prefix_len < 0 || p->kv_len < 0) return HK_ERR_BAD_SHAPE;
    if (p->nh % p->nh_kv) return HK_ERR_BAD_SHAPE;
    if (p->T > (1 << 30) || p->prefix_len > (1 << 30) || p->kv_len > (1 << 30)) return HK_ERR_BAD_SHAPE;
    if ((int64_t)p->B * p->nh > (1 << 24) || (int64_t)p->B * p->nh * p->T > (1LL << 30)) return HK_ERR_BAD_SHAPE;
    if (!std::isfinite(p->scale) || p->scale == 0.f) return HK_ERR_BAD_SHAPE;
    int rc;
    if ((rc = check_view(p->Q, p->B, p->nh, p->T, p->dtype, false)) || (rc = check_view(p->O, p->B, p->nh, p->T, p->dtype, true))) return rc;
    for (const hk_view* v : {&p->Kp, &p->Vp})
        if (p->prefix_len > 0 && (rc = check_view(*v, 1, p->nh_kv, p->prefix_len, p->dtype, false))) return rc;
    for (const hk_view* v : {&p->K, &p->V})
        if (p->kv_len > 0 && (rc = check_view(*v, p->B, p->nh_kv, p->kv_len, p->dtype, false))) return rc;
    if (!p->LSE) return HK_ERR_NULL_POINTER;
    if ((reinterpret_cast<uintptr_t>(p->LSE) | reinterpret_cast<uintptr_t>(p->lengths)) & 3u) return HK_ERR_MISALIGNED;
    return HK_OK;
}

}  // namespace
}  // namespace hk

using namespace hk;

extern "C" {

size_t hk_shared_prefix_workspace_bytes(const hk_shared_prefix_params*) { return 0; }

int hk_shared_prefix_attention(const hk_shared_prefix_params* p, void* stream) {
    const int rc = check(p);
    if (rc != HK_OK) return rc;
    PrefixArgs a{};
    a.Q = p->Q; a.Kp = p->Kp; a.Vp = p->Vp; a.K = p->K; a.V = p->V; a.O = p->O;
    a.LSE = p->LSE; a.lse_sB = p->lse_strideB; a.lse_sH = p->lse_strideH;
    a.lengths = p->lengths;
    a.B = p->B; a.H = p->nh; a.group = p->nh / p->nh_kv; a.T = (int)p->T; a.P = (int)p->prefix_len; a.S = (int)p->kv_len;
    a.scale_log2e = p->scale * LOG2E;
    a.causal = p->is_causal;
    const int64_t rows = (int64_t)p->B * p->nh * p->T;
    auto kernel = p->dtype == HK_F32 ? prefix_rows_kernel<float> : p->dtype == HK_BF16 ? prefix_rows_kernel<__nv_bfloat16> : prefix_rows_kernel<__half>;
    kernel<<<(unsigned)((rows + 7) / 8), 256, 0, static_cast<cudaStream_t>(stream)>>>(a);
    count_launch();
    return check_launch();
}

}  // extern "C"
