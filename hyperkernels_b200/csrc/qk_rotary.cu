// qk_rotary.cu -- what stands between the projections and the attention: rotary positions with several axes and RMS norms of
// every query and key row with the rotation in the same pass, and their backward passes.  include/hk_attention.h has the
// formulas.
//
// Every call is bound by HBM: each row is read and written once, and the arithmetic of a row (about 10 operations an element
// backward) is a fraction of what an SM can do meanwhile.  A warp takes a token and goes through the heads of its queries, or of its
// keys: the 32 lanes compute the 32 pairs' sines and cosines once, and all heads use them.  Eight lanes share a row, each with
// elements 4 s .. 4 s + 3 and 32 + 4 s .. 32 + 4 s + 3, so both halves of a pair are in one lane whether pairs are neighbours or half a
// row apart, and a load instruction of a warp takes whole 128-byte lines of four rows.  The rows of the next step are on their way
// while a step is worked on.
//
// Measured (a plain copy runs at 6.54 TB/s): B8, 12 and 12 heads, T 1024, fp32, rotation 17.9 us (86 % of that rate), norm 19.6 (79 %), its
// backward pass 31.1 (74 %, of which the weights' sums about 2); T 32768, 32 and 32 heads, bf16 rows and fp32 gradients 188 us
// (87 %); T 32767, 32 and 8 heads, fp32 gradients into bf16 84 us (92 %).  One token of 16 or 64 requests 1.9 to 2.3 us.  Three CTAs to an SM
// would leave 80 registers a thread, and what is on its way would not fit them (spills: 37.7 us instead of 20.1, 223 instead of 90).
#include <cmath>

#include "operators.cuh"

namespace hk {
namespace {

enum QkMode { QK_ROTATE = 0, QK_NORM = 1, QK_NORM_BACK = 2 };
constexpr int QK_WARPS = 8;
constexpr int QK_CTAS = 2;  // that an SM holds
constexpr int64_t L2_BYTES = 126 << 20;

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
    int heads[2];
    uint32_t T, tokens, blocks_q;  // CTAs that take queries; the others take keys
    int split;                     // a warp takes one step of a token's heads, not all of them
    int past;                      // results are more than the L2 keeps
    int pos64, w_dtype, back;
    float eps;
    hk_rotary_plan plan;
};

// A lane's part of a row as it is in memory, and as numbers: elements 4 s .. 4 s + 3, then 32 + 4 s ..
template <class T>
struct Raw {
    uint32_t w[2 * sizeof(T)];
    __device__ __forceinline__ void load(const char* p, int sub) {
        if constexpr (sizeof(T) == 4) {
            const uint4 a = __ldcs(reinterpret_cast<const uint4*>(p) + sub), b = __ldcs(reinterpret_cast<const uint4*>(p + 128) + sub);
            w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w; w[4] = b.x; w[5] = b.y; w[6] = b.z; w[7] = b.w;
        } else {
            const uint2 a = __ldcs(reinterpret_cast<const uint2*>(p) + sub), b = __ldcs(reinterpret_cast<const uint2*>(p + 64) + sub);
            w[0] = a.x; w[1] = a.y; w[2] = b.x; w[3] = b.y;
        }
    }
};
struct Row8 {
    float v[8];
};
template <class T>
__device__ __forceinline__ Row8 numbers(const Raw<T>& x) {
    Row8 r;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 8; ++i) r.v[i] = __uint_as_float(x.w[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = unpack<T>(x.w[i]);
            r.v[2 * i] = f.x;
            r.v[2 * i + 1] = f.y;
        }
    }
    return r;
}
// keep: which bits of 16-bit words are those of `raw`; their way through fp32 would give a NaN other ones
struct Keep {
    uint32_t w[4];
};
// With the policy of the results' way through the L2 (two stores to choose from took norm of B8 T1024 from 20.1 to 20.8 us).
__device__ __forceinline__ void store(float4* p, float4 x, uint64_t policy) {
    asm volatile("st.global.L2::cache_hint.v4.f32 [%0], {%1,%2,%3,%4}, %5;" ::"l"(p), "f"(x.x), "f"(x.y), "f"(x.z), "f"(x.w), "l"(policy) : "memory");
}
__device__ __forceinline__ void store(uint2* p, uint2 x, uint64_t policy) {
    asm volatile("st.global.L2::cache_hint.v2.b32 [%0], {%1,%2}, %3;" ::"l"(p), "r"(x.x), "r"(x.y), "l"(policy) : "memory");
}
template <class T, bool KEEPS>
__device__ __forceinline__ void store_row(char* p, int sub, const Row8& r, const uint32_t* raw, const Keep& keep, uint64_t policy) {
    if constexpr (sizeof(T) == 4) {
        store(reinterpret_cast<float4*>(p) + sub, make_float4(r.v[0], r.v[1], r.v[2], r.v[3]), policy);
        store(reinterpret_cast<float4*>(p + 128) + sub, make_float4(r.v[4], r.v[5], r.v[6], r.v[7]), policy);
    } else {
        uint32_t o[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            o[i] = pack<T>(r.v[2 * i], r.v[2 * i + 1]);
            if (KEEPS) o[i] = (o[i] & ~keep.w[i]) | (raw[i] & keep.w[i]);
        }
        store(reinterpret_cast<uint2*>(p) + sub, make_uint2(o[0], o[1]), policy);
        store(reinterpret_cast<uint2*>(p + 64) + sub, make_uint2(o[2], o[3]), policy);
    }
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
// Sums over the eight lanes of a row, of several rows side by side: one after the other, they would be a chain of
// shuffles (norm of B8 T1024 20.3 us instead of 19.5).
template <int U>
__device__ __forceinline__ void sum8(float (&x)[U]) {
#pragma unroll
    for (int off = 4; off > 0; off >>= 1)
#pragma unroll
        for (int i = 0; i < U; ++i) x[i] += __shfl_xor_sync(0xffffffffu, x[i], off);
}
template <class T, int U>
__device__ __forceinline__ void rms_inverse(const Raw<T> (&x)[U], float eps, float (&inv)[U]) {
#pragma unroll
    for (int i = 0; i < U; ++i) {
        const Row8 r = numbers(x[i]);
        inv[i] = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) inv[i] = fmaf(r.v[e], r.v[e], inv[i]);
    }
    sum8(inv);
#pragma unroll
    for (int i = 0; i < U; ++i) inv[i] = rsqrtf(fmaf(inv[i], 1.f / 64.f, eps));
}

// U rows of each of the warp's four groups of lanes are a step.  TOKENS: the groups take four tokens that follow each other, and each
// U heads; otherwise all take the same token, and four heads after each other.  Whichever dimension's rows are next to each other in
// memory: rows of 16 bits, head by head in memory, run at 70 % of the copy rate when a load takes four of them out of four heads.
template <class X, class Y, int MODE, int U, bool TOKENS>
__global__ void __launch_bounds__(QK_WARPS * 32, QK_CTAS) qk_rotary_kernel(const __grid_constant__ QkArgs a) {
    constexpr bool KEEPS = MODE == QK_ROTATE && sizeof(X) == 2 && sizeof(Y) == 2, BACK = MODE == QK_NORM_BACK;
    constexpr int STEP = TOKENS ? U : 4 * U, HOP = TOKENS ? 1 : 4;  // heads of a step, and from a lane's to its next
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, grp = lane >> 3, sub = lane & 7, first_head = TOKENS ? 0 : grp;
    const int k = blockIdx.x >= a.blocks_q;
    const uint32_t block = blockIdx.x - (k ? a.blocks_q : 0u), blocks = k ? gridDim.x - a.blocks_q : a.blocks_q;
    const int heads = a.heads[k];
    const RowView vx = a.x[k], vy = a.y[k], vd = a.dx[k];
    const bool interleaved = a.plan.interleaved != 0;
    // a lane's pairs: with TOKENS the four that it turns; otherwise one of the token's 32, which the lanes hand to each other
    constexpr int PAIRS = TOKENS ? 4 : 1;
    auto turned_by = [&](int i) { return interleaved ? (i < 2 ? 2 * sub + i : 16 + 2 * sub + i - 2) : 4 * sub + i; };
    const uint64_t turn_of_lane = a.plan.turn[lane];
    const int axis_of_lane = a.plan.axis[lane];
    auto my_turn = [&](int i) { return TOKENS ? a.plan.turn[turned_by(i)] : turn_of_lane; };
    auto my_axis = [&](int i) { return TOKENS ? (int)a.plan.axis[turned_by(i)] : axis_of_lane; };
    // strips: all heads of a token (of four), or one step of them
    const uint32_t per_token = a.split ? (heads + STEP - 1) / STEP : 1, strips = TOKENS ? (a.tokens + 3) / 4 : a.tokens * per_token, hop = blocks * QK_WARPS;
    struct Place {
        uint32_t strip;
        int64_t x, y, d;  // offsets of the token's first row
        int64_t pos;
        int head, end;    // first of the step, end of the strip (0: no token for this lane)
    };
    auto place = [&](uint32_t strip) {
        Place p;
        p.strip = strip;
        const uint32_t token = TOKENS ? min(4 * strip + grp, a.tokens - 1) : strip / per_token, b = token / a.T, t = token - b * a.T;
        p.x = b * vx.sB + t * vx.sM;
        p.y = b * vy.sB + t * vy.sM;
        p.d = BACK ? b * vd.sB + t * vd.sM : 0;
        p.pos = b * a.pB + t * a.pT;
        p.head = TOKENS ? 0 : (int)(strip - token * per_token) * STEP;
        p.end = TOKENS ? (4 * strip + grp < a.tokens ? heads : 0) : a.split ? min(p.head + STEP, heads) : heads;
        return p;
    };
    Raw<X> next_x[U] = {};
    Raw<Y> next_g[BACK ? U : 1] = {};
    auto load = [&](const Place& p) {
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const int h = p.head + HOP * i + first_head;
            if (h < p.end) {
                next_x[i].load(vx.ptr + p.x + h * vx.sH, sub);
                if constexpr (BACK) next_g[i].load(vy.ptr + p.y + h * vy.sH, sub);
            }
        }
    };
    // Fractions of a turn (2^-32).  With TOKENS worked out at once, in half the registers: they come once for all heads.
    int64_t next_pos[PAIRS];
    uint32_t next_angle[PAIRS];
    auto angle_of = [&](int i, int64_t pos) { return (uint32_t)((my_turn(i) * (uint64_t)pos) >> 32); };
    auto position = [&](const Place& p) {
#pragma unroll
        for (int i = 0; i < PAIRS; ++i) {
            const int64_t at = p.pos + my_axis(i) * a.pA;
            const int64_t pos = my_axis(i) == HK_ROTARY_STILL ? 0
                                : a.pos64                     ? static_cast<const int64_t*>(a.positions)[at]
                                                              : (int64_t)static_cast<const int32_t*>(a.positions)[at];
            if (TOKENS) next_angle[i] = angle_of(i, pos);
            else next_pos[i] = pos;
        }
    };
    uint64_t policy;
    asm("createpolicy.fractional.L2::evict_normal.b64 %0, 1.0;" : "=l"(policy));
    if (a.past) asm("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(policy));
    Place at = place(block * QK_WARPS + warp);
    pdl_wait();
    pdl_trigger();
    if (at.strip < strips) {
        load(at);
        position(at);
    }
    float w[MODE == QK_ROTATE ? 1 : 8], dw[BACK ? 8 : 1];
    if (MODE != QK_ROTATE)
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = weight_at(a.w[k], a.w_dtype, (i < 4 ? 0 : 28) + 4 * sub + i);
    if (BACK)
#pragma unroll
        for (int i = 0; i < 8; ++i) dw[i] = 0.f;
    float c[4], s[4];
    Keep keep;
    bool fresh = true;  // the angles are another token's
    while (at.strip < strips) {
        Raw<X> x[U];
        Raw<Y> g[BACK ? U : 1];
#pragma unroll
        for (int i = 0; i < U; ++i) {
            x[i] = next_x[i];
            if (BACK) g[i] = next_g[i];
        }
        int64_t pos[PAIRS];
        uint32_t angle[PAIRS];
#pragma unroll
        for (int i = 0; i < PAIRS; ++i) {
            pos[i] = next_pos[i];
            angle[i] = next_angle[i];
        }
        Place next = at;
        next.head += STEP;
        const bool on = next.head >= (TOKENS ? heads : at.end);  // to another strip
        if (on) next = place(at.strip + hop < at.strip ? 0xffffffffu : at.strip + hop);
        if (next.strip < strips) {
            load(next);
            if (on) position(next);
        }
        if (fresh) {
            float mc[PAIRS], ms[PAIRS];
#pragma unroll
            for (int i = 0; i < PAIRS; ++i) {
                sincospif((float)(int32_t)(TOKENS ? angle[i] : angle_of(i, pos[i])) * 0x1p-31f, &ms[i], &mc[i]);
                if (a.back) ms[i] = -ms[i];
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                c[i] = TOKENS ? mc[i % PAIRS] : __shfl_sync(0xffffffffu, mc[0], turned_by(i));
                s[i] = TOKENS ? ms[i % PAIRS] : __shfl_sync(0xffffffffu, ms[0], turned_by(i));
            }
            if (KEEPS) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int lo = (2 * i) & 3, hi = lo + 1;
                    keep.w[i] = interleaved ? (is_still(c[i], s[i]) ? 0xffffffffu : 0u)
                                            : (is_still(c[lo], s[lo]) ? 0xffffu : 0u) | (is_still(c[hi], s[hi]) ? 0xffff0000u : 0u);
                }
            }
        }
        fresh = on;
        float inv[U];  // of rows that are none: anything
        if (MODE != QK_ROTATE) rms_inverse(x, a.eps, inv);
        if (!BACK) {
#pragma unroll
            for (int i = 0; i < U; ++i) {
                const int h = at.head + HOP * i + first_head;
                if (h >= at.end) break;
                Row8 r = numbers(x[i]);
                if (MODE == QK_NORM) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) r.v[e] *= inv[i] * w[e];
                }
                rotate(r, c, s, interleaved);
                store_row<Y, KEEPS>(vy.ptr + at.y + h * vy.sH, sub, r, x[i].w, keep, policy);
            }
        } else {
            Row8 z[U];
            float dot[U];
#pragma unroll
            for (int i = 0; i < U; ++i) {
                const bool valid = at.head + HOP * i + first_head < at.end;
                const Row8 r = numbers(x[i]);
                z[i] = numbers(g[BACK ? i : 0]);
                rotate(z[i], c, s, interleaved);
                dot[i] = 0.f;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float n = r.v[e] * inv[i];
                    if (valid) dw[e] = fmaf(z[i].v[e], n, dw[e]);
                    z[i].v[e] *= w[e];
                    dot[i] = fmaf(z[i].v[e], n, dot[i]);
                }
            }
            sum8(dot);
#pragma unroll
            for (int i = 0; i < U; ++i) {
                const int h = at.head + HOP * i + first_head;
                if (h >= at.end) break;
                const Row8 r = numbers(x[i]);
#pragma unroll
                for (int e = 0; e < 8; ++e) z[i].v[e] = inv[i] * fmaf(-(r.v[e] * inv[i]), dot[i] * (1.f / 64.f), z[i].v[e]);
                store_row<X, false>(vd.ptr + at.d + h * vd.sH, sub, z[i], nullptr, keep, policy);
            }
        }
        at = next;
    }
    if (BACK) {  // sums of the CTA's rows
        __shared__ float sums[QK_WARPS * 4][64];
#pragma unroll
        for (int e = 0; e < 8; ++e) sums[threadIdx.x >> 3][(e < 4 ? 0 : 28) + 4 * sub + e] = dw[e];
        __syncthreads();
        if (threadIdx.x < 64) {
            float x = 0.f;
#pragma unroll
            for (int i = 0; i < QK_WARPS * 4; ++i) x += sums[i][threadIdx.x];
            a.partial[blockIdx.x * 64 + threadIdx.x] = x;
        }
    }
}

// The sums of the CTAs that took queries, and of those that took keys: 16 columns a CTA, 64 threads a column, always in the same
// order.
__global__ void __launch_bounds__(1024) qk_weight_sum_kernel(const float* partial, int n_q, int n, float* dq, float* dk) {
    __shared__ float sums[64][17];
    const int col = threadIdx.x & 15, part = threadIdx.x >> 4, at = (blockIdx.x & 3) * 16 + col;
    const bool keys = blockIdx.x >= 4;
    pdl_wait();
    pdl_trigger();
    float x = 0.f;
    const int end = keys ? n : n_q;
#pragma unroll 4
    for (int i = (keys ? n_q : 0) + part; i < end; i += 64) x += partial[i * 64 + at];
    sums[part][col] = x;
    __syncthreads();
    if (part < 8) {
        x = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) x += sums[8 * part + i][col];
    }
    __syncthreads();
    if (part < 8) sums[part][col] = x;
    __syncthreads();
    if (part == 0) {
#pragma unroll
        for (int i = 1; i < 8; ++i) x += sums[i][col];
        float* to = keys ? dk : dq;
        if (to) to[at] = x;
    }
}

RowView row_view(const hk_view& v, int dtype) {
    const int64_t e = esize(dtype);
    return {static_cast<char*>(v.ptr), v.strideB * e, v.strideM * e, v.strideH * e};
}

typedef void (*QkKernel)(QkArgs);
// Groups of four rows in a step: what fits the registers twice.
template <class X, int MODE>
constexpr int rows_of() { return MODE == QK_NORM_BACK ? 2 : 4; }
template <class X, class Y, int MODE>
QkKernel kernel_of(int& step, bool tokens) {
    step = rows_of<X, MODE>() * (tokens ? 1 : 4);
    if constexpr (sizeof(X) == 2 || sizeof(Y) == 2)
        if (tokens) return qk_rotary_kernel<X, Y, MODE, rows_of<X, MODE>(), true>;
    return qk_rotary_kernel<X, Y, MODE, rows_of<X, MODE>(), false>;
}
template <int MODE>
QkKernel pick(int x, int y, int& step, bool tokens) {
    typedef __nv_bfloat16 bf16;
    if (x == HK_F32 && y == HK_F32) return kernel_of<float, float, MODE>(step, tokens);
    if (x == HK_BF16 && y == HK_BF16) return kernel_of<bf16, bf16, MODE>(step, tokens);
    if (x == HK_F16 && y == HK_F16) return kernel_of<__half, __half, MODE>(step, tokens);
    if (x == HK_BF16 && y == HK_F32) return kernel_of<bf16, float, MODE>(step, tokens);
    if (x == HK_F16 && y == HK_F32) return kernel_of<__half, float, MODE>(step, tokens);
    if constexpr (MODE == QK_ROTATE) {  // gradients from the attention back to the projection's type
        if (x == HK_F32 && y == HK_BF16) return kernel_of<float, bf16, MODE>(step, tokens);
        if (x == HK_F32 && y == HK_F16) return kernel_of<float, __half, MODE>(step, tokens);
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
    if (p->nh_k > 0 && dst[0]->ptr == dst[1]->ptr) return HK_ERR_UNSUPPORTED;  // queries' and keys' results in the same place
    a.positions = p->positions;
    a.pA = p->pos_strideA; a.pB = p->pos_strideB; a.pT = p->pos_strideT;
    a.heads[0] = p->nh; a.heads[1] = p->nh_k;
    a.T = (uint32_t)p->T;
    a.tokens = (uint32_t)(p->B * p->T);
    a.pos64 = p->pos_bits == 64;
    a.w_dtype = p->weight_dtype;
    a.back = back;
    a.eps = p->eps;
    a.plan = p->plan;

    // Warps enough for all that an SM holds; where there are fewer tokens, a warp takes one step of a token's heads.
    const int64_t most = (int64_t)sm_count() * QK_CTAS;
    a.split = (int64_t)a.tokens < most * QK_WARPS;
    // What is next reads the results, out of the L2 if they fit it: there they are stored to stay (norm and attention, 12 heads, T 1024, fp32:
    // B8 59.4 us and B16 104.4, 61.4 and 108.5 with stores that do not ask to).  Results that do not fit would only push each other out
    // (T 32767, 32 and 8 heads, into bf16: 89.3 us, and 84.7 with such stores; norm backward, T 32768, 32 and 32 heads, bf16 193 and 190).
    a.past = (int64_t)a.tokens * (p->nh + p->nh_k) * HEAD_DIM * esize(dst_t) > L2_BYTES;
    // Groups of lanes by tokens where most of the 16-bit tensors lie head by head (B1, 32 and 8 heads, T 32768, bf16 in and out:
    // 65 us instead of 74, fp32 gradients into bf16 86 instead of 95; fp32 alone gains 1 % and its backward pass has no registers for it)
    int by_head = 0, of_16 = 0;
    auto count = [&](const hk_view& v, int dtype) {
        if (dtype == HK_F32) return;
        ++of_16;
        if (v.strideM < v.strideH && p->nh > 1) ++by_head;
    };
    count(*src[0], src_t);
    count(*dst[0], dst_t);
    if (mode == QK_NORM_BACK) count(*grad[0], p->out_dtype);
    const bool tokens = !a.split && 2 * by_head > of_16;
    int step = 0;
    const QkKernel kernel = mode == QK_ROTATE ? pick<QK_ROTATE>(src_t, dst_t, step, tokens)
                            : mode == QK_NORM ? pick<QK_NORM>(src_t, dst_t, step, tokens)
                                              : pick<QK_NORM_BACK>(src_t, p->out_dtype, step, tokens);
    if (!kernel) return HK_ERR_UNSUPPORTED;
    auto strips = [&](int heads) { return tokens ? ((int64_t)a.tokens + 3) / 4 : (int64_t)a.tokens * (a.split ? (heads + step - 1) / step : 1); };
    // CTAs by the steps there are
    int64_t n_q = (strips(p->nh) + QK_WARPS - 1) / QK_WARPS, n_k = (strips(p->nh_k) + QK_WARPS - 1) / QK_WARPS;
    if (p->nh_k == 0) n_k = 0;
    if (n_q + n_k > most) {
        const int64_t s_q = (p->nh + step - 1) / step, s_k = (p->nh_k + step - 1) / step;
        const int64_t for_q = std::max<int64_t>(1, std::min<int64_t>(most - (n_k > 0), (most * s_q + (s_q + s_k) / 2) / (s_q + s_k)));
        n_q = std::min(n_q, for_q);
        n_k = std::min(n_k, most - n_q);
    }
    if (strips(p->nh) > 0xffffffffLL || strips(p->nh_k) > 0xffffffffLL) return HK_ERR_BAD_SHAPE;
    a.blocks_q = (uint32_t)n_q;
    const int blocks = (int)(n_q + n_k);
    LaunchConfig lc(blocks, QK_WARPS * 32, 0, stream, 1, true);
    if (cudaLaunchKernelEx(&lc.cfg, kernel, a) != cudaSuccess) return check_launch();
    count_launch();
    if (mode == QK_NORM_BACK && (p->dq_weight || p->dk_weight)) {
        LaunchConfig sum(8, 1024, 0, stream, 1, true);
        if (cudaLaunchKernelEx(&sum.cfg, qk_weight_sum_kernel, (const float*)a.partial, (int)n_q, blocks, p->dq_weight, p->dk_weight) != cudaSuccess)
            return check_launch();
        count_launch();
    }
    return HK_OK;
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
            // 64 bits of significand up to the rounding of the fraction: the 53 of a power in double would be 2^-57 of a turn off, and the
            // position multiplies that
            const long double f = frequency ? (long double)frequency[n] : std::pow((long double)base, -n / 32.0L);
            if (!std::isfinite(f)) return HK_ERR_BAD_SHAPE;
            // turns per position without whole ones, which an integer position turns into whole turns again
            const long double turns = f / 6.283185307179586476925286766559005768L;
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

size_t hk_qk_norm_rotary_workspace_bytes(const hk_qk_params*) { return (size_t)sm_count() * QK_CTAS * 64 * sizeof(float); }

}  // extern "C"
