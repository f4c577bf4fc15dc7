// few_rows.cuh -- a warp's rows against batches of keys in shared memory (shared_prefix_few.cu, serving_few.cu): up to 16 rows by matrix
// instructions, up to four of fp32 lane by lane.
#pragma once

#include <type_traits>

#include "tile_math.cuh"

namespace hk {

__device__ __forceinline__ void mma_tf32(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <class X>
__device__ __forceinline__ void mma_16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (sizeof(X) == 2 && std::is_same<X, __half>::value)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t tf32_high(uint32_t x) { return x & 0xffffe000u; }
// rounded to nearest where the tensor core cuts off: cut off, with the sign of x, every product would be a little too small
__device__ __forceinline__ uint32_t tf32_low(uint32_t x) { return __float_as_uint(__uint_as_float(x) - __uint_as_float(tf32_high(x))) + 0x1000u; }

__device__ __forceinline__ uint4 query_piece(const void* p, bool late) {
    return late ? __ldcg(static_cast<const uint4*>(p)) : *static_cast<const uint4*>(p);
}

// fp32: x = h + l with h the upper 11 bits of the significand; a product is h h' + (h l' + l h'): what
// is left out is 2^-22 of it.  A batch's weighted values are added to the rest in fp32 adds, since the tensor core's own additions
// cut off instead of rounding.
// Lane (g, c) = (lane / 4, lane % 4) of a matrix instruction: rows g and g + 8, columns and contracted elements by c.
// Which of eight keys (or pieces of a row) column n stands for: neighbours are four apart, so that the eight lanes that read at once
// meet all banks.
__device__ __forceinline__ int order(int n) { return (n >> 1) | ((n & 1) << 2); }
template <class X>
struct FewMath;
template <>
struct FewMath<float> {
    static constexpr int KEYS = 8;
    // Column n of the scores is key order(n); column n of the result has elements 4 order(n) .. and 32 + 4 order(n) ..
    uint4 k[4], v[4];  // k: key order(g), elements 16 i + 4 c ..; v: keys c, c, c + 4, c + 4
    __device__ __forceinline__ void read_k(const uint8_t* at, int g, int c) {  // two boxes of 128 bytes of each row
        const int key = order(g);
#pragma unroll
        for (int i = 0; i < 4; ++i) k[i] = *reinterpret_cast<const uint4*>(at + (i >> 1) * 1024 + key * 128 + ((((i & 1) * 4 + c) ^ key) << 4));
    }
    __device__ __forceinline__ void read_v(const uint8_t* at, int g, int c) {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = *reinterpret_cast<const uint4*>(at + (i & 1) * 1024 + key_v(i, c) * 128 + ((order(g) ^ key_v(i, c)) << 4));
    }
    static __device__ __forceinline__ int key_v(int i, int c) { return c + 4 * (i >> 1); }
    static __device__ __forceinline__ int key_s(int, int c, int e) { return c + 4 * (e & 1); }  // of a lane's scores
    uint32_t qh[8][4], ql[8][4];
    static constexpr int Q_WORDS = 4;
    static __device__ __forceinline__ int at_q(int i, int c) { return 16 * i + 4 * c; }
    __device__ __forceinline__ void set_q(const uint4 (&lo)[4], const uint4 (&hi)[4], uint32_t flip) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint4 &a = lo[i], &b = hi[i];
            const uint32_t q[2][4] = {{a.x ^ flip, b.x ^ flip, a.y ^ flip, b.y ^ flip}, {a.z ^ flip, b.z ^ flip, a.w ^ flip, b.w ^ flip}};
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    qh[2 * i + h][e] = tf32_high(q[h][e]);
                    ql[2 * i + h][e] = tf32_low(q[h][e]);
                }
        }
    }
    // s: rows g, g + 8 of columns 2 c, 2 c + 1
    __device__ __forceinline__ void scores(float (&s)[1][4]) const {
        uint32_t b[16], bl[16];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t w[4] = {k[i].x, k[i].y, k[i].z, k[i].w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                b[4 * i + e] = tf32_high(w[e]);
                bl[4 * i + e] = tf32_low(w[e]);
            }
        }
        // Chains of two and of four, not one of 24: the instruction's latency is what a batch waits for, and an accumulator of scores
        // (they come to 30 and more before they are scaled) loses up to 2^-23 of itself with every addition.
        float h[4][4] = {}, m[4][4] = {};
#pragma unroll
        for (int x = 0; x < 8; ++x) {
            mma_tf32(h[x & 3], qh[x], b[2 * x], b[2 * x + 1]);
            mma_tf32(m[x & 1], ql[x], b[2 * x], b[2 * x + 1]);
            mma_tf32(m[2 + (x & 1)], qh[x], bl[2 * x], bl[2 * x + 1]);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) s[0][e] = ((h[0][e] + h[1][e]) + (h[2][e] + h[3][e])) + ((m[0][e] + m[1][e]) + (m[2][e] + m[3][e]));
    }
    // o[j] = alpha o[j] + p V: rows g, g + 8 of columns n = 2 c, 2 c + 1
    __device__ __forceinline__ void weigh(const float (&p)[1][4], const float (&alpha)[2], bool, float (&o)[8][4]) const {
        uint32_t ph[4], pl[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const uint32_t x = __float_as_uint(p[0][(e & 1) * 2 + (e >> 1)]);  // rows g, g + 8 of key c, then of c + 4
            ph[e] = tf32_high(x);
            pl[e] = tf32_low(x);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const uint4 &x = v[j >> 2], &y = v[2 + (j >> 2)];
            const uint32_t b0 = (j & 3) == 0 ? x.x : (j & 3) == 1 ? x.y : (j & 3) == 2 ? x.z : x.w;
            const uint32_t b1 = (j & 3) == 0 ? y.x : (j & 3) == 1 ? y.y : (j & 3) == 2 ? y.z : y.w;
            float t[4] = {0.f, 0.f, 0.f, 0.f};
            mma_tf32(t, pl, tf32_high(b0), tf32_high(b1));
            mma_tf32(t, ph, tf32_low(b0), tf32_low(b1));
            mma_tf32(t, ph, tf32_high(b0), tf32_high(b1));
#pragma unroll
            for (int e = 0; e < 4; ++e) o[j][e] = fmaf(o[j][e], alpha[e >> 1], t[e]);
        }
    }
    static __device__ __forceinline__ int column(int j, int n) { return (j < 4 ? 0 : 28) + 4 * order(n) + j; }
};
template <class X>
struct FewMath {
    static constexpr int KEYS = 16;
    // Column n of scores t is key 8 t + order(n); column n of the result has elements 8 order(n) ..
    uint4 k[4], v[4];  // k: keys order(g), order(g), 8 + order(g) twice, elements 32 (i & 1) + 8 c ..; v: keys c, c + 4, 8 + c, 12 + c
    __device__ __forceinline__ void read_k(const uint8_t* at, int g, int c) {
        const int key = order(g);
#pragma unroll
        for (int i = 0; i < 4; ++i) k[i] = *reinterpret_cast<const uint4*>(at + ((i >> 1) * 8 + key) * 128 + ((((i & 1) * 4 + c) ^ key) << 4));
    }
    __device__ __forceinline__ void read_v(const uint8_t* at, int g, int c) {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = *reinterpret_cast<const uint4*>(at + key_v(i, c) * 128 + ((order(g) ^ (key_v(i, c) & 7)) << 4));
    }
    static __device__ __forceinline__ int key_v(int i, int c) { return c + 4 * i; }
    static __device__ __forceinline__ int key_s(int t, int c, int e) { return 8 * t + c + 4 * (e & 1); }
    uint32_t q[4][4];
    static constexpr int Q_WORDS = 2;
    static __device__ __forceinline__ int at_q(int i, int c) { return 32 * i + 8 * c; }
    __device__ __forceinline__ void set_q(const uint4 (&lo)[2], const uint4 (&hi)[2], uint32_t flip) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint4 &a = lo[i], &b = hi[i];
            q[2 * i][0] = a.x; q[2 * i][1] = b.x; q[2 * i][2] = a.y; q[2 * i][3] = b.y;
            q[2 * i + 1][0] = a.z; q[2 * i + 1][1] = b.z; q[2 * i + 1][2] = a.w; q[2 * i + 1][3] = b.w;
#pragma unroll
            for (int e = 0; e < 8; ++e) q[2 * i + (e >> 2)][e & 3] ^= flip;
        }
    }
    // s[t]: rows g, g + 8 of columns 2 c, 2 c + 1
    __device__ __forceinline__ void scores(float (&s)[2][4]) const {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const uint4 &x = k[2 * t], &y = k[2 * t + 1];
#pragma unroll
            for (int e = 0; e < 4; ++e) s[t][e] = 0.f;
            mma_16<X>(s[t], q[0], x.x, x.y);
            mma_16<X>(s[t], q[1], x.z, x.w);
            mma_16<X>(s[t], q[2], y.x, y.y);
            mma_16<X>(s[t], q[3], y.z, y.w);
        }
    }
    __device__ __forceinline__ void weigh(const float (&p)[2][4], const float (&alpha)[2], bool rescale, float (&o)[8][4]) const {
        // the weights take the type of the values: half a step of it each
        const uint32_t a[4] = {pack<X>(p[0][0], p[0][1]), pack<X>(p[0][2], p[0][3]), pack<X>(p[1][0], p[1][1]), pack<X>(p[1][2], p[1][3])};
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = j < 2 ? v[i].x : j < 4 ? v[i].y : j < 6 ? v[i].z : v[i].w;
            if (rescale) {
#pragma unroll
                for (int e = 0; e < 4; ++e) o[j][e] *= alpha[e >> 1];
            }
            mma_16<X>(o[j], a, __byte_perm(w[0], w[1], j & 1 ? 0x7632 : 0x5410), __byte_perm(w[2], w[3], j & 1 ? 0x7632 : 0x5410));
        }
    }
    static __device__ __forceinline__ int column(int j, int n) { return 8 * order(n) + j; }
};


// Up to 16 rows of a warp.  Lane (g, c) has rows g and g + 8.
template <class T>
struct RowsOf16 {
    typedef T X;
    typedef FewMath<X> Math;
    static constexpr int ROWS = 16, KEYS = Math::KEYS, PARTS = 1, NT = KEYS / 8;
    static constexpr int STAGES = sizeof(T) == 4 ? 4 : 3, CTAS = sizeof(T) == 4 ? 3 : 4;  // of the ring; CTAs that an SM holds
    Math f;
    float o[8][4], m[2], l[2];

    // a lane's pieces of its rows of Q
    struct Query {
        uint4 row[2][Math::Q_WORDS];
        __device__ __forceinline__ void load(int i, const X* from, int lane, bool late) {
#pragma unroll
            for (int k = 0; k < Math::Q_WORDS; ++k) row[i][k] = from ? query_piece(from + Math::at_q(k, lane & 3), late) : make_uint4(0, 0, 0, 0);
        }
    };
    __device__ __forceinline__ void start(const Query& q, uint32_t flip) {
        f.set_q(q.row[0], q.row[1], flip);
#pragma unroll
        for (int e = 0; e < 2; ++e) m[e] = -INFINITY, l[e] = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[j][e] = 0.f;
    }
    static __device__ __forceinline__ int row(int i, int lane) { return (lane >> 2) + 8 * i; }
    // A batch of keys from `key0` on, of which those below `end` are; rows see those that `sees(i, key)` says, all of them if `all`.
    // copy_next: to be called when the batch has been read.
    template <class S, class F>
    __device__ __forceinline__ void batch(const uint8_t* from, int lane, int key0, int end, bool all, S&& sees, float scale_log2e, F&& copy_next) {
        const int g = lane >> 2, c = lane & 3;
        f.read_k(from, g, c);
        float s[NT][4];
        f.scores(s);
        f.read_v(from + 2048, g, c);
        copy_next();
        if (!__all_sync(0xffffffffu, all)) {
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (!sees(e >> 1, key0 + Math::key_s(t, c, e))) s[t][e] = -INFINITY;
#pragma unroll
            for (int i = 0; i < 4; ++i)  // what is behind the last key may be anything: it has no weight, but 0 times a NaN is one
                if (key0 + Math::key_v(i, c) >= end) f.v[i] = make_uint4(0, 0, 0, 0);
        }
        float mx[2] = {-INFINITY, -INFINITY}, alpha[2], ref[2];
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) mx[e >> 1] = fmaxf(mx[e >> 1], s[t][e]);
        bool raised = false;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 1));
            mx[i] = fmaf(fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 2)), scale_log2e, -lift<X>());
            const float mn = fmaxf(m[i], mx[i]);
            raised |= mn > m[i];
            ref[i] = mn == -INFINITY ? 0.f : mn;
            alpha[i] = ex2_approx(m[i] - ref[i]);  // 0 while m is -inf
            m[i] = mn;
            l[i] *= alpha[i];
        }
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                s[t][e] = ex2_approx(fmaf(s[t][e], scale_log2e, -ref[e >> 1]));
                l[e >> 1] += s[t][e];
            }
        f.weigh(s, alpha, __any_sync(0xffffffffu, raised), o);
    }
    template <class P>
    __device__ __forceinline__ void finish(P* part, float2 (*ml)[ROWS], int warp, int lane) {
        const int c = lane & 3;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int r = row(i, lane);
            l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
            l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
            if (c == 0) ml[warp][r] = make_float2(m[i], l[i]);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int j = (k >> 1) * 4, e = 2 * i + (k & 1);
                *reinterpret_cast<float4*>(&part[warp][r][Math::column(j, 2 * c + (k & 1))]) = make_float4(o[j][e], o[j + 1][e], o[j + 2][e], o[j + 3][e]);
            }
        }
    }
};

// N rows of fp32, in the same half-warp: lane `sub` of 16 has elements 4 sub .. 4 sub + 3 of queries, keys and results.  A batch is
// four keys of each half-warp; their scores are summed over the lanes with five shuffles a row, after which a lane has the score
// of one key and takes its exponential alone.
template <int N>
struct RowsOfOne {
    typedef float X;
    static constexpr int ROWS = N, KEYS = 8, PARTS = 2, STAGES = 3, CTAS = 4;
    // a lane's piece of key i of its half-warp
    static __device__ __forceinline__ float4 piece(const uint8_t* at, int i, int lane) {
        const int key = 2 * i + (lane >> 4);
        return *reinterpret_cast<const float4*>(at + ((lane >> 3) & 1) * 1024 + key * 128 + (((lane & 7) ^ key) << 4));
    }

    float4 q[N], o[N];
    float m[N], l[N];

    static __device__ __forceinline__ int row(int i, int) { return i; }
    struct Query {
        uint4 row[N];
        __device__ __forceinline__ void load(int i, const X* from, int lane, bool late) {
            row[i] = from ? query_piece(from + 4 * (lane & 15), late) : make_uint4(0, 0, 0, 0);
        }
    };
    __device__ __forceinline__ void start(const Query& from, uint32_t flip) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const uint4& x = from.row[i];
            q[i] = make_float4(__uint_as_float(x.x ^ flip), __uint_as_float(x.y ^ flip), __uint_as_float(x.z ^ flip), __uint_as_float(x.w ^ flip));
            o[i] = make_float4(0.f, 0.f, 0.f, 0.f);
            m[i] = -INFINITY;
            l[i] = 0.f;
        }
    }
    template <class S, class F>
    __device__ __forceinline__ void batch(const uint8_t* from, int lane, int key0, int end, bool, S&& sees, float scale_log2e, F&& copy_next) {
        const bool b3 = lane & 8, b2 = lane & 4;
        float s[N];
        {
            float4 k[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) k[i] = piece(from, i, lane);
#pragma unroll
            for (int r = 0; r < N; ++r) {
                float d[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) d[i] = fmaf(q[r].x, k[i].x, q[r].y * k[i].y) + fmaf(q[r].z, k[i].z, q[r].w * k[i].w);
                const float u0 = (b3 ? d[2] : d[0]) + __shfl_xor_sync(0xffffffffu, b3 ? d[0] : d[2], 8);
                const float u1 = (b3 ? d[3] : d[1]) + __shfl_xor_sync(0xffffffffu, b3 ? d[1] : d[3], 8);
                float u = (b2 ? u1 : u0) + __shfl_xor_sync(0xffffffffu, b2 ? u0 : u1, 4);
                u += __shfl_xor_sync(0xffffffffu, u, 2);
                u += __shfl_xor_sync(0xffffffffu, u, 1);
                s[r] = u;  // of key 2 (2 b3 + b2) + the half
            }
        }
        float4 v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = piece(from + 2048, i, lane);
        copy_next();
        const int key = key0 + (b3 ? 4 : 0) + (b2 ? 2 : 0) + (lane >> 4);
        if (key0 + KEYS > end) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (key0 + 2 * i + (lane >> 4) >= end) v[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        }
#pragma unroll
        for (int r = 0; r < N; ++r) {
            if (!sees(r, key)) s[r] = -INFINITY;
            float mx = fmaxf(s[r], __shfl_xor_sync(0xffffffffu, s[r], 8));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4)) * scale_log2e;
            const float mn = fmaxf(m[r], mx), ref = mn == -INFINITY ? 0.f : mn, alpha = ex2_approx(m[r] - ref);
            const float p = ex2_approx(fmaf(s[r], scale_log2e, -ref));
            m[r] = mn;
            l[r] = fmaf(l[r], alpha, p);
            o[r].x *= alpha; o[r].y *= alpha; o[r].z *= alpha; o[r].w *= alpha;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float w = __shfl_sync(0xffffffffu, p, (i & 2) * 4 + (i & 1) * 4, 16);
                o[r].x = fmaf(w, v[i].x, o[r].x); o[r].y = fmaf(w, v[i].y, o[r].y); o[r].z = fmaf(w, v[i].z, o[r].z); o[r].w = fmaf(w, v[i].w, o[r].w);
            }
        }
    }
    template <class P>
    __device__ __forceinline__ void finish(P* part, float2 (*ml)[ROWS], int warp, int lane) {
        const int at = 2 * warp + (lane >> 4);
#pragma unroll
        for (int r = 0; r < N; ++r) {
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 8);
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 4);
            if ((lane & 15) == 0) ml[at][r] = make_float2(m[r], l[r]);
            *reinterpret_cast<float4*>(&part[at][r][4 * (lane & 15)]) = o[r];
        }
    }
};

}  // namespace hk
