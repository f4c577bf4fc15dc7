// shared_prefix_few.cu -- attention over a shared prefix where few rows meet a run of keys (decoding): bound by reading keys and
// values.
//
// A warp takes its rows through batches of 8 (fp32) or 16 keys that TMA brings into a ring of its own, two or three batches ahead: no
// barrier between warps until they merge what they have.  (Copies by the lanes themselves, cp.async, kept the load/store unit busy for
// 112 cycles a batch and warp: 64 requests, 32 heads on 8, 8 192 and up to 1 000 keys, bf16, took 37.7 us instead of 30.5, launches
// behind each other.)  A batch of all warps of an SM takes 0.45 us for 16-bit types, 0.65 for 16 rows of fp32, 0.4 for one or two, and
// a CTA 2.2 us beside its batches.  Sixteen requests of 12 heads on 2 047 and up to 512 keys, fp32: 12.0 us with the launch that adds
// up the slots, for 37.8 MB (48 % of the copy rate); four on 333 and up to 64, in one launch: 5.0 us, of which the keys take one.
//   One or two rows in fp32: a half-warp to a key, four elements a lane (RowsOfOne).
//   Up to 16 rows: matrix instructions (m16n8k8 on TF32, m16n8k16 on 16-bit types).  A lane's part of an operand is whatever
// 16-byte pieces it reads, because the order of the contracted index (head dimension, keys) and of the result's columns is free
// as long as both operands agree on it; the order taken makes every read free of bank conflicts in the layout TMA writes (16-byte
// piece c of row r at c ^ (r % 8)).  The instructions on tensor memory would need 128 rows to a tile.
#include <algorithm>
#include <cmath>
#include <mutex>
#include <type_traits>

#include "shared_prefix.cuh"

namespace hk {
namespace {

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


constexpr int FEW_WARPS = 4;

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
    int limit[2];
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
    template <class F>
    __device__ __forceinline__ void batch(const uint8_t* from, int lane, int key0, int end, bool own, float scale_log2e, F&& copy_next) {
        const int g = lane >> 2, c = lane & 3;
        f.read_k(from, g, c);
        float s[NT][4];
        f.scores(s);
        f.read_v(from + 2048, g, c);
        copy_next();
        const int last[2] = {own ? limit[0] : end, own ? limit[1] : end};
        if (!__all_sync(0xffffffffu, key0 + KEYS <= min(last[0], last[1]))) {
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (key0 + Math::key_s(t, c, e) >= last[e >> 1]) s[t][e] = -INFINITY;
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
    int limit[N];

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
    template <class F>
    __device__ __forceinline__ void batch(const uint8_t* from, int lane, int key0, int end, bool own, float scale_log2e, F&& copy_next) {
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
            if (key >= (own ? limit[r] : end)) s[r] = -INFINITY;
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

// What a CTA takes: a run of the prefix's keys; a run of a request's own, by the keys there are; or the whole prefix and all of the
// request's own, with more warps (small calls, where a second and a third launch would take longer).
enum FewJob { FEW_PREFIX = 0, FEW_OWN = 1, FEW_WHOLE = 2 };
template <class Rows, int JOB>
struct FewShared {
    static constexpr int WARPS = JOB != FEW_WHOLE ? FEW_WARPS : Rows::ROWS < 16 ? 16 : 8, PARTS = WARPS * Rows::PARTS;
    union {
        uint8_t ring[WARPS][Rows::STAGES][4096];  // a batch's keys and values
        float part[PARTS][Rows::ROWS][64 + 4];
    };
    float2 ml[PARTS][Rows::ROWS];
    uint64_t full[WARPS][Rows::STAGES];
    Abort abort;
};

constexpr int W_FEW = 401;

template <class Rows, int JOB>
__device__ __forceinline__ void few_job(const CUtensorMap& map_kp, const CUtensorMap& map_vp, const CUtensorMap& map_k, const CUtensorMap& map_v, const PrefixArgs& a,
                                        const int block, const bool late) {
    typedef typename Rows::X X;
    typedef FewShared<Rows, JOB> Shared;
    constexpr bool OWN = JOB != FEW_PREFIX;
    constexpr int N = Rows::ROWS, KEYS = Rows::KEYS, WARPS = Shared::WARPS, MINE = N < 16 ? N : 2;  // rows that a lane works on
    extern __shared__ __align__(1024) uint8_t few_smem[];
    Shared& sh = *reinterpret_cast<Shared*>(few_smem);
    const int warp = (int)uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (lane == 0) {
        for (int s = 0; s < Rows::STAGES; ++s) mbar_init(&sh.full[warp][s], 1);
        if (warp == 0) sh.abort.id = 0;
        fence_mbar_init();
    }
    if (!late) pdl_wait();
    pdl_trigger();
    // the rows
    const int ns = JOB == FEW_PREFIX ? a.splits_p : JOB == FEW_OWN ? a.splits_o : 1, item = block / ns, split = block - item * ns;
    const int tiles = OWN ? a.tiles_o : a.tiles_p, at = item / tiles, tile = item - at * tiles;
    const int b = OWN ? at / a.Hk : 0, kvh = at - b * a.Hk;
    const int len = OWN ? request_keys(a, b) : 0;
    const int all = OWN ? a.T * a.group : a.R, row0 = b * a.T * a.group + tile * N, rows = min(N, all - tile * N);
    typename Rows::Query query;
    int token_of[MINE];
#pragma unroll
    for (int i = 0; i < MINE; ++i) {
        const int r = Rows::row(i, lane), row = row0 + r, token = row / a.group, bq = OWN ? b : token / a.T;
        token_of[i] = r < rows ? token - bq * a.T : a.T;
        query.load(i, r < rows ? row_of<X>(a.Q, bq, kvh * a.group + (row - token * a.group), token_of[i]) : nullptr, lane, late);
    }
    // the keys: batches of the prefix, then of the request's own
    int p_begin = 0, p_end = 0, o_begin = 0, o_end = 0;
    if (JOB == FEW_PREFIX) {
        p_begin = split * a.per_p;
        p_end = min(a.P, p_begin + a.per_p);
    } else {
        const int seen = token_keys(a, len, (tile * N + rows - 1) / a.group), per = ((seen + ns - 1) / ns + KEYS - 1) / KEYS * KEYS;
        o_begin = min(seen, split * per);
        o_end = min(seen, o_begin + per);
        if (JOB == FEW_WHOLE) p_end = a.P;
    }
    const int n_p = (p_end - p_begin + KEYS - 1) / KEYS, n = n_p + (o_end - o_begin + KEYS - 1) / KEYS;
    auto key_of = [&](int i) { return i < n_p ? p_begin + i * KEYS : o_begin + (i - n_p) * KEYS; };
    int put = 0, put_at = warp;
    auto copy_next = [&] {  // the next batch of this warp, if there is one, into the slot that its lanes have read
        __syncwarp();
        if (put_at < n && lane == 0) {
            const bool own = JOB == FEW_OWN || (JOB == FEW_WHOLE && put_at >= n_p);
            uint64_t* full = &sh.full[warp][put];
            uint8_t* to = sh.ring[warp][put];
            mbar_arrive_expect_tx(full, 4096);
            tma_load_tile(to, own ? &map_k : &map_kp, full, key_of(put_at), kvh, own ? b : 0);
            tma_load_tile(to + 2048, own ? &map_v : &map_vp, full, key_of(put_at), kvh, own ? b : 0);
        }
        put_at += WARPS;
        put = put + 1 == Rows::STAGES ? 0 : put + 1;
    };
#pragma unroll
    for (int i = 0; i < Rows::STAGES - 1; ++i) copy_next();
    Rows w;
    w.start(query, a.flip);
#pragma unroll
    for (int i = 0; i < MINE; ++i) w.limit[i] = OWN && token_of[i] < a.T ? min(o_end, token_keys(a, len, token_of[i])) : o_end;
    __syncthreads();  // the record of waits that gave up
    WaitNote wc{&sh.abort};
    int get = 0;
    uint32_t phase = 0;
    for (int i = warp; i < n; i += WARPS) {
        if (!__all_sync(0xffffffffu, mbar_wait(wc, &sh.full[warp][get], phase, W_FEW, i))) {
            for (const unsigned long long t0 = globaltimer_ns(); globaltimer_ns() - t0 < 100000ull;) {}  // copies in flight land
            break;
        }
        const uint8_t* from = sh.ring[warp][get];
        if (++get == Rows::STAGES) get = 0, phase ^= 1u;
        const bool own = JOB == FEW_OWN || (JOB == FEW_WHOLE && i >= n_p);
        w.batch(from, lane, key_of(i), own ? o_end : p_end, own, a.scale_log2e, copy_next);
    }
    const int64_t slot0 = (int64_t)kvh * a.R + row0, slot_rows = a.slot_rows;
    __syncthreads();  // the ring is the warps' exchange now: every copy has been waited for
    w.finish(sh.part, sh.ml, warp, lane);
    __syncthreads();
    // PER threads a row, 64 / PER elements each
    constexpr int PER = N < 16 ? 16 : 8, E = 64 / PER;
    const int r = threadIdx.x / PER, d = threadIdx.x % PER * E;
    const bool mine = r < rows;
    float M = -INFINITY, L = 0.f, acc[E];
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = 0.f;
    if (mine) {
#pragma unroll
        for (int p = 0; p < Shared::PARTS; ++p) M = fmaxf(M, sh.ml[p][r].x);
        const float ref = M == -INFINITY ? 0.f : M;
#pragma unroll
        for (int p = 0; p < Shared::PARTS; ++p) {
            const float f = ex2_approx(sh.ml[p][r].x - ref);
            L += sh.ml[p][r].y * f;
#pragma unroll
            for (int e = 0; e < E; ++e) acc[e] = fmaf(sh.part[p][r][d + e], f, acc[e]);
        }
    }
    if (threadIdx.x == 0) report_abort(sh.abort, a.status);
    if (mine && JOB != FEW_WHOLE && a.slots > 1) {
        const int64_t to = (OWN ? a.splits_p + split : split) * slot_rows + slot0 + r;
        if (d == 0) a.ml[to] = make_float2(M, L);
#pragma unroll
        for (int e = 0; e < E; e += 4) *reinterpret_cast<float4*>(a.part + to * 64 + d + e) = make_float4(acc[e], acc[e + 1], acc[e + 2], acc[e + 3]);
    } else if (mine) {
        const float f = L != 0.f ? 1.f / L : 0.f;
        const int row = row0 + r, token = row / a.group, bq = OWN ? b : token / a.T, t = token - bq * a.T, h = kvh * a.group + (row - token * a.group);
        X* to = const_cast<X*>(row_of<X>(a.O, bq, h, t)) + d;
#pragma unroll
        for (int e = 0; e < E; e += 4) store4(to + e, make_float4(acc[e] * f, acc[e + 1] * f, acc[e + 2] * f, acc[e + 3] * f));
        if (d == 0) a.LSE[bq * a.lse_sB + h * a.lse_sH + t] = L != 0.f ? (M + log2f(L)) * LN2 : -INFINITY;
    }
}

// late: runs beside the kernel over the prefix.  What was before that is complete when this one begins, and this one when that is.
template <class Rows, int JOB>
__global__ void __launch_bounds__(FewShared<Rows, JOB>::WARPS * 32, JOB == FEW_WHOLE ? 1 : Rows::CTAS)
prefix_few_kernel(const __grid_constant__ CUtensorMap map_kp, const __grid_constant__ CUtensorMap map_vp, const __grid_constant__ CUtensorMap map_k,
                  const __grid_constant__ CUtensorMap map_v, const __grid_constant__ PrefixArgs a) {
    const bool late = JOB == FEW_OWN && a.splits_p > 0;
    few_job<Rows, JOB>(map_kp, map_vp, map_k, map_v, a, blockIdx.x, late);
    if (late && blockIdx.x == gridDim.x - 1) pdl_wait();
}
// The runs of the prefix and those of the requests' own keys in one launch.
template <class Prefix, class Own>
__global__ void __launch_bounds__(FEW_WARPS * 32, Prefix::CTAS < Own::CTAS ? Prefix::CTAS : Own::CTAS)
prefix_few_both_kernel(const __grid_constant__ CUtensorMap map_kp, const __grid_constant__ CUtensorMap map_vp, const __grid_constant__ CUtensorMap map_k,
                       const __grid_constant__ CUtensorMap map_v, const __grid_constant__ PrefixArgs a) {
    const int n = a.Hk * a.tiles_p * a.splits_p;
    if ((int)blockIdx.x < n) few_job<Prefix, FEW_PREFIX>(map_kp, map_vp, map_k, map_v, a, blockIdx.x, false);
    else few_job<Own, FEW_OWN>(map_kp, map_vp, map_k, map_v, a, blockIdx.x - n, false);
}

typedef void (*FewKernel)(CUtensorMap, CUtensorMap, CUtensorMap, CUtensorMap, PrefixArgs);
struct FewEntry {
    FewKernel kernel;
    size_t smem;
    int threads;
};
template <class Rows, int JOB>
FewEntry entry() {
    return {prefix_few_kernel<Rows, JOB>, sizeof(FewShared<Rows, JOB>), FewShared<Rows, JOB>::WARPS * 32};
}
template <int JOB>
FewEntry pick(int dtype, int rows) {
    if (dtype == HK_BF16) return entry<RowsOf16<__nv_bfloat16>, JOB>();
    if (dtype == HK_F16) return entry<RowsOf16<__half>, JOB>();
    return rows == 1 ? entry<RowsOfOne<1>, JOB>() : rows == 2 ? entry<RowsOfOne<2>, JOB>() : entry<RowsOf16<float>, JOB>();
}

template <class Prefix, class Own>
FewEntry both() {
    return {prefix_few_both_kernel<Prefix, Own>, std::max(sizeof(FewShared<Prefix, FEW_PREFIX>), sizeof(FewShared<Own, FEW_OWN>)), FEW_WARPS * 32};
}
FewEntry pick_both(int dtype, int prefix, int own) {  // rows of a tile: own <= prefix
    if (dtype == HK_BF16) return both<RowsOf16<__nv_bfloat16>, RowsOf16<__nv_bfloat16>>();
    if (dtype == HK_F16) return both<RowsOf16<__half>, RowsOf16<__half>>();
    if (prefix == 1) return both<RowsOfOne<1>, RowsOfOne<1>>();
    if (prefix == 2) return own == 1 ? both<RowsOfOne<2>, RowsOfOne<1>>() : both<RowsOfOne<2>, RowsOfOne<2>>();
    return own == 1 ? both<RowsOf16<float>, RowsOfOne<1>>() : own == 2 ? both<RowsOf16<float>, RowsOfOne<2>>() : both<RowsOf16<float>, RowsOf16<float>>();
}

int launch(const FewEntry& k, const PrefixArgs& a, int dtype, bool prefix, bool own, int64_t blocks, cudaStream_t stream) {
    // once per device and kernel: more than 48 KB of shared memory
    static std::mutex mu;
    static FewKernel known[HK_MAX_DEVICES][32];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= HK_MAX_DEVICES) return HK_ERR_CUDA;
    {
        std::lock_guard<std::mutex> lock(mu);
        for (FewKernel& x : known[dev]) {
            if (x == k.kernel) break;
            if (x) continue;
            if (cudaFuncSetAttribute(k.kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)k.smem) != cudaSuccess) return check_launch();
            x = k.kernel;
            break;
        }
    }
    if (blocks > 0x7fffffffLL) return HK_ERR_BAD_SHAPE;
    LaunchConfig lc((unsigned)blocks, k.threads, k.smem, stream, 1, true);
    CUtensorMap kp, vp, mk, mv;
    const int rows = few_plan(dtype, 16).step / FEW_WARPS;
    int rc;
    if ((rc = prefix_tile_map(&kp, a.Kp, dtype, 1, a.Hk, prefix ? a.P : 0, rows, false)) || (rc = prefix_tile_map(&vp, a.Vp, dtype, 1, a.Hk, prefix ? a.P : 0, rows, false)) ||
        (rc = prefix_tile_map(&mk, a.K, dtype, a.B, a.Hk, own ? a.S : 0, rows, false)) || (rc = prefix_tile_map(&mv, a.V, dtype, a.B, a.Hk, own ? a.S : 0, rows, false)))
        return rc;
    if (cudaLaunchKernelEx(&lc.cfg, k.kernel, kp, vp, mk, mv, a) != cudaSuccess) return check_launch();
    count_launch();
    return HK_OK;
}

}  // namespace

FewPlan few_plan(int dtype, int rows) {
    if (dtype != HK_F32) return {16, FEW_WARPS * 16, RowsOf16<__half>::CTAS};
    return {rows <= 2 ? rows : 16, FEW_WARPS * 8, rows <= 2 ? RowsOfOne<1>::CTAS : RowsOf16<float>::CTAS};
}
int launch_prefix_few(const PrefixArgs& a, int dtype, cudaStream_t stream) {
    return launch(pick<FEW_PREFIX>(dtype, few_plan(dtype, a.R).rows), a, dtype, true, false, (int64_t)a.Hk * a.tiles_p * a.splits_p, stream);
}
int launch_own_few(const PrefixArgs& a, int dtype, cudaStream_t stream) {
    const int rows = few_plan(dtype, a.T * a.group).rows;
    if (a.whole) return launch(pick<FEW_WHOLE>(dtype, rows), a, dtype, true, true, (int64_t)a.B * a.Hk * a.tiles_o, stream);
    return launch(pick<FEW_OWN>(dtype, rows), a, dtype, false, true, (int64_t)a.B * a.Hk * a.tiles_o * a.splits_o, stream);
}
int launch_both_few(const PrefixArgs& a, int dtype, cudaStream_t stream) {
    return launch(pick_both(dtype, few_plan(dtype, a.R).rows, few_plan(dtype, a.T * a.group).rows), a, dtype, true, true,
                  (int64_t)a.Hk * a.tiles_p * a.splits_p + (int64_t)a.B * a.Hk * a.tiles_o * a.splits_o, stream);
}

}  // namespace hk
