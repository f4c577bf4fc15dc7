// serving_few.cu -- attention of few new tokens against a cache of pages (decoding, small trees): bound by reading keys and values.
//
// A CTA has an equal stretch of all requests' keys (serving_attention.cuh), each of its four warps a quarter of it, which TMA brings into a
// ring of its own in batches of 8 (fp32) or 16 keys, two or three ahead, over the borders of requests.  A batch lies in one page.  Lengths
// and tables are read where the batches are asked for, 32 entries of a table at a time, so no product waits for them.  What a block of rows has in
// several warps goes to slots; a CTA adds up what its own warps left, and what is left of blocks that fell to several CTAs a second kernel.
// The products of 16-bit types are summed up in the instructions' accumulators, whose additions cut off: with every piece of Pieces batches of a block the sum so far goes to the
// warp's place in the workspace, where the next is added to it in fp32, and back at the block's end.
//   Where key heads come in fours the warps take one each instead, over the whole stretch of the CTA (heads_side_by_side).
//   What bounds it is memory: 64 requests of 4 096 tokens, 32 heads on 8, bf16, 96 us or 5.6 TB/s, of which some 9 are the launch, the search for
// the stretches, the first loads and the sum of the parts.  More than two rows of fp32 are bound by arithmetic: 16 requests of up to 2 047 tokens,
// 12 heads, 1 / 2 / 4 (lane by lane) / 8 / 16 rows (three TF32 products of mma.sync): 24 / 26 / 32 / 34 / 36 us with the keys in memory, 18 / 22 / 31 / 33 / 35 with
// them in the L2; the kernel of many rows takes 53.
#include <algorithm>
#include <cmath>
#include <mutex>

#include "few_rows.cuh"
#include "serving_attention.cuh"

namespace hk {
namespace {

constexpr int WARPS = 4;

template <int KEYS>
using FewWork = Work<KEYS, 2, 4, 3 * KEYS, true>;

// CTAs that an SM holds, by what their threads need of its registers (16 rows by matrix instructions 160, fp32 233), and batches of a warp's
// ring, which share its memory.  With four, and registers spilled, 64 requests of up to 4 096 tokens, 32 heads on 8, bf16, took 56 us instead of
// 53, with two as long or longer; 16 rows of fp32 in three 75 us instead of 56 (16 requests of up to 4 096, 12 heads).
template <class Rows>
struct Shape {
    static constexpr int CTAS = Rows::ROWS == 16 ? (sizeof(typename Rows::X) == 4 ? 2 : 3) : Rows::ROWS > 2 ? 3 : 4, STAGES = 12 / CTAS;
};

// Batches of 16 keys that one sum of weighted values has at most: a cut-off of 8e-8 of it for each comes to less than half a step of the type, 1.6e-4 of fp16 and 1.3e-3
// of bf16.  fp32 adds every batch up by itself, rounded.
template <class X>
struct Pieces {
    static constexpr int BATCHES = std::is_same<X, __half>::value ? 2048 : std::is_same<X, __nv_bfloat16>::value ? 16384 : 0;
};

struct Segment {  // a run as the products need it
    int b, kvh, row0, rows, from, to, old, len, slot;
};
template <class Rows, int SIDE>
struct FewShared {
    uint8_t ring[WARPS][Shape<Rows>::STAGES][4096];  // a batch's keys and values
    Segment segments[WARPS][8];               // as many as can be on their way, and more
    uint64_t full[WARPS][Shape<Rows>::STAGES];
    LineSearch<WARPS / SIDE> search;
    PartRecord records[WARPS];
    Abort abort;
};
static_assert(sizeof(Segment) == 36, "");
constexpr int W_FEW = 601;

// The weighted sum of a row's values from registers to memory, scaled: fp32 in slots, or the result.
template <class T, int M, class P>
__device__ __forceinline__ void store_rows(const RowsOf16<T>& w, int lane, int rows, const float (&f_of)[M], P&& place) {
    typedef typename RowsOf16<T>::Math Math;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int r = RowsOf16<T>::row(i, lane);
        if (r >= rows) continue;
        auto* const to = place(i);
        const float f = f_of[i];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int j = (k >> 1) * 4, e = 2 * i + (k & 1);
            store4(to + Math::column(j, 2 * (lane & 3) + (k & 1)), make_float4(w.o[j][e] * f, w.o[j + 1][e] * f, w.o[j + 2][e] * f, w.o[j + 3][e] * f));
        }
    }
}
template <int N, class P>
__device__ __forceinline__ void store_rows(const RowsOfOne<N>& w, int lane, int rows, const float (&f_of)[N], P&& place) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
        if (i >= rows || lane >= 16) continue;
        auto* const to = place(i);
        const float f = f_of[i];
        store4(to + 4 * lane, make_float4(w.o[i].x * f, w.o[i].y * f, w.o[i].z * f, w.o[i].w * f));
    }
}
// A warp's sums of weighted values that were cut into pieces, in `sum`, and the maxima that they were taken by: with those of the piece that is over,
// which begins anew, or (back) all of them to where they were.
template <class T>
__device__ __forceinline__ void sum_pieces(RowsOf16<T>& w, float4* sum, float (&m_sum)[2], int lane, bool first, bool back) {
    float f[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        f[i] = first ? 0.f : ex2_approx(m_sum[i] - (w.m[i] == -INFINITY ? 0.f : w.m[i]));
        m_sum[i] = w.m[i];
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        float4 x = make_float4(w.o[j][0], w.o[j][1], w.o[j][2], w.o[j][3]);
        if (!first) {
            const float4 y = sum[j * 32 + lane];
            x = make_float4(fmaf(y.x, f[0], x.x), fmaf(y.y, f[0], x.y), fmaf(y.z, f[1], x.z), fmaf(y.w, f[1], x.w));
        }
        if (!back) {
            sum[j * 32 + lane] = x;
            x = make_float4(0.f, 0.f, 0.f, 0.f);
        }
        w.o[j][0] = x.x; w.o[j][1] = x.y; w.o[j][2] = x.z; w.o[j][3] = x.w;
    }
}
// Sums of the lanes that share a row; then every lane of a row has its maximum and sum.
template <class T>
__device__ __forceinline__ void join(RowsOf16<T>& w) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        w.l[i] += __shfl_xor_sync(0xffffffffu, w.l[i], 1);
        w.l[i] += __shfl_xor_sync(0xffffffffu, w.l[i], 2);
    }
}
template <int N>
__device__ __forceinline__ void join(RowsOfOne<N>& w) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
        w.l[i] += __shfl_xor_sync(0xffffffffu, w.l[i], 8);
        w.l[i] += __shfl_xor_sync(0xffffffffu, w.l[i], 4);
        const float other = __shfl_xor_sync(0xffffffffu, w.m[i], 16), m = fmaxf(w.m[i], other), ref = m == -INFINITY ? 0.f : m;
        const float mine = ex2_approx(w.m[i] - ref), its = ex2_approx(other - ref);
        w.l[i] = w.l[i] * mine + __shfl_xor_sync(0xffffffffu, w.l[i], 16) * its;
        w.m[i] = m;
        float* o = &w.o[i].x;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = o[e] * mine + __shfl_xor_sync(0xffffffffu, o[e], 16) * its;
    }
}

// The parts that the CTA's warps left of blocks that go from one to the next, added up in that order, 16 lanes to a row: blocks that end
// here are results, what one has of a block that goes on in another CTA, at either end, goes to the CTA's slots.
template <class X, int ROWS>
__device__ __forceinline__ void join_warps(const ServingArgs& a, const PartRecord (&records)[WARPS]) {
    constexpr int EACH = (ROWS + 7) / 8;  // rows of a thread
    const int sub = threadIdx.x & 15, r0 = threadIdx.x >> 4, first = blockIdx.x * WARPS;
    float4 o[EACH];
    float2 ml[EACH];
    PartRecord mine{PART_EMPTY, 0, 0, 0, 0, 0}, open{PART_EMPTY, 0, 0, 0, 0, 0};  // the CTA's; of the block that is being added up
    bool is_open = false, begun_here = false;
    auto slot_of = [&](int slot, int r) { return (int64_t)slot * a.slot_rows + r; };
    auto put = [&](int slot) {
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            const int r = r0 + 8 * i;
            if (r >= a.slot_rows) continue;
            *reinterpret_cast<float4*>(a.part + slot_of(slot, r) * 64 + 4 * sub) = o[i];
            if (sub == 0) a.ml[slot_of(slot, r)] = ml[i];
        }
    };
    const int done = 2 * WARPS * gridDim.x;  // the CTAs' slots lie behind the warps'
#pragma unroll 1
    for (int w = 0; w < WARPS; ++w) {
        const PartRecord rec = records[w];
        if (rec.head == PART_EMPTY) continue;
        if (rec.head != PART_NONE) {  // goes on with what is open, or with what the CTA in front has
            const int slot = 2 * (first + w);
#pragma unroll
            for (int i = 0; i < EACH; ++i) {
                const int r = r0 + 8 * i;
                if (r >= a.slot_rows) continue;
                const float4 v = *reinterpret_cast<const float4*>(a.part + slot_of(slot, r) * 64 + 4 * sub);
                const float2 x = a.ml[slot_of(slot, r)];
                if (!is_open) {
                    o[i] = v;
                    ml[i] = x;
                    continue;
                }
                const float m = fmaxf(ml[i].x, x.x), ref = m == -INFINITY ? 0.f : m, f = ex2_approx(ml[i].x - ref), g = x.y != 0.f ? ex2_approx(x.x - ref) : 0.f;
                ml[i] = make_float2(m, ml[i].y * f + x.y * g);
                o[i] = make_float4(o[i].x * f + v.x * g, o[i].y * f + v.y * g, o[i].z * f + v.z * g, o[i].w * f + v.w * g);
            }
            if (!is_open) begun_here = false;
            is_open = true;
            if (rec.head == PART_LAST) {
                if (!begun_here) {
                    put(done + 2 * blockIdx.x);
                    mine.head = PART_LAST;
                } else {
#pragma unroll
                    for (int i = 0; i < EACH; ++i) {
                        const int r = r0 + 8 * i;
                        if (r >= open.tokens) continue;
                        const float f = ml[i].y != 0.f ? 1.f / ml[i].y : 0.f;
                        const int row = open.token0 + r, token = (int)(((uint64_t)(uint32_t)row * a.group_mul) >> a.group_shift), h = open.head0 * a.group + row - token * a.group;
                        store4(const_cast<X*>(row_of<X>(a.O, open.b, h, token)) + 4 * sub, make_float4(o[i].x * f, o[i].y * f, o[i].z * f, o[i].w * f));
                        if (sub == 0) a.LSE[open.b * a.lse_sB + h * a.lse_sH + token] = ml[i].y != 0.f ? (ml[i].x + log2f(ml[i].y)) * LN2 : -INFINITY;
                    }
                }
                is_open = false;
            }
        }
        if (mine.head == PART_EMPTY) mine.head = PART_NONE;
        if (rec.tokens > 0) {
            const int slot = 2 * (first + w) + 1;
#pragma unroll
            for (int i = 0; i < EACH; ++i) {
                const int r = r0 + 8 * i;
                if (r >= a.slot_rows) continue;
                o[i] = *reinterpret_cast<const float4*>(a.part + slot_of(slot, r) * 64 + 4 * sub);
                ml[i] = a.ml[slot_of(slot, r)];
            }
            open = rec;
            is_open = begun_here = true;
        }
    }
    if (is_open) {
        if (begun_here) {
            mine.b = open.b; mine.head0 = open.head0; mine.token0 = open.token0; mine.tokens = open.tokens;
            put(done + 2 * blockIdx.x + 1);
        } else {
            mine.head = PART_GOES_ON;
            put(done + 2 * blockIdx.x);
        }
    }
    if (threadIdx.x == 0) a.parts[blockIdx.x] = mine;
}

// SIDE key heads side by side: 1, the warps have a stretch each, or 4, a head each of the CTA's stretch (a.Hk and a.group are then of four
// heads taken for one).  LONG: 16-bit types, where a block can have more batches than a piece; a kernel of its own, for
// it takes 1 % longer (64 requests of 4 096 tokens, 32 heads on 8, fp16: 98.0 us and 97.2; 16 of up to 2 047, 12 heads: 18.2 and 17.9).
template <class Rows, int SIDE, bool LONG>
__global__ void __launch_bounds__(WARPS * 32, Shape<Rows>::CTAS)
tree_few_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_kp,
                const __grid_constant__ CUtensorMap map_vp, const __grid_constant__ ServingArgs a) {
    typedef typename Rows::X X;
    typedef FewWork<Rows::KEYS> W;
    constexpr int KEYS = Rows::KEYS, STAGES = Shape<Rows>::STAGES, MINE = Rows::ROWS < 16 ? Rows::ROWS : 2;  // rows that a lane works on
    extern __shared__ __align__(1024) uint8_t few_smem[];
    FewShared<Rows, SIDE>& sh = *reinterpret_cast<FewShared<Rows, SIDE>*>(few_smem);
    const int warp = (int)uniform(threadIdx.x >> 5), lane = threadIdx.x & 31, me = SIDE == 1 ? blockIdx.x * WARPS + warp : blockIdx.x, group = a.group / SIDE;
    if (lane < (warp == 0 ? 4 : 0)) tma_prefetch_desc(lane == 0 ? &map_kp : lane == 1 ? &map_vp : lane == 2 ? &map_k : &map_v);
    if (lane == 0) {
        for (int s = 0; s < STAGES; ++s) mbar_init(&sh.full[warp][s], 1);
        if (warp == 0) sh.abort.id = 0;
        fence_mbar_init();
    }
    pdl_wait();
    pdl_trigger();
    const W work{a};
    Line<W> line;
    line.template find<WARPS * 32>(work, sh.search, blockIdx.x, gridDim.x, SIDE == 1 ? warp : 0);
    WaitNote wc{&sh.abort};
    PartRecord record{PART_EMPTY, 0, 0, 0, 0, 0};

    // Batches on their way: the run that they come from, the next one's number, 32 entries of the table from page `ids_at` on
    Segment put = {};
    int put_j = 0, put_slot = 0, put_segment = 0, ids = 0, ids_at = 0;
    bool more = true;
    auto copy_next = [&] {
        __syncwarp();
        if (!more) return;
        if (put_j == put.to) {
            Run run;
            more = line.next(work, run);
            if (more) {
                const int rows = min(a.block_tokens, run.r.tokens - run.i * a.block_tokens);
                put = {run.b, SIDE == 1 ? run.kvh : run.kvh * SIDE + warp, run.i * a.block_tokens, rows / SIDE, run.from, run.to, run.n - a.new_tiles, run.r.len, run.slot(me)};
                put_j = run.from;
                ids_at = INT_MAX;
                if (run.from > 0) {
                    record.head = run.to < run.n ? PART_GOES_ON : PART_LAST;
                } else {
                    if (record.head == PART_EMPTY) record.head = PART_NONE;
                    if (run.to < run.n) record.b = put.b, record.head0 = run.kvh, record.token0 = put.row0, record.tokens = rows;
                }
            } else {
                put.rows = 0;
            }
            if (lane == 0) sh.segments[warp][put_segment] = put;
            put_segment = (put_segment + 1) & 7;
            if (!more) return;
        }
        uint64_t* full = &sh.full[warp][put_slot];
        uint8_t* to = sh.ring[warp][put_slot];
        const int key = put_j * KEYS;
        const bool old = put_j < put.old;
        int row, b = put.b;
        if (old) {
            const int page = (int)(((uint64_t)(uint32_t)key * a.page_mul) >> a.page_shift);
            row = key - page * a.pool.page;
            if ((unsigned)(page - ids_at) >= 32u) {
                ids_at = page;
                ids = page + lane < a.pool.width ? __ldcg(a.pool.pages + b * a.pool.pages_stride + page + lane) : -1;
            }
            b = __shfl_sync(0xffffffffu, ids, page - ids_at);
        } else {
            row = key - put.old * KEYS;
        }
        if (lane == 0) {
            mbar_arrive_expect_tx(full, 4096);
            tma_load_tile(to, old ? &map_kp : &map_k, full, row, put.kvh, b);
            tma_load_tile(to + 2048, old ? &map_vp : &map_v, full, row, put.kvh, b);
        }
        ++put_j;
        put_slot = put_slot + 1 == STAGES ? 0 : put_slot + 1;
    };

    int get_slot = 0, get_segment = 0, j = 0;
    uint32_t phase = 0;
    Segment get = {};
    Rows w;
    uint64_t bits[MINE];
    int token_of[MINE], head_of[MINE];
    float m_sum[2] = {0.f, 0.f};
    float4* const sum = LONG ? a.sums + (blockIdx.x * WARPS + warp) * 256 : nullptr;
    constexpr int PIECE = LONG ? Pieces<X>::BATCHES : 1;
    for (int i = 1 - STAGES;; ++i) {
        copy_next();
        if (i < 0) continue;
        if (j == get.to) {  // the next run; between them the result of the one before
            __syncwarp();
            get = sh.segments[warp][get_segment];
            get_segment = (get_segment + 1) & 7;
            if (get.rows == 0) break;
            j = get.from;
            typename Rows::Query query;
#pragma unroll
            for (int k = 0; k < MINE; ++k) {
                const int r = Rows::row(k, lane), row = get.row0 + r;
                token_of[k] = (int)(((uint64_t)(uint32_t)row * a.group_mul) >> a.group_shift);
                head_of[k] = get.kvh * group + row - token_of[k] * group;
                const bool there = r < get.rows;
                query.load(k, there ? row_of<X>(a.Q, get.b, head_of[k], token_of[k]) : nullptr, lane, true);
                bits[k] = there && get.to > get.old ? tree_bits(a, get.b, token_of[k]) : 0ull;
            }
            w.start(query, a.flip);
        }
        if (!__all_sync(0xffffffffu, mbar_wait(wc, &sh.full[warp][get_slot], phase, W_FEW, i))) {
            for (const unsigned long long t0 = globaltimer_ns(); globaltimer_ns() - t0 < 100000ull;) {}  // copies in flight land
            break;
        }
        {
            const bool old = j < get.old;
            const int key0 = (old ? j : j - get.old) * KEYS, end = old ? get.len : a.T;
            w.batch(sh.ring[warp][get_slot], lane, key0, end, old && key0 + KEYS <= end, [&](int k, int key) { return old ? key < end : key < a.T && (bits[k] >> key & 1); }, a.scale_log2e,
                    [] {});
        }
        if (++get_slot == STAGES) get_slot = 0, phase ^= 1u;
        ++j;
        if constexpr (LONG) {
            const int done = j - get.from;
            if (j == get.to ? done > PIECE : done % PIECE == 0) sum_pieces(w, sum, m_sum, lane, done == PIECE, j == get.to);
        }
        if (j == get.to) {
            join(w);
            float f[MINE];
#pragma unroll
            for (int k = 0; k < MINE; ++k) f[k] = get.slot >= 0 ? 1.f : w.l[k] != 0.f ? 1.f / w.l[k] : 0.f;
            if (get.slot >= 0) {
                const int64_t at = (int64_t)get.slot * a.slot_rows;
                auto place = [&](int k) { return at + Rows::row(k, lane) + (SIDE == 1 ? 0 : token_of[k] * (a.group - group) + warp * group); };
                store_rows(w, lane, get.rows, f, [&](int k) { return a.part + place(k) * 64; });
#pragma unroll
                for (int k = 0; k < MINE; ++k)
                    if (Rows::row(k, lane) < get.rows && (Rows::ROWS < 16 ? lane == 0 : (lane & 3) == 0)) a.ml[place(k)] = make_float2(w.m[k], w.l[k]);
            } else {
                store_rows(w, lane, get.rows, f, [&](int k) { return const_cast<X*>(row_of<X>(a.O, get.b, head_of[k], token_of[k])); });
#pragma unroll
                for (int k = 0; k < MINE; ++k)
                    if (Rows::row(k, lane) < get.rows && (Rows::ROWS < 16 ? lane == 0 : (lane & 3) == 0))
                        a.LSE[get.b * a.lse_sB + head_of[k] * a.lse_sH + token_of[k]] = w.l[k] != 0.f ? (w.m[k] + log2f(w.l[k])) * LN2 : -INFINITY;
            }
        }
    }
    if (!a.parts) {
        __syncthreads();
        if (threadIdx.x == 0) report_abort(sh.abort, a.status);
        return;
    }
    if (lane == 0) sh.records[warp] = record;
    __syncthreads();
    if (threadIdx.x == 0) report_abort(sh.abort, a.status);
    if constexpr (SIDE == 1) join_warps<X, Rows::ROWS>(a, sh.records);
    else if (threadIdx.x == 0) a.parts[blockIdx.x] = record;
}

typedef void (*Kernel)(CUtensorMap, CUtensorMap, CUtensorMap, CUtensorMap, ServingArgs);
struct Entry {
    Kernel kernel;
    size_t smem;
    int per_sm, keys, rows;
};
template <class Rows, int SIDE = 1, bool LONG = false>
Entry entry() {
    return {tree_few_kernel<Rows, SIDE, LONG>, sizeof(FewShared<Rows, SIDE>), Shape<Rows>::CTAS, Rows::KEYS, Rows::ROWS};
}
template <class X, int SIDE>
Entry entry_16(bool pieces) {
    return pieces ? entry<RowsOf16<X>, SIDE, true>() : entry<RowsOf16<X>, SIDE>();
}
Entry pick(int dtype, int rows, int side, bool pieces = false) {
    if (side > 1) {
        if (dtype == HK_BF16) return entry_16<__nv_bfloat16, WARPS>(pieces);
        if (dtype == HK_F16) return entry_16<__half, WARPS>(pieces);
        return rows == 1 ? entry<RowsOfOne<1>, WARPS>() : rows == 2 ? entry<RowsOfOne<2>, WARPS>() : rows <= 4 ? entry<RowsOfOne<4>, WARPS>() : entry<RowsOf16<float>, WARPS>();
    }
    if (dtype == HK_BF16) return entry_16<__nv_bfloat16, 1>(pieces);
    if (dtype == HK_F16) return entry_16<__half, 1>(pieces);
    return rows == 1 ? entry<RowsOfOne<1>>() : rows == 2 ? entry<RowsOfOne<2>>() : rows <= 4 ? entry<RowsOfOne<4>>() : entry<RowsOf16<float>>();
}
// Key heads that a CTA takes side by side.  Four: its warps have nothing to add up, and where pools are stored token by token, with the heads
// next to each other, memory is asked for neighbouring lines at once (64 requests of 4 096 tokens, 32 heads on 8, bf16: 96 us, 100 with a head
// at a time; token by token 98 and 111; fp32, 16 requests of up to 2 047, 12 heads: 24 and 26).  But a block is then cut in four times as many
// parts, all of which one CTA adds up: at 14 to 18 for each block the two are alike (one request of 40 000 tokens: 36 and 22).
int heads_side_by_side(const ServingArgs& a, const Entry& e) {
    const int64_t blocks = (int64_t)a.B * a.Hk / WARPS, tiles = (int64_t)a.pool.width * a.pool.page / e.keys;
    return a.Hk % WARPS == 0 && std::min<int64_t>(sm_count() * e.per_sm / blocks, tiles / FewWork<1>::SHARE) <= 16 ? WARPS : 1;
}

}  // namespace

TreeFewPlan tree_few_plan(int dtype, int rows, int64_t keys) {
    const Entry e = pick(dtype, rows, 1);
    const int piece = dtype == HK_F32 ? 0 : dtype == HK_BF16 ? Pieces<__nv_bfloat16>::BATCHES : Pieces<__half>::BATCHES;
    return {std::min(rows, e.rows), e.keys, 2, sm_count() * e.per_sm, 2 * (WARPS + 1), piece > 0 && keys / e.keys + cdiv(16, e.keys) > piece ? WARPS * 16 : 0};
}

namespace {
// The kernel of the call, and how it cuts the work: `side` key heads are one from there on
Entry cut(ServingArgs& a, int dtype, int& side) {
    a.rows = a.T * a.group;
    side = heads_side_by_side(a, pick(dtype, a.rows, 1));
    const Entry e = pick(dtype, a.rows, side, a.sums != nullptr);
    a.block_tokens = std::min(a.rows, e.rows) * side;
    a.chunks = 1;
    divide_by(a.group, a.group_mul, a.group_shift);
    a.Hk /= side;
    a.group *= side;
    a.rows *= side;
    a.slot_rows = a.block_tokens;
    a.new_tiles = cdiv(a.T, e.keys);
    set_line(a, true, e.keys);
    return e;
}
}  // namespace

LineSum tree_few_line(ServingArgs a, int dtype, const int32_t* lens) {
    int side;
    const Entry e = cut(a, dtype, side);
    return e.keys == FewMath<float>::KEYS ? line_sum<FewWork<FewMath<float>::KEYS>>(a, lens) : line_sum<FewWork<FewMath<__half>::KEYS>>(a, lens);
}

int launch_tree_few(ServingArgs a, int dtype, cudaStream_t stream) {
    const int Hk = a.Hk;
    int side;
    const Entry e = cut(a, dtype, side);
    // once per device and kernel: more than 48 KB of shared memory
    static std::mutex mu;
    static Kernel known[HK_MAX_DEVICES][32];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= HK_MAX_DEVICES) return HK_ERR_CUDA;
    {
        std::lock_guard<std::mutex> lock(mu);
        for (Kernel& x : known[dev]) {
            if (x == e.kernel) break;
            if (x) continue;
            if (cudaFuncSetAttribute(e.kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)e.smem) != cudaSuccess) return check_launch();
            x = e.kernel;
            break;
        }
    }
    CUtensorMap k, v, kp, vp;
    int s;
    if ((s = prefix_tile_map(&k, a.K, dtype, a.B, Hk, a.T, e.keys, false)) || (s = prefix_tile_map(&v, a.V, dtype, a.B, Hk, a.T, e.keys, false)) ||
        (s = prefix_tile_map(&kp, a.pool.K, dtype, a.pool.n_pages, Hk, a.pool.page, e.keys, false, a.pool.K.strideM != HEAD_DIM)) ||
        (s = prefix_tile_map(&vp, a.pool.V, dtype, a.pool.n_pages, Hk, a.pool.page, e.keys, false, a.pool.V.strideM != HEAD_DIM)))
        return s;
    divide_by(a.pool.page, a.page_mul, a.page_shift);
    const int ctas = sm_count() * e.per_sm;
    LaunchConfig lc(ctas, WARPS * 32, e.smem, stream, 1, true);
    if (cudaLaunchKernelEx(&lc.cfg, e.kernel, k, v, kp, vp, a) != cudaSuccess) return check_launch();
    count_launch();
    if (!a.parts) return HK_OK;
    if (side == 1) {
        a.part += (size_t)2 * WARPS * ctas * a.slot_rows * 64;  // the CTAs' slots
        a.ml += (size_t)2 * WARPS * ctas * a.slot_rows;
    }
    return launch_combine(a, dtype, ctas, stream);
}

}  // namespace hk
