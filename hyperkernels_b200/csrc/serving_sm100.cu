// serving_sm100.cu -- attention within packed prompts, and of many new tokens against a cache of pages: blocks of 128 rows (fp32) or 256
// (16-bit types: two streams of 128) against tiles of keys, on tcgen05.
//
// A row is a token under one of the query heads that share a key head; 128 rows of a block are as many whole tokens as fit, their heads
// side by side (of more than 128 heads, each 128 are blocks of their own), so TMA brings the queries of a stream in one copy and a key is
// loaded once for all of them.  Lengths are on the device, so the work is cut there: block by block, head by
// head, request by request the tiles of keys make one line, of which every CTA takes an equal stretch.  A block of rows whose tiles fall to
// several CTAs leaves its parts (maximum, sum, weighted values) in slots of the workspace, a pair to a CTA, and a second kernel adds
// them up in their order.
//   Warp 0 cuts the stretch into items (a block of rows, a run of its tiles), makes them known to the other warps in a ring and loads
// their queries and tiles of keys by TMA, another the tiles of values, warp 1 issues the products S = Q K^T and, two products behind, O += P V (tcgen05, operands in shared and tensor memory),
// four warps to a stream take S through the softmax, a row to a thread.  All of them go from one item to the next without a barrier: the
// queries and the first tiles of the next are there, and its first scores under way, when the last weights of this one are worked out.
// Scores are three deep in tensor memory; P takes the place of its S.
//   fp32: x = h + l with h the upper 11 bits of the significand, which is what the tensor core reads of an fp32 word.  Q lies in tensor memory
// with its l parts, four warps write those of each tile beside it; a product is l h' + h l' + h h', in this order: what is left out is 2^-22 of it.  P V of
// a tile comes back into registers and is added there in fp32: the tensor core's additions cut off instead of rounding.
//   What bounds it: with 16-bit types the softmax warps, whose exponentials (four fifths on the special function units, 62 % of what these can do)
// take longer than the products (38 % of the tensor pipe): a tile of 256 rows by 128 keys takes 1.38 us, 0.85 the exponentials alone.  fp32:
// the tensor pipe (43 %) and, with it, the port of shared memory; a tile of 128 by 64 takes 1.3 us.  Beginning and end of a block are 1.6 us (fp32 3.7), of
// a CTA 6.  4 prompts of 4 096 tokens, 32 heads on 8, bf16: 363 us, 760 TFLOP/s, call after call with other inputs.
// How fast instructions come counts too: the loops are some 70 KB of code.  With fp32 trees the softmax warps are 80 bytes a thread short of registers.
#include <climits>
#include <cmath>
#include <mutex>
#include <numeric>

#include "serving_attention.cuh"

namespace hk {
namespace {

template <class X>
struct Rows {
    static constexpr bool LOW = sizeof(X) == 4;  // products in three parts
    static constexpr int STREAMS = LOW ? 1 : 2;  // blocks of 128 rows
    static constexpr int BLOCK = STREAMS * TILE;
    static constexpr int KEYS = LOW ? 64 : 128;  // of a tile
    static constexpr int SLOTS = LOW ? 3 : 4;    // of the rings of tiles of keys and of values
    static constexpr int THREADS = 384;
    static constexpr int SOFTMAX_WARPS = LOW ? 4 : 8;
    static constexpr int LEAST = LOW ? 4 : 2;    // tiles of a part of a block
    static constexpr int KV_RAW = KEYS * 64 * (int)sizeof(X), KV_BYTES = KV_RAW * (LOW ? 2 : 1);
    static constexpr int KV_BOX = KEYS * 128;    // 128 bytes of each row
    static constexpr int Q_BYTES = TILE * 64 * (int)sizeof(X), Q_BUFFERS = LOW ? 1 : 2;  // of a stream: K-major operands two items deep; fp32: on their way to tensor memory
    static constexpr int ITEMS = 8;
    // Tiles that one sum of O in tensor memory has at most.  Its additions cut off, 8e-8 of the sum for every 16 keys (6.4e-3 for 2^20): with so many less than
    // half a step of the type, 1.6e-4 of fp16 and 1.3e-3 of bf16.
    static constexpr int PIECE = LOW ? 0 : std::is_same<X, __half>::value ? 256 : 2048;
};

// Half a tile is masked, and a block's beginning and end take as long as a tile (fp32: 3.7 us, nearly three; where both streams have the same rows a tile
// takes half as long: 16 requests of up to 4 096 tokens, 32 drafts, 12 heads, bf16: 3.7 us less than with 3 / 2).
template <class X, bool TREE, bool SPLIT>
using RowsWork = Work<Rows<X>::KEYS, Rows<X>::LEAST, 3 * Rows<X>::LEAST, Rows<X>::KEYS * (sizeof(X) == 4 ? 6 : SPLIT ? 8 : 3) / 2, TREE, TREE ? 0 : 5>;

struct __align__(16) Item {
    int b, kvh, chunk;   // request, key head, which 128 of its query heads
    int token0, tokens;  // of the request; no tokens: the end
    int begin, len;      // of the packed rows; keys of the sequence, or in pages
    int key0;            // of the first tile
    int n0, n1;          // tiles of each stream
    int slot;            // of the workspace, -1: the result
    int new_tile;        // number of the tile that is the new tokens'
    int piece;           // of a longer run: GOES_ON with what the third slot has, NOT_LAST: what there is then comes there
};
enum { GOES_ON = 1, NOT_LAST = 2 };

template <class X, bool TREE, bool SPLIT>
struct __align__(16) RowsShared {
    typedef Rows<X> C;
    uint64_t q_full[C::Q_BUFFERS], q_empty[C::Q_BUFFERS], q_ready, p_full[3];
    uint64_t s_full[C::STREAMS][3], o_full[C::STREAMS][3];  // of a stream's own products: it does not see the other's
    uint64_t item_full[C::ITEMS], item_empty[C::ITEMS];
    uint64_t full[2][C::SLOTS], empty[2][C::SLOTS];  // keys, values
    uint64_t ready[2][C::SLOTS];                     // tended: low parts are there, what is behind a last key is cleared
    Item items[C::ITEMS];
    uint64_t pair_full[2][4], pair_done[2][4];       // what a warp has for that of the other stream's with the same rows; it has read that of it
    LineSearch<1> search;
    typename Line<RowsWork<X, TREE, SPLIT>>::Saved line;
    int keep[2][C::SLOTS];  // rows of the tile that are values, LAST: none follows
    uint32_t tmem_base;
    Abort abort;
};
constexpr int LAST = -1;

template <class X>
struct RowsSpace {
    typedef Rows<X> C;
    static constexpr int OFF_Q = 2 * C::SLOTS * C::KV_BYTES, OFF_O = OFF_Q + C::STREAMS * C::Q_BUFFERS * C::Q_BYTES, OFF_SH = OFF_O + (C::LOW ? 0 : C::SOFTMAX_WARPS * 4096), SMEM = OFF_SH + (int)sizeof(RowsShared<X, false, false>);
    static_assert(sizeof(RowsShared<X, false, false>) == sizeof(RowsShared<X, true, false>), "");
    static_assert(SMEM <= 232448, "exceeds the 227 KiB a CTA may opt in to");
};
// Tensor memory.  16-bit types: three buffers of 128 columns for scores and weights, O of two streams.  fp32: three buffers of
// 64 for scores and weights, two for the weights' low parts, O of a tile, Q and its low parts.
constexpr uint32_t COL_O = 384, LOW_COL_LOW = 192, LOW_COL_O = 320, LOW_COL_Q = 384;

enum RowsWait { W_Q = 501, W_Q_EMPTY, W_KV, W_READY, W_EMPTY, W_S, W_P, W_O, W_ITEM, W_ITEM_EMPTY, W_PAIR, W_PAIR_DONE };

// A product's place in the CTA's items, in the order they are issued in: tile by tile, stream by stream
template <bool SPLIT>  // of tiles of their own
struct Cursor {
    int j, t, n0, n1;
    __device__ __forceinline__ void start(int streams0, int streams1) {
        j = 0;
        n0 = streams0;
        n1 = streams1;
        t = n0 > 0 ? 0 : 1;
    }
    __device__ __forceinline__ bool first() const { return SPLIT || t == 0 || j >= n0; }  // of the tile's streams
    __device__ __forceinline__ bool last() const { return SPLIT || t == 1 || j >= n1; }
    __device__ __forceinline__ bool next() {  // false: the item is over
        if (t == 0 && j < n1) {
            t = 1;
            return true;
        }
        ++j;
        t = j < n0 ? 0 : 1;
        return j < max(n0, n1);
    }
};
struct Turn {  // a ring's place
    int at;
    uint32_t phase;
    __device__ __forceinline__ void next(int n) {
        if (++at == n) {
            at = 0;
            phase ^= 1u;
        }
    }
};
// 1 / x and log2 x of a row's sum, from 1 on.  fp32: rounded like those of blocks that are added up from parts.  16-bit types: 2^-22 off, which is a 2^11th of the
// result's rounding and less than the polynomial's exponentials leave in LSE; rounded ones on the way out of every block took 5 % of 16 prompts' time (56.0 and 59.3 us).
template <class X>
__device__ __forceinline__ float rcp_of(float x) {
    if constexpr (sizeof(X) == 4) return 1.f / x;
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
template <class X>
__device__ __forceinline__ float log2_of(float x) {
    if constexpr (sizeof(X) == 4) return log2f(x);
    return __log2f(x);
}

constexpr int BEHIND = 2;  // products that O is behind S
// Whether S may be issued when it is so many items in front of O.  fp32: the queries of an item come to tensor memory when the softmax is
// through with the item before the last, which waits for all of O of that.
template <bool LOW>
__device__ __forceinline__ bool may_go(int between) { return !LOW || between < 2; }

// The queries of `stream_tokens` tokens from `token` on under the heads from `head` on, 128 bytes of each (piece `x`)
__device__ __forceinline__ void tma_load_queries(void* to, const CUtensorMap* map, uint64_t* bar, int head, int token, int x, int b) {
    asm volatile(
        "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6, %7}], [%2];"
        ::"r"(smem_u32(to)), "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(0), "r"(head), "r"(token), "r"(x), "r"(b)
        : "memory");
}

// What the pieces of a run before this one came to (maximum and sum in `ml`, weighted values in `part`) added to O of a row in tensor memory; x: its maximum
// and sum, before and after.  Not inlined: in place it costs the blocks that have no pieces another 1 to 3 %.
__device__ __noinline__ float2 add_pieces(uint32_t at_o, const float* part, const float2* ml, bool valid, float2 x) {
    float f_old = 0.f, f_new = 1.f;
    if (valid) {
        const float2 before = *ml;
        const float mn = fmaxf(x.x, before.x), ref = mn == -INFINITY ? 0.f : mn;
        f_new = x.y != 0.f ? ex2_approx(x.x - ref) : 0.f;
        f_old = before.y != 0.f ? ex2_approx(before.x - ref) : 0.f;
        x = make_float2(mn, x.y * f_new + before.y * f_old);
    }
#pragma unroll 1
    for (int c = 0; c < 64; c += 16) {
        uint32_t y[16];
        tmem_ld16(at_o + c, y);
        tmem_wait_ld();
        const float4* const old = reinterpret_cast<const float4*>(part + c);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float4 v = valid ? old[i] : make_float4(0.f, 0.f, 0.f, 0.f);
            y[4 * i] = __float_as_uint(fmaf(v.x, f_old, __uint_as_float(y[4 * i]) * f_new));
            y[4 * i + 1] = __float_as_uint(fmaf(v.y, f_old, __uint_as_float(y[4 * i + 1]) * f_new));
            y[4 * i + 2] = __float_as_uint(fmaf(v.z, f_old, __uint_as_float(y[4 * i + 2]) * f_new));
            y[4 * i + 3] = __float_as_uint(fmaf(v.w, f_old, __uint_as_float(y[4 * i + 3]) * f_new));
        }
        tmem_st16(at_o + c, y);
    }
    tmem_wait_st();
    return x;
}
// SPLIT: the rows of a block are a stream's at most, and both streams have them, every other tile each.
// LONG: 16-bit types, where a block can have more than PIECE tiles.  A run of more is taken in pieces of PIECE, items of their own, which are added up in fp32 with the
// worker's third slot on their way out; each row by the thread that has it in all of them.  A kernel of its own, for where there can be such runs: what may have to be added up costs
// the ends of all blocks 0.2 us (512 prompts of 128 tokens, 32 heads on 8, bf16: 178 us and 168).
template <class X, bool TREE, bool SPLIT, bool LONG>
__global__ void __launch_bounds__(Rows<X>::THREADS, 1)
serving_rows_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_kp,
                    const __grid_constant__ CUtensorMap map_vp, const __grid_constant__ ServingArgs a) {
    typedef Rows<X> C;
    typedef RowsSpace<X> Space;
    constexpr bool LOW = C::LOW, BF16 = std::is_same<X, __nv_bfloat16>::value;
    constexpr int KEYS = C::KEYS, SLOTS = C::SLOTS, ITEMS = C::ITEMS;
    extern __shared__ __align__(1024) uint8_t smem[];
    uint8_t *sKV = smem, *sQ = smem + Space::OFF_Q;
    RowsShared<X, TREE, SPLIT>& sh = *reinterpret_cast<RowsShared<X, TREE, SPLIT>*>(smem + Space::OFF_SH);
    const int warp = (int)uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;

    if (warp == 2 && lane < (TREE ? 5 : 3)) tma_prefetch_desc(lane == 0 ? &map_q : lane == 1 ? &map_k : lane == 2 ? &map_v : lane == 3 ? &map_kp : &map_vp);
    if (threadIdx.x == 0) {
        for (int i = 0; i < C::Q_BUFFERS; ++i) {
            mbar_init(&sh.q_full[i], 1);
            mbar_init(&sh.q_empty[i], LOW ? 4 : 1);
        }
        mbar_init(&sh.q_ready, 4);
        for (int s = 0; s < SLOTS; ++s) {
            for (int v = 0; v < 2; ++v) {
                mbar_init(&sh.full[v][s], 1);
                mbar_init(&sh.empty[v][s], LOW || v == 0 ? 1 : 2);
                mbar_init(&sh.ready[v][s], LOW ? 2 : 1);
            }
        }
        for (int b = 0; b < 3; ++b) {
            mbar_init(&sh.p_full[b], 4);
            for (int t = 0; t < C::STREAMS; ++t) {
                mbar_init(&sh.s_full[t][b], 1);
                mbar_init(&sh.o_full[t][b], 1);
            }
        }
        for (int i = 0; i < ITEMS; ++i) {
            mbar_init(&sh.item_full[i], 1);
            mbar_init(&sh.item_empty[i], 2 + C::SOFTMAX_WARPS);
        }
        sh.abort.id = 0;
        for (int w = 0; w < 8; ++w) {
            mbar_init(&sh.pair_full[w >> 2][w & 3], 1);
            mbar_init(&sh.pair_done[w >> 2][w & 3], 1);
        }
        fence_mbar_init();
    }
    // rows that no query comes to stay zero
    if (!LOW)
        for (int i = threadIdx.x; i < C::STREAMS * C::Q_BUFFERS * C::Q_BYTES / 16; i += C::THREADS) reinterpret_cast<uint4*>(sQ)[i] = make_uint4(0, 0, 0, 0);
    fence_proxy_async_smem();
    if (warp == 1) {
        tmem_alloc(&sh.tmem_base, 512);
        tmem_relinquish();
        tc_fence_before_sync();
    }
    pdl_wait();
    pdl_trigger();
    {
        Line<RowsWork<X, TREE, SPLIT>> line;
        const RowsWork<X, TREE, SPLIT> work{a};
        line.template find<C::THREADS>(work, sh.search, blockIdx.x, gridDim.x, 0);
        if (threadIdx.x == 0) sh.line.line = line;
        if (line.dealt && threadIdx.x < line.DEAL_REQUESTS) sh.line.blocks[threadIdx.x] = threadIdx.x < a.B ? work.request(threadIdx.x).blocks : 0;
        __syncthreads();
    }
    tc_fence_after_sync();
    constexpr uint32_t tmem = 0;  // all columns are this CTA's
    if (sh.tmem_base != tmem) sh.abort.id = 598;
    WaitNote wc{&sh.abort};

    // three groups of warps, 168 registers a thread at the launch
    if (warp >= 4 && (!LOW || warp < 8)) {
        // ------------------------------ softmax ------------------------------
        if constexpr (LOW) asm volatile("setmaxnreg.inc.sync.aligned.u32 240;\n");
        else asm volatile("setmaxnreg.inc.sync.aligned.u32 216;\n");
        // The row of this thread: of the item's tokens the `my_token`-th, of the heads the `my_head`-th
        const int t = (warp - 4) >> 2, quarter = warp & 3, in_stream = quarter * 32 + lane, r = (SPLIT ? 0 : t * TILE) + in_stream;
        const int box_heads = min(a.group, TILE), my_token_in = in_stream / box_heads, my_head = in_stream - my_token_in * box_heads;
        const int my_token = my_token_in < a.stream_tokens ? (SPLIT ? 0 : t * a.stream_tokens) + my_token_in : INT_MAX;
        const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16);
        const float2 scale2 = make_float2(a.scale_log2e, a.scale_log2e);
        bool ok = true;
        int q0 = 0, own = 0;  // products of the items before; the stream's own ones so far
        int pairs = 0;        // items that both streams had
        auto wait = [&](uint64_t (&bar)[3], int c, int id) {  // of the stream's product c
            ok = __all_sync(0xffffffffu, mbar_wait(wc, &bar[c % 3], (c / 3) & 1, id, c));
            if (ok) tc_fence_after_sync();
            return ok;
        };
        // fp32: the queries of item n to tensor memory, from where those before are read no longer
        int fetched = 0;
        Turn fetch{0, 0u};
        auto fetch_queries = [&] {
            if constexpr (LOW) {
                if (!(ok = __all_sync(0xffffffffu, mbar_wait(wc, &sh.item_full[fetch.at], fetch.phase, W_ITEM, fetched)))) return;
                const int tokens = sh.items[fetch.at].tokens;
                fetch.next(ITEMS);
                if (tokens == 0) return;
                if (!(ok = __all_sync(0xffffffffu, mbar_wait(wc, &sh.q_full[0], fetched & 1, W_Q, fetched)))) return;
                ++fetched;
                const bool mine = my_token < tokens;
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    uint32_t y[32], z[32];
#pragma unroll
                    for (int c = 0; c < 8; ++c) {
                        const uint4 v = mine ? *reinterpret_cast<const uint4*>(sQ + (half * TILE + in_stream) * 128 + ((c ^ (in_stream & 7)) << 4)) : make_uint4(0, 0, 0, 0);
                        y[4 * c] = v.x ^ a.flip; y[4 * c + 1] = v.y ^ a.flip; y[4 * c + 2] = v.z ^ a.flip; y[4 * c + 3] = v.w ^ a.flip;
                    }
#pragma unroll
                    for (int i = 0; i < 32; ++i) z[i] = tf32_rest(y[i]);
                    tmem_st32(lanes + LOW_COL_Q + 32 * half, y);
                    tmem_st32(lanes + LOW_COL_Q + 64 + 32 * half, z);
                }
                tmem_wait_st();
                tc_fence_before_sync();
                mbar_arrive_warp(&sh.q_ready, lane);
                if (fetched == 1) mbar_arrive_warp(&sh.q_empty[0], lane);  // later ones' place is needed for O first
            }
        };
        // The result of an item, or a part of it, from O of its tiles: 32 columns at a time, in loops, for this runs once an item and what bounds it
        // is how fast its instructions come.  Where it goes is looked up again, not kept in registers all the while.
        auto finish = [&](int place_of_item, float m, float l, int n, const float* o) {
            asm volatile("" ::: "memory");
            const Item& it = sh.items[place_of_item];
            const bool valid = my_token < it.tokens && my_head < a.group - it.chunk * TILE && !(SPLIT && t && it.n1 == 0), live = __any_sync(0xffffffffu, valid);
            if (!LOW && n > 0 && !wait(sh.o_full[t], own - 1, W_O)) return;
            const int slot = it.slot;
            // A piece of a longer run, each stream's for itself
            const bool not_last = LONG && (it.piece & NOT_LAST);
            const int64_t at_sum = (2 * gridDim.x + blockIdx.x) * (int64_t)C::BLOCK + t * TILE + in_stream;
            if (LONG && (it.piece & GOES_ON)) {
                const float2 x = add_pieces(lanes + COL_O + t * 64, a.part + at_sum * 64, a.ml + at_sum, valid, make_float2(m, l));
                m = x.x;
                l = x.y;
            }
            // Both streams' rows: each warp adds half of the columns up.  O is in tensor memory for both to read, their maxima and sums go
            // through the place that rows of O leave by.
            const bool both = SPLIT && it.n1 > 0 && !not_last;
            float f0 = 1.f, f1 = 0.f;
            auto pair = [&](uint64_t (&bar)[2][4], int id) {
                tc_fence_before_sync();
                mbar_arrive_warp(&bar[t][quarter], lane);
                ok = __all_sync(0xffffffffu, mbar_wait(wc, &bar[t ^ 1][quarter], pairs & 1, id, pairs));
                tc_fence_after_sync();
            };
            if (both) {
                float2* const room = reinterpret_cast<float2*>(smem + Space::OFF_O) + quarter * 512 + lane;
                room[t * 2048] = make_float2(m, l);
                pair(sh.pair_full, W_PAIR);
                if (!ok) return;
                const float2 other = room[(t ^ 1) * 2048];
                const float mn = fmaxf(m, other.x), ref = mn == -INFINITY ? 0.f : mn;
                f0 = l != 0.f ? ex2_approx(m - ref) : 0.f;
                f1 = other.y != 0.f ? ex2_approx(other.x - ref) : 0.f;
                l = l * f0 + other.y * f1;
                m = mn;
            }
            const bool kept = slot >= 0 || not_last;  // as a part
            const float f = kept ? 1.f : l != 0.f ? rcp_of<X>(l) : 0.f;
            const int b = TREE ? it.b : 0, row = it.begin + it.token0 + (valid ? my_token : 0), h = it.kvh * a.group + it.chunk * TILE + my_head;
            X* const to = const_cast<X*>(row_of<X>(a.O, b, h, row));
            const int64_t at_slot = not_last ? at_sum : (int64_t)slot * (SPLIT ? TILE : C::BLOCK) + r;
            // Through shared memory, so that 8 lanes store 128 bytes of a row: a row to a lane is 32 lines an instruction.  fp32: in place of the
            // warp's rows of the queries that have just gone to tensor memory, 16 lanes to a row.
            if constexpr (LOW) {
                if (live) {
                    uint8_t* const stage = sQ + quarter * 4096;
#pragma unroll
                    for (int c = 0; c < 16; ++c)
                        *reinterpret_cast<float4*>(stage + (c >> 3) * (TILE * 128) + lane * 128 + (((c & 7) ^ (lane & 7)) << 4)) =
                            make_float4(o[4 * c] * f, o[4 * c + 1] * f, o[4 * c + 2] * f, o[4 * c + 3] * f);
                    __syncwarp();
                    const uint64_t place = !valid ? 0ull : slot >= 0 ? reinterpret_cast<uint64_t>(a.part + at_slot * 64) : reinterpret_cast<uint64_t>(to);
#pragma unroll 4
                    for (int i = 0; i < 16; ++i) {
                        const int from = 2 * i + (lane >> 4), c = lane & 15;
                        const uint64_t at = __shfl_sync(0xffffffffu, place, from);
                        const float4 v = *reinterpret_cast<const float4*>(stage + (c >> 3) * (TILE * 128) + from * 128 + (((c & 7) ^ (from & 7)) << 4));
                        if (at) reinterpret_cast<float4*>(at)[c] = v;
                    }
                }
                fence_proxy_async_smem();
                mbar_arrive_warp(&sh.q_empty[0], lane);
            } else if (both) {
                uint32_t y[32], z[32];
                tmem_ld32(lanes + COL_O + t * 64 + 32 * t, y);
                tmem_ld32(lanes + COL_O + (t ^ 1) * 64 + 32 * t, z);
                tmem_wait_ld();
                pair(sh.pair_done, W_PAIR_DONE);  // before a product writes over O, and rows over what the other warp reads
                ++pairs;
                if (!ok) return;
                f0 *= f;
                f1 *= f;
#pragma unroll
                for (int i = 0; i < 32; ++i) y[i] = __float_as_uint(fmaf(__uint_as_float(z[i]), f1, __uint_as_float(y[i]) * f0));
                if (slot >= 0) {
                    uint4* const whole = reinterpret_cast<uint4*>(a.part + at_slot * 64) + 8 * t;
                    if (valid) {
#pragma unroll
                        for (int i = 0; i < 8; ++i) whole[i] = make_uint4(y[4 * i], y[4 * i + 1], y[4 * i + 2], y[4 * i + 3]);
                    }
                } else if (live) {  // four lanes to half a row
                    uint4* const mine = reinterpret_cast<uint4*>(smem + Space::OFF_O + (warp - 4) * 4096);
#pragma unroll
                    for (int i = 0; i < 16; ++i) y[i] = pack<X>(__uint_as_float(y[2 * i]), __uint_as_float(y[2 * i + 1]));
#pragma unroll
                    for (int i = 0; i < 4; ++i) mine[lane * 4 + (i ^ (lane >> 1 & 3))] = make_uint4(y[4 * i], y[4 * i + 1], y[4 * i + 2], y[4 * i + 3]);
                    __syncwarp();
                    const uint64_t place = valid ? reinterpret_cast<uint64_t>(to + 32 * t) : 0ull;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int from = 8 * i + (lane >> 2);
                        const uint64_t at = __shfl_sync(0xffffffffu, place, from);
                        const uint4 v = mine[from * 4 + ((lane ^ (from >> 1)) & 3)];
                        if (at) reinterpret_cast<uint4*>(at)[lane & 3] = v;
                    }
                    __syncwarp();
                }
            } else if (kept) {
                uint4* const whole = reinterpret_cast<uint4*>(a.part + at_slot * 64);
#pragma unroll 1
                for (int half = 0; half < 2; ++half) {
                    uint32_t y[32];
                    if (n > 0) {
                        tmem_ld32(lanes + COL_O + t * 64 + 32 * half, y);
                        tmem_wait_ld();
                    } else {
#pragma unroll
                        for (int i = 0; i < 32; ++i) y[i] = 0u;
                    }
                    if (valid) {
#pragma unroll
                        for (int i = 0; i < 8; ++i) whole[8 * half + i] = make_uint4(y[4 * i], y[4 * i + 1], y[4 * i + 2], y[4 * i + 3]);
                    }
                }
            } else if (live) {
                uint4* const mine = reinterpret_cast<uint4*>(smem + Space::OFF_O + (warp - 4) * 4096);
#pragma unroll 1
                for (int half = 0; half < 2; ++half) {
                    uint32_t y[32];
                    tmem_ld32(lanes + COL_O + t * 64 + 32 * half, y);
                    tmem_wait_ld();
#pragma unroll
                    for (int i = 0; i < 16; ++i) y[i] = pack<X>(__uint_as_float(y[2 * i]) * f, __uint_as_float(y[2 * i + 1]) * f);
#pragma unroll
                    for (int i = 0; i < 4; ++i) mine[lane * 8 + ((4 * half + i) ^ (lane & 7))] = make_uint4(y[4 * i], y[4 * i + 1], y[4 * i + 2], y[4 * i + 3]);
                }
                __syncwarp();
                const uint64_t place = valid ? reinterpret_cast<uint64_t>(to) : 0ull;
#pragma unroll 4
                for (int i = 0; i < 8; ++i) {
                    const int from = 4 * i + (lane >> 3);
                    const uint64_t at = __shfl_sync(0xffffffffu, place, from);
                    const uint4 v = mine[from * 8 + ((lane ^ from) & 7)];
                    if (at) reinterpret_cast<uint4*>(at)[lane & 7] = v;
                }
                __syncwarp();
            }
            if (!LOW) tc_fence_before_sync();
            if (valid && (!(SPLIT && t) || not_last)) {
                if (kept) a.ml[at_slot] = make_float2(m, l);
                else a.LSE[b * a.lse_sB + h * a.lse_sH + row] = l != 0.f ? (m + log2_of<X>(l)) * LN2 : -INFINITY;
            }
            mbar_arrive_warp(&sh.item_empty[place_of_item], lane);
        };
        int last_at = -1, last_n = 0;  // 16-bit types: the item before this one, whose O is taken out under the first tile of this
        float last_m = 0.f, last_l = 0.f;
        Turn get{0, 0u};
        while (ok) {
            if (!(ok = __all_sync(0xffffffffu, mbar_wait(wc, &sh.item_full[get.at], get.phase, W_ITEM, q0)))) break;
            const Item& it = sh.items[get.at];
            const int tokens = it.tokens;
            if (LOW && tokens == 0) break;
            const bool valid = my_token < tokens && my_head < a.group - it.chunk * TILE, live = __any_sync(0xffffffffu, valid);
            const int token = it.token0 + (valid ? my_token : 0);
            constexpr int STEP = SPLIT ? 2 * KEYS : KEYS;  // keys from a tile of the stream's to the next
            const int new_tile = SPLIT ? it.new_tile - t : it.new_tile, n = tokens == 0 ? 0 : t == 0 ? it.n0 : it.n1;
            const int limit = (!valid ? INT_MAX / 2 : !TREE && a.causal ? token + 1 : it.len) - it.key0 - (SPLIT ? t * KEYS : 0);  // keys that the row sees, from the first tile's on
            const uint64_t bits = TREE && valid ? tree_bits(a, it.b, token) : 0ull;
            // the item's product of tile j: the other stream's come in between
            const int between = t == 1 ? it.n0 : it.n1 > 0 ? INT_MAX : 0;
            auto product = [&](int j) { return q0 + j + min(j + t, between); };
            float o[LOW ? 64 : 1], m = -INFINITY, l = 0.f;
            if constexpr (LOW) {
                // O_j of every tile comes back and is added here: o = o * before + O_j
                float before = 0.f, alpha = 0.f;
#pragma unroll
                for (int i = 0; i < 64; ++i) o[i] = 0.f;
                auto add = [&](int j) {
                    if (!wait(sh.o_full[0], q0 + j, W_O) || !live) return;
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        uint32_t x[32];
                        tmem_ld32(lanes + LOW_COL_O + 32 * half, x);
                        tmem_wait_ld();
#pragma unroll
                        for (int i = 0; i < 32; i += 2) {
                            float2& y = reinterpret_cast<float2&>(o[32 * half + i]);
                            y = __ffma2_rn(y, make_float2(before, before), make_float2(__uint_as_float(x[i]), __uint_as_float(x[i + 1])));
                        }
                    }
                };
                for (int j = fetched == 0 ? -1 : 0; j <= n; ++j) {  // a step behind the last tile, for its O; one in front of the first item's, for its queries
                    if (j >= 0 && j < n && !wait(sh.s_full[0], q0 + j, W_S)) break;
                    if (j < 0 || j == n - 1) {  // the next item's: all scores of this one are there
                        fetch_queries();
                        if (!ok) break;
                        if (j < 0) continue;
                    }
                    const int q = q0 + j;
                    const uint32_t at_s = lanes + q % 3 * 64, at_low = lanes + LOW_COL_LOW + (q & 1) * 64;
                    if (live && j < n) {
                        const bool fresh = TREE && j == new_tile;
                        const int lim = fresh ? 0 : limit - j * KEYS;  // columns the row sees
                        uint32_t x[64];
                        tmem_ld32p(at_s, x);
                        tmem_ld32p(at_s + 32, x + 32);
                        tmem_wait_ld();
                        if (lim < KEYS) {
#pragma unroll
                            for (int i = 0; i < 64; ++i)
                                if (fresh ? !(bits >> i & 1) : i >= lim) x[i] = __float_as_uint(-INFINITY);
                        }
                        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                        for (int i = 0; i < 64; i += 2) mx[(i >> 1) & 3] = fmax3(mx[(i >> 1) & 3], __uint_as_float(x[i]), __uint_as_float(x[i + 1]));
                        const float mn = fmaxf(m, fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * a.scale_log2e), ref = mn == -INFINITY ? 0.f : mn;
                        alpha = ex2_approx(m - ref);  // 0 while m is -inf
                        m = mn;
                        const float2 nm = make_float2(-ref, -ref);
                        float2 sum[2] = {};
#pragma unroll
                        for (int c = 0; c < 64; c += 32) {
                            uint32_t z[32];
#pragma unroll
                            for (int i = 0; i < 32; i += 2) {
                                const float2 e = __ffma2_rn(make_float2(__uint_as_float(x[c + i]), __uint_as_float(x[c + i + 1])), scale2, nm);
                                const float2 w = make_float2(ex2_approx(e.x), ex2_approx(e.y));
                                sum[(i >> 1) & 1] = __fadd2_rn(sum[(i >> 1) & 1], w);
                                x[c + i] = __float_as_uint(w.x);
                                x[c + i + 1] = __float_as_uint(w.y);
                                z[i] = __float_as_uint(w.x - __uint_as_float(x[c + i] & 0xffffe000u));
                                z[i + 1] = __float_as_uint(w.y - __uint_as_float(x[c + i + 1] & 0xffffe000u));
                            }
                            tmem_st32p(at_s + c, x + c);
                            tmem_st32(at_low + c, z);
                        }
                        l = fmaf(l, alpha, (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y));
                        tmem_wait_st();
                    }
                    if (j > 0) add(j - 1);  // before O_j may come to the same place
                    if (!ok || j == n) break;
                    tc_fence_before_sync();
                    mbar_arrive_warp(&sh.p_full[q % 3], lane);
                    before = alpha;
                }
            } else {
                // O stays in tensor memory and is scaled there when a tile's weights come to more than MOST: a stale maximum makes them larger,
                // which neither fp32 sums nor 16-bit types mind up to there
                constexpr float MOST = lift<X>() > 0.f ? 32768.f : 256.f;  // 2^8 of the reference's own weight
                constexpr int POLY_OF = 5;  // of so many pairs of weights, one by the polynomial
                const uint32_t at_o = lanes + COL_O + t * 64;
                uint32_t x[128];
                for (int j = 0; j < max(n, 1); ++j) {
                    if (n > 0 && !wait(sh.s_full[t], own, W_S)) break;
                    const int q = product(j);
                    const uint32_t at_s = lanes + q % 3 * 128;
                    if (live && n > 0) {
                        const bool fresh = TREE && j * STEP == new_tile * KEYS;
                        const int lim = fresh ? 0 : limit - j * STEP;  // columns the row sees
                        auto load = [&] {
#pragma unroll
                            for (int c = 0; c < 128; c += 32) tmem_ld32p(at_s + c, x + c);
                            tmem_wait_ld();
                        };
                        float2 sum[2];
                        // The weights take the type of the values: half a step of it each.  A run of them is summed and packed while the next
                        // one's exponentials are under way.
                        auto weights = [&] {
                            constexpr int RUN = 16;
                            const float2 nm = make_float2(lift<X>() - m, lift<X>() - m);
                            sum[0] = sum[1] = make_float2(0.f, 0.f);
#pragma unroll
                            for (int c = 0; c < 128 + RUN; c += RUN) {
#pragma unroll
                                for (int i = c; i < c + RUN && i < 128; i += 2) {
                                    const float2 e = __ffma2_rn(make_float2(__uint_as_float(x[i]), __uint_as_float(x[i + 1])), scale2, nm);
                                    const float2 w = (i >> 1) % POLY_OF == POLY_OF - 1 ? ex2_poly(e) : make_float2(ex2_approx(e.x), ex2_approx(e.y));
                                    x[i] = __float_as_uint(w.x);
                                    x[i + 1] = __float_as_uint(w.y);
                                }
#pragma unroll
                                for (int i = c - RUN; i >= 0 && i < c; i += 2) {
                                    const float2 w = make_float2(__uint_as_float(x[i]), __uint_as_float(x[i + 1]));
                                    sum[(i >> 1) & 1] = __fadd2_rn(sum[(i >> 1) & 1], w);
                                    x[i / 2] = pack<X>(w.x, w.y);
                                }
                            }
                            return (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
                        };
                        // Most tiles raise no maximum by much: their weights are taken by the one there is (of the first tile: by its own), and
                        // their sum tells if it was too low.  The polynomial would make small numbers of a large argument and of a NaN.
                        float alpha = 1.f, add = 0.f;
                        bool done = false;
                        if (__all_sync(0xffffffffu, lim >= KEYS)) {
                            load();
                            if (j == 0) {
                                float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                                for (int i = 0; i < 128; i += 2) mx[(i >> 1) & 3] = fmax3(mx[(i >> 1) & 3], __uint_as_float(x[i]), __uint_as_float(x[i + 1]));
                                m = fmaxf(fmax3(mx[0], mx[1], mx[2]), mx[3]) * a.scale_log2e;
                            }
                            float poly_top = -INFINITY;
#pragma unroll
                            for (int i = 2 * (POLY_OF - 1); i < 128; i += 2 * POLY_OF) poly_top = max3_or_nan(poly_top, __uint_as_float(x[i]), __uint_as_float(x[i + 1]));
                            add = weights();
                            done = __all_sync(0xffffffffu, !valid || (add <= MOST && fmaf(poly_top, a.scale_log2e, -m) <= 8.f));
                            if (done) {
                                tmem_st32p(at_s, x);
                                tmem_st32p(at_s + 32, x + 32);
                            } else if (j == 0) {
                                m = -INFINITY;
                            }
                        }
                        if (!done) {
                            // The others, masked ones among them, 32 columns at a time: the maximum, then the weights.  Columns that no row of the
                            // warp sees are not worked on.
                            const int all_see = fresh ? 0 : __reduce_min_sync(0xffffffffu, lim), some_see = fresh ? a.T : __reduce_max_sync(0xffffffffu, valid ? lim : 0);
                            auto scores = [&](int c) {
                                tmem_ld32p(at_s + c, x);
                                tmem_wait_ld();
                                if (c + 32 > all_see) {
                                    const int left = lim - c;
                                    const uint32_t own_bits = (uint32_t)(bits >> (c & 63));
#pragma unroll
                                    for (int i = 0; i < 32; ++i)
                                        if (fresh ? !(own_bits >> i & 1) : i >= left) x[i] = __float_as_uint(-INFINITY);
                                }
                            };
                            float top = -INFINITY;
#pragma unroll 1
                            for (int c = 0; c < 128 && c < some_see; c += 32) {
                                scores(c);
                                float mx[4] = {top, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                                for (int i = 0; i < 32; i += 2) mx[(i >> 1) & 3] = fmax3(mx[(i >> 1) & 3], __uint_as_float(x[i]), __uint_as_float(x[i + 1]));
                                top = fmaxf(fmax3(mx[0], mx[1], mx[2]), mx[3]);
                            }
                            top *= a.scale_log2e;
                            const bool raise = top > m;
                            if (raise) {
                                alpha = ex2_approx(m - top);  // 0 from -inf
                                m = top;
                            }
                            if (j > 0 && __any_sync(0xffffffffu, raise)) {
                                if (!wait(sh.o_full[t], own - 1, W_O)) break;
#pragma unroll 1
                                for (int c = 0; c < 64; c += 32) {
                                    uint32_t y[32];
                                    tmem_ld32(at_o + c, y);
                                    tmem_wait_ld();
#pragma unroll
                                    for (int i = 0; i < 32; ++i) y[i] = __float_as_uint(__uint_as_float(y[i]) * alpha);
                                    tmem_st32(at_o + c, y);
                                }
                            }
                            const float up = m == -INFINITY ? 0.f : lift<X>() - m;
                            const float2 nm = make_float2(up, up);
                            sum[0] = sum[1] = make_float2(0.f, 0.f);
#pragma unroll 1
                            for (int c = 0; c < 128; c += 32) {  // 16 columns of weights take the place of scores that are done with
                                uint32_t w16[16];
                                if (c < some_see) {
                                    scores(c);
#pragma unroll
                                    for (int i = 0; i < 32; i += 2) {
                                        const float2 e = __ffma2_rn(make_float2(__uint_as_float(x[i]), __uint_as_float(x[i + 1])), scale2, nm);
                                        const float2 w = make_float2(ex2_approx(e.x), ex2_approx(e.y));
                                        sum[(i >> 1) & 1] = __fadd2_rn(sum[(i >> 1) & 1], w);
                                        w16[i / 2] = pack<X>(w.x, w.y);
                                    }
                                } else {
#pragma unroll
                                    for (int i = 0; i < 16; ++i) w16[i] = 0u;
                                }
                                tmem_st16(at_s + c / 2, w16);
                            }
                            add = (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
                        }
                        l = fmaf(l, alpha, add);
                        tmem_wait_st();
                    }
                    if (j == 0 && last_at >= 0) finish(last_at, last_m, last_l, last_n, nullptr);
                    if (n == 0 || !ok) break;
                    tc_fence_before_sync();
                    mbar_arrive_warp(&sh.p_full[q % 3], lane);
                    ++own;
                }
                if (tokens == 0) break;
            }
            q0 += it.n0 + it.n1;
            if (!ok) break;
            if constexpr (LOW) {
                finish(get.at, m, l, n, o);
            } else {
                last_at = get.at;
                last_n = n;
                last_m = m - lift<X>();  // what the weights were taken by
                last_l = l;
            }
            get.next(ITEMS);
        }
    } else {
        if constexpr (LOW) asm volatile("setmaxnreg.dec.sync.aligned.u32 120;\n");
        else asm volatile("setmaxnreg.dec.sync.aligned.u32 72;\n");
        if (warp == 0 || warp == (LOW ? 10 : 3)) {
            // ------------------------------ items, tiles of keys; tiles of values ------------------------------
            const RowsWork<X, TREE, SPLIT> work{a};
            Line<RowsWork<X, TREE, SPLIT>> line;
            line = sh.line.line;
            bool ok = true;
            const bool v = warp != 0;
            PartRecord record{PART_EMPTY, 0, 0, 0, 0, 0};
            Turn get{0, 0u}, at{0, 0u};  // of the items, of the ring
            int left = 0;  // LONG: tiles of the run behind the piece before
            // An item's tiles for each stream, of the next `count`
            auto share_out = [&](Item& it, int count) {
                if constexpr (LONG) {
                    left = count;
                    if (count >= C::PIECE + C::LEAST) {
                        count = C::PIECE;
                        it.piece |= NOT_LAST;
                    }
                    left -= count;
                }
                it.n0 = count;
                it.n1 = 0;
                if (!LOW && it.tokens > a.stream_tokens) {
                    it.n1 = count;
                    if (!TREE && a.causal) it.n0 = max(0, min((it.token0 + a.stream_tokens + KEYS - 1 - it.key0) / KEYS, count));
                }
                if (SPLIT) {
                    it.n0 = (count + 1) / 2;
                    it.n1 = count / 2;
                }
            };
            // The next item into the ring; one without tokens at the end of the stretch
            auto publish = [&](Item& it) {
                if (LONG && left > 0) {  // the next piece of what the item before began
                    __syncwarp();
                    it = sh.items[get.at == 0 ? ITEMS - 1 : get.at - 1];
                    it.key0 += C::PIECE * KEYS;
                    it.new_tile -= C::PIECE;
                    it.piece = GOES_ON;
                    share_out(it, left);
                    return;
                }
                Run run;
                it.tokens = 0;
                it.piece = 0;
                if (!line.next(work, run, sh.line.blocks)) return;
                it.b = run.b; it.kvh = run.kvh; it.chunk = run.chunk;
                it.token0 = run.i * a.block_tokens;
                it.tokens = min(a.block_tokens, run.r.tokens - it.token0);
                it.begin = run.r.begin; it.len = run.r.len; it.key0 = run.from * KEYS;
                it.new_tile = TREE ? run.n - 1 - run.from : -1;
                share_out(it, run.to - run.from);
                it.slot = run.slot(blockIdx.x);
                if (run.from > 0) {
                    record.head = run.to < run.n ? PART_GOES_ON : PART_LAST;
                } else {
                    if (record.head == PART_EMPTY) record.head = PART_NONE;
                    if (run.to < run.n) {
                        record.b = TREE ? it.b : 0; record.head0 = it.kvh * a.group + it.chunk * TILE; record.heads = min(TILE, a.group - it.chunk * TILE);
                        record.token0 = it.begin + it.token0; record.tokens = it.tokens;
                    }
                }
            };
            int made = 0;
            bool filled = false;         // each place of the ring once
            int ids_b = -1, ids_from = 0, ids = 0;  // entry ids_from + lane of request ids_b's row of the table
            uint8_t* const ring = sKV + (v ? SLOTS * C::KV_BYTES : 0);
            while (true) {
                Item it;
                if (v) {
                    if (!(ok = __all_sync(0xffffffffu, mbar_wait(wc, &sh.item_full[get.at], get.phase, W_ITEM, made)))) break;
                    it = sh.items[get.at];
                    mbar_arrive_warp(&sh.item_empty[get.at], lane);
                } else {
                    publish(it);
                    if (!(ok = __all_sync(0xffffffffu, mbar_wait(wc, &sh.item_empty[get.at], get.phase ^ 1u, W_ITEM_EMPTY, made)))) break;
                    if (lane == 0) {
                        sh.items[get.at] = it;
                        mbar_arrive(&sh.item_full[get.at]);
                    }
                }
                get.next(ITEMS);
                if (it.tokens == 0) break;
                if (!v) {  // its queries, in the place of those of the item before, or before that
                    const int buf = made & (C::Q_BUFFERS - 1), use = made / C::Q_BUFFERS;
                    if (use > 0 && !(ok = __all_sync(0xffffffffu, mbar_wait(wc, &sh.q_empty[buf], (use - 1) & 1, W_Q_EMPTY, made)))) break;
                    if (lane == 0) {
                        const int streams = it.n1 > 0 && !SPLIT ? 2 : 1, head = it.kvh * a.group + it.chunk * TILE;
                        mbar_arrive_expect_tx(&sh.q_full[buf], streams * a.q_bytes);
#pragma unroll
                        for (int x = 0; x < 2; ++x) {  // streams, or halves of the rows
                            if (LOW || x < streams)
                                tma_load_queries(sQ + (buf * 2 + x) * (TILE * 128), &map_q, &sh.q_full[buf], head, it.begin + it.token0 + (LOW ? 0 : x * a.stream_tokens), LOW ? x : 0, TREE ? it.b : 0);
                        }
                    }
                }
                ++made;
                const int n = SPLIT ? it.n0 + it.n1 : max(it.n0, it.n1);
                int key = it.key0;
                for (int j = 0; j < n; ++j, key += KEYS) {
                    if (filled && !(ok = __all_sync(0xffffffffu, mbar_wait(wc, &sh.empty[v][at.at], at.phase ^ 1u, W_EMPTY, j)))) break;
                    uint64_t* const full = &sh.full[v][at.at];
                    uint8_t* const to = ring + at.at * C::KV_BYTES;
                    const bool fresh = TREE && j == it.new_tile;
                    if (lane == 0) {
                        sh.keep[v][at.at] = v && !fresh ? min(KEYS, it.len - key) : KEYS;
                        mbar_arrive_expect_tx(full, C::KV_RAW);
                        if (!TREE || fresh) tma_load_tile(to, v ? &map_v : &map_k, full, TREE ? 0 : it.begin + key, it.kvh, TREE ? it.b : 0);
                    }
                    if constexpr (TREE) {
                        if (!fresh) {
                            // A box of a page to a lane; pages that are none, and those behind the last, read as zeros.  The table is looked up 32
                            // entries at a time: a look for every tile took longer than the tile.
                            const int k = key + lane * a.box, page = (int)(((uint64_t)(uint32_t)k * a.page_mul) >> a.page_shift);
                            const int first = __shfl_sync(0xffffffffu, page, 0), last = __shfl_sync(0xffffffffu, page, KEYS / a.box - 1);
                            if (it.b != ids_b || first < ids_from || last >= ids_from + 32) {
                                ids_b = it.b;
                                ids_from = first;
                                ids = first + lane < a.pool.width ? __ldcg(a.pool.pages + it.b * a.pool.pages_stride + first + lane) : -1;
                            }
                            const int id = __shfl_sync(0xffffffffu, ids, (page - ids_from) & 31);
                            if (lane < KEYS / a.box) {
#pragma unroll
                                for (int half = 0; half < (LOW ? 2 : 1); ++half)
                                    tma_load_box(to + half * C::KV_BOX + lane * a.box * 128, v ? &map_vp : &map_kp, full, k - page * a.pool.page, half, it.kvh, k < it.len ? id : -1);
                            }
                        }
                    }
                    at.next(SLOTS);
                    filled |= at.at == 0;
                }
                if (!ok) break;
            }
            if (ok && (LOW || v)) {  // to those who tend the tiles: no more
                ok = !filled || __all_sync(0xffffffffu, mbar_wait(wc, &sh.empty[v][at.at], at.phase ^ 1u, W_EMPTY, -1));
                if (ok && lane == 0) {
                    sh.keep[v][at.at] = LAST;
                    mbar_arrive(&sh.full[v][at.at]);
                }
            }
            if (!v && a.parts && lane == 0) a.parts[blockIdx.x] = record;
            // a CTA that gave up may have copies in flight: they get time to land
            if (!ok)
                for (const unsigned long long t0 = globaltimer_ns(); globaltimer_ns() - t0 < 100000ull;) {}
        } else if (warp == 1) {
            // ------------------------------ products ------------------------------
            const uint32_t leader = elect_one_sync();
            struct Barrier {
                uint64_t* bar;
                uint32_t parity;
            };
            // each barrier is looked at while the products before it are still being issued, and waited for if that look came too early
            auto seen = [&](const Barrier& x) { return mbar_test_wait(x.bar, x.parity); };
            auto wait = [&](bool was_seen, const Barrier& x, int id, int aux) {
                return __all_sync(0xffffffffu, was_seen) || (bool)__all_sync(0xffffffffu, mbar_wait(wc, x.bar, x.parity, id, aux));
            };
            const uint32_t kv_addr = smem_u32(sKV);
            const Desc q_desc = make_smem_desc(smem_u32(sQ), 16, 1024, DESC_SW128), k_desc = make_smem_desc(kv_addr, 16, 1024, DESC_SW128),
                       v_desc = LOW ? mnmajor_desc(kv_addr + SLOTS * C::KV_BYTES, 0, C::KV_BOX) : make_smem_desc(kv_addr + SLOTS * C::KV_BYTES, 16, 1024, DESC_SW128);
            const uint32_t negate = a.flip ? IDESC_NEGATE_A : 0u;
            Turn k_tile{0, 0u}, v_tile{0, 0u}, p{0, 0u}, s_item{0, 0u}, o_item{0, 0u};
            Cursor<SPLIT> s, o;
            int ahead = 0, k_slot = 0, v_slot = 0, s_buf = 0, items = 0, low_buf = 0;
            int s_own[2] = {0, 0}, o_own[2] = {0, 0};  // the next barriers of a stream's own
            auto after = [&](int (&own)[2], int t) {
                const int x = t ? own[1] : own[0], y = x == 2 ? 0 : x + 1;
                if (t) own[1] = y;
                else own[0] = y;
                return t * 3 + x;
            };
            bool ok = true, s_on = false, new_queries = false;
            auto key_tile = [&]() -> Barrier { return LOW ? Barrier{&sh.ready[0][k_tile.at], k_tile.phase} : Barrier{&sh.full[0][k_tile.at], k_tile.phase}; };
            auto value_tile = [&]() -> Barrier { return {&sh.ready[1][v_tile.at], v_tile.phase}; };
            auto next_item = [&](Turn& turn, Cursor<SPLIT>& c) -> bool {  // false: the end, or gave up
                if (!(ok = wait(false, {&sh.item_full[turn.at], turn.phase}, W_ITEM, items))) return false;
                const Item& it = sh.items[turn.at];
                if ((int)uniform(it.tokens) == 0) return false;
                c.start((int)uniform(it.n0), (int)uniform(it.n1));
                return true;
            };
            bool s_new = true, o_new = true, seen_k = false, seen_v = false, seen_p = false;
            int between = -1;
#pragma unroll 1
            while (ok) {
                const bool fresh = s_new;
                if (s_new) {
                    s_on = next_item(s_item, s);
                    if (!ok) break;
                    s_new = false;
                    ++between;
                }
                if (!s_on && ahead == 0) break;
                if (o_new) {
                    if (!next_item(o_item, o)) break;
                    o_new = false;
                }
                const bool go = s_on && may_go<LOW>(between);
                new_queries |= fresh;
                if (go) {
                    if (new_queries) {
                        if (!(ok = wait(false, LOW ? Barrier{&sh.q_ready, (uint32_t)items & 1u} : Barrier{&sh.q_full[items & 1 & (C::Q_BUFFERS - 1)], (uint32_t)(items >> 1) & 1u}, W_Q, items))) break;
                        new_queries = false;
                    }
                    if (s.first()) {
                        if (!(ok = wait(seen_k, key_tile(), W_READY, items))) break;
                        k_slot = k_tile.at;
                        k_tile.next(SLOTS);
                    }
                    seen_k = false;
                    tc_fence_after_sync();
                    const Desc kd = k_desc + k_slot * C::KV_BYTES;
                    const bool both = ahead >= BEHIND;  // O follows
                    auto look = [&] {
                        seen_v = o.first() && seen(value_tile());
                        seen_p = seen({&sh.p_full[p.at], p.phase});
                    };
                    if constexpr (LOW) {
                        constexpr uint32_t IDESC = make_idesc_tf32(TILE, KEYS, false, false);
                        const uint32_t d = tmem + s_buf * 64;
                        auto eight = [&](uint32_t x, uint32_t y, uint32_t acc) {
                            umma_ts4<KMAJOR_STEP>(leader, d, tmem + LOW_COL_Q + x, kd + y, IDESC, acc);
                            umma_ts4<KMAJOR_STEP>(leader, d, tmem + LOW_COL_Q + x + 32, kd + (y + C::KV_BOX), IDESC, 1u);
                        };
                        eight(64, 0, 0u);
                        eight(0, C::KV_RAW, 1u);
                        if (both) look();
                        eight(0, 0, 1u);
                    } else {
                        const uint32_t IDESC = make_idesc_16(TILE, KEYS, BF16, false) | negate;
                        const uint32_t d = tmem + s_buf * 128;
                        const Desc qd = q_desc + ((items & 1) * C::STREAMS + (SPLIT ? 0 : s.t)) * C::Q_BYTES;
                        umma_ss_16(leader, d, qd.d, kd.d, IDESC, 0u);
                        umma_ss_16(leader, d, qd.d + 2, kd.d + 2, IDESC, 1u);
                        if (both) look();
                        umma_ss_16(leader, d, qd.d + 4, kd.d + 4, IDESC, 1u);
                        umma_ss_16(leader, d, qd.d + 6, kd.d + 6, IDESC, 1u);
                    }
                    umma_commit_lead(leader, &sh.s_full[0][0] + after(s_own, s.t));
                    if (s.last()) umma_commit_lead(leader, &sh.empty[0][k_slot]);
                    s_buf = s_buf == 2 ? 0 : s_buf + 1;
                    ++ahead;
                    if (!s.next()) {
                        if (!LOW) umma_commit_lead(leader, &sh.q_empty[items & (C::Q_BUFFERS - 1)]);
                        ++items;
                        s_item.next(ITEMS);
                        s_new = true;
                    }
                }
                if (ahead > BEHIND || !go) {  // O
                    if (o.first()) {
                        if (!(ok = wait(seen_v, value_tile(), W_READY, items))) break;
                        v_slot = v_tile.at;
                        v_tile.next(SLOTS);
                    }
                    if (!(ok = wait(seen_p, {&sh.p_full[p.at], p.phase}, W_P, items))) break;
                    tc_fence_after_sync();
                    seen_v = seen_p = false;
                    const Desc vd = v_desc + v_slot * C::KV_BYTES;
                    const uint32_t acc = o.j > 0;
                    const bool look_k = s_on && !s_new && s.first() && o.last();
                    if constexpr (LOW) {
                        constexpr uint32_t IDESC = make_idesc_tf32(TILE, HEAD_DIM, false, true);
                        const uint32_t high = tmem + p.at * 64, low = tmem + LOW_COL_LOW + low_buf * 64, d = tmem + LOW_COL_O;
                        auto eight = [&](uint32_t x, uint32_t y, uint32_t acc) {
                            umma_ts4<MNMAJOR_STEP>(leader, d, x, vd + y, IDESC, acc);
                            umma_ts4<MNMAJOR_STEP>(leader, d, x + 32, vd + (y + 4096), IDESC, 1u);
                        };
                        eight(low, 0, 0u);
                        eight(high, C::KV_RAW, 1u);
                        seen_k = look_k && seen(key_tile());
                        eight(high, 0, 1u);
                        low_buf ^= 1;
                    } else {
                        constexpr uint32_t IDESC = make_idesc_16(TILE, HEAD_DIM, BF16, true);
                        const uint32_t w = tmem + p.at * 128, d = tmem + COL_O + o.t * 64;
#pragma unroll
                        for (int k = 0; k < 8; ++k) {
                            if (k == 4) seen_k = look_k && seen(key_tile());
                            umma_ts_16(leader, d, w + 8 * k, vd.d + (2048 >> 4) * k, IDESC, k > 0 ? 1u : acc);
                        }
                    }
                    umma_commit_lead(leader, &sh.o_full[0][0] + after(o_own, o.t));
                    if (o.last()) umma_commit_lead(leader, &sh.empty[1][v_slot]);
                    p.next(3);
                    --ahead;
                    if (!o.next()) {
                        if (lane == 0) mbar_arrive(&sh.item_empty[o_item.at]);
                        o_item.next(ITEMS);
                        --between;
                        o_new = true;
                    }
                }
            }
        } else if (warp == 2 || (LOW && (warp == 3 || warp == 8 || warp == 9))) {
            // What the tiles need beside the loads.  Rows behind the request's last key may hold anything, and 0 times a NaN is one: they are
            // cleared among the values.  fp32: the tiles' low parts, by a pair of warps each for keys and values.
            const int me = LOW ? threadIdx.x & 63 : lane, v = !LOW || warp >= 8;
            Turn at{0, 0u};
            while (true) {
                if (!__all_sync(0xffffffffu, mbar_wait(wc, &sh.full[v][at.at], at.phase, W_KV, at.at))) break;
                const int keep = sh.keep[v][at.at];
                if (keep == LAST) break;
                uint4* raw = reinterpret_cast<uint4*>(sKV + (v * SLOTS + at.at) * C::KV_BYTES);
                if constexpr (LOW) {
                    constexpr int EACH = C::KV_RAW / 16 / 64;
                    uint4 *from = raw + me, *low = from + C::KV_RAW / 16, x[EACH];
#pragma unroll
                    for (int k = 0; k < EACH; ++k) x[k] = from[k * 64];
                    if (keep < KEYS) {
#pragma unroll
                        for (int k = 0; k < EACH; ++k)
                            if (((k * 64 + me) & (C::KV_BOX / 16 - 1)) / 8 >= keep) from[k * 64] = x[k] = make_uint4(0, 0, 0, 0);  // row of the box
                    }
#pragma unroll
                    for (int k = 0; k < EACH; ++k) low[k * 64] = make_uint4(tf32_rest(x[k].x), tf32_rest(x[k].y), tf32_rest(x[k].z), tf32_rest(x[k].w));
                    fence_proxy_async_smem();
                    mbar_arrive_warp(&sh.ready[v][at.at], lane);
                } else {
                    if (keep < KEYS) {
                        for (int k = keep * 8 + me; k < C::KV_RAW / 16; k += 32) raw[k] = make_uint4(0, 0, 0, 0);
                        fence_proxy_async_smem();
                    }
                    mbar_arrive_warp(&sh.ready[v][at.at], lane);
                    if (lane == 0) mbar_arrive(&sh.empty[v][at.at]);  // a slot is filled again when this warp has seen what it held
                }
                at.next(SLOTS);
            }
        }
    }
    tc_fence_before_sync();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after_sync();
        tmem_dealloc(tmem, 512);
        if (lane == 0) report_abort(sh.abort, a.status);
    }
}

// Boxes of `rows` rows of a page, 128 bytes of each
int page_map(CUtensorMap* map, const hk_view& v, int dtype, int n_pages, int H, int page, int rows, bool mn_major) {
    EncodeTiledFn enc = get_encode_tiled();
    if (!enc) return HK_ERR_CUDA;
    const int e = esize(dtype), inner = 128 / e;
    const int64_t sM = v.strideM, sH = H == 1 ? sM * page : v.strideH, sB = n_pages == 1 ? std::max(sH * H, sM * page) : v.strideB;
    cuuint64_t dims[5] = {(cuuint64_t)inner, (cuuint64_t)page, (cuuint64_t)(64 / inner), (cuuint64_t)H, (cuuint64_t)n_pages};
    cuuint64_t strides[4] = {(cuuint64_t)sM * e, 128, (cuuint64_t)sH * e, (cuuint64_t)sB * e};
    cuuint32_t box[5] = {(cuuint32_t)inner, (cuuint32_t)rows, 1, 1, 1}, ones[5] = {1, 1, 1, 1, 1};
    const CUtensorMapDataType type = dtype == HK_F32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : dtype == HK_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    const CUresult r = enc(map, type, 5, v.ptr, dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, mn_major ? CU_TENSOR_MAP_SWIZZLE_128B_ATOM_32B : CU_TENSOR_MAP_SWIZZLE_128B,
                           e == 2 && v.strideM != HEAD_DIM ? CU_TENSOR_MAP_L2_PROMOTION_L2_128B : CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? HK_OK : HK_ERR_CUDA;
}

// `tokens` tokens under `heads` heads, 128 bytes of each
int query_map(CUtensorMap* map, const hk_view& v, int dtype, int B, int H, int64_t T, int heads, int tokens) {
    EncodeTiledFn enc = get_encode_tiled();
    if (!enc) return HK_ERR_CUDA;
    const int e = esize(dtype), inner = 128 / e;
    const int64_t sM = T == 1 ? HEAD_DIM : v.strideM, sH = H == 1 ? HEAD_DIM : v.strideH, sB = B == 1 ? HEAD_DIM : v.strideB;
    cuuint64_t dims[5] = {(cuuint64_t)inner, (cuuint64_t)H, (cuuint64_t)T, (cuuint64_t)(64 / inner), (cuuint64_t)B};
    cuuint64_t strides[4] = {(cuuint64_t)sH * e, (cuuint64_t)sM * e, 128, (cuuint64_t)sB * e};
    cuuint32_t box[5] = {(cuuint32_t)inner, (cuuint32_t)heads, (cuuint32_t)tokens, 1, 1}, ones[5] = {1, 1, 1, 1, 1};
    const CUtensorMapDataType type = dtype == HK_F32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : dtype == HK_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    const CUresult r = enc(map, type, 5, v.ptr, dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? HK_OK : HK_ERR_CUDA;
}

// How the work is cut
template <class X, bool TREE, bool SPLIT>
void cut(ServingArgs& a) {
    typedef Rows<X> C;
    a.stream_tokens = std::max(1, TILE / a.group);
    a.block_tokens = C::STREAMS * a.stream_tokens;
    a.chunks = cdiv(a.group, TILE);
    a.new_tiles = 1;
    a.slot_rows = SPLIT ? TILE : C::BLOCK;
    set_line(a, TREE, C::KEYS);
}

template <class X, bool TREE, bool SPLIT, bool LONG>
int launch(ServingArgs a, int dtype, cudaStream_t stream) {
    typedef Rows<X> C;
    static std::once_flag once[HK_MAX_DEVICES];
    static cudaError_t rc[HK_MAX_DEVICES];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= HK_MAX_DEVICES) return HK_ERR_CUDA;
    std::call_once(once[dev], [dev] { rc[dev] = cudaFuncSetAttribute(serving_rows_kernel<X, TREE, SPLIT, LONG>, cudaFuncAttributeMaxDynamicSharedMemorySize, RowsSpace<X>::SMEM); });
    if (rc[dev] != cudaSuccess) return HK_ERR_CUDA;
    cut<X, TREE, SPLIT>(a);
    CUtensorMap k, v, kp, vp;
    const int B = TREE ? a.B : 1;
    const int64_t T = TREE ? a.T : a.N;
    int s;
    if ((s = prefix_tile_map(&k, a.K, dtype, B, a.Hk, T, C::KEYS, false)) || (s = prefix_tile_map(&v, a.V, dtype, B, a.Hk, T, C::KEYS, true))) return s;
    kp = k;
    vp = v;
    if (TREE) {
        a.box = std::gcd(a.pool.page, C::KEYS);
        divide_by(a.pool.page, a.page_mul, a.page_shift);
        if ((s = page_map(&kp, a.pool.K, dtype, a.pool.n_pages, a.Hk, a.pool.page, a.box, false)) ||
            (s = page_map(&vp, a.pool.V, dtype, a.pool.n_pages, a.Hk, a.pool.page, a.box, C::LOW)))
            return s;
    }
    CUtensorMap q;
    if ((s = query_map(&q, a.Q, dtype, B, a.Hk * a.group, T, std::min(a.group, TILE), a.stream_tokens)) != HK_OK) return s;
    a.q_bytes = std::min(a.group, TILE) * a.stream_tokens * 64 * (int)sizeof(X);
    const int ctas = sm_count();
    LaunchConfig lc(ctas, C::THREADS, RowsSpace<X>::SMEM, stream, 1, true);
    if (cudaLaunchKernelEx(&lc.cfg, serving_rows_kernel<X, TREE, SPLIT, LONG>, q, k, v, kp, vp, a) != cudaSuccess) return check_launch();
    count_launch();
    return a.parts ? launch_combine(a, dtype, ctas, stream) : HK_OK;
}
template <class X, bool TREE, bool SPLIT>
LineSum line(ServingArgs a, const int32_t* lens) {
    cut<X, TREE, SPLIT>(a);
    return line_sum<RowsWork<X, TREE, SPLIT>>(a, lens);
}
template <bool TREE, bool SPLIT>
LineSum line(const ServingArgs& a, int dtype, const int32_t* lens) {
    return dtype == HK_F32 ? line<float, TREE, false>(a, lens) : line<__half, TREE, SPLIT>(a, lens);
}
template <bool TREE, bool SPLIT, bool LONG>
int launch_16(const ServingArgs& a, int dtype, cudaStream_t stream) {
    return dtype == HK_BF16 ? launch<__nv_bfloat16, TREE, SPLIT, LONG>(a, dtype, stream) : launch<__half, TREE, SPLIT, LONG>(a, dtype, stream);
}
template <bool TREE, bool SPLIT>
int launch(const ServingArgs& a, int dtype, cudaStream_t stream) {
    if (dtype == HK_F32) return launch<float, TREE, false, false>(a, dtype, stream);
    const RowsPlan plan = rows_plan(dtype);
    const int64_t tiles = TREE ? cdiv((int64_t)a.pool.width * a.pool.page, plan.keys) + 1 : cdiv(a.N, plan.keys);  // that a block can have
    return plan.slots(tiles) > 2 ? launch_16<TREE, SPLIT, true>(a, dtype, stream) : launch_16<TREE, SPLIT, false>(a, dtype, stream);
}

}  // namespace

template <class C>
static RowsPlan plan_of() { return {C::BLOCK, C::KEYS, C::LEAST, C::PIECE}; }
RowsPlan rows_plan(int dtype) { return dtype == HK_F32 ? plan_of<Rows<float>>() : dtype == HK_BF16 ? plan_of<Rows<__nv_bfloat16>>() : plan_of<Rows<__half>>(); }
int launch_prompt_rows(const ServingArgs& a, int dtype, cudaStream_t stream) { return launch<false, false>(a, dtype, stream); }
// Up to 128 rows of a request under a key head: both streams have them, every other tile each (16 requests of up to 4 096 tokens, 16 new ones,
// 32 heads on 8, bf16: 25 us, 29 where the second stream has nothing to do; 32 new ones of 12 heads 30 and 39).
static bool one_stream(const ServingArgs& a) { return a.T <= std::max(1, TILE / a.group); }
int launch_tree_rows(const ServingArgs& a, int dtype, cudaStream_t stream) {
    return one_stream(a) ? launch<true, true>(a, dtype, stream) : launch<true, false>(a, dtype, stream);
}
LineSum prompt_rows_line(const ServingArgs& a, int dtype, const int32_t* lens) { return line<false, false>(a, dtype, lens); }
LineSum tree_rows_line(const ServingArgs& a, int dtype, const int32_t* lens) { return one_stream(a) ? line<true, true>(a, dtype, lens) : line<true, false>(a, dtype, lens); }

}  // namespace hk
