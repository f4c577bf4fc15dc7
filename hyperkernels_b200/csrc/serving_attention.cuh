// serving_attention.cuh -- what the kernels of the attention within packed prompts and against a cache of pages have in common.
#pragma once

#include <climits>

#include "cache_pages.cuh"
#include "tile_math.cuh"

namespace hk {

// How the work is cut.  The tiles of keys that the rows meet, block of rows by block, key head by key head, request by request, make one
// line, of which every worker (a CTA, a warp) takes an equal stretch.  A block whose tiles fall to several workers leaves its parts
// in slots of the workspace, two to a worker: what it has of a block that it has not begun itself, and of one that it has begun
// and not ended.  What a worker has of a block in several pieces (16-bit types) is added up in a third, behind those of all workers.
enum PartHead { PART_NONE, PART_LAST, PART_GOES_ON, PART_EMPTY /* nothing of any block */ };
struct PartRecord {
    int head;                             // what the first slot holds: the last part of its block, one in between, or nothing
    int b, head0, heads, token0, tokens;  // whose first part the second slot holds (no tokens: none)
};

struct ServingArgs {
    hk_view Q, K, V, O;  // K, V: of the packed prompts, or of the new tokens
    hk_pool pool;        // tree only
    float* LSE;
    int64_t lse_sB, lse_sH;
    const int32_t* starts;   // prompts
    const int32_t* lengths;  // tree
    const int64_t* tree;
    int64_t tree_stride;
    int rows;                // few rows: of a request under a key head; many: 0
    int B, Hk, group, T, N;  // sequences, key heads, query heads of each, new tokens of each, tokens of all prompts
    float scale_log2e;  // the scale's size; a negative one turns the queries' signs (flip)
    uint32_t flip;
    int causal;
    // a block's tokens (few rows: its rows) and 128s of query heads, tiles of new tokens; x / block_tokens is x * block_mul >> block_shift for x below 2^31
    int block_tokens, chunks, new_tiles;
    uint32_t block_mul;
    int block_shift, unit_shift;
    uint32_t group_mul, page_mul;  // x / group (few rows) and x / page likewise
    int group_shift, page_shift;
    int stream_tokens, q_bytes;  // many rows: tokens of a stream, bytes of its queries
    int box;            // rows of a page that are loaded at once
    // slots of the workspace, and who has what in them; no parts: blocks are not cut
    int slot_rows;
    int sum_rows;       // that can be any block's
    float2* ml;         // [slots][slot_rows]
    float* part;        // the same, [64]
    PartRecord* parts;
    float4* sums;       // few rows: of what a warp has of a block in several pieces, [16][64] of each
    DeviceStatus* status;
};

// keys that request b has in its pages
__device__ __forceinline__ int cache_keys(const ServingArgs& a, int b) { return min(max(a.lengths[b], 0), a.pool.width * a.pool.page); }
// new tokens that token t of request b sees
__device__ __forceinline__ uint64_t tree_bits(const ServingArgs& a, int b, int t) {
    return (a.tree ? (uint64_t)a.tree[b * a.tree_stride + t] : (2ull << t) - 1) & (~0ull >> (64 - a.T));
}

struct Request {
    int begin, len, tokens, blocks;  // of the packed rows; keys of the sequence, or in pages; tokens (few rows: rows); blocks of them
    int units;                       // of all of its blocks, under one key head
};
// A block counts as the keys that it meets and EXTRA for its beginning and end, in units of 2^unit_shift keys, so that all of them fit 32
// bits: a division of 64-bit numbers takes a warp some 300 cycles.  EXTRA is up to a unit more where a unit is several keys: every block is then at least as
// wide as what it counts as, so none lies on the line without a width, taken by nobody, and a worker that has all of a block's units has all of its tiles.
template <int KEYS_, int LEAST_, int SHARE_, int EXTRA, bool TREE, int DEAL_ = 0>
struct Work {
    // keys of a tile; tiles that a part of a block has, and a worker, at least; blocks for each worker from which on they are dealt out (0: never)
    static constexpr int KEYS = KEYS_, LEAST = LEAST_, SHARE = SHARE_, DEAL = DEAL_;
    const ServingArgs& a;
    __host__ __device__ __forceinline__ int all_tiles(const Request& r) const { return (r.len + KEYS - 1) / KEYS + (TREE ? a.new_tiles : 0); }
    __host__ __device__ __forceinline__ int tiles(const Request& r, int i) const {
        return TREE || !a.causal ? all_tiles(r) : (((i + 1) * a.block_tokens < r.len ? (i + 1) * a.block_tokens : r.len) + KEYS - 1) / KEYS;
    }
    // units in front of block i, of one chunk of heads
    __host__ __device__ __forceinline__ int before(const Request& r, int i) const {
        const int extra = EXTRA - 1 + (1 << a.unit_shift);
        const int64_t keys = TREE || !a.causal ? (int64_t)i * (all_tiles(r) * KEYS + extra) : (int64_t)i * (i + 1) / 2 * a.block_tokens + (int64_t)i * extra;
        return (int)(keys >> a.unit_shift);
    }
    // A border inside a block is moved to its beginning or end where a part of less than LEAST tiles would be left.
    __host__ __device__ __forceinline__ int border(int units, int n) const {
        const int64_t at = ((int64_t)units << a.unit_shift) / KEYS;
        const int j = at < n ? (int)at : n;
        return j == n ? n : j < LEAST ? 0 : n - j < LEAST ? n : j;
    }
    __host__ __device__ __forceinline__ Request sized(int begin, int len, int tokens) const {
        Request r;
        r.begin = begin;
        r.len = len;
        r.tokens = tokens;
        r.blocks = (int)(((uint64_t)(uint32_t)(r.tokens + a.block_tokens - 1) * a.block_mul) >> a.block_shift);
        r.units = before(r, r.blocks) * a.chunks;
        return r;
    }
    __device__ __forceinline__ Request request(int b) const {
        if (TREE) return sized(0, cache_keys(a, b), a.rows ? a.rows : a.T);
        const int begin = min(max(a.starts[b], 0), a.N), len = max(0, min(max(a.starts[b + 1], 0), a.N) - begin);
        return sized(begin, len, len);
    }
};
// What a worker takes at once: tiles [from, to) of block i's n.
struct Run {
    Request r;
    int b, kvh, chunk, i, from, to, n;
    __device__ __forceinline__ int slot(int worker) const { return from > 0 ? 2 * worker : to < n ? 2 * worker + 1 : -1; }  // -1: the result
};
// Where N stretches of the line begin, found by a whole CTA.
template <int N>
struct LineSearch {
    int sums[32], blocks[32];  // of the warps' requests
    Request r[N];              // a stretch's first request, and how far behind its beginning
    int b[N], left[N];
};
// A worker's stretch of the line: it begins in block i of request b under key head kvh (blocks of the first chunk of heads, of the second,
// ..), `done` units behind the block's beginning, and goes on for `units`.
// Where causal prompts make many blocks, these are dealt out whole instead, the longest first, there and back along the workers: no parts, and the
// workers' shares differ by less than their last blocks (16 prompts of 17 to 1 000 tokens, 32 heads on 8, bf16: 56 us, 66 in equal stretches;
// 16 of 1 024: 116 and 129).  With fewer than five blocks to a worker the stretches are the more even; more than 128 prompts, which is what four ballots
// tell apart, go in stretches whatever their blocks.
template <class W>
struct Line {
    Request r;
    int b, kvh, chunk, i, done, units;
    bool dealt;  // to this CTA, in rounds: the next is b, and the level that it comes to i, with `done` blocks in the levels in front

    static constexpr int DEAL_REQUESTS = 128;  // 32 k + lane
    // Put down for the time until a warp takes it up: held in registers it costs those of the others.
    struct Saved;

    // The stretches of worker `me` of at most `most`, cut in N (of a CTA's warps, say), by all THREADS threads.  Stretch k is made for the
    // threads that ask for it; those of a warp have to ask for the same.
    template <int THREADS, int N>
    __device__ __forceinline__ void find(const W& work, LineSearch<N>& sh, int worker, int most, int k) {
        const ServingArgs& a = work.a;
        constexpr int WARPS = THREADS / 32;
        const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, each = (a.B + THREADS - 1) / THREADS;
        int sum = 0, n = 0;
        Request one = {};
        for (int x = 0; x < each; ++x) {
            if (tid * each + x >= a.B) break;
            one = work.request(tid * each + x);
            sum += one.units;
            n += min(one.blocks * a.chunks, 1 << 20);
        }
        int upto = sum;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, upto, off);
            if (lane >= off) upto += y;
        }
        n = __reduce_add_sync(0xffffffffu, n);
        if (lane == 31) {
            sh.sums[warp] = upto;
            sh.blocks[warp] = n;
        }
        if (tid < N) sh.b[tid] = -1;
        __syncthreads();
        int all = 0, from = upto - sum;
        n = 0;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            if (w < warp) from += sh.sums[w];
            all += sh.sums[w];
            n = min(n + sh.blocks[w], 1 << 20);
        }
        all *= a.Hk;
        const int64_t n_blocks = (int64_t)n * a.Hk;
        dealt = W::DEAL > 0 && a.causal && a.B <= DEAL_REQUESTS && n_blocks >= (int64_t)W::DEAL * most;
        if (dealt) {
            i = 0;
#pragma unroll
            for (int x = 0; x < DEAL_REQUESTS / 32; ++x) i = max(i, 32 * x + lane < a.B ? work.request(32 * x + lane).blocks : 0);
            i = __reduce_max_sync(0xffffffffu, i) - 1;
            r = {};
            b = kvh = chunk = done = units = 0;
            return;
        }
        // a worker to N blocks, more if the blocks are long, as many as there are
        const int workers = min(most, max((int)min((int64_t)most, (n_blocks + N - 1) / N), all / max(1, N * W::SHARE * W::KEYS >> a.unit_shift)));
        const bool mine = worker < workers;
        const int share = mine ? (unsigned)all / (unsigned)workers : 0, more = all - share * workers, begin = worker * share + min(worker, more), length = mine ? share + (worker < more) : 0;
        auto border = [&](int k) { return k == N ? begin + length : begin + length / N * k; };
#pragma unroll
        for (int x = 0; x < N; ++x) {
            int left = border(x) - from * a.Hk;
            if (!mine || left < 0 || left >= sum * a.Hk) continue;
            for (int y = 0; y < each; ++y) {
                if (each > 1) one = work.request(tid * each + y);
                if (left < one.units * a.Hk) {
                    sh.b[x] = tid * each + y;
                    sh.left[x] = left;
                    sh.r[x] = one;
                    break;
                }
                left -= one.units * a.Hk;
            }
        }
        __syncthreads();
        b = sh.b[k];
        units = mine && b >= 0 ? border(k + 1) - border(k) : 0;
        if (units <= 0) return;
        int left = sh.left[k];
        r = sh.r[k];
        kvh = r.units > 0 ? (unsigned)left / (unsigned)r.units : a.Hk;
        if (kvh >= a.Hk) {  // starts that do not ascend can come to more than 32 bits: such a call gives nothing of use, but stays inside
            units = 0;
            return;
        }
        left -= kvh * r.units;
        chunk = 0;
        if (a.chunks > 1) {
            const int one = r.units / a.chunks;
            chunk = left / one;
            left -= chunk * one;
        }
        int lo = 0, len = r.blocks;  // the last block that begins at or before it
        while (len > 1) {
            const int step = (len + 31) / 32;
            const int c = __popc(__ballot_sync(0xffffffffu, lane * step < len && work.before(r, lo + lane * step) <= left));
            lo += (c - 1) * step;
            len = min(step, len - (c - 1) * step);
        }
        i = lo;
        done = left - work.before(r, lo);
    }
    // The next block that is dealt to this CTA, by a warp: number x of all in the order of the levels, each of the blocks i of all requests
    // that have so many (blocks: of every request, in shared memory)
    __device__ __forceinline__ bool next_dealt(const W& work, Run& run, const int* blocks) {
        const int lane = threadIdx.x & 31, x = b * gridDim.x + (b & 1 ? gridDim.x - 1 - blockIdx.x : blockIdx.x), each = work.a.Hk * work.a.chunks;
        ++b;
        while (i >= 0) {
            unsigned have[DEAL_REQUESTS / 32];
            int n = 0;
#pragma unroll
            for (int k = 0; k < DEAL_REQUESTS / 32; ++k) {
                have[k] = __ballot_sync(0xffffffffu, blocks[32 * k + lane] > i);
                n += __popc(have[k]);
            }
            if (x >= done + n * each) {
                done += n * each;
                --i;
                continue;
            }
            int rest = x - done, q = rest / each;  // the q-th of them
            rest -= q * each;
            int request = 0;
#pragma unroll
            for (int k = 0; k < DEAL_REQUESTS / 32; ++k) {
                const int c = __popc(have[k]);
                if (q >= 0 && q < c) {
                    const unsigned it = __ballot_sync(0xffffffffu, (have[k] >> lane & 1) && __popc(have[k] & ((1u << lane) - 1)) == q);
                    request = 32 * k + __ffs(it) - 1;
                    q = -1;
                } else if (q >= 0) {
                    q -= c;
                }
            }
            run.r = work.request(request);
            run.b = request;
            run.kvh = rest / work.a.chunks;
            run.chunk = rest - run.kvh * work.a.chunks;
            run.i = i;
            run.from = 0;
            run.to = run.n = work.tiles(run.r, i);
            return true;
        }
        return false;
    }
    // The next run; false: the stretch is over
    __device__ __forceinline__ bool next(const W& work, Run& run, const int* blocks = nullptr) {
        if (W::DEAL > 0 && dealt) return next_dealt(work, run, blocks);
        while (units > 0) {
            if (i >= r.blocks) {
                i = 0;
                if (r.blocks == 0 || ++chunk == work.a.chunks) {
                    chunk = 0;
                    if (r.blocks == 0 || ++kvh == work.a.Hk) {
                        kvh = 0;
                        if (++b >= work.a.B) break;
                        r = work.request(b);
                    }
                }
                continue;
            }
            const int n = work.tiles(r, i), from = work.border(done, n), to = work.border(done + units, n);
            units -= work.before(r, i + 1) - work.before(r, i) - done;
            done = 0;
            run = {r, b, kvh, chunk, i, from, to, n};
            ++i;
            if (to > from) return true;
        }
        return false;
    }
};
template <class W>
struct Line<W>::Saved {
    Line line;
    int blocks[DEAL_REQUESTS];  // dealt: of each request
};
// Host: the constants of the line; the sum of the parts of blocks that fell to several of `workers`
void set_line(ServingArgs& a, bool tree, int keys);
// For tests: what the line of requests of these lengths comes to under all key heads, in units; units of its narrowest block; tiles that its blocks
// would lose at their ends.  2^unit_shift is a unit.
struct LineSum {
    int64_t units, narrowest, lost, unit_shift;
};
template <class W>
LineSum line_sum(const ServingArgs& a, const int32_t* lens) {
    const W work{a};
    LineSum sum{0, INT_MAX, 0, a.unit_shift};
    for (int b = 0; b < a.B; ++b) {
        const Request r = work.sized(0, lens[b], a.T == 0 ? lens[b] : a.rows ? a.rows : a.T);
        sum.units += (int64_t)r.units * a.Hk;
        for (int i = 0; i < r.blocks; ++i) {
            const int width = work.before(r, i + 1) - work.before(r, i), n = work.tiles(r, i);
            sum.narrowest = std::min<int64_t>(sum.narrowest, width);
            sum.lost += n - work.border(width, n);
        }
    }
    return sum;
}
int launch_combine(ServingArgs a, int dtype, int workers, cudaStream_t stream);

struct RowsPlan {
    int rows;   // of a block
    int keys;   // of a tile
    int least;  // tiles of a part of a block
    int piece;  // tiles that are taken at once of a longer run, 0: all
    int slots(int64_t tiles) const { return piece > 0 && tiles >= piece + least ? 3 : 2; }  // of a worker, for blocks of up to so many tiles
};
RowsPlan rows_plan(int dtype);
struct TreeFewPlan {
    int rows;  // of a slot
    int keys, least;
    int workers, slots;  // CTAs; slots of each
    int sums;  // rows of 64 floats of each for sums of blocks' pieces, 0: no block can have several
};
TreeFewPlan tree_few_plan(int dtype, int rows, int64_t keys);  // keys: that a request can have
int launch_tree_few(ServingArgs a, int dtype, cudaStream_t stream);
int launch_prompt_rows(const ServingArgs& a, int dtype, cudaStream_t stream);
int launch_tree_rows(const ServingArgs& a, int dtype, cudaStream_t stream);
LineSum tree_few_line(ServingArgs a, int dtype, const int32_t* lens);
LineSum prompt_rows_line(const ServingArgs& a, int dtype, const int32_t* lens);
LineSum tree_rows_line(const ServingArgs& a, int dtype, const int32_t* lens);

}  // namespace hk
