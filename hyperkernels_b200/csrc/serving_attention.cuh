// serving_attention.cuh -- what the kernels of the attention within packed prompts and against a cache of pages have in common.
#pragma once

#include "cache_pages.cuh"
#include "tile_math.cuh"

namespace hk {

// How the work is cut.  The tiles of keys that the rows meet, block of rows by block, key head by key head, request by request, make one
// line, of which every worker (a CTA, a warp) takes an equal stretch.  A block whose tiles fall to several workers leaves its parts
// in slots of the workspace, two to a worker: what it has of a block that it has not begun itself, and of one that it has begun
// and not ended.
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
    float scale;
    float scale_log2e;  // its size; a negative scale turns the queries' signs (flip)
    uint32_t flip;
    int causal;
    // a block's tokens (few rows: its rows) and 128s of query heads, tiles of new tokens; x / block_tokens is x * block_mul >> block_shift for x below 2^31
    int block_tokens, chunks, new_tiles;
    uint32_t block_mul;
    int block_shift, unit_shift;
    uint32_t group_mul, page_mul;  // few rows: x / group, x / page likewise
    int group_shift, page_shift;
    int stream_tokens, q_bytes;  // many rows: tokens of a stream, bytes of its queries
    int box;            // rows of a page that are loaded at once
    // slots of the workspace, and who has what in them; no parts: blocks are not cut
    float2* ml;         // [slots][rows]
    float* part;        // the same, [64]
    PartRecord* parts;
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
// bits: a division of 64-bit numbers takes a warp some 300 cycles.
template <int KEYS_, int LEAST_, int SHARE_, int EXTRA, bool TREE>
struct Work {
    static constexpr int KEYS = KEYS_, LEAST = LEAST_, SHARE = SHARE_;  // of a tile; tiles that a part of a block has, and a worker, at least
    const ServingArgs& a;
    __device__ __forceinline__ int all_tiles(const Request& r) const { return (r.len + KEYS - 1) / KEYS + (TREE ? a.new_tiles : 0); }
    __device__ __forceinline__ int tiles(const Request& r, int i) const {
        return TREE || !a.causal ? all_tiles(r) : (min((i + 1) * a.block_tokens, r.len) + KEYS - 1) / KEYS;
    }
    // units in front of block i, of one chunk of heads
    __device__ __forceinline__ int before(const Request& r, int i) const {
        const int64_t keys = TREE || !a.causal ? (int64_t)i * (all_tiles(r) * KEYS + EXTRA) : (int64_t)i * (i + 1) / 2 * a.block_tokens + (int64_t)i * EXTRA;
        return (int)(keys >> a.unit_shift);
    }
    __device__ __forceinline__ Request request(int b) const {
        Request r;
        if (TREE) {
            r.begin = 0;
            r.len = cache_keys(a, b);
            r.tokens = a.rows ? a.rows : a.T;
        } else {
            r.begin = min(max(a.starts[b], 0), a.N);
            r.len = r.tokens = max(0, min(max(a.starts[b + 1], 0), a.N) - r.begin);
        }
        r.blocks = (int)(((uint64_t)(uint32_t)(r.tokens + a.block_tokens - 1) * a.block_mul) >> a.block_shift);
        r.units = before(r, r.blocks) * a.chunks;
        return r;
    }
};
// What a worker takes at once: tiles [from, to) of block i's n.
struct Run {
    Request r;
    int b, kvh, chunk, i, from, to, n;
    __device__ __forceinline__ int slot(int worker) const { return from > 0 ? 2 * worker : to < n ? 2 * worker + 1 : -1; }  // -1: the result
};
// A worker's stretch of the line: it begins in block i of request b under key head kvh (blocks of the first chunk of heads, of the second,
// ..), `done` units behind the block's beginning, and goes on for `units`.
template <class W>
struct Line {
    Request r;
    int b, kvh, chunk, i, done, units;

    // By one warp.
    __device__ __forceinline__ void find(const W& work, int lane, int me, int workers) {
        const ServingArgs& a = work.a;
        constexpr int EACH = 2;  // requests of a lane
        int each[EACH], sum = 0, all = 0, blocks = 0;
        auto take = [&](int b0) {
            sum = 0;
#pragma unroll
            for (int k = 0; k < EACH; ++k) {
                const int b = b0 + lane * EACH + k;
                each[k] = 0;
                if (b < a.B) {
                    const Request x = work.request(b);
                    each[k] = x.units;
                    blocks += x.blocks * a.chunks;
                }
                sum += each[k];
            }
            int upto = sum;
#pragma unroll
            for (int off = 1; off < 32; off <<= 1) {
                const int y = __shfl_up_sync(0xffffffffu, upto, off);
                if (lane >= off) upto += y;
            }
            return upto;
        };
        units = 0;
        int upto = 0;
        for (int b0 = 0; b0 < a.B; b0 += 32 * EACH) {
            upto = take(b0);
            all += __shfl_sync(0xffffffffu, upto, 31);
        }
        all *= a.Hk;
        // a worker to a block, more if the blocks are long, as many as there are
        const int n_blocks = (int)min((int64_t)workers, (int64_t)__reduce_add_sync(0xffffffffu, min(blocks, 1 << 20)) * a.Hk);
        workers = min(workers, max(n_blocks, all / max(1, W::SHARE * W::KEYS >> a.unit_shift)));
        if (me >= workers) return;
        const int share = (unsigned)all / (unsigned)workers, more = all - share * workers;
        int left = me * share + min(me, more);
        units = share + (me < more);
        b = -1;
        for (int b0 = 0; b0 < a.B; b0 += 32 * EACH) {
            if (a.B > 32 * EACH) upto = take(b0);  // otherwise they are here still
            const unsigned here = __ballot_sync(0xffffffffu, left < upto * a.Hk);
            if (!here) {
                left -= __shfl_sync(0xffffffffu, upto, 31) * a.Hk;
                continue;
            }
            const int l = __ffs(here) - 1;
            left -= (upto - sum) * a.Hk;
            int k = 0;
#pragma unroll
            for (int m = 0; m < EACH - 1; ++m)
                if (k == m && left >= each[m] * a.Hk) left -= each[m] * a.Hk, ++k;
            left = __shfl_sync(0xffffffffu, left, l);
            b = b0 + l * EACH + __shfl_sync(0xffffffffu, k, l);
            break;
        }
        r = b >= 0 ? work.request(b) : Request{};
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
    // A border inside a block is moved to its beginning or end where a part of less than LEAST tiles would be left.
    __device__ __forceinline__ int border(const W& work, int units, int n) const {
        const int j = (int)min((int64_t)n, ((int64_t)units << work.a.unit_shift) / W::KEYS);
        return j == n ? n : j < W::LEAST ? 0 : n - j < W::LEAST ? n : j;
    }
    // The next run; false: the stretch is over
    __device__ __forceinline__ bool next(const W& work, Run& run) {
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
            const int n = work.tiles(r, i), from = border(work, done, n), to = border(work, done + units, n);
            units -= work.before(r, i + 1) - work.before(r, i) - done;
            done = 0;
            run = {r, b, kvh, chunk, i, from, to, n};
            ++i;
            if (to > from) return true;
        }
        return false;
    }
};
// The worker that has the last part of the block that this one has begun, by whole warps.
__device__ __forceinline__ int last_part(const ServingArgs& a, int worker, int workers) {
    const int lane = threadIdx.x & 31;
    for (int w0 = worker + 1;; w0 += 32) {
        const int w = min(w0 + lane, workers - 1), head = a.parts[w].head;
        const unsigned stops = __ballot_sync(0xffffffffu, w == workers - 1 || (head != PART_GOES_ON && head != PART_EMPTY));
        if (stops) return min(w0 + __ffs(stops) - 1, workers - 1);
    }
}
// Host: the constants of the line
void set_line(ServingArgs& a, bool tree, int keys);

struct RowsPlan {
    int rows;   // of a block
    int keys;   // of a tile
    int least;  // tiles of a part of a block
};
RowsPlan rows_plan(int dtype);
struct TreeFewPlan {
    int rows;     // of a slot
    int keys, least;
    int workers;
};
TreeFewPlan tree_few_plan(int dtype, int rows);
int launch_tree_few(ServingArgs a, int dtype, cudaStream_t stream);
int launch_prompt_rows(const ServingArgs& a, int dtype, cudaStream_t stream);
int launch_tree_rows(const ServingArgs& a, int dtype, cudaStream_t stream);

}  // namespace hk
