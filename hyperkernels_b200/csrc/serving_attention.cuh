// serving_attention.cuh -- what the kernels of the attention within packed prompts and against a cache of pages have in common.
#pragma once

#include "cache_pages.cuh"
#include "tile_math.cuh"

namespace hk {

// What a CTA of the kernel of many rows has of blocks that fell to several: how the first one goes on that it has not begun itself, and the
// one that it has begun and not ended (no tokens: none).
enum PartHead { PART_NONE, PART_LAST, PART_GOES_ON, PART_EMPTY /* nothing of any block */ };
struct PartRecord {
    int head;
    int b, head0, heads, token0, tokens;
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
    int B, Hk, group, T, N;  // sequences, key heads, query heads of each, new tokens of each, tokens of all prompts
    float scale;
    float scale_log2e;  // its size; a negative scale turns the queries' signs (flip)
    uint32_t flip;
    int causal;
    // kernel of many rows: tokens of a stream and of a block, 128s of query heads, bytes of a stream's queries; x / block_tokens is x *
    // block_mul >> block_shift for x below 2^31
    int stream_tokens, block_tokens, chunks, q_bytes;
    uint32_t block_mul;
    int block_shift, unit_shift;
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

struct RowsPlan {
    int rows;   // of a block
    int keys;   // of a tile
    int least;  // tiles of a part of a block
};
RowsPlan rows_plan(int dtype);
int launch_prompt_rows(const ServingArgs& a, int dtype, cudaStream_t stream);
int launch_tree_rows(const ServingArgs& a, int dtype, cudaStream_t stream);

}  // namespace hk
