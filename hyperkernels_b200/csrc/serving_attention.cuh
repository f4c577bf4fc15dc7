// serving_attention.cuh -- what the kernels of the attention within packed prompts and against a cache of pages have in common.
#pragma once

#include "cache_pages.cuh"

namespace hk {

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
    int causal;
};

// keys that request b has in its pages
__device__ __forceinline__ int cache_keys(const ServingArgs& a, int b) { return min(max(a.lengths[b], 0), a.pool.width * a.pool.page); }
// new tokens that token t of request b sees
__device__ __forceinline__ uint64_t tree_bits(const ServingArgs& a, int b, int t) {
    return (a.tree ? (uint64_t)a.tree[b * a.tree_stride + t] : (2ull << t) - 1) & (~0ull >> (64 - a.T));
}

}  // namespace hk
