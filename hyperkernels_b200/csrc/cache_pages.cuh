// cache_pages.cuh -- what the operators over a cache of pages (cache_pages.cu) and the attention against it (serving_attention.cuh) share.
#pragma once

#include "operators.cuh"

namespace hk {

// The sequence of token n among those that begin at starts[0 .. B], ascending: how many end at or before it.
__device__ __forceinline__ int sequence_of(const int32_t* starts, int B, int n, int lane) {
    int lo = 0, len = B;
    while (len > 0) {
        const int step = (len + 31) / 32, at = lane * step;
        const int c = __popc(__ballot_sync(0xffffffffu, at < len && starts[lo + at + 1] <= n));
        if (c == 0) break;
        const int skip = (c - 1) * step + 1;
        len = min(c * step, len) - skip;
        lo += skip;
    }
    return lo;
}

// Host: x / d is x * mul >> shift for x below 2^31.
inline void divide_by(int d, uint32_t& mul, int& shift) {
    for (shift = 31; (1LL << (shift - 31)) < d;) ++shift;
    mul = (uint32_t)(((1ULL << shift) + d - 1) / d);
}

int check_pool_sizes(const hk_pool& pool, int64_t B, int nh_kv, int dtype);
int check_pool(const hk_pool& pool, int64_t B, int nh_kv, int dtype, bool written);

}  // namespace hk
