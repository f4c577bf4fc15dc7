// shared_prefix.cuh -- what the kernels of the attention over a shared prefix (hk_shared_prefix_attention) have in common.
#pragma once

#include <type_traits>

#include "tile_math.cuh"

namespace hk {

// The rows of a key head: row r = (b * T + i) * group + g is token i of request b under query head kvh * group + g, so that a
// request's rows follow each other; R of them.  What a run of keys, of the prefix or of a request's own, gives for row
// kvh * R + r is left in a slot of the workspace: the maximum and the sum of its weights (log2 units), and the weighted sum of
// the values.  The last kernel adds the slots of a row in their order.
struct PrefixArgs {
    hk_view Q, Kp, Vp, K, V, O;
    float* LSE;
    int64_t lse_sB, lse_sH;
    const int32_t* lengths;
    int B, Hk, group, T, P, S;  // batch, key heads, query heads of each, new tokens, prefix keys, rows of the requests' caches
    int R;
    float scale_log2e;  // its size; a negative scale turns the queries' signs (flip)
    uint32_t flip;
    int causal;
    int splits_p, per_p, tiles_p;  // over the prefix: runs of keys, keys of a run, row tiles of a key head
    int splits_o, tiles_o;         // over the requests' own keys
    int slots;                     // of a row; one: the result is written where it is worked out
    // Blocks of rows that take the prefix and the request's own keys in one go (`whole`): of many rows the last ones, which would not
    // fill the SMs, in parts of their keys, as many as there are slots.  Only they have slots then, block by block.
    int whole, first_split, block_rows;
    int64_t slot_rows;             // rows that have slots
    float2* ml;                    // [slots][slot_rows]
    float* part;                   // the same, [64]
    DeviceStatus* status;
};

// Lengths and queries are what the launch before this call wrote a moment ago: they are read behind pdl_wait, in program order.  The kernel
// over the own keys next to the prefix's (late) begins when that one's wait is over and has none of its own; nothing says that its SM's
// L1 has no older line of them, so it does not take them from there.  Few rows read past the L1, many have a fence in front (a row to a
// thread comes in pieces of lines that the L1 keeps meanwhile): chunk 51.6 us with the fence, 52.5 with the other; decoding of 64 26.1
// and 25.3.
// keys that request b has
__device__ __forceinline__ int request_keys(const PrefixArgs& a, int b) { return a.lengths ? min(max(__ldcg(a.lengths + b), 0), a.S) : a.S; }
// own keys that token t of a request of `len` keys sees
__device__ __forceinline__ int token_keys(const PrefixArgs& a, int len, int t) { return a.causal ? min(len, max(0, len - a.T + t + 1)) : len; }

// Launchers.  The kernel over the requests' own keys runs beside the one over the prefix, if that is launched just before it; it does
// not wait for it, so a launch that does has to follow (there are slots to add up then).
struct FewPlan {
    int rows;      // rows of a tile: 1, 2 (fp32 arithmetic lane by lane) or 16 (matrix instructions)
    int step;      // keys that a CTA takes at once
    int per_sm;    // CTAs that an SM holds
};
FewPlan few_plan(int dtype, int rows);
int launch_prefix_few(const PrefixArgs& a, int dtype, cudaStream_t stream);
int launch_own_few(const PrefixArgs& a, int dtype, cudaStream_t stream);   // and the prefix's before them, if `whole`
int launch_both_few(const PrefixArgs& a, int dtype, cudaStream_t stream);  // the two in one launch
struct ManyPlan {
    int rows;  // of a CTA's blocks
    int keys;  // of a tile
};
ManyPlan many_plan(int dtype);
int launch_prefix_many(const PrefixArgs& a, int dtype, cudaStream_t stream);
int launch_own_many(const PrefixArgs& a, int dtype, cudaStream_t stream);  // and the prefix's before them, if `whole`

}  // namespace hk
