// shared_prefix.cuh -- what the kernels of the attention over a shared prefix (hk_shared_prefix_attention) have in common.
#pragma once

#include <type_traits>

#include "operators.cuh"

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

// The 2^ of what a softmax's reference lies below the row's largest score.  A weight takes the type of the values, and fp16 has none below
// 2^-24: with the largest at 2^7 (2^15 where a stale maximum may lie 2^8 lower), those down to 2^-31 of it are kept, where many of
// them would be lost beside one that is large.  The sums and the LSE take it back by themselves.
template <class X>
__host__ __device__ constexpr float lift() { return std::is_same<X, __half>::value ? 7.f : 0.f; }

template <class X>
__device__ __forceinline__ void store4(X* p, float4 v) {
    if constexpr (sizeof(X) == 4) *reinterpret_cast<float4*>(p) = v;
    else *reinterpret_cast<uint2*>(p) = make_uint2(pack<X>(v.x, v.y), pack<X>(v.z, v.w));
}

// Tiles of `rows` rows of a view of keys or values, all heads and batches (tma_load_tile): 128 bytes of each row side by side,
// swizzled; fp32 rows are two such pieces.  mn_major: the values as an MN-major operand of fp32 products.
int prefix_tile_map(CUtensorMap* map, const hk_view& v, int dtype, int64_t B, int H, int64_t T, int rows, bool mn_major);

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
