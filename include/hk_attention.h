/*
 * hk_attention.h -- C ABI of the sm_100a (B200) fused attention forward/backward.
 *
 * Drop-in boundary for the launch surface of BlubridgeAI/HyperKernels
 * kernels/attention.  The reference exposes no host API: its boundary is
 * "kernel symbol + by-value POD argument block + launch geometry", visible in
 * kernels/tests/kernels_test.cu:509-530 (forward), :475-477 (D pre-pass) and
 * :580-584 (backward).  Each entry point below replaces one of those launches
 * and takes an argument block whose leading bytes are exactly the reference
 * block, followed by an extension tail.  A caller holding a reference block
 * copies it into the head of ours, zeroes the tail, and calls.
 *
 * Conventions
 *   - head_dim is 64, I/O is fp32, MMA operands are TF32 rounded to nearest
 *     (Q, K, V, dO by the TMA copies that load them, ties to even; P and dS in
 *     registers by bit pattern + 0x1000, as the reference rounds everything),
 *     accumulation is fp32.
 *   - All pointers are device pointers owned by the caller; the library never
 *     allocates device memory.  Scratch comes from `workspace`.
 *   - Strides are in elements; the last-dimension stride is 1.  Every pointer
 *     and every stride*4 must be a multiple of 16 bytes.  A batch or head
 *     stride of 0 (one slice broadcast over several batches or heads, which
 *     the reference's pointer arithmetic allows) is refused with
 *     HK_ERR_UNSUPPORTED when that dimension is larger than 1: the TMA tensor
 *     maps the kernels read through cannot express it.
 *   - Bits: the same call gives the same O, LSE, D, dK, dV on every run (dQ:
 *     HK_FLAG_DETERMINISTIC_DQ).  At training lengths -- forward with
 *     kv_len <= 4096 and kv_len < 2 T, backward with T < 2 kv_len -- a (batch,
 *     head) slice also gives them whatever other slices are in the call, so a
 *     batch may be cut into several calls.  Outside these the keys (backward:
 *     the queries) of a slice may be shared by several CTAs, by a number that
 *     depends on B * nh: the same slice in another batch then differs by the
 *     rounding of sums in another order, a decoding step (T <= 2) included.
 *   - Re-entrant: no call keeps state between calls except per-device caches
 *     that are filled once under a lock, so any number of host threads may
 *     drive any number of devices and streams.  Device ordinals 0..63.
 *   - Every function returns HK_OK (0) or a negative hk_status; nothing exits
 *     the process or throws.  Kernel launches are asynchronous on `stream`;
 *     device-side faults surface on the caller's next synchronisation, and the
 *     bounded-wait guard of the kernels is read back with hk_attn_last_device_status.
 *   - No CPU fallback: without a CUDA device every compute call returns
 *     HK_ERR_CUDA.
 */
#ifndef HK_ATTENTION_H_
#define HK_ATTENTION_H_

#include <stdbool.h>
#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef enum hk_status {
    HK_OK = 0,
    HK_ERR_NULL_POINTER = -1,
    HK_ERR_BAD_SHAPE = -2,     /* B, nh, T <= 0, T too large, kv_len < 0 */
    HK_ERR_MISALIGNED = -3,    /* pointer or stride not 16-byte aligned */
    HK_ERR_BAD_DROPOUT = -4,   /* p outside [0,1), or both mask and Philox requested */
    HK_ERR_WORKSPACE = -5,     /* workspace missing or smaller than hk_attn_*_workspace_bytes */
    HK_ERR_UNSUPPORTED = -6,   /* combination the kernels do not implement */
    HK_ERR_CUDA = -7,          /* CUDA runtime/driver error (no device, launch failure) */
    HK_ERR_DEVICE_TIMEOUT = -8, /* a bounded wait inside a kernel gave up */
    HK_ERR_STATIC_SCRATCH = -9  /* problem too large for the built-in scratch of hk_attn_forward_static_scratch */
} hk_status;

/* Size limit of hk_attn_forward_static_scratch. */
#define HK_STATIC_SCRATCH_BYTES ((size_t)24 << 20)

enum {
    /* dropout keep-mask is generated in the kernel from (dropout_seed, dropout_offset)
     * with Philox4x32-10; see hk_attn_dropout_mask for the host twin. */
    HK_FLAG_PHILOX_DROPOUT = 1u << 0,
    /* Q, K, V (and dO) already hold TF32-representable values (low 13 mantissa
     * bits zero): no workspace is asked for. */
    HK_FLAG_OPERANDS_PREROUNDED = 1u << 1,
    /* backward: add into dK/dV instead of overwriting them (a K/V block that
     * travels round a sequence-sharded ring carries its gradients with it). */
    HK_FLAG_ACCUM_DKDV = 1u << 2,
    /* backward: do not zero dQ before accumulating into it. */
    HK_FLAG_ACCUM_DQ = 1u << 3,
    /* backward: D is supplied by the caller (reference behaviour of the unified
     * kernel taken alone); otherwise hk_attn_backward computes it from dO and O. */
    HK_FLAG_D_PRECOMPUTED = 1u << 4,
    /* backward: `workspace` is the one hk_attn_forward was given for these same Q, K, V.  Accepted and without
     * effect: the operands are rounded as they are loaded, there is nothing to reuse. */
    HK_FLAG_REUSE_FWD_ROUNDED = 1u << 5,
    /* forward and backward: inverted dropout instead of the reference's drop-then-renormalise
     * (no reference counterpart).  The softmax is normalised over ALL visible keys, the kept
     * probabilities are multiplied by 1/(1-p) and the dropped ones are zero in O; LSE does not
     * depend on the mask.  p is dropout_p for a dense mask and floor(dropout_p * 65536) / 65536
     * for the Philox mask.  Without active dropout the flag changes nothing. */
    HK_FLAG_DROPOUT_SCALED = 1u << 6,
    /* forward: O and LSE already hold the attention result over the keys seen so far (LSE = -inf, any O, for a
     * row that has seen none); the call folds the keys of THIS call in and leaves the combined result in O and
     * LSE -- the previous result acts as one more "key" of weight exp(LSE) and value O.  A caller that shards the
     * key sequence (a KV ring) chains its calls this way instead of merging partial results afterwards.  Not
     * available together with HK_FLAG_DROPOUT_SCALED.  No counterpart in the reference. */
    HK_FLAG_CONTINUE_SOFTMAX_STATE = 1u << 7,
    /* forward: ask for the workspace at every size.  The operands are rounded to TF32 by the TMA copies that load
     * them and the workspace is not touched; by default it is required except for 512 <= T <= 2048 (causal) or
     * <= 1024 (otherwise). */
    HK_FLAG_ROUND_IN_HBM = 1u << 8,
    /* backward: deterministic dQ.  By default the KV-tile CTAs add their dQ tiles into dQ with bulk reductions whose
     * order is not fixed (run-to-run differences of the order of 1e-5); with this flag every CTA stores its tiles
     * into the workspace instead (ceil(kv_len / 128) slabs of B*nh*T*256 bytes behind the rounded operands:
     * hk_attn_bwd_workspace_bytes counts them) and a second kernel adds the slabs in KV-tile order: the same
     * inputs give the same bits on every run.  The slabs are ceil(kv_len / 128) times the size of dQ: meant for
     * the sequence lengths of training batches, not for a 32k-token single sequence.  The reference's own dQ is
     * accumulated with atomicAdd
     * (mem_efficient_bwd_unified_kernel_exp12.cu:239-260) and is not reproducible either. */
    HK_FLAG_DETERMINISTIC_DQ = 1u << 9
};

/* ---- forward ------------------------------------------------------------
 * Head (192 bytes) == MemEfficientFwdParams,
 * kernels/attention/fused_attn_forward_kernel_tc_sm89.cu:8-29. */
typedef struct hk_attn_fwd_params {
    const float* Q;
    const float* K;
    const float* V;
    float* O;
    float* LSE;
    int B;
    int nh;
    int64_t T; /* query rows per (b,h) */
    float scale;
    bool is_causal;
    float dropout_p;
    const float* dropout_mask; /* dense [B*nh, T, kv_len] 1.0/0.0 floats, or NULL */
    int64_t q_strideB, q_strideM, q_strideH;
    int64_t k_strideB, k_strideM, k_strideH;
    int64_t v_strideB, v_strideM, v_strideH;
    int64_t o_strideB, o_strideM, o_strideH;
    int64_t lse_strideB, lse_strideH;
    /* ---- extension tail (all-zero == reference behaviour) ---- */
    uint64_t dropout_seed;
    uint64_t dropout_offset;
    void* workspace;
    size_t workspace_bytes;
    int64_t kv_len; /* key rows per (b,h); 0 means T */
    int64_t q_pos0; /* global position of query row 0 (causal mask, dropout counter) */
    int64_t k_pos0; /* global position of key row 0 */
    uint32_t flags;
    uint32_t bh_pos0; /* global index of (batch 0, head 0) of this call in the Philox counter: a caller that
                       * cuts one problem into several calls over runs of (batch, head) slices passes the
                       * first slice's index, so every cut draws the mask of the single call; 0 otherwise */
} hk_attn_fwd_params;

/* ---- backward -----------------------------------------------------------
 * Head (328 bytes) == MemEfficientBwdParams, declared twice in the reference
 * with one layout: kernels/attention/mem_efficient_bwd_precompute_D_sm89.cu:7-33
 * and OwnTensor:: kernels/attention/mem_efficient_bwd_unified_kernel_exp12.cu:11-38. */
typedef struct hk_attn_bwd_params {
    const float* Q;
    const float* K;
    const float* V;
    const float* O;
    const float* dO;
    const float* LSE;
    float* D;
    float* dQ;
    float* dK;
    float* dV;
    int B;
    int nh;
    int T;
    float scale;
    bool is_causal;
    int64_t q_strideB, q_strideM, q_strideH;
    int64_t k_strideB, k_strideM, k_strideH;
    int64_t v_strideB, v_strideM, v_strideH;
    int64_t o_strideB, o_strideM, o_strideH;
    int64_t do_strideB, do_strideM, do_strideH;
    int64_t dq_strideB, dq_strideM, dq_strideH;
    int64_t dk_strideB, dk_strideM, dk_strideH;
    int64_t dv_strideB, dv_strideM, dv_strideH;
    int64_t lse_strideB, lse_strideH;
    int64_t d_strideB, d_strideH;
    /* ---- extension tail ---- */
    float dropout_p; /* the reference backward has no dropout; 0 reproduces it */
    uint32_t flags;
    const float* dropout_mask; /* dense [B*nh, T, kv_len] or NULL */
    uint64_t dropout_seed;
    uint64_t dropout_offset;
    void* workspace;
    size_t workspace_bytes;
    int64_t kv_len;
    int64_t q_pos0;
    int64_t k_pos0;
    uint32_t bh_pos0; /* as in hk_attn_fwd_params */
    uint32_t reserved;
} hk_attn_bwd_params;

/* Replaces the launch of fused_attn_forward_kernel_tc_sm89<64,64,64,1>
 * (kernels/tests/kernels_test.cu:509-530; kernel at
 * kernels/attention/fused_attn_forward_kernel_tc_sm89.cu:72-426).
 * Writes O and LSE.  `stream` is a cudaStream_t (NULL = default stream). */
int hk_attn_forward(const hk_attn_fwd_params* p, void* stream);

/* hk_attn_forward for callers that cannot allocate device memory (it has no
 * counterpart in the reference, whose kernels need no scratch).  Same arguments
 * and results as hk_attn_forward, but `workspace`/`workspace_bytes` are ignored and
 * the call allocates nothing (no cudaMalloc, no cudaFree).  Meant for plug-ins
 * living inside a framework that owns all device memory, and for serving loops
 * where an allocation would stall the GPU.
 * Limits: B*nh*(T + 2*kv_len)*256 bytes must fit in HK_STATIC_SCRATCH_BYTES,
 * otherwise HK_ERR_STATIC_SCRATCH. */
int hk_attn_forward_static_scratch(const hk_attn_fwd_params* p, void* stream);

/* Replaces the launch of mem_efficient_bwd_precompute_D_sm89<64>
 * (kernels/tests/kernels_test.cu:475-477; kernel at
 * kernels/attention/mem_efficient_bwd_precompute_D_sm89.cu:45-91).
 * Reads dO, O and their strides, B, nh, T; writes D. */
int hk_attn_bwd_precompute_D(const hk_attn_bwd_params* p, void* stream);

/* The same pre-pass for the other head dimensions the reference instantiates it for
 * (mem_efficient_bwd_precompute_D_sm89<16|32|48|64|80|96|128|160|192|256>,
 * kernels/attention/mem_efficient_bwd_precompute_D_sm89.cu:93-102): dO and O rows hold
 * `head_dim` floats.  The attention kernels themselves are head_dim 64 only. */
int hk_attn_bwd_precompute_D_hd(const hk_attn_bwd_params* p, int head_dim, void* stream);

/* Replaces the launch of OwnTensor::mem_efficient_bwd_unified_kernel_exp12<64,Causal>
 * (kernels/tests/kernels_test.cu:562-584; kernel at
 * kernels/attention/mem_efficient_bwd_unified_kernel_exp12.cu:54-329) together
 * with the steps its caller performs around it: the D pre-pass (unless
 * HK_FLAG_D_PRECOMPUTED) and the zeroing of dQ (unless HK_FLAG_ACCUM_DQ).
 * Writes dQ, dK, dV (and D). */
int hk_attn_backward(const hk_attn_bwd_params* p, void* stream);

/* Scratch the two calls ask for with the given block, flags included (0 when none).  Forward: room for Q, K, V, by size
 * (HK_FLAG_ROUND_IN_HBM).  Backward: room for Q, K, V, dO, then, with HK_FLAG_DETERMINISTIC_DQ, one slab of partial dQ
 * per 128-key tile.  The slabs are the only part that is written. */
size_t hk_attn_fwd_workspace_bytes(const hk_attn_fwd_params* p);
size_t hk_attn_bwd_workspace_bytes(const hk_attn_bwd_params* p);

/* Merges the result of a forward over one more block of keys into a running
 * result: (O_acc, LSE_acc) <- softmax-merge of (O_acc, LSE_acc) and
 * (O_part, LSE_part), rows contiguous [rows, 64] / [rows].  Used by callers that
 * shard the key sequence (ring attention).  No counterpart in the reference,
 * whose forward always sees all keys. */
int hk_attn_merge_partial(float* O_acc, float* LSE_acc, const float* O_part, const float* LSE_part, int64_t rows,
                          void* stream);

/* Rounds `rows` contiguous rows of 64 floats to TF32 (round to nearest, the reference's
 * `+0x1000`, fused_attn_forward_kernel_tc_sm89.cu:197) from src into dst (dst may be src: in place).  A caller
 * that feeds the same tensor to several calls (the ring schedule does) rounds it once and passes
 * HK_FLAG_OPERANDS_PREROUNDED.  No counterpart in the reference, which rounds at every load. */
int hk_attn_round_tf32(const float* src, float* dst, int64_t rows, void* stream);

/* Host twin of the in-kernel Philox keep-mask: fills the dense mask the
 * reference forward consumes (fused_attn_forward_kernel_tc_sm89.cu:321-324),
 * mask[(bh*Tq + i)*Tk + j] = 1.0f keep / 0.0f drop.  `mask` is HOST memory. */
int hk_attn_dropout_mask(float* mask, int BH, int64_t Tq, int64_t Tk, float p, uint64_t seed, uint64_t offset,
                         int64_t q_pos0, int64_t k_pos0);
/* The same for (batch, head) slices bh_pos0 .. bh_pos0 + BH - 1 of a larger problem (the mask a call with that
 * bh_pos0 in its argument block draws). */
int hk_attn_dropout_mask_slices(float* mask, uint32_t bh_pos0, int BH, int64_t Tq, int64_t Tk, float p, uint64_t seed,
                                uint64_t offset, int64_t q_pos0, int64_t k_pos0);

/* Reads (and clears) the status word the kernels of this process wrote on the
 * current device: HK_OK, or HK_ERR_DEVICE_TIMEOUT if a bounded wait gave up.
 * Synchronises the device. */
int hk_attn_last_device_status(void);

/* Number of kernels this library has launched in this process (all devices). */
uint64_t hk_attn_launch_count(void);

/* Per-kernel timing for benchmarks: while enabled, CUDA events are recorded on the
 * launching stream around the forward (kind 0) and backward (kind 1) tensor-core
 * kernels; _read waits for them, returns their summed duration and count since
 * the last read, and releases them.  The reference has no counterpart (its
 * timing lives in its benchmark programs, blas/tests/test_sgemm_addmm_sm89.cu:131-145). */
void hk_attn_kernel_timing_enable(int on);
int hk_attn_kernel_timing_read(int kind, double* total_ms, int* launches);

/* Runs the tensor-core self-test on the current device: small TF32 products
 * through each operand path the attention kernels use (K-major and MN-major
 * shared-memory operands, tensor-memory A operand).  out[0..n) receives the
 * raw results of case `which` (0..2); case 3 computes nothing and makes one
 * bounded wait run out on purpose (about 2 s), after which
 * hk_attn_last_device_status() reports HK_ERR_DEVICE_TIMEOUT once; see
 * hyperkernels_b200/csrc/umma_selftest.cu. */
int hk_attn_selftest(int which, const float* A, const float* B, float* out, void* stream);

/* ---- operators round the attention -------------------------------------------
 * No counterpart in the reference.  They read and write fp32, bf16 or fp16.  What is in between is fp32, but for the products
 * of the shared prefix: 16-bit types multiply values by weights that are rounded to their type too (half a step each; the sums
 * that divide, and LSE, are of the weights before that), fp32 tensors may go through the tensor core in two parts, which leaves
 * out 2^-22 of a product.  A fifth of the 16-bit types' exponentials may come from a polynomial that is 2.7e-6 of them off. */
typedef enum hk_dtype { HK_F32 = 0, HK_BF16 = 1, HK_F16 = 2 } hk_dtype;

/* A [B, heads, T, 64] tensor: pointer and element strides, last stride 1.  The pointer and the bytes of every stride
 * are multiples of 16; the stride of a dimension of one is not used. */
typedef struct hk_view {
    void* ptr;
    int64_t strideB, strideM, strideH;
} hk_view;

/* Rotary positions with several axes.  The 64 elements of a row are 32 pairs (p, p + 32), or (2 p, 2 p + 1) with
 * `interleaved`; pair p turns by positions[axis[p], b, t] * turn[p] / 2^64 of a full turn.  An integer position times an
 * integer fraction of a turn, modulo one turn, has no error however far the position is.  turn[p] itself is rounded: half
 * of 2^-64 of a turn and, from hk_rotary_plan_fill, 2^-62 of the turns per position, which the position multiplies.  A pair of axis
 * HK_ROTARY_STILL is left as it is. */
#define HK_ROTARY_STILL 255
typedef struct hk_rotary_plan {
    uint64_t turn[32];
    uint8_t axis[32];
    int32_t n_axes;
    int32_t interleaved;
} hk_rotary_plan;

/* Fills a plan: the first sections[0] pairs turn with axis 0, the next sections[1] with axis 1, and so on; pairs behind
 * the last section are left as they are.  `frequency` holds radians per position for each turning pair, or is NULL for
 * base^(-p / 32), p counted over all axes. */
int hk_rotary_plan_fill(hk_rotary_plan* plan, int n_axes, const int* sections, double base, const double* frequency,
                        int interleaved);

typedef struct hk_qk_params {
    hk_view q, k;           /* what the projection gives, `dtype`; the rotary backward does not read it */
    hk_view q_out, k_out;   /* forward, written: `out_dtype` */
    hk_view dq_out, dk_out; /* backward, read: gradients of q_out, k_out, `out_dtype` */
    hk_view dq, dk;         /* backward, written: gradients of q, k, `dtype` */
    const void* q_weight;   /* norm: [64] of weight_dtype, or NULL for ones */
    const void* k_weight;
    float* dq_weight; /* norm, backward, written: [64], or NULL if not wanted */
    float* dk_weight;
    const void* positions; /* [n_axes, B, T] with the element strides below (0 broadcasts), 32- or 64-bit integers */
    int64_t pos_strideA, pos_strideB, pos_strideT;
    int B, nh, nh_k; /* nh_k = 0: no keys */
    int pos_bits;    /* 32 or 64 */
    int64_t T;
    int dtype, out_dtype, weight_dtype; /* hk_dtype; the norm's out_dtype is HK_F32 or dtype, and so is weight_dtype;
                                         * 16-bit types are not mixed with each other */
    float eps;
    hk_rotary_plan plan;
    void* workspace; /* norm, backward: hk_qk_norm_rotary_workspace_bytes, 16-byte aligned */
    size_t workspace_bytes;
} hk_qk_params;

/* q_out = the rotation of q, k_out that of k.  The result may be the argument itself (same pointer, strides, type). */
int hk_rotary_forward(const hk_qk_params* p, void* stream);
/* dq = the rotation of dq_out by the opposite angles, dk that of dk_out. */
int hk_rotary_backward(const hk_qk_params* p, void* stream);
/* The same behind an RMS norm of every row: x -> x / sqrt(mean(x^2) + eps) * weight. */
int hk_qk_norm_rotary_forward(const hk_qk_params* p, void* stream);
/* Gradients of q, k and of the weights (sums over all rows, in an order that depends on sizes and device alone: the same
 * call gives the same bits). */
int hk_qk_norm_rotary_backward(const hk_qk_params* p, void* stream);
size_t hk_qk_norm_rotary_workspace_bytes(const hk_qk_params* p);

/* Attention of a batch whose requests share a prefix.  Row (b, i) of a head sees every prefix key and the keys
 * j < lengths[b] of its request, with is_causal those with j <= lengths[b] - T + i.  Heads in groups of nh / nh_kv
 * share a head of keys and values.  A row that sees nothing gives O = 0, LSE = -inf.  A key that is_causal alone hides from
 * a row takes part in it with weight 0, so its values have to be finite.
 * A NaN among a row's scores makes O and LSE of the row NaN; so may an infinite score.  An infinite value that a row sees makes
 * its element of O infinite or NaN.
 * Keys and values are read by TMA: a stride of 0 over a dimension larger than 1 is refused (HK_ERR_UNSUPPORTED), and so are
 * results whose rows lie on top of each other.  The same call gives the same bits: the kernels and how many runs they cut the keys
 * into depend on the sizes of the call and the device's SMs alone, where the runs of a request's own keys begin on its length too. */
typedef struct hk_shared_prefix_params {
    hk_view Q;        /* [B, nh, T, 64], `dtype` */
    hk_view Kp, Vp;   /* [1, nh_kv, prefix_len, 64], once for the whole batch; strideB is not used */
    hk_view K, V;     /* [B, nh_kv, kv_len, 64] */
    hk_view O;        /* [B, nh, T, 64], `dtype`, written */
    float* LSE;       /* [B, nh, T], written */
    int64_t lse_strideB, lse_strideH;
    const int32_t* lengths; /* device, [B]: keys each request has, taken into [0, kv_len]; NULL: kv_len.  Rows of K and V
                             * behind them are not part of any result, whatever they hold. */
    int B, nh, nh_kv, dtype;
    int64_t T, prefix_len, kv_len; /* prefix_len or kv_len may be 0 */
    float scale;
    bool is_causal;
    void* workspace; /* hk_shared_prefix_workspace_bytes, 256-byte aligned */
    size_t workspace_bytes;
} hk_shared_prefix_params;
int hk_shared_prefix_attention(const hk_shared_prefix_params* p, void* stream);
size_t hk_shared_prefix_workspace_bytes(const hk_shared_prefix_params* p);

/* ---- serving from a cache of pages ----------------------------------------------
 * No counterpart in the reference.  Prompts of different lengths behind each other, new tokens (drafted ones, or one) of each request against
 * keys and values that lie in pages, and what happens to the pages in between.
 *
 * A pool holds n_pages pages of `page` tokens (a multiple of 16) of every key head, [n_pages, nh_kv, page, 64], as a view whose strideB
 * leads from page to page: pages stored token by token are one with strideM > strideH.  Request b's token i is row i % page of the page
 * pages[b * pages_stride + i / page].  An entry outside [0, n_pages) stands for no page: nothing is written there, and as keys and values
 * it counts as rows of zeros.  The tables are read by the kernels: a captured call follows what they hold when it is replayed. */
typedef struct hk_pool {
    hk_view K, V;
    const int32_t* pages; /* device, [B, width] */
    int64_t pages_stride;
    int width;
    int n_pages, page;
} hk_pool;

/* Attention within whole prompts, packed: sequence b is rows starts[b] <= i < starts[b + 1] of Q, K, V and O; the starts are taken into
 * [0, N] and have to ascend.  Row i sees the keys j of its sequence, with is_causal those with j <= i.  Rows in no sequence are left as
 * they are, in O and LSE.  Heads in groups of nh / nh_kv share a head of keys and values.  NaN, infinities and bits: as in
 * hk_shared_prefix_attention; a key that is_causal alone hides from a row has to have finite values, other sequences' may hold
 * anything.  O and LSE may not overlap what is read. */
typedef struct hk_prompt_params {
    hk_view Q, K, V;  /* [1, nh or nh_kv, N, 64], `dtype`; strideB is not used */
    hk_view O;        /* the same, written */
    float* LSE;       /* [nh, N], written */
    int64_t lse_strideH;
    const int32_t* starts; /* device, [B + 1] */
    int B, nh, nh_kv, dtype;
    int64_t N;
    float scale;
    bool is_causal;
    void* workspace; /* hk_prompt_workspace_bytes, 256-byte aligned */
    size_t workspace_bytes;
} hk_prompt_params;
int hk_prompt_attention(const hk_prompt_params* p, void* stream);
size_t hk_prompt_workspace_bytes(const hk_prompt_params* p);

/* Attention of T <= 64 new tokens of each request.  Token i of request b sees the lengths[b] keys that lie in its pages (taken into [0,
 * width * page]) and of the new tokens those j with bit j of tree[b * tree_stride + i]: its ancestors in a tree of drafts, and itself.
 * Without `tree` it sees j <= i.  T = 1 is plain decoding.  A row that sees nothing gives O = 0, LSE = -inf.  Rows of pages behind a
 * request's last key may hold anything; a new token that the tree hides from a row takes part with weight 0, so its values have to be finite.
 * O and LSE may not overlap what is read. */
#define HK_TREE_TOKENS 64
typedef struct hk_tree_params {
    hk_view Q;        /* [B, nh, T, 64], `dtype` */
    hk_view K, V;     /* [B, nh_kv, T, 64], the new tokens' */
    hk_view O;        /* [B, nh, T, 64], written */
    float* LSE;       /* [B, nh, T], written */
    int64_t lse_strideB, lse_strideH;
    hk_pool pool;
    const int32_t* lengths; /* device, [B] */
    const int64_t* tree;    /* device, [B, T], or NULL */
    int64_t tree_stride;
    int B, nh, nh_kv, dtype;
    int64_t T;
    float scale;
    void* workspace; /* hk_tree_workspace_bytes, 256-byte aligned */
    size_t workspace_bytes;
} hk_tree_params;
int hk_tree_attention(const hk_tree_params* p, void* stream);
size_t hk_tree_workspace_bytes(const hk_tree_params* p);

/* Brings keys and values of new tokens into the pages, behind the lengths[b] that are there: new token k of request b becomes token
 * lengths[b] + k.  Which rows these are: with `starts`, taken into [0, T] and ascending, rows starts[b] <= i < starts[b + 1] of a packed
 * [1, nh_kv, T, 64] (k = i - starts[b]); otherwise of [B, nh_kv, T, 64] the rows picks[b * T + k] (NULL: k), k < counts[b] (NULL: T).  A pick outside [0, T) is
 * left out, and so is a token that has no page.  No two tokens may come to the same place. */
typedef struct hk_append_params {
    hk_view K, V;
    hk_pool pool;           /* written */
    const int32_t* lengths; /* device, [B] */
    const int32_t* starts;  /* device, [B + 1], or NULL */
    const int32_t* picks;   /* device, [B, T], or NULL */
    const int32_t* counts;  /* device, [B], or NULL */
    int B, nh_kv, dtype;
    int64_t T;
} hk_append_params;
int hk_cache_append(const hk_append_params* p, void* stream);

/* The next batch of B_out requests out of one of B: request i of it goes on where source[i] is (an entry outside [0, B): it starts
 * anew, with a length of 0).  users[p] counts who holds page p: the entries of the tables, and whoever else keeps pages (it counts on; of
 * a begun page the rows that there are stay, and one request goes on behind them).  Pages
 * that are full of a request's tokens are shared by all that go on with it.  One that is begun stays with the first of these; the others
 * get a page of their own with its rows copied, in every layer; if it is no page, all of them get one, whose rows are zeros, as they counted.
 * Then each request gets pages until it has room for room[i] tokens more,
 * out of those that nobody holds any longer: the lowest first, to the requests in their order.  What does not fit, because the pool is
 * empty or a row of the table at its end, is -1 in the table and counted in `missing` (up to 2^31 - 1).
 * Pages of requests that do not go on are free at once, and may be the ones that are given.  The tables that are written may not overlap
 * those that are read. */
typedef struct hk_fork_params {
    hk_pool pool;             /* of the first layer, with the old table; rows of pages are written */
    int64_t k_strideL, v_strideL; /* from layer to layer */
    const int32_t* lengths;   /* device, [B] */
    const int32_t* users;     /* device, [n_pages] */
    const int32_t* source;    /* device, [B_out] */
    const int32_t* room;      /* device, [B_out], or NULL: room_all for each */
    int32_t* pages_out;       /* device, [B_out, width], contiguous, written */
    int32_t* lengths_out;     /* device, [B_out], written */
    int32_t* users_out;       /* device, [n_pages], written */
    int32_t* missing;         /* device, [1], written */
    int B, B_out, layers, nh_kv, dtype;
    int64_t room_all;
    void* workspace; /* hk_cache_fork_workspace_bytes, 256-byte aligned */
    size_t workspace_bytes;
} hk_fork_params;
int hk_cache_fork(const hk_fork_params* p, void* stream);
size_t hk_cache_fork_workspace_bytes(const hk_fork_params* p);

/* Brings the n pages that somebody holds (users > 0) to the front of the pools, in every layer: those at n and behind it are copied, in
 * their order, to the free ones before it, in theirs.  where[p] is page p's new place, -1 if it is free; pages_out and users_out are the table
 * and the users as they are then.  The same restrictions as above; the rows of pages that are free then are left as they are. */
typedef struct hk_compact_params {
    hk_pool pool;
    int64_t k_strideL, v_strideL;
    const int32_t* users;
    int32_t* pages_out; /* device, [B, width], contiguous, written */
    int32_t* users_out; /* device, [n_pages], written */
    int32_t* where;     /* device, [n_pages], written */
    int B, layers, nh_kv, dtype;
    void* workspace; /* hk_cache_compact_workspace_bytes, 256-byte aligned */
    size_t workspace_bytes;
} hk_compact_params;
int hk_cache_compact(const hk_compact_params* p, void* stream);
size_t hk_cache_compact_workspace_bytes(const hk_compact_params* p);

const char* hk_status_string(int status);

#ifdef __cplusplus
}
#endif

#endif /* HK_ATTENTION_H_ */
