// serving_attention.cu -- attention within packed prompts (hk_prompt_attention) and of drafted tokens against a cache of pages
// (hk_tree_attention), include/hk_attention.h: checks of arguments and how the work is cut.
#include <cmath>

#include "serving_attention.cuh"

namespace hk {
namespace {

// ---------------------------------------------------------------------------
// The parts of each block that fell to several workers, added up in an order of their own: 16 lanes to a part of a row, and as many parts
// of a row at once as there are lanes left.  The block begins in the second slot of a worker and goes on in the first ones of those behind it.
// Latency bounds it: what is looked up is asked for at once, whether there turns out to be such a part or not.
// ---------------------------------------------------------------------------
constexpr int GROUPS = 16;

template <class X>
__global__ void __launch_bounds__(GROUPS * 16) combine_kernel(const __grid_constant__ ServingArgs a, const int workers) {
    __shared__ float4 sums[GROUPS][16];
    __shared__ float2 mls[GROUPS];
    pdl_wait();
    pdl_trigger();
    const int first = blockIdx.x;
    const PartRecord rec = a.parts[first];
    int n = 0;  // parts: up to the first worker behind that has the last one
    for (int w0 = first + 1; n == 0; w0 += 32) {
        const int w = min(w0 + (int)(threadIdx.x & 31), workers - 1), head = a.parts[w].head;
        if (rec.tokens == 0) return;
        const unsigned stops = __ballot_sync(0xffffffffu, w == workers - 1 || (head != PART_GOES_ON && head != PART_EMPTY));
        if (stops) n = min(w0 + __ffs(stops) - 1, workers - 1) - first + 1;
    }
    const int sub = threadIdx.x & 15, g = threadIdx.x >> 4;
    const uint32_t together = threadIdx.x & 16 ? 0xffff0000u : 0xffffu;
    const int rows = a.rows ? rec.tokens : a.sum_rows, per = (rows + gridDim.y - 1) / gridDim.y, r_end = min(rows, (int)(blockIdx.y + 1) * per);
    int side = 1;  // groups to a row
    while (side * 2 * per <= GROUPS && side < n) side *= 2;
    for (int r0 = blockIdx.y * per; r0 < r_end; r0 += GROUPS / side) {
        const int r = r0 + g / side, p_first = g % side;
        // the token and the head that row r is
        int token, h;
        bool valid = r < r_end;
        if (a.rows) {
            const int row = rec.token0 + r;
            token = row / a.group;
            h = rec.head0 * a.group + row - token * a.group;
        } else {
            const int t = r / TILE, box_heads = min(a.group, TILE), in_stream = r - t * TILE, token_in = in_stream / box_heads, head = in_stream - token_in * box_heads;
            token = t * a.stream_tokens + token_in;
            valid = valid && token_in < a.stream_tokens && token < rec.tokens && head < rec.heads;
            token += rec.token0;
            h = rec.head0 + head;
        }
        float M = -INFINITY, L = 0.f;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
        if (valid) {
            for (int p0 = p_first; p0 < n; p0 += 8 * side) {
                // eight parts; a lane looks up one
                const int p = p0 + (sub & 7) * side, worker = min(first + p, workers - 1), slot = 2 * worker + (p == 0);
                const int head = p == 0 ? PART_GOES_ON : a.parts[worker].head;
                const float2 ml = a.ml[(int64_t)slot * a.slot_rows + r];
                float4 v[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const int q = p0 + k * side, from = 2 * min(first + q, workers - 1) + (q == 0);
                    v[k] = q < n ? *reinterpret_cast<const float4*>(a.part + ((int64_t)from * a.slot_rows + r) * 64 + 4 * sub) : make_float4(0.f, 0.f, 0.f, 0.f);
                }
                const bool there = p < n && (head == PART_GOES_ON || head == PART_LAST);
                const float2 x = there ? ml : make_float2(-INFINITY, 0.f);
                float mx = x.x;
#pragma unroll
                for (int off = 4; off > 0; off >>= 1) mx = fmaxf(mx, __shfl_xor_sync(together, mx, off));
                mx = fmaxf(mx, M);
                const float ref = mx == -INFINITY ? 0.f : mx, old = ex2_approx(M - ref), w = there && x.y != 0.f ? ex2_approx(x.x - ref) : 0.f;
                M = mx;
                float sum = x.y * w;
#pragma unroll
                for (int off = 4; off > 0; off >>= 1) sum += __shfl_xor_sync(together, sum, off);
                L = L * old + sum;
                o.x *= old; o.y *= old; o.z *= old; o.w *= old;
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const float f = __shfl_sync(together, w, k, 16);
                    if (!__shfl_sync(together, (int)there, k, 16)) continue;  // what nobody wrote may be anything
                    o.x = fmaf(v[k].x, f, o.x); o.y = fmaf(v[k].y, f, o.y); o.z = fmaf(v[k].z, f, o.z); o.w = fmaf(v[k].w, f, o.w);
                }
            }
        }
        if (side > 1) {
            __syncthreads();
            sums[g][sub] = o;
            if (sub == 0) mls[g] = make_float2(M, L);
            __syncthreads();
            if (p_first == 0) {
                for (int k = 1; k < side; ++k) M = fmaxf(M, mls[g + k].x);
                const float ref = M == -INFINITY ? 0.f : M;
                L = 0.f;
                o = make_float4(0.f, 0.f, 0.f, 0.f);
                for (int k = 0; k < side; ++k) {
                    const float2 x = mls[g + k];
                    const float f = ex2_approx(x.x - ref);
                    const float4 v = sums[g + k][sub];
                    L = fmaf(x.y, f, L);
                    o.x = fmaf(v.x, f, o.x); o.y = fmaf(v.y, f, o.y); o.z = fmaf(v.z, f, o.z); o.w = fmaf(v.w, f, o.w);
                }
            }
        }
        if (valid && p_first == 0) {
            const float f = L != 0.f ? 1.f / L : 0.f;
            store4(const_cast<X*>(row_of<X>(a.O, rec.b, h, token)) + 4 * sub, make_float4(o.x * f, o.y * f, o.z * f, o.w * f));
            if (sub == 0) a.LSE[rec.b * a.lse_sB + h * a.lse_sH + token] = L != 0.f ? (M + log2f(L)) * LN2 : -INFINITY;
        }
    }
}

int check_heads(int64_t B, int nh, int nh_kv, int dtype, float scale) {
    if (dtype < HK_F32 || dtype > HK_F16) return HK_ERR_UNSUPPORTED;
    if (B <= 0 || nh <= 0 || nh_kv <= 0 || nh % nh_kv) return HK_ERR_BAD_SHAPE;
    if (!std::isfinite(scale) || scale == 0.f) return HK_ERR_BAD_SHAPE;
    return HK_OK;
}
// What is read by TMA: tensor maps do not know a stride of 0
int check_read(const hk_view& v, int64_t B, int H, int64_t T, int dtype) {
    const int rc = check_view(v, B, H, T, dtype, false);
    if (rc != HK_OK) return rc;
    return (B == 1 || v.strideB > 0) && (H == 1 || v.strideH > 0) && (T == 1 || v.strideM > 0) ? HK_OK : HK_ERR_UNSUPPORTED;
}
bool odd(const void* ints, uintptr_t size) { return reinterpret_cast<uintptr_t>(ints) & (size - 1); }

int check_sizes(const hk_prompt_params* p) {
    if (!p) return HK_ERR_NULL_POINTER;
    const int rc = check_heads(p->B, p->nh, p->nh_kv, p->dtype, p->scale);
    if (rc != HK_OK) return rc;
    return p->N <= 0 || p->B > (1 << 20) || p->nh > (1 << 20) || p->N * p->nh > (1LL << 30) ? HK_ERR_BAD_SHAPE : HK_OK;
}
int check_sizes(const hk_tree_params* p) {
    if (!p) return HK_ERR_NULL_POINTER;
    int rc = check_heads(p->B, p->nh, p->nh_kv, p->dtype, p->scale);
    if (rc != HK_OK || (rc = check_pool_sizes(p->pool, p->B, p->nh_kv, p->dtype)) != HK_OK) return rc;
    if (p->T <= 0 || p->B > (1 << 24) || p->nh > (1 << 20) || (int64_t)p->B * p->nh * 64 > (1LL << 30)) return HK_ERR_BAD_SHAPE;
    return p->T > HK_TREE_TOKENS ? HK_ERR_UNSUPPORTED : HK_OK;
}

// Slots for what workers leave of blocks that fell to several, if any can: `tiles` are the most that a block meets.
struct Parts {
    int workers, slots, rows;  // slots: of a worker
    bool any;
    int sums;                  // of a worker, rows of 64 floats
    size_t all_rows() const { return (size_t)workers * slots * rows; }
    size_t bytes() const { return any ? all_rows() * (64 * sizeof(float) + sizeof(float2)) + (size_t)workers * (sums * 64 * sizeof(float) + sizeof(PartRecord)) : 0; }
};
Parts parts_of(const hk_prompt_params* p) {
    const RowsPlan plan = rows_plan(p->dtype);
    const int64_t tiles = (p->N + plan.keys - 1) / plan.keys;
    return {sm_count(), plan.slots(tiles), plan.rows, tiles >= 2 * plan.least, 0};
}
bool few_rows(const hk_tree_params* p) { return p->T * (p->nh / p->nh_kv) <= 16; }
Parts parts_of(const hk_tree_params* p) {
    const int64_t keys = (int64_t)p->pool.width * p->pool.page;
    if (few_rows(p)) {
        const TreeFewPlan plan = tree_few_plan(p->dtype, (int)(p->T * (p->nh / p->nh_kv)), keys);
        return {plan.workers, plan.slots, plan.rows, keys / plan.keys + cdiv(p->T, plan.keys) >= 2 * plan.least, plan.sums};
    }
    const RowsPlan plan = rows_plan(p->dtype);
    const int64_t tiles = (keys + plan.keys - 1) / plan.keys + 1;
    return {sm_count(), plan.slots(tiles), plan.rows, tiles >= 2 * plan.least, 0};
}
int set_parts(ServingArgs& a, const Parts& parts, void* workspace, size_t bytes) {
    if (!parts.any) return HK_OK;
    if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 255u) || bytes < parts.bytes()) return HK_ERR_WORKSPACE;
    const size_t rows = parts.all_rows();
    a.sums = parts.sums > 0 ? static_cast<float4*>(workspace) : nullptr;
    a.part = static_cast<float*>(workspace) + (size_t)parts.workers * parts.sums * 64;
    a.ml = reinterpret_cast<float2*>(a.part + rows * 64);
    a.parts = reinterpret_cast<PartRecord*>(a.ml + rows);
    return HK_OK;
}
int set_scale(ServingArgs& a, int dtype, float scale) {
    a.scale_log2e = std::fabs(scale) * LOG2E;
    a.flip = scale > 0.f ? 0u : dtype == HK_F32 ? 0x80000000u : 0x80008000u;
    a.status = device_status_ptr();
    return a.status ? HK_OK : HK_ERR_CUDA;
}
ServingArgs sizes_of(const hk_prompt_params* p) {
    ServingArgs a{};
    a.B = p->B; a.Hk = p->nh_kv; a.group = p->nh / p->nh_kv; a.N = (int)p->N;
    a.causal = p->is_causal;
    return a;
}
ServingArgs sizes_of(const hk_tree_params* p) {
    ServingArgs a{};
    a.pool = p->pool;
    a.B = p->B; a.Hk = p->nh_kv; a.group = p->nh / p->nh_kv; a.T = (int)p->T;
    return a;
}
void put_line(const LineSum& x, int64_t* out) { out[0] = x.units; out[1] = x.narrowest; out[2] = x.lost; out[3] = x.unit_shift; }
}  // namespace

void set_line(ServingArgs& a, bool tree, int keys) {
    divide_by(a.block_tokens, a.block_mul, a.block_shift);
    // What all requests can come to: blocks, those of prompts without tokens left out; the keys that they meet, of prompts most where one has all the tokens; of
    // each block 5 tiles beside them (its beginning and end count up to 4, and its last tile as a whole), and up to a unit.
    const double heads = (double)a.Hk * a.chunks, blocks = heads * (tree ? (double)a.B * cdiv(a.rows ? a.rows : a.T, a.block_tokens) : (double)a.N / a.block_tokens + std::min(a.B, a.N));
    const double met = tree ? blocks * ((double)a.pool.width * a.pool.page + a.new_tiles * keys) : heads * ((double)a.N * a.N / a.block_tokens + 2.0 * a.N + (double)std::min(a.B, a.N) * a.block_tokens);
    double all = met + blocks * 5.0 * keys;
    for (a.unit_shift = 0; all + (a.unit_shift > 0 ? blocks : 0.0) >= 2e9; all /= 2) ++a.unit_shift;
}

// Sixteen rows to a CTA, 32 of blocks of 256: those that find nothing to add up cost time too (6 prompts of 300 tokens, 32 heads on 8, bf16: 18.5 us,
// 19.8 with sixteen; 64 rows are slower where there is something: 4 prompts of up to 1 000, 12 heads 25.7 and 23.6).
int launch_combine(ServingArgs a, int dtype, int workers, cudaStream_t stream) {
    typedef void (*Kernel)(ServingArgs, int);
    static const Kernel kernels[] = {combine_kernel<float>, combine_kernel<__nv_bfloat16>, combine_kernel<__half>};
    LaunchConfig lc(workers, GROUPS * 16, 0, stream, 1, true);
    a.sum_rows = a.T > 0 && a.T <= a.stream_tokens ? a.T * std::min(a.group, TILE) : a.slot_rows;
    lc.cfg.gridDim.y = cdiv(a.sum_rows, a.sum_rows > TILE ? 2 * GROUPS : GROUPS);
    if (cudaLaunchKernelEx(&lc.cfg, kernels[dtype], a, workers) != cudaSuccess) return check_launch();
    count_launch();
    return HK_OK;
}

}  // namespace hk

using namespace hk;

extern "C" {

size_t hk_prompt_workspace_bytes(const hk_prompt_params* p) { return check_sizes(p) == HK_OK ? parts_of(p).bytes() : 0; }

int hk_prompt_attention(const hk_prompt_params* p, void* stream) {
    int rc = check_sizes(p);
    if (rc != HK_OK) return rc;
    if ((rc = check_read(p->Q, 1, p->nh, p->N, p->dtype)) || (rc = check_read(p->K, 1, p->nh_kv, p->N, p->dtype)) ||
        (rc = check_read(p->V, 1, p->nh_kv, p->N, p->dtype)) || (rc = check_view(p->O, 1, p->nh, p->N, p->dtype, true)))
        return rc;
    if (!p->LSE || !p->starts) return HK_ERR_NULL_POINTER;
    if (odd(p->LSE, 4) || odd(p->starts, 4)) return HK_ERR_MISALIGNED;
    if (p->nh > 1 && p->lse_strideH < p->N) return HK_ERR_UNSUPPORTED;  // rows on top of each other
    ServingArgs a = sizes_of(p);
    a.Q = p->Q; a.K = p->K; a.V = p->V; a.O = p->O;
    a.LSE = p->LSE; a.lse_sH = p->lse_strideH;
    a.starts = p->starts;
    if ((rc = set_parts(a, parts_of(p), p->workspace, p->workspace_bytes)) || (rc = set_scale(a, p->dtype, p->scale))) return rc;
    return launch_prompt_rows(a, p->dtype, static_cast<cudaStream_t>(stream));
}

size_t hk_tree_workspace_bytes(const hk_tree_params* p) { return check_sizes(p) == HK_OK ? parts_of(p).bytes() : 0; }

int hk_tree_attention(const hk_tree_params* p, void* stream) {
    int rc = check_sizes(p);
    if (rc != HK_OK) return rc;
    if ((rc = check_read(p->Q, p->B, p->nh, p->T, p->dtype)) || (rc = check_read(p->K, p->B, p->nh_kv, p->T, p->dtype)) ||
        (rc = check_read(p->V, p->B, p->nh_kv, p->T, p->dtype)) || (rc = check_view(p->O, p->B, p->nh, p->T, p->dtype, true)) ||
        (rc = check_pool(p->pool, p->B, p->nh_kv, p->dtype, false)) || (rc = check_read(p->pool.K, p->pool.n_pages, p->nh_kv, p->pool.page, p->dtype)) ||
        (rc = check_read(p->pool.V, p->pool.n_pages, p->nh_kv, p->pool.page, p->dtype)))
        return rc;
    if (!p->LSE || !p->lengths) return HK_ERR_NULL_POINTER;
    if (odd(p->LSE, 4) || odd(p->lengths, 4) || odd(p->tree, 8)) return HK_ERR_MISALIGNED;
    if (p->tree && p->tree_stride < 0) return HK_ERR_BAD_SHAPE;
    Dim lse[] = {{p->B, p->lse_strideB}, {p->nh, p->lse_strideH}};
    if (!lie_apart(lse, p->T)) return HK_ERR_UNSUPPORTED;  // rows on top of each other
    ServingArgs a = sizes_of(p);
    a.Q = p->Q; a.K = p->K; a.V = p->V; a.O = p->O;
    a.LSE = p->LSE; a.lse_sB = p->lse_strideB; a.lse_sH = p->lse_strideH;
    a.lengths = p->lengths; a.tree = p->tree; a.tree_stride = p->tree_stride;
    if ((rc = set_parts(a, parts_of(p), p->workspace, p->workspace_bytes)) || (rc = set_scale(a, p->dtype, p->scale))) return rc;
    return few_rows(p) ? launch_tree_few(a, p->dtype, static_cast<cudaStream_t>(stream)) : launch_tree_rows(a, p->dtype, static_cast<cudaStream_t>(stream));
}

// For tests: the line (LineSum) of a call of these sizes whose prompts, or requests in their pages, have `lens` keys (host, [B])
int hk_prompt_line(const hk_prompt_params* p, const int32_t* lens, int64_t* out) {
    const int rc = check_sizes(p);
    if (rc == HK_OK) put_line(prompt_rows_line(sizes_of(p), p->dtype, lens), out);
    return rc;
}
int hk_tree_line(const hk_tree_params* p, const int32_t* lens, int64_t* out) {
    const int rc = check_sizes(p);
    if (rc == HK_OK) put_line(few_rows(p) ? tree_few_line(sizes_of(p), p->dtype, lens) : tree_rows_line(sizes_of(p), p->dtype, lens), out);
    return rc;
}

}  // extern "C"
