// serving_attention.cu -- attention within packed prompts (hk_prompt_attention) and of drafted tokens against a cache of pages
// (hk_tree_attention), include/hk_attention.h: checks of arguments and how the work is cut.
#include <cmath>

#include "serving_attention.cuh"

namespace hk {
namespace {

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
    int workers, rows;
    bool any;
    size_t bytes() const { return any ? (size_t)workers * (2 * rows * (64 * sizeof(float) + sizeof(float2)) + sizeof(PartRecord)) : 0; }
};
Parts parts_of(const hk_prompt_params* p) {
    const RowsPlan plan = rows_plan(p->dtype);
    return {sm_count(), plan.rows, (p->N + plan.keys - 1) / plan.keys >= 2 * plan.least};
}
bool few_rows(const hk_tree_params* p) { return p->T * (p->nh / p->nh_kv) <= 16; }
Parts parts_of(const hk_tree_params* p) {
    const int64_t keys = (int64_t)p->pool.width * p->pool.page;
    if (few_rows(p)) {
        const TreeFewPlan plan = tree_few_plan(p->dtype, (int)(p->T * (p->nh / p->nh_kv)));
        return {plan.workers, plan.rows, keys / plan.keys + cdiv(p->T, plan.keys) >= 2 * plan.least};
    }
    const RowsPlan plan = rows_plan(p->dtype);
    return {sm_count(), plan.rows, (keys + plan.keys - 1) / plan.keys + 1 >= 2 * plan.least};
}
int set_parts(ServingArgs& a, const Parts& parts, void* workspace, size_t bytes) {
    if (!parts.any) return HK_OK;
    if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 255u) || bytes < parts.bytes()) return HK_ERR_WORKSPACE;
    const size_t rows = (size_t)parts.workers * 2 * parts.rows;
    a.part = static_cast<float*>(workspace);
    a.ml = reinterpret_cast<float2*>(a.part + rows * 64);
    a.parts = reinterpret_cast<PartRecord*>(a.ml + rows);
    return HK_OK;
}
int set_scale(ServingArgs& a, int dtype, float scale) {
    a.scale = scale;
    a.scale_log2e = std::fabs(scale) * LOG2E;
    a.flip = scale > 0.f ? 0u : dtype == HK_F32 ? 0x80000000u : 0x80008000u;
    a.status = device_status_ptr();
    return a.status ? HK_OK : HK_ERR_CUDA;
}
}  // namespace

void set_line(ServingArgs& a, bool tree, int keys) {
    a.block_shift = 31;
    while ((1LL << (a.block_shift - 31)) < a.block_tokens) ++a.block_shift;
    a.block_mul = (uint32_t)(((1ULL << a.block_shift) + a.block_tokens - 1) / a.block_tokens);
    // what all requests can come to, in keys: blocks, and what each counts at most
    const double blocks = (tree ? (double)a.B * cdiv(a.rows ? a.rows : a.T, a.block_tokens) : (double)a.N / a.block_tokens + a.B) * a.Hk * a.chunks;
    double all = blocks * ((tree ? (double)a.pool.width * a.pool.page + a.new_tiles * keys : a.N + a.block_tokens) + 4.0 * keys);
    for (a.unit_shift = 0; all >= 2e9; all /= 2) ++a.unit_shift;
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
    ServingArgs a{};
    a.Q = p->Q; a.K = p->K; a.V = p->V; a.O = p->O;
    a.LSE = p->LSE; a.lse_sH = p->lse_strideH;
    a.starts = p->starts;
    a.B = p->B; a.Hk = p->nh_kv; a.group = p->nh / p->nh_kv; a.N = (int)p->N;
    a.causal = p->is_causal;
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
    ServingArgs a{};
    a.Q = p->Q; a.K = p->K; a.V = p->V; a.O = p->O; a.pool = p->pool;
    a.LSE = p->LSE; a.lse_sB = p->lse_strideB; a.lse_sH = p->lse_strideH;
    a.lengths = p->lengths; a.tree = p->tree; a.tree_stride = p->tree_stride;
    a.B = p->B; a.Hk = p->nh_kv; a.group = p->nh / p->nh_kv; a.T = (int)p->T;
    if ((rc = set_parts(a, parts_of(p), p->workspace, p->workspace_bytes)) || (rc = set_scale(a, p->dtype, p->scale))) return rc;
    return few_rows(p) ? launch_tree_few(a, p->dtype, static_cast<cudaStream_t>(stream)) : launch_tree_rows(a, p->dtype, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
