// serving_attention.cu -- attention within packed prompts (hk_prompt_attention) and of drafted tokens against a cache of pages
// (hk_tree_attention), include/hk_attention.h: checks of arguments and how the work is cut.
#include <cmath>

#include "serving_attention.cuh"

namespace hk {
namespace {

template <class X>
__device__ __forceinline__ float2 two(const X* p) {
    if constexpr (sizeof(X) == 4) return *reinterpret_cast<const float2*>(p);
    else return unpack<X>(*reinterpret_cast<const uint32_t*>(p));
}

// A warp to a row: 32 keys at a time, a key to a lane for the scores, two elements to a lane for the values.
template <class X, bool TREE>
__global__ void __launch_bounds__(128) rows_kernel(const __grid_constant__ ServingArgs a) {
    const int lane = threadIdx.x & 31;
    pdl_wait();
    pdl_trigger();
    const int64_t item = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    const int h = (int)(item % (a.Hk * a.group)), kvh = h / a.group;
    const int64_t token = item / (a.Hk * a.group);
    if (token >= (TREE ? (int64_t)a.B * a.T : a.N)) return;
    int b, t, old, n;  // keys of the pages or the sequence, and all of them
    int64_t base = 0;
    uint64_t sees = ~0ull;
    if (TREE) {
        b = (int)(token / a.T);
        t = (int)(token - (int64_t)b * a.T);
        old = cache_keys(a, b);
        n = old + a.T;
        sees = tree_bits(a, b, t);
    } else {
        t = (int)token;
        b = sequence_of(a.starts, a.B, t, lane);
        if (b >= a.B || a.starts[b] > t) return;
        base = max(a.starts[b], 0);
        old = n = (a.causal ? t + 1 : min(max(a.starts[b + 1], 0), a.N)) - (int)base;
    }
    auto key = [&](int j, bool v) -> const X* {
        if (!TREE) return row_of<X>(v ? a.V : a.K, 0, kvh, base + j);
        if (j >= old) return row_of<X>(v ? a.V : a.K, b, kvh, j - old);
        const int page = a.pool.pages[b * a.pool.pages_stride + j / a.pool.page];
        return (unsigned)page < (unsigned)a.pool.n_pages ? row_of<X>(v ? a.pool.V : a.pool.K, page, kvh, j % a.pool.page) : nullptr;
    };
    const X* q = row_of<X>(a.Q, TREE ? b : 0, h, t);
    float m = -INFINITY, l = 0.f;
    float2 o = make_float2(0.f, 0.f);
    for (int j0 = 0; j0 < n; j0 += 32) {
        const int j = j0 + lane;
        const bool seen = j < n && (j < old || (sees >> (j - old) & 1));
        float s = 0.f;
        const X* k = seen ? key(j, false) : nullptr;
        for (int d = 0; d < 64; d += 2) {
            const float2 x = two(q + d), y = k ? two(k + d) : make_float2(0.f, 0.f);
            s = fmaf(x.x, y.x, fmaf(x.y, y.y, s));
        }
        s = seen ? s * a.scale : -INFINITY;
        float mx = s;
        for (int off = 16; off > 0; off >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
        mx = fmaxf(mx, m);
        const float ref = mx == -INFINITY ? 0.f : mx, alpha = expf(m - ref), w = expf(s - ref);
        m = mx;
        l = l * alpha + w;
        o.x *= alpha;
        o.y *= alpha;
        for (int i = 0; i < 32 && j0 + i < n; ++i) {
            const X* v = key(j0 + i, true);
            const float wi = __shfl_sync(0xffffffffu, w, i);
            if (!v || !(j0 + i < old || (sees >> (j0 + i - old) & 1))) continue;
            const float2 y = two(v + 2 * lane);
            o.x = fmaf(wi, y.x, o.x);
            o.y = fmaf(wi, y.y, o.y);
        }
    }
    for (int off = 16; off > 0; off >>= 1) l += __shfl_xor_sync(0xffffffffu, l, off);
    const float f = l != 0.f ? 1.f / l : 0.f;
    X* to = const_cast<X*>(row_of<X>(a.O, TREE ? b : 0, h, t)) + 2 * lane;
    if constexpr (sizeof(X) == 4) *reinterpret_cast<float2*>(to) = make_float2(o.x * f, o.y * f);
    else *reinterpret_cast<uint32_t*>(to) = pack<X>(o.x * f, o.y * f);
    if (lane == 0) a.LSE[(TREE ? b * a.lse_sB : 0) + h * a.lse_sH + t] = l != 0.f ? m + logf(l) : -INFINITY;
}

template <bool TREE>
int launch_rows(const ServingArgs& a, int dtype, int64_t tokens, cudaStream_t stream) {
    typedef void (*Kernel)(ServingArgs);
    static const Kernel kernels[] = {rows_kernel<float, TREE>, rows_kernel<__nv_bfloat16, TREE>, rows_kernel<__half, TREE>};
    const int64_t blocks = (tokens * a.Hk * a.group + 3) / 4;
    if (blocks > 0x7fffffffLL) return HK_ERR_BAD_SHAPE;
    LaunchConfig lc((unsigned)blocks, 128, 0, stream, 1, true);
    if (cudaLaunchKernelEx(&lc.cfg, kernels[dtype], a) != cudaSuccess) return check_launch();
    count_launch();
    return HK_OK;
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

// What the kernel of many rows leaves of blocks that fell to several CTAs; nothing where no block can: `keys` are the most that there are.
size_t parts_bytes(int dtype, int64_t keys, bool more) {
    const RowsPlan plan = rows_plan(dtype);
    if ((keys + plan.keys - 1) / plan.keys + more < 2 * plan.least) return 0;
    return (size_t)sm_count() * (2 * plan.rows * (64 * sizeof(float) + sizeof(float2)) + sizeof(PartRecord));
}
int set_parts(ServingArgs& a, int dtype, size_t need, void* workspace, size_t bytes) {
    if (need == 0) return HK_OK;
    if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 255u) || bytes < need) return HK_ERR_WORKSPACE;
    const size_t rows = (size_t)sm_count() * 2 * rows_plan(dtype).rows;
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
bool few_rows(const hk_tree_params* p) { return p->T * (p->nh / p->nh_kv) <= 16; }

}  // namespace
}  // namespace hk

using namespace hk;

extern "C" {

size_t hk_prompt_workspace_bytes(const hk_prompt_params* p) { return check_sizes(p) == HK_OK ? parts_bytes(p->dtype, p->N, false) : 0; }

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
    if ((rc = set_parts(a, p->dtype, hk_prompt_workspace_bytes(p), p->workspace, p->workspace_bytes)) || (rc = set_scale(a, p->dtype, p->scale))) return rc;
    return launch_prompt_rows(a, p->dtype, static_cast<cudaStream_t>(stream));
}

size_t hk_tree_workspace_bytes(const hk_tree_params* p) {
    return check_sizes(p) == HK_OK && !few_rows(p) ? parts_bytes(p->dtype, (int64_t)p->pool.width * p->pool.page, true) : 0;
}

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
    if ((rc = set_parts(a, p->dtype, hk_tree_workspace_bytes(p), p->workspace, p->workspace_bytes)) || (rc = set_scale(a, p->dtype, p->scale))) return rc;
    if (!few_rows(p)) return launch_tree_rows(a, p->dtype, static_cast<cudaStream_t>(stream));
    return launch_rows<true>(a, p->dtype, (int64_t)a.B * a.T, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
