// shared_prefix.cu -- attention of a batch whose requests share a prefix (include/hk_attention.h: hk_shared_prefix_attention):
// checks of arguments and how the work is cut.
#include <cmath>
#include <cstring>

#include "shared_prefix.cuh"

namespace hk {
namespace {

// ---------------------------------------------------------------------------
// The slots of each row, added up in an order of their own: 16 lanes a row, four elements a lane, or a warp, a half of it to every
// other slot.  What bounds it is the latency of one round of loads and of the launch: up to 16 slots are loaded at once by 16 lanes, 32
// by a warp (B16 H12, 18 slots of 192 rows: 0.8 us less than 16 lanes take; 3 slots of 7 392 rows: 2 us more).
// ---------------------------------------------------------------------------
template <class X, int HALVES>
__global__ void __launch_bounds__(128) prefix_combine_kernel(const __grid_constant__ PrefixArgs a) {
    constexpr int LANES = 16 * HALVES;
    const int lane = threadIdx.x & (LANES - 1), half = lane >> 4, sub = lane & 15;
    const uint32_t together = HALVES == 2 ? 0xffffffffu : threadIdx.x & 16 ? 0xffff0000u : 0xffffu;
    const int64_t rows = a.slot_rows, row = (int64_t)blockIdx.x * (128 / LANES) + threadIdx.x / LANES;
    if (row >= rows) return;
    int kvh, b, r;  // the row among those of its key head and request
    bool valid = true;
    if (a.whole) {
        const int item = a.first_split + (int)(row / a.block_rows), at = item / a.tiles_o;
        b = at / a.Hk;
        kvh = at - b * a.Hk;
        r = (a.tiles_o - 1 - (item - at * a.tiles_o)) * a.block_rows + (int)(row % a.block_rows);
        valid = r < a.T * a.group;  // the last block of a request is not full
    } else {
        kvh = (int)(row / a.R);
        r = (int)(row - (int64_t)kvh * a.R);
        b = r / (a.T * a.group);
        r -= b * a.T * a.group;
    }
    if (!valid) return;
    const int t = r / a.group, h = kvh * a.group + r - t * a.group;
    X* const O = const_cast<X*>(row_of<X>(a.O, b, h, t)) + 4 * sub;
    float* const LSE = a.LSE + b * a.lse_sB + h * a.lse_sH + t;
    pdl_wait();
    pdl_trigger();
    float M = -INFINITY, L = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int s0 = 0; s0 < a.slots; s0 += LANES) {
        const float2 x = s0 + lane < a.slots ? a.ml[(s0 + lane) * rows + row] : make_float2(-INFINITY, 0.f);  // a lane looks up one slot
        const float* from = a.part + ((int64_t)(s0 + half) * rows + row) * 64 + 4 * sub;
        float4 v[16];
#pragma unroll
        for (int i = 0; i < 16; ++i)
            v[i] = s0 + HALVES * i + half < a.slots ? *reinterpret_cast<const float4*>(from + HALVES * i * rows * 64) : make_float4(0.f, 0.f, 0.f, 0.f);
        float mx = x.x;
#pragma unroll
        for (int off = LANES / 2; off > 0; off >>= 1) mx = fmaxf(mx, __shfl_xor_sync(together, mx, off));
        mx = fmaxf(mx, M);
        const float ref = mx == -INFINITY ? 0.f : mx, old = ex2_approx(M - ref), w = x.y == 0.f ? 0.f : ex2_approx(x.x - ref);
        M = mx;
        L = L * old + x.y * w;
        o.x *= old; o.y *= old; o.z *= old; o.w *= old;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            if (s0 + HALVES * i >= a.slots) break;
            const float f = __shfl_sync(together, w, HALVES * i + half, LANES);
            o.x = fmaf(v[i].x, f, o.x); o.y = fmaf(v[i].y, f, o.y); o.z = fmaf(v[i].z, f, o.z); o.w = fmaf(v[i].w, f, o.w);
        }
    }
#pragma unroll
    for (int off = LANES / 2; off > 0; off >>= 1) L += __shfl_xor_sync(together, L, off);
    if (HALVES == 2) {
        o.x += __shfl_xor_sync(together, o.x, 16); o.y += __shfl_xor_sync(together, o.y, 16);
        o.z += __shfl_xor_sync(together, o.z, 16); o.w += __shfl_xor_sync(together, o.w, 16);
    }
    const float f = L != 0.f ? 1.f / L : 0.f;
    if (half == 0) store4(O, make_float4(o.x * f, o.y * f, o.z * f, o.w * f));
    if (lane == 0) *LSE = L != 0.f ? (M + log2f(L)) * LN2 : -INFINITY;
}

int check_sizes(const hk_shared_prefix_params* p) {
    if (!p) return HK_ERR_NULL_POINTER;
    if (p->dtype < HK_F32 || p->dtype > HK_F16) return HK_ERR_UNSUPPORTED;
    if (p->B <= 0 || p->nh <= 0 || p->nh_kv <= 0 || p->T <= 0 || p->prefix_len < 0 || p->kv_len < 0) return HK_ERR_BAD_SHAPE;
    if (p->nh % p->nh_kv) return HK_ERR_BAD_SHAPE;
    if (p->T > (1 << 30) || p->prefix_len > (1 << 30) || p->kv_len > (1 << 30)) return HK_ERR_BAD_SHAPE;
    if ((int64_t)p->B * p->nh > (1 << 24) || (int64_t)p->B * p->nh * p->T > (1LL << 30)) return HK_ERR_BAD_SHAPE;
    if (!std::isfinite(p->scale) || p->scale == 0.f) return HK_ERR_BAD_SHAPE;
    return HK_OK;
}
int check(const hk_shared_prefix_params* p) {
    int rc = check_sizes(p);
    if (rc != HK_OK) return rc;
    if ((rc = check_view(p->Q, p->B, p->nh, p->T, p->dtype, false)) || (rc = check_view(p->O, p->B, p->nh, p->T, p->dtype, true))) return rc;
    auto keys = [&](const hk_view& v, int B, int64_t T) {
        const int rc = T > 0 ? check_view(v, B, p->nh_kv, T, p->dtype, false) : HK_OK;
        // tensor maps do not know a stride of 0
        const bool spread = T == 0 || ((B == 1 || v.strideB > 0) && (p->nh_kv == 1 || v.strideH > 0) && (T == 1 || v.strideM > 0));
        return rc != HK_OK ? rc : spread ? HK_OK : (int)HK_ERR_UNSUPPORTED;
    };
    if ((rc = keys(p->Kp, 1, p->prefix_len)) || (rc = keys(p->Vp, 1, p->prefix_len)) || (rc = keys(p->K, p->B, p->kv_len)) || (rc = keys(p->V, p->B, p->kv_len))) return rc;
    if (!p->LSE) return HK_ERR_NULL_POINTER;
    Dim lse[] = {{p->B, p->lse_strideB}, {p->nh, p->lse_strideH}};
    if (!lie_apart(lse, p->T)) return HK_ERR_UNSUPPORTED;  // rows on top of each other
    if ((reinterpret_cast<uintptr_t>(p->LSE) | reinterpret_cast<uintptr_t>(p->lengths)) & 3u) return HK_ERR_MISALIGNED;
    return HK_OK;
}

// How the work is cut: kernels and numbers of runs depend on sizes and the number of SMs alone (lengths are on the device), the borders of
// the runs of a request's own keys on its length too.  The same call gives the same bits.
struct Plan {
    bool prefix_many, own_many;  // which kernels
};

// Estimates, in microseconds, from calls taken apart with the clock of one B200; the choice they make was then compared with its
// neighbours (runs of the prefix 1 to 32, requests' own keys in 1 to 8 runs) at a dozen sizes.
constexpr double BLOCK_US = 4.4;                   // many rows: to start and end a CTA
constexpr double FEW_US = 2.2, COMBINE_US = 3.0;  // few rows: to start and end a CTA; the last kernel
double tile_us(int dtype, bool own) { return dtype == HK_F32 ? (own ? 1.3 : 1.15) : own ? 1.7 : 1.28; }  // many rows: a tile; own keys are masked
double batch_us(int dtype, int rows) { return dtype != HK_F32 ? 0.45 : rows <= 2 ? 0.4 : 0.65; }  // few rows: a batch of every warp

// One kind of work: CTAs, microseconds of each, how many an SM holds.
struct Work {
    double ctas, us, per_sm;
    double rounds(int sms) const { return std::ceil(ctas / (sms * per_sm)) * us; }
    double sm_time() const { return ctas * us / per_sm; }
};
// Two kinds side by side.  They do not fit each other without gaps: a part of all the work on top.
double together(const Work& x, const Work& y, int sms) {
    const double all = (x.sm_time() + y.sm_time()) / sms;
    return std::max({x.rounds(sms), y.rounds(sms), all}) + 0.15 * all;
}
// CTAs of few rows through `keys` keys each: by the batches of a warp, or by what the memory gives to all that run at once
Work few_work(double ctas, double keys, const FewPlan& f, int dtype, int sms) {
    return {ctas, FEW_US + std::max(std::ceil(keys / f.step) * batch_us(dtype, f.rows), keys * 2 * HEAD_DIM * esize(dtype) * std::min(ctas, (double)sms * f.per_sm) / 6e6),
            (double)f.per_sm};
}

// `items` blocks of many rows through all of their keys: of `mean` microseconds, the longest of `longest` and `tiles` tiles.  The last
// ones, which do not fill the SMs, in `parts` by their keys.
double whole_time(int64_t items, double mean, double longest, double tiles, int sms, int& parts) {
    const int64_t full = items / sms, tail = items % sms;
    double best = 0.0;
    parts = 1;
    for (int k = 1; tail > 0 && k <= 16 && (k == 1 || tiles >= 1.5 * k); ++k) {
        const double time = cdiv(tail * k, sms) * (longest / k + BLOCK_US) + (k > 1 ? COMBINE_US : 0.0);
        if (k > 1 && time >= best) continue;
        best = time;
        parts = k;
    }
    return full * (mean + BLOCK_US) + best;
}

Plan make_plan(const hk_shared_prefix_params* p, PrefixArgs& a) {
    a.B = p->B; a.Hk = p->nh_kv; a.group = p->nh / p->nh_kv; a.T = (int)p->T; a.P = (int)p->prefix_len; a.S = (int)p->kv_len;
    a.R = p->B * a.T * a.group;
    const int own_rows = a.T * a.group, sms = sm_count(), dtype = p->dtype;
    const ManyPlan mp = many_plan(dtype);
    const FewPlan fp = few_plan(dtype, a.R), fo = few_plan(dtype, own_rows);
    const int64_t requests = (int64_t)a.B * a.Hk;
    const double mean_own = 0.5 * a.S;  // the caches are taken to be half full
    const bool own = a.S > 0 || a.P == 0;  // without keys of their own, the prefix alone

    // the requests' own keys, by few or by many rows: CTAs and runs
    const int few_tiles = cdiv(own_rows, fo.rows), many_tiles = cdiv(own_rows, mp.rows);
    int few_splits = 1;
    while (few_splits < 16 && requests * few_tiles * few_splits * 2 <= sms * fo.per_sm && few_splits * 2 * 4 * fo.step <= a.S) few_splits *= 2;
    const Work own_few = few_work((double)requests * few_tiles * few_splits, mean_own / few_splits, fo, dtype, sms);
    const Work own_many{(double)requests * many_tiles, BLOCK_US + std::ceil(mean_own / mp.keys) * tile_us(dtype, true), 1.0}, nothing{0.0, 0.0, 1.0};

    struct Choice {
        double us;
        Plan plan;
        int whole, per_p;
    } best{1e30, {false, false}, 0, 0};
    auto consider = [&](const Choice& c) {
        if (c.us < best.us) best = c;
    };
    int parts = 1;
    // every block of rows takes the prefix and then its request's keys: nothing goes through memory, in one launch
    if (own) {
        const int warps = fo.rows < 16 ? 16 : 8, keys = fo.step / 4 * warps;
        const double items = (double)requests * few_tiles, all_keys = a.P + mean_own, bytes = all_keys * 2 * HEAD_DIM * esize(dtype);
        // a batch of every warp takes longer beside more warps; an SM reads 80 GB/s, all of them 6 TB/s
        const double us = FEW_US + 1.0 + std::max({std::ceil(all_keys / keys) * 1.3 * batch_us(dtype, fo.rows), bytes / 80e3, bytes * std::min(items, (double)sms) / 6e6});
        consider({std::ceil(items / sms) * us, {false, false}, 1, 0});
        if (a.P == 0) consider({together(own_few, nothing, sms) + (few_splits > 1 ? COMBINE_US : 0.0), {false, false}, 0, 0});
        if (own_rows > 16) {
            const double prefix = std::ceil((double)a.P / mp.keys), most = std::ceil((double)a.S / mp.keys), us = prefix * tile_us(dtype, false), own_us = most * tile_us(dtype, true);
            consider({whole_time(requests * many_tiles, us + 0.5 * own_us, us + own_us, prefix + most, sms, parts), {false, true}, 1, 0});
        }
    }
    // the prefix once for all rows, in runs: as many as make the longer of its waves of CTAs and all of the work spread over the SMs
    // shortest
    for (int k = 0; a.P > 0 && k < 2; ++k) {
        if (k == 1 && a.R <= 32) break;
        const int64_t items = (int64_t)a.Hk * cdiv(a.R, k ? mp.rows : fp.rows);
        const int step = k ? mp.keys : fp.step, most = std::min(64, std::max(1, cdiv(a.P, (k ? 2 : 4) * step)));
        if (!k && a.R > 32 && items > 16 * sms) continue;  // far from few rows
        for (int n = 1; n <= most; ++n) {
            const int per = cdiv(a.P, (int64_t)n * step) * step;
            const Work w = k ? Work{(double)items * n, BLOCK_US + per / step * tile_us(dtype, false), 1.0}
                             : few_work((double)items * n, per, fp, dtype, sms);
            const double last = COMBINE_US + 0.07 * n;
            consider({together(w, own ? own_few : nothing, sms) + last + (k && own ? 1.0 : 0.0), {k == 1, false}, 0, per});
            if (own && own_rows > 16) consider({together(w, own_many, sms) + last + 1.0, {k == 1, true}, 0, per});
        }
    }
    a.tiles_o = best.plan.own_many ? many_tiles : few_tiles;
    a.whole = best.whole;
    a.per_p = best.per_p;
    a.splits_p = a.per_p ? cdiv(a.P, a.per_p) : 0;
    a.tiles_p = a.per_p ? cdiv(a.R, best.plan.prefix_many ? mp.rows : fp.rows) : 0;
    if (a.whole) {
        const int64_t items = requests * a.tiles_o;
        a.splits_o = 1;
        a.slots = best.plan.own_many ? parts : 1;
        a.first_split = (int)(a.slots > 1 ? items / sms * sms : items);
        a.block_rows = mp.rows;
        a.slot_rows = (items - a.first_split) * mp.rows;
    } else {
        a.splits_o = !own ? 0 : best.plan.own_many ? 1 : few_splits;
        a.slots = a.splits_p + a.splits_o;
        a.slot_rows = (int64_t)a.Hk * a.R;
    }
    return best.plan;
}
// rows of all slots in the workspace
size_t slot_rows(const PrefixArgs& a) { return a.slots > 1 ? (size_t)a.slots * a.slot_rows : 0; }
constexpr size_t SLOT_BYTES = 64 * sizeof(float) + sizeof(float2);

}  // namespace

int prefix_tile_map(CUtensorMap* map, const hk_view& v, int dtype, int64_t B, int H, int64_t T, int rows, bool mn_major) {
    if (T == 0) {
        memset(map, 0, sizeof(*map));  // no tile of it is loaded
        return HK_OK;
    }
    const int64_t sM = T == 1 ? HEAD_DIM : v.strideM, sH = H == 1 ? sM * T : v.strideH, sB = B == 1 ? std::max(sH * H, sM * T) : v.strideB;
    if (dtype == HK_F32) return make_tile_map(map, static_cast<const float*>(v.ptr), HEAD_DIM, (int)B, H, T, sB, sM, sH, rows, mn_major);
    EncodeTiledFn enc = get_encode_tiled();
    if (!enc) return HK_ERR_CUDA;
    cuuint64_t dims[5] = {HEAD_DIM, (cuuint64_t)T, 1, (cuuint64_t)H, (cuuint64_t)B};
    cuuint64_t strides[4] = {(cuuint64_t)sM * 2, 128, (cuuint64_t)sH * 2, (cuuint64_t)sB * 2};
    cuuint32_t box[5] = {HEAD_DIM, (cuuint32_t)rows, 1, 1, 1}, ones[5] = {1, 1, 1, 1, 1};
    const CUresult r = enc(map, dtype == HK_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 5, v.ptr, dims, strides, box, ones,
                           CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? HK_OK : HK_ERR_CUDA;
}

}  // namespace hk

using namespace hk;

extern "C" {

size_t hk_shared_prefix_workspace_bytes(const hk_shared_prefix_params* p) {
    if (check_sizes(p) != HK_OK) return 0;
    PrefixArgs a{};
    make_plan(p, a);
    return slot_rows(a) * SLOT_BYTES;
}

// For tests: which kernels take the call's blocks of rows (many rows against the prefix, against the own keys; both in one go), the runs
// of the prefix and of the own keys, and the slots of a row.
int hk_shared_prefix_plan(const hk_shared_prefix_params* p, int* plan) {
    const int rc = check_sizes(p);
    if (rc != HK_OK) return rc;
    PrefixArgs a{};
    const Plan x = make_plan(p, a);
    const int out[] = {x.prefix_many, x.own_many, a.whole, a.splits_p, a.splits_o, a.slots};
    std::copy(out, out + 6, plan);
    return HK_OK;
}

int hk_shared_prefix_attention(const hk_shared_prefix_params* p, void* stream_) {
    int rc = check(p);
    if (rc != HK_OK) return rc;
    cudaStream_t stream = static_cast<cudaStream_t>(stream_);
    PrefixArgs a{};
    const Plan plan = make_plan(p, a);
    const size_t n = slot_rows(a);
    if (n > 0 && (!p->workspace || (reinterpret_cast<uintptr_t>(p->workspace) & 255u) || p->workspace_bytes < n * SLOT_BYTES)) return HK_ERR_WORKSPACE;
    a.part = static_cast<float*>(p->workspace);
    a.ml = reinterpret_cast<float2*>(a.part + n * 64);
    a.Q = p->Q; a.Kp = p->Kp; a.Vp = p->Vp; a.K = p->K; a.V = p->V; a.O = p->O;
    a.LSE = p->LSE; a.lse_sB = p->lse_strideB; a.lse_sH = p->lse_strideH;
    a.lengths = p->lengths;
    a.scale_log2e = std::fabs(p->scale) * LOG2E;
    a.flip = p->scale > 0.f ? 0u : p->dtype == HK_F32 ? 0x80000000u : 0x80008000u;
    a.causal = p->is_causal;
    a.status = device_status_ptr();
    if (!a.status) return HK_ERR_CUDA;
    if (a.splits_p > 0 && a.splits_o > 0 && !plan.prefix_many && !plan.own_many) {
        rc = launch_both_few(a, p->dtype, stream);
    } else {
        if (a.splits_p > 0) rc = plan.prefix_many ? launch_prefix_many(a, p->dtype, stream) : launch_prefix_few(a, p->dtype, stream);
        if (rc == HK_OK && a.splits_o > 0) rc = plan.own_many ? launch_own_many(a, p->dtype, stream) : launch_own_few(a, p->dtype, stream);
    }
    if (rc != HK_OK) return rc;
    if (a.slots == 1) return HK_OK;
    typedef void (*Kernel)(PrefixArgs);
    static const Kernel combine[2][3] = {{prefix_combine_kernel<float, 1>, prefix_combine_kernel<__nv_bfloat16, 1>, prefix_combine_kernel<__half, 1>},
                                         {prefix_combine_kernel<float, 2>, prefix_combine_kernel<__nv_bfloat16, 2>, prefix_combine_kernel<__half, 2>}};
    const int wide = a.slots > 16;
    LaunchConfig lc((unsigned)cdiv(a.slot_rows, wide ? 4 : 8), 128, 0, stream, 1, true);
    if (cudaLaunchKernelEx(&lc.cfg, combine[wide][p->dtype], a) != cudaSuccess) return check_launch();
    count_launch();
    return HK_OK;
}

}  // extern "C"
