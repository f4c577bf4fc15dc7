// shared_prefix.cu -- attention of a batch whose requests share a prefix (include/hk_attention.h: hk_shared_prefix_attention):
// checks of arguments and how the work is cut.
#include <cmath>

#include "shared_prefix.cuh"

namespace hk {
namespace {

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
    for (const hk_view* v : {&p->Kp, &p->Vp})
        if (p->prefix_len > 0 && (rc = check_view(*v, 1, p->nh_kv, p->prefix_len, p->dtype, false))) return rc;
    for (const hk_view* v : {&p->K, &p->V})
        if (p->kv_len > 0 && (rc = check_view(*v, p->B, p->nh_kv, p->kv_len, p->dtype, false))) return rc;
    if (!p->LSE) return HK_ERR_NULL_POINTER;
    if ((reinterpret_cast<uintptr_t>(p->LSE) | reinterpret_cast<uintptr_t>(p->lengths)) & 3u) return HK_ERR_MISALIGNED;
    return HK_OK;
}

// How the work is cut.  The runs of keys depend on sizes, lengths and the number of SMs alone: the same call gives the same bits.
struct Plan {
    bool prefix_many, own_many;  // which kernels
    bool whole;                  // a block of rows takes the prefix and the request's own keys in one go
};
// a view that a tensor map can describe
bool mappable(const hk_view& v, int64_t B, int64_t H, int64_t T) { return (B == 1 || v.strideB > 0) && (H == 1 || v.strideH > 0) && (T == 1 || v.strideM > 0); }

Plan make_plan(const hk_shared_prefix_params* p, PrefixArgs& a, bool many) {
    a.B = p->B; a.Hk = p->nh_kv; a.group = p->nh / p->nh_kv; a.T = (int)p->T; a.P = (int)p->prefix_len; a.S = (int)p->kv_len;
    a.R = p->B * a.T * a.group;
    const int own_rows = a.T * a.group, sms = sm_count();
    const ManyPlan mp = many_plan(p->dtype);
    Plan plan{many && a.P > 0 && a.R > 32, many && own_rows > 16, false};
    a.splits_p = a.per_p = a.tiles_p = 0;
    double prefix_time = 0.0;
    if (a.P > 0 && plan.prefix_many) {
        // as many runs as make the waves of CTAs shortest, four tiles to start and end one
        a.tiles_p = cdiv(a.R, mp.rows);
        const int64_t items = (int64_t)a.Hk * a.tiles_p;
        const int most = std::min(64, std::max(1, cdiv(a.P, 2 * mp.keys)));
        for (int n = 1; n <= most; ++n) {
            const int tiles = cdiv(cdiv(a.P, n), mp.keys);
            const double time = (double)cdiv(items * n, sms) * (tiles + 4) + 0.25 * n;
            if (n > 1 && time >= prefix_time) continue;
            prefix_time = time;
            a.per_p = tiles * mp.keys;
        }
        a.splits_p = cdiv(a.P, a.per_p);
    } else if (a.P > 0) {
        const FewPlan fp = few_plan(p->dtype, a.R);
        a.tiles_p = cdiv(a.R, fp.rows);
        const int64_t items = (int64_t)a.Hk * a.tiles_p, places = sms * fp.per_sm;
        const int n = (int)std::max<int64_t>(1, std::min<int64_t>({64, places / items, cdiv(a.P, 4 * fp.step)}));
        a.per_p = cdiv(cdiv(a.P, n), fp.step) * fp.step;
        a.splits_p = cdiv(a.P, a.per_p);
    }
    a.splits_o = 1;
    if (plan.own_many) {
        a.tiles_o = cdiv(own_rows, mp.rows);
        const int64_t items = (int64_t)a.B * a.Hk * a.tiles_o;
        // the prefix again for every request, or once and its results through memory: in tiles, as above
        const double whole = (double)cdiv(items, sms) * cdiv(a.P, mp.keys);
        if (a.P > 0 && plan.prefix_many && whole <= prefix_time + 4) {
            plan.whole = true;
            a.splits_p = a.per_p = a.tiles_p = 0;
        }
    } else {
        const FewPlan fo = few_plan(p->dtype, own_rows);
        a.tiles_o = cdiv(own_rows, fo.rows);
        const int64_t items = (int64_t)a.B * a.Hk * a.tiles_o, places = sms * fo.per_sm;
        while (a.splits_o < 8 && items * a.splits_o * 2 <= places && a.splits_o * 2 * 2 * fo.step <= a.S) a.splits_o *= 2;
    }
    return plan;
}
size_t slots(const PrefixArgs& a) { return (size_t)a.splits_p * a.Hk * a.R; }
constexpr size_t SLOT_BYTES = 64 * sizeof(float) + sizeof(float2);

}  // namespace
}  // namespace hk

using namespace hk;

extern "C" {

size_t hk_shared_prefix_workspace_bytes(const hk_shared_prefix_params* p) {
    if (check_sizes(p) != HK_OK) return 0;
    PrefixArgs a{};
    size_t n = 0;
    for (bool many : {false, true}) {  // by sizes alone: whichever the views allow
        make_plan(p, a, many);
        n = std::max(n, slots(a));
    }
    return n * SLOT_BYTES;
}

int hk_shared_prefix_attention(const hk_shared_prefix_params* p, void* stream_) {
    int rc = check(p);
    if (rc != HK_OK) return rc;
    cudaStream_t stream = static_cast<cudaStream_t>(stream_);
    PrefixArgs a{};
    const Plan plan = make_plan(p, a, (p->prefix_len == 0 || (mappable(p->Kp, 1, p->nh_kv, p->prefix_len) && mappable(p->Vp, 1, p->nh_kv, p->prefix_len))) &&
                                          (p->kv_len == 0 || (mappable(p->K, p->B, p->nh_kv, p->kv_len) && mappable(p->V, p->B, p->nh_kv, p->kv_len))));
    const size_t n = slots(a);
    if (n > 0 && (!p->workspace || (reinterpret_cast<uintptr_t>(p->workspace) & 255u) || p->workspace_bytes < n * SLOT_BYTES)) return HK_ERR_WORKSPACE;
    a.part = static_cast<float*>(p->workspace);
    a.ml = reinterpret_cast<float2*>(a.part + n * 64);
    a.Q = p->Q; a.Kp = p->Kp; a.Vp = p->Vp; a.K = p->K; a.V = p->V; a.O = p->O;
    a.LSE = p->LSE; a.lse_sB = p->lse_strideB; a.lse_sH = p->lse_strideH;
    a.lengths = p->lengths;
    a.scale_log2e = std::fabs(p->scale) * LOG2E;
    a.flip = p->scale > 0.f ? 0u : p->dtype == HK_F32 ? 0x80000000u : 0x80008000u;
    a.causal = p->is_causal;
    if (a.splits_p > 0 && (rc = plan.prefix_many ? launch_prefix_many(a, p->dtype, stream) : launch_prefix_few(a, p->dtype, stream))) return rc;
    return plan.own_many ? launch_own_many(a, p->dtype, plan.whole, stream) : launch_own_few(a, p->dtype, stream);
}

}  // extern "C"
