// shared_prefix_few.cu -- attention over a shared prefix where few rows meet a run of keys (decoding): bound by reading keys and
// values.
//
// A warp takes its rows through batches of 8 (fp32) or 16 keys that TMA brings into a ring of its own, two or three batches ahead: no
// barrier between warps until they merge what they have.  (Copies by the lanes themselves, cp.async, kept the load/store unit busy for
// 112 cycles a batch and warp: 64 requests, 32 heads on 8, 8 192 and up to 1 000 keys, bf16, took 37.7 us instead of 30.5, launches
// behind each other.)  A batch of all warps of an SM takes 0.45 us for 16-bit types, 0.65 for 16 rows of fp32, 0.4 for one or two, and
// a CTA 2.2 us beside its batches.  Sixteen requests of 12 heads on 2 047 and up to 512 keys, fp32: 12.0 us with the launch that adds
// up the slots, for 37.8 MB (48 % of the copy rate); four on 333 and up to 64, in one launch: 5.0 us, of which the keys take one.
//   One or two rows in fp32: a half-warp to a key, four elements a lane (RowsOfOne).
//   Up to 16 rows: matrix instructions (m16n8k8 on TF32, m16n8k16 on 16-bit types).  A lane's part of an operand is whatever
// 16-byte pieces it reads, because the order of the contracted index (head dimension, keys) and of the result's columns is free
// as long as both operands agree on it; the order taken makes every read free of bank conflicts in the layout TMA writes (16-byte
// piece c of row r at c ^ (r % 8)).  The instructions on tensor memory would need 128 rows to a tile.
#include <algorithm>
#include <cmath>
#include <mutex>
#include <type_traits>

#include "few_rows.cuh"
#include "shared_prefix.cuh"

namespace hk {
namespace {

constexpr int FEW_WARPS = 4;

// What a CTA takes: a run of the prefix's keys; a run of a request's own, by the keys there are; or the whole prefix and all of the
// request's own, with more warps (small calls, where a second and a third launch would take longer).
enum FewJob { FEW_PREFIX = 0, FEW_OWN = 1, FEW_WHOLE = 2 };
template <class Rows, int JOB>
struct FewShared {
    static constexpr int WARPS = JOB != FEW_WHOLE ? FEW_WARPS : Rows::ROWS < 16 ? 16 : 8, PARTS = WARPS * Rows::PARTS;
    union {
        uint8_t ring[WARPS][Rows::STAGES][4096];  // a batch's keys and values
        float part[PARTS][Rows::ROWS][64 + 4];
    };
    float2 ml[PARTS][Rows::ROWS];
    uint64_t full[WARPS][Rows::STAGES];
    Abort abort;
};

constexpr int W_FEW = 401;

template <class Rows, int JOB>
__device__ __forceinline__ void few_job(const CUtensorMap& map_kp, const CUtensorMap& map_vp, const CUtensorMap& map_k, const CUtensorMap& map_v, const PrefixArgs& a,
                                        const int block, const bool late) {
    typedef typename Rows::X X;
    typedef FewShared<Rows, JOB> Shared;
    constexpr bool OWN = JOB != FEW_PREFIX;
    constexpr int N = Rows::ROWS, KEYS = Rows::KEYS, WARPS = Shared::WARPS, MINE = N < 16 ? N : 2;  // rows that a lane works on
    extern __shared__ __align__(1024) uint8_t few_smem[];
    Shared& sh = *reinterpret_cast<Shared*>(few_smem);
    const int warp = (int)uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (lane == 0) {
        for (int s = 0; s < Rows::STAGES; ++s) mbar_init(&sh.full[warp][s], 1);
        if (warp == 0) sh.abort.id = 0;
        fence_mbar_init();
    }
    if (!late) pdl_wait();
    pdl_trigger();
    // the rows
    const int ns = JOB == FEW_PREFIX ? a.splits_p : JOB == FEW_OWN ? a.splits_o : 1, item = block / ns, split = block - item * ns;
    const int tiles = OWN ? a.tiles_o : a.tiles_p, at = item / tiles, tile = item - at * tiles;
    const int b = OWN ? at / a.Hk : 0, kvh = at - b * a.Hk;
    const int len = OWN ? request_keys(a, b) : 0;
    const int all = OWN ? a.T * a.group : a.R, row0 = b * a.T * a.group + tile * N, rows = min(N, all - tile * N);
    typename Rows::Query query;
    int token_of[MINE];
#pragma unroll
    for (int i = 0; i < MINE; ++i) {
        const int r = Rows::row(i, lane), row = row0 + r, token = row / a.group, bq = OWN ? b : token / a.T;
        token_of[i] = r < rows ? token - bq * a.T : a.T;
        query.load(i, r < rows ? row_of<X>(a.Q, bq, kvh * a.group + (row - token * a.group), token_of[i]) : nullptr, lane, late);
    }
    // the keys: batches of the prefix, then of the request's own
    int p_begin = 0, p_end = 0, o_begin = 0, o_end = 0;
    if (JOB == FEW_PREFIX) {
        p_begin = split * a.per_p;
        p_end = min(a.P, p_begin + a.per_p);
    } else {
        const int seen = token_keys(a, len, (tile * N + rows - 1) / a.group), per = ((seen + ns - 1) / ns + KEYS - 1) / KEYS * KEYS;
        o_begin = min(seen, split * per);
        o_end = min(seen, o_begin + per);
        if (JOB == FEW_WHOLE) p_end = a.P;
    }
    const int n_p = (p_end - p_begin + KEYS - 1) / KEYS, n = n_p + (o_end - o_begin + KEYS - 1) / KEYS;
    auto key_of = [&](int i) { return i < n_p ? p_begin + i * KEYS : o_begin + (i - n_p) * KEYS; };
    int put = 0, put_at = warp;
    auto copy_next = [&] {  // the next batch of this warp, if there is one, into the slot that its lanes have read
        __syncwarp();
        if (put_at < n && lane == 0) {
            const bool own = JOB == FEW_OWN || (JOB == FEW_WHOLE && put_at >= n_p);
            uint64_t* full = &sh.full[warp][put];
            uint8_t* to = sh.ring[warp][put];
            mbar_arrive_expect_tx(full, 4096);
            tma_load_tile(to, own ? &map_k : &map_kp, full, key_of(put_at), kvh, own ? b : 0);
            tma_load_tile(to + 2048, own ? &map_v : &map_vp, full, key_of(put_at), kvh, own ? b : 0);
        }
        put_at += WARPS;
        put = put + 1 == Rows::STAGES ? 0 : put + 1;
    };
#pragma unroll
    for (int i = 0; i < Rows::STAGES - 1; ++i) copy_next();
    Rows w;
    w.start(query, a.flip);
    int limit[MINE];
#pragma unroll
    for (int i = 0; i < MINE; ++i) limit[i] = OWN && token_of[i] < a.T ? min(o_end, token_keys(a, len, token_of[i])) : o_end;
    __syncthreads();  // the record of waits that gave up
    WaitNote wc{&sh.abort};
    int get = 0;
    uint32_t phase = 0;
    for (int i = warp; i < n; i += WARPS) {
        if (!__all_sync(0xffffffffu, mbar_wait(wc, &sh.full[warp][get], phase, W_FEW, i))) {
            for (const unsigned long long t0 = globaltimer_ns(); globaltimer_ns() - t0 < 100000ull;) {}  // copies in flight land
            break;
        }
        const uint8_t* from = sh.ring[warp][get];
        if (++get == Rows::STAGES) get = 0, phase ^= 1u;
        const bool own = JOB == FEW_OWN || (JOB == FEW_WHOLE && i >= n_p);
        const int key0 = key_of(i), end = own ? o_end : p_end;
        int last[MINE], least = end;
#pragma unroll
        for (int k = 0; k < MINE; ++k) {
            last[k] = own ? limit[k] : end;
            least = min(least, last[k]);
        }
        w.batch(from, lane, key0, end, key0 + KEYS <= least, [&](int k, int key) { return key < last[k]; }, a.scale_log2e, copy_next);
    }
    const int64_t slot0 = (int64_t)kvh * a.R + row0, slot_rows = a.slot_rows;
    __syncthreads();  // the ring is the warps' exchange now: every copy has been waited for
    w.finish(sh.part, sh.ml, warp, lane);
    __syncthreads();
    // PER threads a row, 64 / PER elements each
    constexpr int PER = N < 16 ? 16 : 8, E = 64 / PER;
    const int r = threadIdx.x / PER, d = threadIdx.x % PER * E;
    const bool mine = r < rows;
    float M = -INFINITY, L = 0.f, acc[E];
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = 0.f;
    if (mine) {
#pragma unroll
        for (int p = 0; p < Shared::PARTS; ++p) M = fmaxf(M, sh.ml[p][r].x);
        const float ref = M == -INFINITY ? 0.f : M;
#pragma unroll
        for (int p = 0; p < Shared::PARTS; ++p) {
            const float f = ex2_approx(sh.ml[p][r].x - ref);
            L += sh.ml[p][r].y * f;
#pragma unroll
            for (int e = 0; e < E; ++e) acc[e] = fmaf(sh.part[p][r][d + e], f, acc[e]);
        }
    }
    if (threadIdx.x == 0) report_abort(sh.abort, a.status);
    if (mine && JOB != FEW_WHOLE && a.slots > 1) {
        const int64_t to = (OWN ? a.splits_p + split : split) * slot_rows + slot0 + r;
        if (d == 0) a.ml[to] = make_float2(M, L);
#pragma unroll
        for (int e = 0; e < E; e += 4) *reinterpret_cast<float4*>(a.part + to * 64 + d + e) = make_float4(acc[e], acc[e + 1], acc[e + 2], acc[e + 3]);
    } else if (mine) {
        const float f = L != 0.f ? 1.f / L : 0.f;
        const int row = row0 + r, token = row / a.group, bq = OWN ? b : token / a.T, t = token - bq * a.T, h = kvh * a.group + (row - token * a.group);
        X* to = const_cast<X*>(row_of<X>(a.O, bq, h, t)) + d;
#pragma unroll
        for (int e = 0; e < E; e += 4) store4(to + e, make_float4(acc[e] * f, acc[e + 1] * f, acc[e + 2] * f, acc[e + 3] * f));
        if (d == 0) a.LSE[bq * a.lse_sB + h * a.lse_sH + t] = L != 0.f ? (M + log2f(L)) * LN2 : -INFINITY;
    }
}

// late: runs beside the kernel over the prefix.  What was before that is complete when this one begins, and this one when that is.
template <class Rows, int JOB>
__global__ void __launch_bounds__(FewShared<Rows, JOB>::WARPS * 32, JOB == FEW_WHOLE ? 1 : Rows::CTAS)
prefix_few_kernel(const __grid_constant__ CUtensorMap map_kp, const __grid_constant__ CUtensorMap map_vp, const __grid_constant__ CUtensorMap map_k,
                  const __grid_constant__ CUtensorMap map_v, const __grid_constant__ PrefixArgs a) {
    const bool late = JOB == FEW_OWN && a.splits_p > 0;
    few_job<Rows, JOB>(map_kp, map_vp, map_k, map_v, a, blockIdx.x, late);
    if (late && blockIdx.x == gridDim.x - 1) pdl_wait();
}
// The runs of the prefix and those of the requests' own keys in one launch.
template <class Prefix, class Own>
__global__ void __launch_bounds__(FEW_WARPS * 32, Prefix::CTAS < Own::CTAS ? Prefix::CTAS : Own::CTAS)
prefix_few_both_kernel(const __grid_constant__ CUtensorMap map_kp, const __grid_constant__ CUtensorMap map_vp, const __grid_constant__ CUtensorMap map_k,
                       const __grid_constant__ CUtensorMap map_v, const __grid_constant__ PrefixArgs a) {
    const int n = a.Hk * a.tiles_p * a.splits_p;
    if ((int)blockIdx.x < n) few_job<Prefix, FEW_PREFIX>(map_kp, map_vp, map_k, map_v, a, blockIdx.x, false);
    else few_job<Own, FEW_OWN>(map_kp, map_vp, map_k, map_v, a, blockIdx.x - n, false);
}

typedef void (*FewKernel)(CUtensorMap, CUtensorMap, CUtensorMap, CUtensorMap, PrefixArgs);
struct FewEntry {
    FewKernel kernel;
    size_t smem;
    int threads;
};
template <class Rows, int JOB>
FewEntry entry() {
    return {prefix_few_kernel<Rows, JOB>, sizeof(FewShared<Rows, JOB>), FewShared<Rows, JOB>::WARPS * 32};
}
template <int JOB>
FewEntry pick(int dtype, int rows) {
    if (dtype == HK_BF16) return entry<RowsOf16<__nv_bfloat16>, JOB>();
    if (dtype == HK_F16) return entry<RowsOf16<__half>, JOB>();
    return rows == 1 ? entry<RowsOfOne<1>, JOB>() : rows == 2 ? entry<RowsOfOne<2>, JOB>() : entry<RowsOf16<float>, JOB>();
}

template <class Prefix, class Own>
FewEntry both() {
    return {prefix_few_both_kernel<Prefix, Own>, std::max(sizeof(FewShared<Prefix, FEW_PREFIX>), sizeof(FewShared<Own, FEW_OWN>)), FEW_WARPS * 32};
}
FewEntry pick_both(int dtype, int prefix, int own) {  // rows of a tile: own <= prefix
    if (dtype == HK_BF16) return both<RowsOf16<__nv_bfloat16>, RowsOf16<__nv_bfloat16>>();
    if (dtype == HK_F16) return both<RowsOf16<__half>, RowsOf16<__half>>();
    if (prefix == 1) return both<RowsOfOne<1>, RowsOfOne<1>>();
    if (prefix == 2) return own == 1 ? both<RowsOfOne<2>, RowsOfOne<1>>() : both<RowsOfOne<2>, RowsOfOne<2>>();
    return own == 1 ? both<RowsOf16<float>, RowsOfOne<1>>() : own == 2 ? both<RowsOf16<float>, RowsOfOne<2>>() : both<RowsOf16<float>, RowsOf16<float>>();
}

int launch(const FewEntry& k, const PrefixArgs& a, int dtype, bool prefix, bool own, int64_t blocks, cudaStream_t stream) {
    // once per device and kernel: more than 48 KB of shared memory
    static std::mutex mu;
    static FewKernel known[HK_MAX_DEVICES][32];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= HK_MAX_DEVICES) return HK_ERR_CUDA;
    {
        std::lock_guard<std::mutex> lock(mu);
        for (FewKernel& x : known[dev]) {
            if (x == k.kernel) break;
            if (x) continue;
            if (cudaFuncSetAttribute(k.kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)k.smem) != cudaSuccess) return check_launch();
            x = k.kernel;
            break;
        }
    }
    if (blocks > 0x7fffffffLL) return HK_ERR_BAD_SHAPE;
    LaunchConfig lc((unsigned)blocks, k.threads, k.smem, stream, 1, true);
    CUtensorMap kp, vp, mk, mv;
    const int rows = few_plan(dtype, 16).step / FEW_WARPS;
    int rc;
    if ((rc = prefix_tile_map(&kp, a.Kp, dtype, 1, a.Hk, prefix ? a.P : 0, rows, false)) || (rc = prefix_tile_map(&vp, a.Vp, dtype, 1, a.Hk, prefix ? a.P : 0, rows, false)) ||
        (rc = prefix_tile_map(&mk, a.K, dtype, a.B, a.Hk, own ? a.S : 0, rows, false)) || (rc = prefix_tile_map(&mv, a.V, dtype, a.B, a.Hk, own ? a.S : 0, rows, false)))
        return rc;
    if (cudaLaunchKernelEx(&lc.cfg, k.kernel, kp, vp, mk, mv, a) != cudaSuccess) return check_launch();
    count_launch();
    return HK_OK;
}

}  // namespace

FewPlan few_plan(int dtype, int rows) {
    if (dtype != HK_F32) return {16, FEW_WARPS * 16, RowsOf16<__half>::CTAS};
    return {rows <= 2 ? rows : 16, FEW_WARPS * 8, rows <= 2 ? RowsOfOne<1>::CTAS : RowsOf16<float>::CTAS};
}
int launch_prefix_few(const PrefixArgs& a, int dtype, cudaStream_t stream) {
    return launch(pick<FEW_PREFIX>(dtype, few_plan(dtype, a.R).rows), a, dtype, true, false, (int64_t)a.Hk * a.tiles_p * a.splits_p, stream);
}
int launch_own_few(const PrefixArgs& a, int dtype, cudaStream_t stream) {
    const int rows = few_plan(dtype, a.T * a.group).rows;
    if (a.whole) return launch(pick<FEW_WHOLE>(dtype, rows), a, dtype, true, true, (int64_t)a.B * a.Hk * a.tiles_o, stream);
    return launch(pick<FEW_OWN>(dtype, rows), a, dtype, false, true, (int64_t)a.B * a.Hk * a.tiles_o * a.splits_o, stream);
}
int launch_both_few(const PrefixArgs& a, int dtype, cudaStream_t stream) {
    return launch(pick_both(dtype, few_plan(dtype, a.R).rows, few_plan(dtype, a.T * a.group).rows), a, dtype, true, true,
                  (int64_t)a.Hk * a.tiles_p * a.splits_p + (int64_t)a.B * a.Hk * a.tiles_o * a.splits_o, stream);
}

}  // namespace hk
