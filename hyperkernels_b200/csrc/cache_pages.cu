// cache_pages.cu -- what happens to a cache's pages between the attention calls (include/hk_attention.h): rows of new tokens are
// appended (hk_cache_append), requests are continued, forked and freed (hk_cache_fork), the pages in use come to the front of the pools
// (hk_cache_compact).
//
// Elements are copied as they are, whatever their type.
#include <climits>

#include "cache_pages.cuh"

namespace hk {
namespace {

__device__ __forceinline__ bool is_page(int e, int n_pages) { return (unsigned)e < (unsigned)n_pages; }

// ---------------------------------------------------------------------------
// Rows of new tokens into the pages: a warp to a token, 16 bytes to a lane, all heads of keys and values.
// ---------------------------------------------------------------------------
struct AppendArgs {
    hk_pool pool;
    hk_view K, V;
    const int32_t *lengths, *starts, *picks, *counts;
    int B, Hk, T, esize;
};

template <int PIECES>  // of 16 bytes in a row
__global__ void __launch_bounds__(256) append_kernel(const __grid_constant__ AppendArgs a) {
    pdl_wait();
    pdl_trigger();
    const int lane = threadIdx.x & 31;
    const int64_t item = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    int b, row;  // the row of K and V, and of which batch
    int64_t pos, from_b;
    if (a.starts) {
        if (item >= a.T) return;
        row = (int)item;
        b = sequence_of(a.starts, a.B, row, lane);
        if (b >= a.B || a.starts[b] > row) return;
        pos = (int64_t)row - a.starts[b];
        from_b = 0;
    } else {
        if (item >= (int64_t)a.B * a.T) return;
        b = (int)(item / a.T);
        const int k = (int)(item - (int64_t)b * a.T);
        if (a.counts && k >= a.counts[b]) return;
        row = a.picks ? a.picks[item] : k;
        if ((unsigned)row >= (unsigned)a.T) return;
        pos = k;
        from_b = b;
    }
    pos += max(a.lengths[b], 0);
    const int64_t at = pos / a.pool.page;
    if (at >= a.pool.width) return;
    const int page = a.pool.pages[b * a.pool.pages_stride + at];
    if (!is_page(page, a.pool.n_pages)) return;
    const int64_t in_page = pos - at * a.pool.page, e = a.esize;
    const char *k = static_cast<const char*>(a.K.ptr) + (from_b * a.K.strideB + row * a.K.strideM) * e,
               *v = static_cast<const char*>(a.V.ptr) + (from_b * a.V.strideB + row * a.V.strideM) * e;
    char *kp = static_cast<char*>(a.pool.K.ptr) + (page * a.pool.K.strideB + in_page * a.pool.K.strideM) * e,
         *vp = static_cast<char*>(a.pool.V.ptr) + (page * a.pool.V.strideB + in_page * a.pool.V.strideM) * e;
    constexpr int HEADS = 32 / PIECES, RUN = 4;
    for (int h0 = lane / PIECES; h0 < a.Hk; h0 += HEADS * RUN) {
        uint4 x[RUN], y[RUN];
#pragma unroll
        for (int i = 0; i < RUN; ++i) {
            const int64_t h = h0 + i * HEADS;
            if (h >= a.Hk) break;
            x[i] = reinterpret_cast<const uint4*>(k + h * a.K.strideH * e)[lane % PIECES];
            y[i] = reinterpret_cast<const uint4*>(v + h * a.V.strideH * e)[lane % PIECES];
        }
#pragma unroll
        for (int i = 0; i < RUN; ++i) {
            const int64_t h = h0 + i * HEADS;
            if (h >= a.Hk) break;
            reinterpret_cast<uint4*>(kp + h * a.pool.K.strideH * e)[lane % PIECES] = x[i];
            reinterpret_cast<uint4*>(vp + h * a.pool.V.strideH * e)[lane % PIECES] = y[i];
        }
    }
}

// ---------------------------------------------------------------------------
// Copies of pages, of the first `rows` rows of every head in every layer, and the table's new entries.
// ---------------------------------------------------------------------------
struct Pair {
    int from, to, rows, pad;
};
struct CopyArgs {
    hk_pool pool;
    int64_t k_strideL, v_strideL;
    int layers, Hk, esize, parts;
    const Pair* pairs;
    const int* n_pairs;
    const int32_t* where;  // compaction: the pages' new places
    int32_t* pages_out;
    int B;
};

template <int PIECES>
__global__ void __launch_bounds__(256) copy_pages_kernel(const __grid_constant__ CopyArgs a) {
    constexpr int ROWS = 32 / PIECES, RUN = 8;  // rows that a warp copies at once, and how often
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    pdl_wait();
    pdl_trigger();
    if (a.where) {
        for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < (int64_t)a.B * a.pool.width; i += (int64_t)gridDim.x * 256) {
            const int64_t b = i / a.pool.width;
            const int e = a.pool.pages[b * a.pool.pages_stride + (i - b * a.pool.width)];
            a.pages_out[i] = is_page(e, a.pool.n_pages) ? a.where[e] : -1;
        }
    }
    const int64_t items = (int64_t)*a.n_pairs * a.layers * 2 * a.parts, e = a.esize;
    for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
        const int part = (int)(item % a.parts), kv = (int)(item / a.parts & 1), layer = (int)(item / a.parts / 2 % a.layers);
        const Pair pair = a.pairs[item / a.parts / 2 / a.layers];
        const hk_view& v = kv ? a.pool.V : a.pool.K;
        // rows of the page in the order they lie in
        const bool by_token = v.strideH < v.strideM;
        const int inner = by_token ? a.Hk : pair.rows, all = a.Hk * pair.rows;
        const int64_t s_in = by_token ? v.strideH : v.strideM, s_out = by_token ? v.strideM : v.strideH;
        const char* base = static_cast<const char*>(v.ptr) + layer * (kv ? a.v_strideL : a.k_strideL) * e + lane % PIECES * 16;
        const char* from = base + pair.from * v.strideB * e;
        char* to = const_cast<char*>(base) + pair.to * v.strideB * e;
        const int first = (part * 8 + warp) * ROWS * RUN + lane / PIECES;
        uint4 x[RUN];
        int64_t at[RUN];
#pragma unroll
        for (int i = 0; i < RUN; ++i) {
            const int r = first + i * ROWS, outer = r / inner;
            at[i] = (outer * s_out + (r - outer * inner) * s_in) * e;
            if (r < all) x[i] = *reinterpret_cast<const uint4*>(from + at[i]);
        }
#pragma unroll
        for (int i = 0; i < RUN; ++i)
            if (first + i * ROWS < all) *reinterpret_cast<uint4*>(to + at[i]) = x[i];
    }
}
int parts_of(int Hk, int page, int esize) { return cdiv((int64_t)Hk * page, 8 * (esize == 4 ? 2 : 4) * 8); }

// ---------------------------------------------------------------------------
// Tables: one CTA, since every step needs all of the one before.
// ---------------------------------------------------------------------------
constexpr int THREADS = 1024;

// Sum of x over the threads in front of this one, and of all
struct Sums {
    int warp[32];
};
__device__ __forceinline__ int block_scan(Sums& sh, int x, int& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int s = x;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, s, off);
        if (lane >= off) s += y;
    }
    __syncthreads();
    if (lane == 31) sh.warp[warp] = s;
    __syncthreads();
    int w = lane < blockDim.x / 32 ? sh.warp[lane] : 0;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, w, off);
        if (lane >= off) w += y;
    }
    total = __shfl_sync(0xffffffffu, w, 31);
    return s - x + (warp ? __shfl_sync(0xffffffffu, w, warp - 1) : 0);
}

struct Request {  // of the new batch
    int source;   // row of the old table, -1: none
    int kept;     // pages it has
    int need;     // pages up to where it has room
    int first;    // number of its first new page
};
struct ForkArgs {
    hk_pool pool;
    const int32_t *lengths, *users, *source, *room;
    int32_t *pages_out, *lengths_out, *users_out, *missing;
    int B, B_out;
    int64_t room_all;
    int* owner;    // [B]: the first of the new batch that goes on with a request
    Request* request;  // [B_out]
    int* free;     // [n_pages]
    Pair* pairs;   // [B_out]
    int* n_pairs;
};

__global__ void __launch_bounds__(THREADS) fork_kernel(const __grid_constant__ ForkArgs a) {
    __shared__ Sums sums;
    __shared__ int lacking, n_pairs;
    const int tid = threadIdx.x, M = a.pool.width, P = a.pool.n_pages;
    pdl_wait();
    pdl_trigger();
    if (tid == 0) lacking = n_pairs = 0;
    for (int p = tid; p < P; p += THREADS) a.users_out[p] = a.users[p];
    for (int b = tid; b < a.B; b += THREADS) a.owner[b] = INT_MAX;
    __syncthreads();
    // what the old table held is nobody's, and who goes on with a request first
    for (int64_t i = tid; i < (int64_t)a.B * M; i += THREADS) {
        const int64_t b = i / M;
        const int e = a.pool.pages[b * a.pool.pages_stride + (i - b * M)];
        if (is_page(e, P)) atomicSub(a.users_out + e, 1);
    }
    for (int i = tid; i < a.B_out; i += THREADS)
        if ((unsigned)a.source[i] < (unsigned)a.B) atomicMin(a.owner + a.source[i], i);
    __syncthreads();
    int given = 0;
    for (int i0 = 0; i0 < a.B_out; i0 += THREADS) {
        const int i = i0 + tid;
        Request r = {-1, 0, 0, 0};
        int len = 0;
        if (i < a.B_out) {
            const int s = a.source[i];
            if ((unsigned)s < (unsigned)a.B) {
                r.source = s;
                len = (int)min((int64_t)max(a.lengths[s], 0), (int64_t)M * a.pool.page);
                r.kept = len / a.pool.page + (len % a.pool.page && a.owner[s] == i);
            }
            const int64_t need = (len + (a.room ? (int64_t)max(a.room[i], 0) : a.room_all) + a.pool.page - 1) / a.pool.page;
            r.need = (int)max((int64_t)r.kept, min(need, (int64_t)M));
            if (need > M) atomicAdd(&lacking, (int)min(need - M, (int64_t)1 << 20));
        }
        int total;
        r.first = given + block_scan(sums, r.need - r.kept, total);
        given += total;
        if (i < a.B_out) {
            a.lengths_out[i] = len;
            a.request[i] = r;
        }
    }
    __syncthreads();
    // pages that are kept
    for (int64_t k = tid; k < (int64_t)a.B_out * M; k += THREADS) {
        const int i = (int)(k / M), j = (int)(k - (int64_t)i * M);
        const Request r = a.request[i];
        int e = -1;
        if (j < r.kept) {
            e = a.pool.pages[r.source * a.pool.pages_stride + j];
            if (is_page(e, P)) atomicAdd(a.users_out + e, 1);
            else e = -1;
        }
        a.pages_out[k] = e;
    }
    __syncthreads();
    // the free ones in their order
    const int each = (P + THREADS - 1) / THREADS, p0 = min(P, tid * each), p1 = min(P, p0 + each);
    int n = 0, n_free;
    for (int p = p0; p < p1; ++p) n += a.users_out[p] == 0;
    n = block_scan(sums, n, n_free);
    for (int p = p0; p < p1; ++p)
        if (a.users_out[p] == 0) a.free[n++] = p;
    __syncthreads();
    for (int64_t k = tid; k < (int64_t)a.B_out * M; k += THREADS) {
        const int i = (int)(k / M), j = (int)(k - (int64_t)i * M);
        const Request r = a.request[i];
        if (j < r.kept || j >= r.need) continue;
        const int f = r.first + j - r.kept, page = f < n_free ? a.free[f] : -1;
        a.pages_out[k] = page;
        if (page >= 0) a.users_out[page] = 1;
        const int len = a.lengths_out[i], rows = len % a.pool.page;
        if (page >= 0 && j == len / a.pool.page && rows) {  // a begun page of which another has the original
            const int from = a.pool.pages[r.source * a.pool.pages_stride + j];
            if (is_page(from, P)) a.pairs[atomicAdd(&n_pairs, 1)] = {from, page, rows, 0};
        }
    }
    __syncthreads();
    if (tid == 0) {
        *a.missing = lacking + max(0, given - n_free);
        *a.n_pairs = n_pairs;
    }
}

struct CompactArgs {
    const int32_t* users;
    int32_t *users_out, *where;
    int P, page;
    int* hole;    // [n_pages]
    Pair* pairs;  // [n_pages / 2 + 1]
    int* n_pairs;
};
__global__ void __launch_bounds__(THREADS) compact_kernel(const __grid_constant__ CompactArgs a) {
    __shared__ Sums sums;
    const int tid = threadIdx.x, P = a.P, each = (P + THREADS - 1) / THREADS, p0 = min(P, tid * each), p1 = min(P, p0 + each);
    pdl_wait();
    pdl_trigger();
    int used = 0, n, holes = 0, moves = 0, n_holes, n_moves;
    for (int p = p0; p < p1; ++p) used += a.users[p] > 0;
    block_scan(sums, used, n);
    for (int p = p0; p < p1; ++p) {
        const bool u = a.users[p] > 0;
        holes += !u && p < n;
        moves += u && p >= n;
    }
    holes = block_scan(sums, holes, n_holes);
    moves = block_scan(sums, moves, n_moves);  // as many
    for (int p = p0; p < p1; ++p) {
        const int u = a.users[p];
        if (p < n && u <= 0) a.hole[holes++] = p;
        if (p >= n && u > 0) a.pairs[moves++].from = p;
        if (p >= n) a.users_out[p] = 0;
        else if (u > 0) a.users_out[p] = u;
        a.where[p] = u > 0 && p < n ? p : -1;
    }
    __syncthreads();
    for (int k = tid; k < n_moves; k += THREADS) {
        const int from = a.pairs[k].from, to = a.hole[k];
        a.pairs[k] = {from, to, a.page, 0};
        a.where[from] = to;
        a.users_out[to] = a.users[from];
    }
    if (tid == 0) *a.n_pairs = n_moves;
}

size_t up(size_t n) { return (n + 255) / 256 * 256; }

int launch_copy(const CopyArgs& a, int64_t most_pairs, cudaStream_t stream) {
    const int64_t items = std::max<int64_t>(1, most_pairs * a.layers * 2 * a.parts);
    LaunchConfig lc((unsigned)std::min<int64_t>(items, (int64_t)sm_count() * 8), 256, 0, stream, 1, true);
    if (cudaLaunchKernelEx(&lc.cfg, a.esize == 4 ? copy_pages_kernel<16> : copy_pages_kernel<8>, a) != cudaSuccess) return check_launch();
    count_launch();
    return HK_OK;
}

// Pools of several layers: the pages of all of them lie apart.
int check_layers(const hk_pool& pool, int64_t kL, int64_t vL, int layers, int nh_kv, int dtype) {
    for (int i = 0; i < 2; ++i) {
        const hk_view& v = i ? pool.V : pool.K;
        const int64_t sL = i ? vL : kL;
        if (layers > 1 && (sL < 0 || sL % (16 / esize(dtype)))) return HK_ERR_MISALIGNED;
        Dim d[] = {{layers, sL}, {pool.n_pages, v.strideB}, {pool.page, v.strideM}, {nh_kv, v.strideH}};
        if (!lie_apart(d, HEAD_DIM)) return HK_ERR_UNSUPPORTED;
    }
    return HK_OK;
}
int check_fork_sizes(const hk_fork_params* p) {
    if (!p) return HK_ERR_NULL_POINTER;
    if (p->B <= 0 || p->B_out <= 0 || p->layers <= 0 || p->layers > (1 << 20) || p->room_all < 0 || p->room_all > (1 << 30)) return HK_ERR_BAD_SHAPE;
    return check_pool_sizes(p->pool, std::max(p->B, p->B_out), p->nh_kv, p->dtype);
}
struct ForkSpace {
    size_t owner, request, free, pairs, n_pairs, bytes;
    explicit ForkSpace(const hk_fork_params* p) {
        owner = 0;
        request = owner + up(sizeof(int) * p->B);
        free = request + up(sizeof(Request) * p->B_out);
        pairs = free + up(sizeof(int) * p->pool.n_pages);
        n_pairs = pairs + up(sizeof(Pair) * p->B_out);
        bytes = n_pairs + 256;
    }
};
int check_compact_sizes(const hk_compact_params* p) {
    if (!p) return HK_ERR_NULL_POINTER;
    if (p->B <= 0 || p->layers <= 0 || p->layers > (1 << 20)) return HK_ERR_BAD_SHAPE;
    return check_pool_sizes(p->pool, p->B, p->nh_kv, p->dtype);
}
struct CompactSpace {
    size_t hole, pairs, n_pairs, bytes;
    explicit CompactSpace(const hk_compact_params* p) {
        hole = 0;
        pairs = up(sizeof(int) * p->pool.n_pages);
        n_pairs = pairs + up(sizeof(Pair) * (p->pool.n_pages / 2 + 1));
        bytes = n_pairs + 256;
    }
};
bool workspace_fits(const void* ws, size_t have, size_t need) { return ws && !(reinterpret_cast<uintptr_t>(ws) & 255u) && have >= need; }
bool odd(std::initializer_list<const void*> ints) {
    for (const void* x : ints)
        if (reinterpret_cast<uintptr_t>(x) & 3u) return true;
    return false;
}

}  // namespace

int check_pool_sizes(const hk_pool& pool, int64_t B, int nh_kv, int dtype) {
    if (dtype < HK_F32 || dtype > HK_F16) return HK_ERR_UNSUPPORTED;
    if (nh_kv <= 0 || nh_kv > (1 << 20) || pool.n_pages <= 0 || pool.n_pages > (1 << 28) || pool.page <= 0 || pool.page > (1 << 20) || pool.width <= 0) return HK_ERR_BAD_SHAPE;
    if (pool.page % 16) return HK_ERR_UNSUPPORTED;
    if ((int64_t)pool.width * pool.page > (1 << 30) || B * pool.width > (1LL << 30) || (int64_t)nh_kv * pool.page > (1 << 28)) return HK_ERR_BAD_SHAPE;
    return HK_OK;
}
int check_pool(const hk_pool& pool, int64_t B, int nh_kv, int dtype, bool written) {
    int rc = check_pool_sizes(pool, B, nh_kv, dtype);
    if (rc != HK_OK) return rc;
    if ((rc = check_view(pool.K, pool.n_pages, nh_kv, pool.page, dtype, written)) || (rc = check_view(pool.V, pool.n_pages, nh_kv, pool.page, dtype, written))) return rc;
    if (!pool.pages) return HK_ERR_NULL_POINTER;
    if (odd({pool.pages})) return HK_ERR_MISALIGNED;
    return pool.pages_stride < 0 ? HK_ERR_BAD_SHAPE : HK_OK;
}

}  // namespace hk

using namespace hk;

extern "C" {

int hk_cache_append(const hk_append_params* p, void* stream) {
    if (!p) return HK_ERR_NULL_POINTER;
    if (p->B <= 0 || p->B > (1 << 24) || p->T <= 0 || p->T > (1 << 30) || (int64_t)p->B * (p->starts ? 1 : p->T) > (1LL << 30)) return HK_ERR_BAD_SHAPE;
    int rc = check_pool(p->pool, p->B, p->nh_kv, p->dtype, true);
    if (rc != HK_OK) return rc;
    const int64_t B = p->starts ? 1 : p->B;
    if ((rc = check_view(p->K, B, p->nh_kv, p->T, p->dtype, false)) || (rc = check_view(p->V, B, p->nh_kv, p->T, p->dtype, false))) return rc;
    if (!p->lengths) return HK_ERR_NULL_POINTER;
    if (p->starts && (p->picks || p->counts)) return HK_ERR_UNSUPPORTED;
    if (odd({p->lengths, p->starts, p->picks, p->counts})) return HK_ERR_MISALIGNED;
    const AppendArgs a{p->pool, p->K, p->V, p->lengths, p->starts, p->picks, p->counts, p->B, p->nh_kv, (int)p->T, esize(p->dtype)};
    LaunchConfig lc((unsigned)cdiv(B * p->T, 8), 256, 0, static_cast<cudaStream_t>(stream), 1, true);
    if (cudaLaunchKernelEx(&lc.cfg, a.esize == 4 ? append_kernel<16> : append_kernel<8>, a) != cudaSuccess) return check_launch();
    count_launch();
    return HK_OK;
}

size_t hk_cache_fork_workspace_bytes(const hk_fork_params* p) { return check_fork_sizes(p) == HK_OK ? ForkSpace(p).bytes : 0; }

int hk_cache_fork(const hk_fork_params* p, void* stream_) {
    int rc = check_fork_sizes(p);
    if (rc != HK_OK) return rc;
    if ((rc = check_pool(p->pool, std::max(p->B, p->B_out), p->nh_kv, p->dtype, true)) || (rc = check_layers(p->pool, p->k_strideL, p->v_strideL, p->layers, p->nh_kv, p->dtype))) return rc;
    if (!p->lengths || !p->users || !p->source || !p->pages_out || !p->lengths_out || !p->users_out || !p->missing) return HK_ERR_NULL_POINTER;
    if (odd({p->lengths, p->users, p->source, p->room, p->pages_out, p->lengths_out, p->users_out, p->missing})) return HK_ERR_MISALIGNED;
    const ForkSpace at(p);
    if (!workspace_fits(p->workspace, p->workspace_bytes, at.bytes)) return HK_ERR_WORKSPACE;
    cudaStream_t stream = static_cast<cudaStream_t>(stream_);
    char* ws = static_cast<char*>(p->workspace);
    const ForkArgs a{p->pool, p->lengths, p->users, p->source, p->room, p->pages_out, p->lengths_out, p->users_out, p->missing, p->B, p->B_out, p->room_all,
                     reinterpret_cast<int*>(ws + at.owner), reinterpret_cast<Request*>(ws + at.request), reinterpret_cast<int*>(ws + at.free),
                     reinterpret_cast<Pair*>(ws + at.pairs), reinterpret_cast<int*>(ws + at.n_pairs)};
    LaunchConfig lc(1, THREADS, 0, stream, 1, true);
    if (cudaLaunchKernelEx(&lc.cfg, fork_kernel, a) != cudaSuccess) return check_launch();
    count_launch();
    const int e = esize(p->dtype);
    return launch_copy(CopyArgs{p->pool, p->k_strideL, p->v_strideL, p->layers, p->nh_kv, e, parts_of(p->nh_kv, p->pool.page, e), a.pairs, a.n_pairs, nullptr, nullptr, 0}, p->B_out, stream);
}

size_t hk_cache_compact_workspace_bytes(const hk_compact_params* p) { return check_compact_sizes(p) == HK_OK ? CompactSpace(p).bytes : 0; }

int hk_cache_compact(const hk_compact_params* p, void* stream_) {
    int rc = check_compact_sizes(p);
    if (rc != HK_OK) return rc;
    if ((rc = check_pool(p->pool, p->B, p->nh_kv, p->dtype, true)) || (rc = check_layers(p->pool, p->k_strideL, p->v_strideL, p->layers, p->nh_kv, p->dtype))) return rc;
    if (!p->users || !p->pages_out || !p->users_out || !p->where) return HK_ERR_NULL_POINTER;
    if (odd({p->users, p->pages_out, p->users_out, p->where})) return HK_ERR_MISALIGNED;
    const CompactSpace at(p);
    if (!workspace_fits(p->workspace, p->workspace_bytes, at.bytes)) return HK_ERR_WORKSPACE;
    cudaStream_t stream = static_cast<cudaStream_t>(stream_);
    char* ws = static_cast<char*>(p->workspace);
    const CompactArgs a{p->users, p->users_out, p->where, p->pool.n_pages, p->pool.page, reinterpret_cast<int*>(ws + at.hole), reinterpret_cast<Pair*>(ws + at.pairs),
                        reinterpret_cast<int*>(ws + at.n_pairs)};
    LaunchConfig lc(1, THREADS, 0, stream, 1, true);
    if (cudaLaunchKernelEx(&lc.cfg, compact_kernel, a) != cudaSuccess) return check_launch();
    count_launch();
    const int e = esize(p->dtype);
    return launch_copy(CopyArgs{p->pool, p->k_strideL, p->v_strideL, p->layers, p->nh_kv, e, parts_of(p->nh_kv, p->pool.page, e), a.pairs, a.n_pairs, p->where, p->pages_out, p->B},
                       p->pool.n_pages / 2, stream);
}

}  // extern "C"
