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
// Rows of new tokens into the pages: a warp to a token, 16 bytes to a lane, all heads of keys and values.  HBM bounds it: 8 192 tokens of 12
// heads, fp32, 100 MB, in 18.8 us (with CTAs of 8 warps 19.7: the last of them are alone for longer).
// ---------------------------------------------------------------------------
constexpr int APPEND_WARPS = 4;
struct AppendArgs {
    hk_pool pool;
    hk_view K, V;
    const int32_t *lengths, *starts, *picks, *counts;
    int B, Hk, T, esize;
};

template <int PIECES>  // of 16 bytes in a row
__global__ void __launch_bounds__(APPEND_WARPS * 32, 6) append_kernel(const __grid_constant__ AppendArgs a) {
    pdl_wait();
    pdl_trigger();
    const int lane = threadIdx.x & 31;
    const int64_t item = (int64_t)blockIdx.x * APPEND_WARPS + (threadIdx.x >> 5);
    int b, row;  // the row of K and V, and of which batch
    int64_t pos, from_b;
    if (a.starts) {
        if (item >= a.T) return;
        row = (int)item;
        b = sequence_of(a.starts, a.B, row, lane);
        if (b >= a.B || a.starts[b] > row) return;
        pos = row - max(a.starts[b], 0);
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
// Copies of pages, of the first `rows` rows of every head in every layer: a piece of a page's keys or values of a layer to 8 warps, RUN times 16
// bytes to a thread.
// ---------------------------------------------------------------------------
struct Pair {
    int from, to, rows, pad;
};
struct Copies {
    hk_pool pool;
    int64_t k_strideL, v_strideL;
    int layers, Hk, esize;
    int parts;     // pieces of a page
    int of_pair;   // and of all that belongs to it
    int most;      // pairs, at most
};
template <int RUN>
__device__ __forceinline__ void copy_piece(const Copies& a, const Pair& pair, unsigned piece, int warp, int lane) {
    if (pair.rows == 0) return;  // there was no page to copy to
    const unsigned part = piece % a.parts, rest = piece / a.parts;
    const int kv = rest & 1, layer = rest >> 1, shift = a.esize == 4 ? 4 : 3, inside = lane & ((1 << shift) - 1), rows = 32 >> shift;
    const hk_view& v = kv ? a.pool.V : a.pool.K;
    // rows of the page in the order they lie in
    const bool by_token = v.strideH < v.strideM;
    const int inner = by_token ? a.Hk : pair.rows, all = a.Hk * pair.rows;
    const int64_t s_in = by_token ? v.strideH : v.strideM, s_out = by_token ? v.strideM : v.strideH, e = a.esize;
    const char* base = static_cast<const char*>(v.ptr) + layer * (kv ? a.v_strideL : a.k_strideL) * e + inside * 16;
    const char* from = base + pair.from * v.strideB * e;
    char* to = const_cast<char*>(base) + pair.to * v.strideB * e;
    const int first = ((int)part * 8 + warp) * rows * RUN + (lane >> shift);
    uint4 x[RUN];
    int64_t at[RUN];
#pragma unroll
    for (int i = 0; i < RUN; ++i) {
        const int r = first + i * rows, outer = r / inner;
        at[i] = (outer * s_out + (r - outer * inner) * s_in) * e;
        if (r < all) x[i] = *reinterpret_cast<const uint4*>(from + at[i]);
    }
#pragma unroll
    for (int i = 0; i < RUN; ++i)
        if (first + i * rows < all) *reinterpret_cast<uint4*>(to + at[i]) = x[i];
}

// Pieces first, first + step, .. of those of pairs(k), k < n, of which there may be more than 32 bits count
template <int RUN, class F>
__device__ __forceinline__ void copy_all(const Copies& a, unsigned first, unsigned step, int n, F pairs) {
    const unsigned of_pair = a.of_pair, pairs_on = step / of_pair, on = step % of_pair;
    unsigned k = first / of_pair, piece = first % of_pair;
    while (k < (unsigned)n) {
        copy_piece<RUN>(a, pairs(k), piece, threadIdx.x >> 5 & 7, threadIdx.x & 31);
        k += pairs_on;
        piece += on;
        if (piece >= of_pair) {
            piece -= of_pair;
            ++k;
        }
    }
}

// By a kernel of their own, and the table's new entries
constexpr int OWN_RUN = 8;
struct CopyArgs {
    Copies copies;
    const Pair* pairs;
    const int* n_pairs;
    const int32_t* where;  // compaction: the pages' new places
    int32_t* pages_out;
    int B;
};
__global__ void __launch_bounds__(256, 3) copy_pages_kernel(const __grid_constant__ CopyArgs a) {
    const hk_pool& pool = a.copies.pool;
    pdl_wait();
    pdl_trigger();
    if (a.where) {
        for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < (int64_t)a.B * pool.width; i += (int64_t)gridDim.x * 256) {
            const int64_t b = i / pool.width;
            const int e = pool.pages[b * pool.pages_stride + (i - b * pool.width)];
            a.pages_out[i] = is_page(e, pool.n_pages) ? a.where[e] : -1;
        }
    }
    copy_all<OWN_RUN>(a.copies, blockIdx.x, gridDim.x, *a.n_pairs, [&](int k) { return a.pairs[k]; });
}

// ---------------------------------------------------------------------------
// Tables.  Every step needs all of the one before, so one CTA takes them, with what the steps hand on in shared memory where it fits: a
// step then waits for the entries it reads, not for what the last one wrote.  Where few pages can have to be copied, every CTA of a grid works the
// tables out and copies its share: no second kernel, and nobody waits for another (64 requests of 64 pages, a call: 7.1 us, 9.5 with
// two kernels; 512 of 256: 58 us, most of it in the steps over the entries).
// ---------------------------------------------------------------------------
constexpr int THREADS = 1024;
constexpr size_t ROOM = 220 << 10;  // of the 227 KiB that a CTA may have
constexpr int RUN = 4;              // 64 registers to a thread

// A thread's share of n, in a row: an odd number, so that the threads of a warp meet different banks of shared memory
__device__ __forceinline__ int share(int n) { return (n + THREADS - 1) / THREADS | 1; }
// f(x, at(x)) for x < n by all threads, four of each thread's at a time, so that their loads are under way together
template <class At, class F>
__device__ __forceinline__ void for_all(int n, At at, F f) {
    for (int x0 = threadIdx.x; x0 < n; x0 += 4 * THREADS) {
        int e[4];
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if (x0 + u * THREADS < n) e[u] = at(x0 + u * THREADS);
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if (x0 + u * THREADS < n) f(x0 + u * THREADS, e[u]);
    }
}

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

// The first rows of a page to zeros, in every layer, by a warp
__device__ __forceinline__ void clear_rows(const Copies& a, int page, int rows, int lane) {
    const int64_t e = a.esize;
    const int each = 4 * a.esize;  // 16-byte parts of a row
    for (int kv = 0; kv < 2; ++kv) {
        const hk_view& v = kv ? a.pool.V : a.pool.K;
        for (int layer = 0; layer < a.layers; ++layer) {
            for (int h = 0; h < a.Hk; ++h) {
                char* const to = static_cast<char*>(v.ptr) + (layer * (kv ? a.v_strideL : a.k_strideL) + page * v.strideB + h * v.strideH) * e;
                for (int i = lane; i < rows * each; i += 32) reinterpret_cast<uint4*>(to + i / each * v.strideM * e)[i % each] = make_uint4(0, 0, 0, 0);
            }
        }
    }
}

struct Request {  // of the new batch
    int source;   // row of the old table, -1: none
    int len;
    int kept;     // pages it has
    int need;     // pages up to where it has room
    int first;    // number of its first new page
    int copy;     // number of its copy, -1: none, CLEARED: its begun page is none, it gets one whose rows are zeros
};
constexpr int CLEARED = -2;
struct ForkArgs {
    Copies copies;
    const int32_t *lengths, *users, *source, *room;
    int32_t *pages_out, *lengths_out, *users_out, *missing;
    int B, B_out;
    int64_t room_all;
    uint32_t width_mul;  // x / width is x * width_mul >> width_shift for x below 2^31
    int width_shift;
    int* owner;    // [B]: the first of the new batch that goes on with a request
    Request* request;  // [B_out]
    int* free;     // [n_pages]
    Pair* pairs;   // [B_out]
    int* n_pairs;
    int copies_too;  // this kernel makes them
    static size_t shared_bytes(int64_t P, int64_t B, int64_t B_out) { return B_out * (sizeof(Pair) + sizeof(Request)) + (2 * P + B) * sizeof(int); }
};

template <bool SHARED>
__global__ void __launch_bounds__(THREADS, 1) fork_kernel(const __grid_constant__ ForkArgs a) {
    __shared__ Sums sums;
    __shared__ unsigned long long lacking;
    extern __shared__ Pair room[];
    const hk_pool& pool = a.copies.pool;
    const int tid = threadIdx.x, M = pool.width, P = pool.n_pages;
    Request* const request = SHARED ? reinterpret_cast<Request*>(room + a.B_out) : a.request;
    int* const users = SHARED ? reinterpret_cast<int*>(request + a.B_out) : a.users_out;
    int *const free = SHARED ? users + P : a.free, *const owner = SHARED ? users + 2 * P : a.owner;
    const bool writes = blockIdx.x == 0;
    auto row = [&](int x) { return (int)(((uint64_t)(uint32_t)x * a.width_mul) >> a.width_shift); };
    auto nobody = [&] {
        for (int b = tid; b < a.B; b += THREADS) owner[b] = INT_MAX;
    };
    if (tid == 0) lacking = 0;
    if (SHARED) nobody();
    pdl_wait();
    pdl_trigger();
    if (!SHARED) nobody();  // the call before may still have used the workspace
    // a thread's first request is on its way while the tables are read
    struct Wish {
        int source, len, begun;  // begun: the page that is, -1: none
        int64_t room;
    };
    auto wish = [&](int i) {
        Wish w = {-1, 0, -1, 0};
        if (i < a.B_out) {
            const int s = a.source[i];
            w.room = a.room ? (int64_t)max(a.room[i], 0) : a.room_all;
            if ((unsigned)s < (unsigned)a.B) {
                w.source = s;
                w.len = (int)min((int64_t)max(a.lengths[s], 0), (int64_t)M * pool.page);
                const int full = w.len / pool.page;
                if (w.len - full * pool.page) w.begun = pool.pages[s * pool.pages_stride + full];
            }
        }
        return w;
    };
    const Wish first = wish(tid);
    for_all(P, [&](int p) { return a.users[p]; }, [&](int p, int n) { users[p] = n; });
    __syncthreads();
    // what the old table held is nobody's, and who goes on with a request first
    for_all(a.B * M, [&](int x) { const int b = row(x); return pool.pages[b * pool.pages_stride + (x - b * M)]; },
            [&](int, int e) { if (is_page(e, P)) atomicSub(users + e, 1); });
    for (int i = tid; i < a.B_out; i += THREADS) {
        const int s = i == tid ? first.source : a.source[i];
        if ((unsigned)s < (unsigned)a.B) atomicMin(owner + s, i);
    }
    __syncthreads();
    int given = 0, n_pairs = 0;
    for (int i0 = 0; i0 < a.B_out; i0 += THREADS) {
        const int i = i0 + tid;
        const Wish w = i0 == 0 ? first : wish(i);
        Request r = {w.source, w.len, 0, 0, 0, -1};
        bool copy = false, cleared = false;
        if (i < a.B_out) {
            const bool begun = w.len % pool.page != 0;
            if (w.source >= 0) {
                const bool there = begun && is_page(w.begun, P), owns = there && owner[w.source] == i;
                r.kept = w.len / pool.page + owns;
                copy = there && !owns;  // another has the original
                cleared = begun && !there;
            }
            const int64_t need = (w.len + w.room + pool.page - 1) / pool.page;
            r.need = (int)max((int64_t)r.kept, min(need, (int64_t)M));
            if (need > M) atomicAdd(&lacking, (unsigned long long)(need - M));
        }
        int total, copies;
        r.first = given + block_scan(sums, r.need - r.kept, total);
        given += total;
        const int number = n_pairs + block_scan(sums, copy, copies);
        n_pairs += copies;
        if (copy) r.copy = number;
        if (cleared) r.copy = CLEARED;
        if (i < a.B_out) {
            if (writes) a.lengths_out[i] = w.len;
            request[i] = r;
        }
    }
    __syncthreads();
    // pages that are kept
    for_all(a.B_out * M,
            [&](int x) {
                const int i = row(x), j = x - i * M;
                const Request r = request[i];
                return j < r.kept ? pool.pages[r.source * pool.pages_stride + j] : -1;
            },
            [&](int x, int e) {
                if (is_page(e, P)) atomicAdd(users + e, 1);
                else e = -1;
                if (writes) a.pages_out[x] = e;
            });
    __syncthreads();
    // the free ones in their order
    const int each = share(P), p0 = min(P, tid * each), p1 = min(P, p0 + each);
    int n = 0, n_free;
    for (int p = p0; p < p1; ++p) n += users[p] == 0;
    n = block_scan(sums, n, n_free);
    for (int p = p0; p < p1; ++p)
        if (users[p] == 0) free[n++] = p;
    __syncthreads();
    Pair* const pairs = SHARED && a.copies_too ? room : a.pairs;
    for (int i = tid / 32; i < a.B_out; i += THREADS / 32) {  // a warp to a request
        const Request r = request[i];
        const int begun = r.copy >= 0 ? r.len / pool.page : -1;
        for (int j = r.kept + tid % 32; j < r.need; j += 32) {
            const int f = r.first + j - r.kept, page = f < n_free ? free[f] : -1;
            if (page >= 0) users[page] = 1;
            if (writes) a.pages_out[(int64_t)i * M + j] = page;
            if (j == begun) pairs[r.copy] = {pool.pages[r.source * pool.pages_stride + j], page, page >= 0 ? r.len % pool.page : 0, 0};
        }
        // here, not among the copies: there a choice of what to store costs 2 to 4 % of their rate
        if (writes && r.copy == CLEARED && r.first < n_free) clear_rows(a.copies, free[r.first], r.len % pool.page, tid % 32);
    }
    __syncthreads();
    if (writes) {
        if (SHARED)
            for (int p = tid; p < P; p += THREADS) a.users_out[p] = users[p];
        if (tid == 0) {
            *a.missing = (int)min(lacking + max(0, given - n_free), (unsigned long long)INT_MAX);
            *a.n_pairs = n_pairs;
        }
    }
    if (SHARED && a.copies_too) copy_all<RUN>(a.copies, blockIdx.x + gridDim.x * (tid >> 8), gridDim.x * (THREADS / 256), n_pairs, [&](int k) { return room[k]; });
}

struct CompactArgs {
    Copies copies;
    const int32_t* users;
    int32_t *pages_out, *users_out, *where;
    int B;
    int* hole;    // [n_pages]
    Pair* pairs;  // [n_pages / 2 + 1]
    int* n_pairs;
    int copies_too;  // this kernel makes them, and the table
    static size_t shared_bytes(int64_t P) { return 4 * P * sizeof(int); }
};
template <bool SHARED>
__global__ void __launch_bounds__(THREADS) compact_kernel(const __grid_constant__ CompactArgs a) {
    __shared__ Sums sums;
    extern __shared__ Pair room[];
    const hk_pool& pool = a.copies.pool;
    const int tid = threadIdx.x, P = pool.n_pages, each = share(P), p0 = min(P, tid * each), p1 = min(P, p0 + each);
    int *const mine = reinterpret_cast<int*>(room), *const hole = SHARED ? mine + P : a.hole, *const from = mine + 2 * P, *const where = SHARED ? mine + 3 * P : a.where;
    const int* const users = SHARED ? mine : a.users;
    const bool writes = blockIdx.x == 0;
    pdl_wait();
    pdl_trigger();
    if (SHARED) {
        for_all(P, [&](int p) { return a.users[p]; }, [&](int p, int n) { mine[p] = n; });
        __syncthreads();
    }
    int used = 0, n, holes = 0, moves = 0, n_holes, n_moves;
    for (int p = p0; p < p1; ++p) used += users[p] > 0;
    block_scan(sums, used, n);
    for (int p = p0; p < p1; ++p) {
        const bool u = users[p] > 0;
        holes += !u && p < n;
        moves += u && p >= n;
    }
    holes = block_scan(sums, holes, n_holes);
    moves = block_scan(sums, moves, n_moves);  // as many
    for (int p = p0; p < p1; ++p) {
        const int u = users[p];
        if (p < n && u <= 0) hole[holes++] = p;
        if (p >= n && u > 0) {
            if (SHARED) from[moves++] = p;
            else a.pairs[moves++].from = p;
        }
        if (writes && p >= n) a.users_out[p] = 0;
        else if (writes && u > 0) a.users_out[p] = u;
        if (p < n || u <= 0) where[p] = u > 0 ? p : -1;
    }
    __syncthreads();
    for (int k = tid; k < n_moves; k += THREADS) {
        const int x = SHARED ? from[k] : a.pairs[k].from, to = hole[k];
        if (!SHARED || !a.copies_too) a.pairs[k] = {x, to, pool.page, 0};
        where[x] = to;
        if (writes) a.users_out[to] = users[x];
    }
    if (writes && tid == 0) *a.n_pairs = n_moves;
    if (!SHARED) return;
    __syncthreads();
    if (writes)
        for (int p = tid; p < P; p += THREADS) a.where[p] = where[p];
    if (!a.copies_too) return;
    for (int64_t i = (int64_t)blockIdx.x * THREADS + tid; i < (int64_t)a.B * pool.width; i += (int64_t)gridDim.x * THREADS) {
        const int64_t b = i / pool.width;
        const int e = pool.pages[b * pool.pages_stride + (i - b * pool.width)];
        a.pages_out[i] = is_page(e, P) ? where[e] : -1;
    }
    copy_all<RUN>(a.copies, blockIdx.x + gridDim.x * (tid >> 8), gridDim.x * (THREADS / 256), n_moves, [&](int k) { return Pair{from[k], hole[k], pool.page, 0}; });
}

size_t up(size_t n) { return (n + 255) / 256 * 256; }

template <class Args>
int launch_tables(void (*kernel)(Args), const Args& a, int ctas, size_t bytes, cudaStream_t stream) {
    if (bytes > (40 << 10) && cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)ROOM) != cudaSuccess) return check_launch();
    LaunchConfig lc((unsigned)ctas, THREADS, bytes, stream, 1, true);
    if (cudaLaunchKernelEx(&lc.cfg, kernel, a) != cudaSuccess) return check_launch();
    count_launch();
    return HK_OK;
}
int pieces(int Hk, int page, int esize, int run) { return cdiv((int64_t)Hk * page, 8 * (esize == 4 ? 2 : 4) * run); }
template <class Params>
Copies copies_of(const Params* p, int most, int run) {
    const int e = esize(p->dtype), parts = pieces(p->nh_kv, p->pool.page, e, run);
    return {p->pool, p->k_strideL, p->v_strideL, p->layers, p->nh_kv, e, parts, p->layers * 2 * parts, most};
}
// CTAs of a kernel that makes the copies too; 0: a kernel of their own does, which keeps more loads under way (5.9 TB/s, not 5.5) but costs 2 us
int copiers(const Copies& a) {
    const int64_t rounds = cdiv((int64_t)a.most * a.of_pair, THREADS / 256), sms = sm_count();
    return rounds > 16 * sms ? 0 : (int)std::min(rounds, sms);
}

int launch_copy(const CopyArgs& a, cudaStream_t stream) {
    const int64_t items = (int64_t)a.copies.most * a.copies.of_pair;
    LaunchConfig lc((unsigned)std::min<int64_t>(items, (int64_t)sm_count() * 8), 256, 0, stream, 1, true);
    if (cudaLaunchKernelEx(&lc.cfg, copy_pages_kernel, a) != cudaSuccess) return check_launch();
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
// pages that can be copied at once
int fork_pairs(const hk_fork_params* p) { return std::min(p->B_out, p->pool.n_pages); }
int compact_pairs(const hk_compact_params* p) { return std::max(1, p->pool.n_pages / 2); }
// what belongs to a page is counted in 32 bits: no memory holds as much
int check_pieces(int64_t layers, int nh_kv, int page, int dtype) { return layers * 2 * pieces(nh_kv, page, esize(dtype), RUN) <= INT_MAX ? HK_OK : HK_ERR_BAD_SHAPE; }
int check_fork_sizes(const hk_fork_params* p) {
    if (!p) return HK_ERR_NULL_POINTER;
    if (p->B <= 0 || p->B_out <= 0 || p->layers <= 0 || p->layers > (1 << 20) || p->room_all < 0 || p->room_all > (1 << 30)) return HK_ERR_BAD_SHAPE;
    const int rc = check_pool_sizes(p->pool, std::max(p->B, p->B_out), p->nh_kv, p->dtype);
    return rc == HK_OK ? check_pieces(p->layers, p->nh_kv, p->pool.page, p->dtype) : rc;
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
    const int rc = check_pool_sizes(p->pool, p->B, p->nh_kv, p->dtype);
    return rc == HK_OK ? check_pieces(p->layers, p->nh_kv, p->pool.page, p->dtype) : rc;
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
    LaunchConfig lc((unsigned)cdiv(B * p->T, APPEND_WARPS), APPEND_WARPS * 32, 0, static_cast<cudaStream_t>(stream), 1, true);
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
    ForkArgs a{copies_of(p, fork_pairs(p), RUN), p->lengths, p->users, p->source, p->room, p->pages_out, p->lengths_out, p->users_out, p->missing, p->B, p->B_out, p->room_all, 0, 0,
               reinterpret_cast<int*>(ws + at.owner), reinterpret_cast<Request*>(ws + at.request), reinterpret_cast<int*>(ws + at.free),
               reinterpret_cast<Pair*>(ws + at.pairs), reinterpret_cast<int*>(ws + at.n_pairs), 0};
    divide_by(p->pool.width, a.width_mul, a.width_shift);
    const size_t shared = ForkArgs::shared_bytes(p->pool.n_pages, p->B, p->B_out);
    const int ctas = shared <= ROOM ? copiers(a.copies) : 0;
    a.copies_too = ctas > 0;
    rc = shared <= ROOM ? launch_tables(fork_kernel<true>, a, std::max(1, ctas), shared, stream) : launch_tables(fork_kernel<false>, a, 1, 0, stream);
    return rc != HK_OK || ctas ? rc : launch_copy(CopyArgs{copies_of(p, fork_pairs(p), OWN_RUN), a.pairs, a.n_pairs, nullptr, nullptr, 0}, stream);
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
    CompactArgs a{copies_of(p, compact_pairs(p), RUN), p->users, p->pages_out, p->users_out, p->where, p->B, reinterpret_cast<int*>(ws + at.hole),
                  reinterpret_cast<Pair*>(ws + at.pairs), reinterpret_cast<int*>(ws + at.n_pairs), 0};
    const size_t shared = CompactArgs::shared_bytes(p->pool.n_pages);
    const int ctas = shared <= ROOM ? copiers(a.copies) : 0;
    a.copies_too = ctas > 0;
    rc = shared <= ROOM ? launch_tables(compact_kernel<true>, a, std::max(1, ctas), shared, stream) : launch_tables(compact_kernel<false>, a, 1, 0, stream);
    return rc != HK_OK || ctas ? rc : launch_copy(CopyArgs{copies_of(p, compact_pairs(p), OWN_RUN), a.pairs, a.n_pairs, p->where, p->pages_out, p->B}, stream);
}

}  // extern "C"
