// shared_prefix_sm100.cu -- attention over a shared prefix where many rows meet a run of keys: chunks of new tokens, or the rows of
// a whole batch against the prefix.
//
// A CTA takes blocks of 128 rows of one key head (two of 16-bit types, one of fp32) through tiles of keys: a run of the prefix, the
// request's own keys, or the prefix and then those.  Rows of a block are whatever rows of the key head follow each other (tokens
// and query heads of one request, or of several against the prefix), so every key is loaded once for 128 or 256 of them.
//   Warp 0 loads tiles with TMA, warp 1 issues the products S = Q K^T and, a tile or two behind, O += P V (tcgen05, operands in
// shared and tensor memory), four warps to a block of rows take S through the softmax, a row to a thread.  Scores are three deep
// in tensor memory; P takes the place of its S.
//   fp32: x = h + l with h the upper 11 bits of the significand, which is what the tensor core reads of an fp32 word.  Q lies in tensor memory
// with its l parts, four warps write those of each tile beside it; a product is l h' + h l' + h h', in this order: what is left out is 2^-22 of it.  P V of
// a tile comes back into registers and is added there in fp32: the tensor core's additions cut off instead of rounding, and over
// thousands of keys in one accumulator that would be seen.
//
// 16-bit types are bound by the softmax: scaling, exponentials, sums and rounding of 256 rows x 128 keys take 1 930 to 2 120 cycles by
// themselves, whether none or a third of the exponentials goes by a polynomial (the special functions alone need 2 048 or less, packed
// arithmetic takes two issue slots), and a tile takes 2 400 to 2 500 (masked 0.4 us more).  fp32 is bound by the tensor core: 1 680 cycles of a tile's 2 030 (1.1 us).  A
// CTA takes about 5 us beside its tiles.  8 requests of 512 tokens, 32 heads on 8, 8 192 and up to 1 024 keys, bf16: 326 us alone, 363
// under load (800 TFLOP/s; 175 us for the products, 196 for four fifths of the exponentials at 16 a clock and SM).  8 requests of 77 tokens, 12 heads,
// 4 096 and up to 333 keys, fp32: 45.4 us (51.7 from Python, 29 for the products); that kernel spills 36 bytes a thread.
// A row of Q and of O to a thread: with eight lanes to a row, through shared memory, the two took 351 and 48.6 instead of 346 and 47.0.
#include <cmath>
#include <mutex>
#include <type_traits>

#include "shared_prefix.cuh"

namespace hk {
namespace {

template <class X>
struct Many {
    static constexpr bool LOW = sizeof(X) == 4;      // products in three parts
    static constexpr int STREAMS = LOW ? 1 : 2;      // blocks of rows
    static constexpr int KEYS = LOW ? 64 : 128;      // of a tile
    static constexpr int SLOTS = LOW ? 7 : 8;
    static constexpr int THREADS = LOW ? 320 : 384;
    static constexpr int AHEAD = LOW ? 2 : 1;        // tiles that the scores are ahead of the weighted values
    static constexpr int Q_BYTES = LOW ? 0 : TILE * 64 * (int)sizeof(X);  // fp32: in tensor memory
    static constexpr int KV_RAW = KEYS * 64 * (int)sizeof(X), KV_BYTES = KV_RAW * (LOW ? 2 : 1);
    static constexpr int KV_BOX = KEYS * 128;        // 128 bytes of each row
    struct __align__(16) Shared {
        uint64_t q_full[STREAMS], kv_full[SLOTS], kv_empty[SLOTS], s_full[3], p_full[3], o_full[3];
        uint64_t kv_ready[LOW ? SLOTS : 1];  // low parts are there
        uint64_t last_full, last_ready;      // the request's last tile of values, with and without what is behind its last key
        uint32_t tmem_base;
        Abort abort;
    };
    static constexpr int OFF_KV = STREAMS * Q_BYTES, OFF_SH = OFF_KV + SLOTS * KV_BYTES, SMEM = OFF_SH + (int)sizeof(Shared);
    static_assert(SMEM <= 232448, "exceeds the 227 KiB a CTA may opt in to");
};
// Tensor memory.  16-bit types: three buffers of 128 columns for scores and weights, O of two blocks of rows.  fp32: three buffers of
// 64 for scores and weights, two for the weights' low parts, O of a tile, Q and its low parts.
constexpr uint32_t COL_O = 384, LOW_COL_LOW = 192, LOW_COL_O = 320, LOW_COL_Q = 384;

enum ManyWait { W_Q = 301, W_KV, W_READY, W_EMPTY, W_S, W_P, W_O };

struct ManyArgs {
    PrefixArgs p;
    int own;           // the request's own keys are part of it
    int prefix;        // the prefix is: a run of it if not `own`, all of it otherwise
    int late;          // runs beside the kernel over the prefix; what was before that is complete when this one begins
    int tiles;         // items of row blocks: of a key head, or of a request's
};

template <class X>
__global__ void __launch_bounds__(Many<X>::THREADS, 1)
prefix_many_kernel(const __grid_constant__ CUtensorMap map_kp, const __grid_constant__ CUtensorMap map_vp, const __grid_constant__ CUtensorMap map_k,
                   const __grid_constant__ CUtensorMap map_v, const __grid_constant__ ManyArgs args) {
    typedef Many<X> C;
    constexpr bool LOW = C::LOW, BF16 = std::is_same<X, __nv_bfloat16>::value;
    constexpr int KEYS = C::KEYS, SLOTS = C::SLOTS;
    const PrefixArgs& a = args.p;
    extern __shared__ __align__(1024) uint8_t smem[];
    uint8_t *sQ = smem, *sKV = smem + C::OFF_KV;
    typename C::Shared& sh = *reinterpret_cast<typename C::Shared*>(smem + C::OFF_SH);
    const int warp = (int)uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int t = 0; t < C::STREAMS; ++t) mbar_init(&sh.q_full[t], 4);
        for (int s = 0; s < SLOTS; ++s) {
            mbar_init(&sh.kv_full[s], 1);
            if (LOW) mbar_init(&sh.kv_ready[s], 2);
            mbar_init(&sh.kv_empty[s], 1);
        }
        for (int b = 0; b < 3; ++b) {
            mbar_init(&sh.s_full[b], 1);
            mbar_init(&sh.p_full[b], 4);
            mbar_init(&sh.o_full[b], 1);
        }
        mbar_init(&sh.last_full, 1);
        mbar_init(&sh.last_ready, 1);
        sh.abort.id = 0;
        fence_mbar_init();
    }
    if (warp == 1) {
        tmem_alloc(&sh.tmem_base, 512);
        tmem_relinquish();
        tc_fence_before_sync();
    }
    if (args.late) __threadfence();
    else pdl_wait();
    pdl_trigger();
    // the item: rows
    int item = blockIdx.x, split = 0, parts = 1;
    if (!args.own) {
        item = blockIdx.x / a.splits_p;
        split = blockIdx.x - item * a.splits_p;
    } else if (a.whole && item >= a.first_split) {
        parts = a.slots;
        item = a.first_split + (blockIdx.x - a.first_split) / parts;
        split = (blockIdx.x - a.first_split) % parts;
    }
    const int at = item / args.tiles;
    const int tile = args.tiles - 1 - (item - at * args.tiles);  // the last rows see the most keys
    const int b = args.own ? at / a.Hk : 0, kvh = at - b * a.Hk, BLOCK = C::STREAMS * TILE;
    const int all = args.own ? a.T * a.group : a.R, first = tile * BLOCK, row0 = b * a.T * a.group + first, rows = min(BLOCK, all - first);
    const int len = args.own ? request_keys(a, b) : 0;
    // a row of Q to a softmax thread
    const int t = (warp - 4) >> 2, quarter = warp & 3, in_block = quarter * 32 + lane, r = t * TILE + in_block;
    const bool valid = warp >= 4 && r < rows;
    struct Where {
        int b, h, t;
    };
    auto where = [&](int row) -> Where {  // row of the key head
        const int token = row / a.group, bq = args.own ? b : token / a.T;
        return {bq, kvh * a.group + row - token * a.group, token - bq * a.T};
    };
    constexpr int CHUNKS = 64 * sizeof(X) / 16;
    uint4 x_q[CHUNKS];
    if (warp >= 4) {
        const Where at_q = valid ? where(row0 + r) : Where{0, 0, 0};
        const uint4* from = reinterpret_cast<const uint4*>(row_of<X>(a.Q, at_q.b, at_q.h, at_q.t));
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) x_q[c] = valid ? from[c] : make_uint4(0, 0, 0, 0);
    }
    // and keys: tiles of the prefix, then the request's own
    int p_begin = args.own ? 0 : split * a.per_p, own_begin = 0;
    const int p_end = !args.prefix ? 0 : args.own ? a.P : min(a.P, p_begin + a.per_p);
    const int seen = args.own ? token_keys(a, len, (first + rows - 1) / a.group) : 0;
    int n_p = (p_end - p_begin + KEYS - 1) / KEYS, n = n_p + (seen + KEYS - 1) / KEYS;
    if (parts > 1) {  // a run of the block's tiles
        const int per = (n + parts - 1) / parts, from = min(n, split * per);
        own_begin = max(0, from - n_p) * KEYS;
        p_begin = from * KEYS;
        n = min(per, n - from);
        n_p = min(n, max(0, n_p - from));
    }
    const int streams = C::STREAMS == 2 && rows > TILE ? 2 : 1;
    __syncthreads();
    tc_fence_after_sync();
    constexpr uint32_t tmem = 0;  // all columns are this CTA's
    if (sh.tmem_base != tmem) sh.abort.id = 398;
    WaitNote wc{&sh.abort};
    // 16-bit types: the last tile of a request's values goes by a warp that clears it (fp32: every tile does), on barriers of its
    // own, for that warp sees no other phase of the slots' ones
    auto by_hand = [&](int i) { return !LOW && i == 2 * n - 1 && n > n_p; };
    // Tiles go through the ring in the order of their use, keys a tile (fp32: two) ahead: K0 .. K(A) V0 K(A+1) V1 ..
    constexpr int A = C::AHEAD;
    struct Entry {
        int j;
        bool v;
    };
    auto entry = [&](int i) -> Entry {
        if (i < min(n, A + 1)) return {i, false};
        const int k = i - (A + 1);
        return k < 2 * (n - A - 1) ? (k & 1 ? Entry{A + 1 + (k >> 1), false} : Entry{k >> 1, true}) : Entry{i - n, true};
    };
    // first key of tile j, in the prefix or of the request's own
    auto key_of = [&](int j) { return j < n_p ? p_begin + j * KEYS : own_begin + (j - n_p) * KEYS; };

    // What the tiles need beside the loads.  Rows behind the request's last key may hold anything, and 0 times a NaN is one: they are
    // cleared among the values.  fp32: the tiles' low parts, by two pairs of warps.  A pair has every other slot of the ring, not every
    // other tile: a barrier is waited for by the parity of its phase, and who does not see all phases of a slot can take the one before the
    // last for its own.
    auto tend = [&](int me, int first_entry) {
        auto following = [&](int i) { return i % SLOTS + 2 < SLOTS ? i + 2 : (i / SLOTS + 1) * SLOTS + first_entry; };
        bool ok = true;
        for (int i = first_entry; ok && n > (LOW ? 0 : n_p) && i < 2 * n; i = LOW ? following(i) : 2 * n) {
            const auto [j, is_v] = entry(i);
            const int s = i % SLOTS;
            ok = __all_sync(0xffffffffu, LOW ? mbar_wait(wc, &sh.kv_full[s], (i / SLOTS) & 1, W_KV, i) : mbar_wait(wc, &sh.last_full, 0, W_KV, i));
            if (!ok) break;
            const int keep = is_v && j >= n_p ? min(KEYS, len - key_of(j)) : KEYS;  // rows that are values
            uint4* raw = reinterpret_cast<uint4*>(sKV + s * C::KV_BYTES);
            if constexpr (LOW) {
                constexpr int EACH = C::KV_RAW / 16 / 64;
                uint4 *from = raw + me, *low = from + C::KV_RAW / 16, x[EACH];
#pragma unroll
                for (int k = 0; k < EACH; ++k) x[k] = from[k * 64];
                if (keep < KEYS) {
#pragma unroll
                    for (int k = 0; k < EACH; ++k)
                        if (((k * 64 + me) & (C::KV_BOX / 16 - 1)) / 8 >= keep) from[k * 64] = x[k] = make_uint4(0, 0, 0, 0);  // row of the box
                }
#pragma unroll
                for (int k = 0; k < EACH; ++k) low[k * 64] = make_uint4(tf32_rest(x[k].x), tf32_rest(x[k].y), tf32_rest(x[k].z), tf32_rest(x[k].w));
            } else {
                for (int k = keep * 8 + me; k < C::KV_RAW / 16; k += 32) raw[k] = make_uint4(0, 0, 0, 0);
            }
            fence_proxy_async_smem();
            mbar_arrive_warp(LOW ? &sh.kv_ready[s] : &sh.last_ready, lane);
        }
    };

    if (warp < 4) {
        if constexpr (!LOW) asm volatile("setmaxnreg.dec.sync.aligned.u32 72;\n");
        if (warp == 0) {
            // ------------------------------ tiles of keys and values ------------------------------
            if (lane == 0) {
                bool ok = true;
                for (int i = 0; ok && i < 2 * n; ++i) {
                    const auto [j, is_v] = entry(i);
                    const int s = i % SLOTS;
                    if (i >= SLOTS && !(ok = mbar_wait(wc, &sh.kv_empty[s], (i / SLOTS - 1) & 1, W_EMPTY, i))) break;
                    uint64_t* full = by_hand(i) ? &sh.last_full : &sh.kv_full[s];
                    mbar_arrive_expect_tx(full, C::KV_RAW);
                    const CUtensorMap* map = j < n_p ? (is_v ? &map_vp : &map_kp) : (is_v ? &map_v : &map_k);
                    tma_load_tile(sKV + s * C::KV_BYTES, map, full, key_of(j), kvh, j < n_p ? 0 : b);
                }
                // a CTA that gave up may have copies in flight: they get time to land
                if (!ok)
                    for (const unsigned long long t0 = globaltimer_ns(); globaltimer_ns() - t0 < 100000ull;) {}
            }
        } else if (warp == 1) {
            // ------------------------------ products ------------------------------
            const uint32_t leader = elect_one_sync();
            const int total = n * streams, ahead = A * streams;  // products, and those that S is ahead of O
            bool ok = true;
            // The tensor pipe queues next to nothing, and a wait takes some 100 cycles even when its barrier is long complete: each
            // is looked at while the products before it are still being issued, and waited for if that look came too early.  For
            // the same reason nothing is divided here: the tiles come in the order of the ring.
            struct Barrier {
                uint64_t* bar;
                uint32_t parity;
            };
            auto seen = [&](const Barrier& x) { return mbar_test_wait(x.bar, x.parity); };
            auto wait = [&](bool was_seen, const Barrier& x, int id, int aux) {
                return __all_sync(0xffffffffu, was_seen) || (bool)__all_sync(0xffffffffu, mbar_wait(wc, x.bar, x.parity, id, aux));
            };
            struct Cursor {
                int at;
                uint32_t phase;
                __device__ __forceinline__ void next(int n) {
                    if (++at == n) {
                        at = 0;
                        phase ^= 1u;
                    }
                }
            };
            Cursor tile{0, 0u}, p{0, 0u};  // the next tile in the ring, the next weights
            int s_buf = 0, k_slot = 0, v_slot = 0;
            int t_s = 0, t_o = 0, v_left = n;  // block of rows of the next S and O; tiles of values that have not been taken
            auto tile_barrier = [&](bool v) -> Barrier {
                if (LOW) return {&sh.kv_ready[tile.at], tile.phase};
                return v && v_left == 1 && n > n_p ? Barrier{&sh.last_ready, 0u} : Barrier{&sh.kv_full[tile.at], tile.phase};
            };
            bool seen_k = false, seen_v = false, seen_p = false;
            const uint32_t kv_addr = smem_u32(sKV);
            const Desc q_desc = make_smem_desc(smem_u32(sQ), 16, 1024, DESC_SW128), k_desc = make_smem_desc(kv_addr, 16, 1024, DESC_SW128),
                       v_desc = LOW ? mnmajor_desc(kv_addr, 0, C::KV_BOX) : make_smem_desc(kv_addr, 16, 1024, DESC_SW128);
            auto look = [&] {  // for what O needs
                seen_v = t_o == 0 && seen(tile_barrier(true));
                seen_p = seen({&sh.p_full[p.at], p.phase});
            };
#pragma unroll 1
            for (int q = 0; q < total + ahead; ++q) {
                if (q < total) {  // S
                    if (q < streams && !(ok = wait(false, {&sh.q_full[t_s], 0u}, W_Q, t_s))) break;
                    if (t_s == 0) {
                        if (!(ok = wait(seen_k, tile_barrier(false), W_READY, q))) break;
                        k_slot = tile.at;
                        tile.next(SLOTS);
                    }
                    tc_fence_after_sync();
                    const Desc kd = k_desc + k_slot * C::KV_BYTES;
                    if constexpr (LOW) {
                        constexpr uint32_t IDESC = make_idesc_tf32(TILE, KEYS, false, false);
                        const uint32_t d = tmem + s_buf * 64;
                        auto eight = [&](uint32_t x, uint32_t y, uint32_t acc) {
                            umma_ts4<KMAJOR_STEP>(leader, d, tmem + LOW_COL_Q + x, kd + y, IDESC, acc);
                            umma_ts4<KMAJOR_STEP>(leader, d, tmem + LOW_COL_Q + x + 32, kd + (y + C::KV_BOX), IDESC, 1u);
                        };
                        eight(64, 0, 0u);
                        eight(0, C::KV_RAW, 1u);
                        if (q >= ahead) look();
                        eight(0, 0, 1u);
                    } else {
                        constexpr uint32_t IDESC = make_idesc_16(TILE, KEYS, BF16, false);
                        const uint32_t d = tmem + s_buf * 128;
                        const Desc qd = q_desc + t_s * C::Q_BYTES;
                        umma_ss_16(leader, d, qd.d, kd.d, IDESC, 0u);
                        umma_ss_16(leader, d, qd.d + 2, kd.d + 2, IDESC, 1u);
                        if (q >= ahead) look();
                        umma_ss_16(leader, d, qd.d + 4, kd.d + 4, IDESC, 1u);
                        umma_ss_16(leader, d, qd.d + 6, kd.d + 6, IDESC, 1u);
                    }
                    umma_commit_lead(leader, &sh.s_full[s_buf]);
                    if (t_s == streams - 1) umma_commit_lead(leader, &sh.kv_empty[k_slot]);
                    s_buf = s_buf == 2 ? 0 : s_buf + 1;
                    t_s ^= streams - 1;
                }
                if (q >= ahead) {  // O
                    if (t_o == 0) {
                        if (!(ok = wait(seen_v, tile_barrier(true), W_READY, q))) break;
                        v_slot = tile.at;
                        tile.next(SLOTS);
                        --v_left;
                    }
                    if (!(ok = wait(seen_p, {&sh.p_full[p.at], p.phase}, W_P, q))) break;
                    tc_fence_after_sync();
                    seen_v = seen_p = false;
                    const bool look_k = t_s == 0 && q + 1 < total;
                    const Desc vd = v_desc + v_slot * C::KV_BYTES;
                    if constexpr (LOW) {
                        constexpr uint32_t IDESC = make_idesc_tf32(TILE, HEAD_DIM, false, true);
                        const uint32_t high = tmem + p.at * 64, low = tmem + LOW_COL_LOW + ((q - ahead) & 1) * 64, d = tmem + LOW_COL_O;
                        auto eight = [&](uint32_t x, uint32_t y, uint32_t acc) {
                            umma_ts4<MNMAJOR_STEP>(leader, d, x, vd + y, IDESC, acc);
                            umma_ts4<MNMAJOR_STEP>(leader, d, x + 32, vd + (y + 4096), IDESC, 1u);
                        };
                        eight(low, 0, 0u);
                        eight(high, C::KV_RAW, 1u);
                        seen_k = look_k && seen(tile_barrier(false));
                        eight(high, 0, 1u);
                    } else {
                        constexpr uint32_t IDESC = make_idesc_16(TILE, HEAD_DIM, BF16, true);
                        const uint32_t w = tmem + p.at * 128, d = tmem + COL_O + t_o * 64, acc = q >= ahead + streams;
#pragma unroll
                        for (int k = 0; k < 8; ++k) {
                            if (k == 4) seen_k = look_k && seen(tile_barrier(false));
                            umma_ts_16(leader, d, w + 8 * k, vd.d + (2048 >> 4) * k, IDESC, k > 0 ? 1u : acc);
                        }
                    }
                    umma_commit_lead(leader, &sh.o_full[p.at]);
                    if (t_o == streams - 1) umma_commit_lead(leader, &sh.kv_empty[v_slot]);
                    p.next(3);
                    t_o ^= streams - 1;
                }
            }
        } else if (LOW) {
            tend(threadIdx.x & 63, 0);
        } else if (warp == 2) {
            tend(lane, 2 * n - 1);
        }
    } else if (LOW && warp >= 8) {
        tend(threadIdx.x & 63, 1);
    } else {
        // ------------------------------ softmax ------------------------------
        if constexpr (!LOW) asm volatile("setmaxnreg.inc.sync.aligned.u32 216;\n");
        const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16);
        const bool live = t * TILE + quarter * 32 < rows;
        const int limit = args.own && valid ? token_keys(a, len, (first + r) / a.group) : 0;  // own keys the row sees
        if (t < streams) {  // the row of Q
            if constexpr (LOW) {
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    uint32_t y[32], z[32];
#pragma unroll
                    for (int c = 0; c < 8; ++c) {
                        const uint4& v = x_q[8 * half + c];
                        y[4 * c] = v.x ^ a.flip; y[4 * c + 1] = v.y ^ a.flip; y[4 * c + 2] = v.z ^ a.flip; y[4 * c + 3] = v.w ^ a.flip;
                    }
#pragma unroll
                    for (int i = 0; i < 32; ++i) z[i] = tf32_rest(y[i]);
                    tmem_st32(lanes + LOW_COL_Q + 32 * half, y);
                    tmem_st32(lanes + LOW_COL_Q + 64 + 32 * half, z);
                }
                tmem_wait_st();
                tc_fence_before_sync();
            } else {
                uint8_t* to = sQ + t * C::Q_BYTES + in_block * 128;  // in the layout of a K-major operand
#pragma unroll
                for (int c = 0; c < CHUNKS; ++c)
                    *reinterpret_cast<uint4*>(to + ((c ^ (in_block & 7)) << 4)) = make_uint4(x_q[c].x ^ a.flip, x_q[c].y ^ a.flip, x_q[c].z ^ a.flip, x_q[c].w ^ a.flip);
                fence_proxy_async_smem();
            }
            mbar_arrive_warp(&sh.q_full[t], lane);
        }
        float o[64], m = -INFINITY, l = 0.f;
        bool ok = true;
        // 16-bit types: a block of rows waits for every other use of a buffer's barrier.  The use in between, of the other block, is
        // complete: it was issued before products that this thread has waited for already.
        auto wait = [&](uint64_t* bar, int q, int id, int j) {  // of product q
            ok = __all_sync(0xffffffffu, mbar_wait(wc, &bar[q % 3], (q / 3) & 1, id, j));
            if (ok) tc_fence_after_sync();
            return ok;
        };
        const float2 scale2 = make_float2(a.scale_log2e, a.scale_log2e);
        if constexpr (LOW) {
            // O_j of every tile comes back and is added here: o = o * before + O_j
            float before = 0.f, alpha = 0.f;
#pragma unroll
            for (int i = 0; i < 64; ++i) o[i] = 0.f;
            auto add = [&](int j) {
                if (!wait(sh.o_full, j, W_O, j) || !live) return;
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    uint32_t x[32];
                    tmem_ld32(lanes + LOW_COL_O + 32 * half, x);
                    tmem_wait_ld();
#pragma unroll
                    for (int i = 0; i < 32; i += 2) {
                        float2& y = reinterpret_cast<float2&>(o[32 * half + i]);
                        y = __ffma2_rn(y, make_float2(before, before), make_float2(__uint_as_float(x[i]), __uint_as_float(x[i + 1])));
                    }
                }
            };
            for (int j = 0; j < n && wait(sh.s_full, j, W_S, j); ++j) {
                const uint32_t at_s = lanes + j % 3 * 64, at_low = lanes + LOW_COL_LOW + (j & 1) * 64;
                if (live) {
                    const int lim = (j < n_p ? p_end : limit) - key_of(j);  // columns the row sees
                    uint32_t x[64];
                    tmem_ld32p(at_s, x);
                    tmem_ld32p(at_s + 32, x + 32);
                    tmem_wait_ld();
                    if (lim < KEYS) {
#pragma unroll
                        for (int i = 0; i < 64; ++i)
                            if (i >= lim) x[i] = __float_as_uint(-INFINITY);
                    }
                    float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                    for (int i = 0; i < 64; i += 2) mx[(i >> 1) & 3] = fmax3(mx[(i >> 1) & 3], __uint_as_float(x[i]), __uint_as_float(x[i + 1]));
                    const float mn = fmaxf(m, fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * a.scale_log2e), ref = mn == -INFINITY ? 0.f : mn;
                    alpha = ex2_approx(m - ref);  // 0 while m is -inf
                    m = mn;
                    const float2 nm = make_float2(-ref, -ref);
                    float2 sum[2] = {};
#pragma unroll
                    for (int c = 0; c < 64; c += 32) {
                        uint32_t z[32];
#pragma unroll
                        for (int i = 0; i < 32; i += 2) {
                            const float2 e = __ffma2_rn(make_float2(__uint_as_float(x[c + i]), __uint_as_float(x[c + i + 1])), scale2, nm);
                            const float2 w = make_float2(ex2_approx(e.x), ex2_approx(e.y));
                            sum[(i >> 1) & 1] = __fadd2_rn(sum[(i >> 1) & 1], w);
                            x[c + i] = __float_as_uint(w.x);
                            x[c + i + 1] = __float_as_uint(w.y);
                            z[i] = __float_as_uint(w.x - __uint_as_float(x[c + i] & 0xffffe000u));
                            z[i + 1] = __float_as_uint(w.y - __uint_as_float(x[c + i + 1] & 0xffffe000u));
                        }
                        tmem_st32p(at_s + c, x + c);
                        tmem_st32(at_low + c, z);
                    }
                    l = fmaf(l, alpha, (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y));
                    tmem_wait_st();
                }
                if (j > 0) add(j - 1);  // before O_j may come to the same place
                if (!ok) break;
                tc_fence_before_sync();
                mbar_arrive_warp(&sh.p_full[j % 3], lane);
                before = alpha;
            }
            if (ok && n > 0) add(n - 1);
        } else if (t < streams) {
            // O stays in tensor memory and is scaled there when a tile's weights come to more than MOST: a stale maximum makes them larger,
            // which neither fp32 sums nor 16-bit types mind up to there
            constexpr float MOST = lift<X>() > 0.f ? 32768.f : 256.f;  // 2^8 of the reference's own weight
            constexpr int POLY_OF = 5;  // of so many pairs of weights, one by the polynomial (3, 4, 5, 6, 8: 336, 324, 326, 329, 332 us, prefill; under load 4 takes 369, 5 365)
            const uint32_t at_o = lanes + COL_O + t * 64;
            uint32_t x[128];
            for (int j = 0; j < n && wait(sh.s_full, j * streams + t, W_S, j); ++j) {
                const int q = j * streams + t;
                const uint32_t at_s = lanes + q % 3 * 128;
                if (live) {
                    const int lim = (j < n_p ? p_end : limit) - key_of(j);  // columns the row sees
                    auto load = [&] {
#pragma unroll
                        for (int c = 0; c < 128; c += 32) tmem_ld32p(at_s + c, x + c);
                        tmem_wait_ld();
                    };
                    float2 sum[2];
                    // The weights take the type of the values: half a step of it each.  A run of them is summed and packed while the next
                    // one's exponentials are under way (runs of 16: prefill 342 us, each pair at once 348).
                    auto weights = [&](auto poly) {
                        constexpr int RUN = 16;
                        const float up = m == -INFINITY ? 0.f : lift<X>() - m;
                        const float2 nm = make_float2(up, up);
                        sum[0] = sum[1] = make_float2(0.f, 0.f);
#pragma unroll
                        for (int c = 0; c < 128 + RUN; c += RUN) {
#pragma unroll
                            for (int i = c; i < c + RUN && i < 128; i += 2) {
                                const float2 e = __ffma2_rn(make_float2(__uint_as_float(x[i]), __uint_as_float(x[i + 1])), scale2, nm);
                                const float2 w = decltype(poly)::value && (i >> 1) % POLY_OF == POLY_OF - 1 ? ex2_poly(e) : make_float2(ex2_approx(e.x), ex2_approx(e.y));
                                x[i] = __float_as_uint(w.x);
                                x[i + 1] = __float_as_uint(w.y);
                            }
#pragma unroll
                            for (int i = c - RUN; i >= 0 && i < c; i += 2) {
                                const float2 w = make_float2(__uint_as_float(x[i]), __uint_as_float(x[i + 1]));
                                sum[(i >> 1) & 1] = __fadd2_rn(sum[(i >> 1) & 1], w);
                                x[i / 2] = pack<X>(w.x, w.y);
                            }
                        }
                        return (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
                    };
                    load();
                    // Most tiles raise no maximum by much: their weights are taken by the one there is, and their sum tells if it was too
                    // low.  Then, and where keys are masked, the maximum is sought first.  (Always to seek it took 342 us instead of 327,
                    // to seek it beside the weights 354.)  The polynomial would make small numbers of a large argument and of a NaN.
                    float alpha = 1.f, add = 0.f;
                    bool done = false;
                    if (__all_sync(0xffffffffu, lim >= KEYS && m > -INFINITY)) {
                        float poly_top = -INFINITY;
#pragma unroll
                        for (int i = 2 * (POLY_OF - 1); i < 128; i += 2 * POLY_OF) poly_top = max3_or_nan(poly_top, __uint_as_float(x[i]), __uint_as_float(x[i + 1]));
                        add = weights(std::true_type{});
                        done = __all_sync(0xffffffffu, add <= MOST && fmaf(poly_top, a.scale_log2e, -m) <= 8.f);
                        if (!done) load();
                    }
                    if (!done) {
                        if (lim < KEYS) {
#pragma unroll
                            for (int i = 0; i < 128; ++i)
                                if (i >= lim) x[i] = __float_as_uint(-INFINITY);
                        }
                        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                        for (int i = 0; i < 128; i += 2) mx[(i >> 1) & 3] = fmax3(mx[(i >> 1) & 3], __uint_as_float(x[i]), __uint_as_float(x[i + 1]));
                        const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * a.scale_log2e;
                        const bool raise = top > m;
                        if (raise) {
                            alpha = ex2_approx(m - top);  // 0 from -inf
                            m = top;
                        }
                        if (j > 0 && __any_sync(0xffffffffu, raise)) {
                            if (!wait(sh.o_full, q - streams, W_O, j)) break;
#pragma unroll 1
                            for (int c = 0; c < 64; c += 32) {
                                uint32_t y[32];
                                tmem_ld32(at_o + c, y);
                                tmem_wait_ld();
#pragma unroll
                                for (int i = 0; i < 32; ++i) y[i] = __float_as_uint(__uint_as_float(y[i]) * alpha);
                                tmem_st32(at_o + c, y);
                            }
                        }
                        add = weights(std::false_type{});
                    }
                    tmem_st32p(at_s, x);
                    tmem_st32p(at_s + 32, x + 32);
                    l = fmaf(l, alpha, add);
                    tmem_wait_st();
                }
                tc_fence_before_sync();
                mbar_arrive_warp(&sh.p_full[q % 3], lane);
            }
            m -= lift<X>();  // what the weights were taken by
#pragma unroll
            for (int i = 0; i < 64; ++i) o[i] = 0.f;
            if (ok && n > 0 && wait(sh.o_full, (n - 1) * streams + t, W_O, n) && live) {
                tmem_ld32p(at_o, reinterpret_cast<uint32_t*>(o));
                tmem_ld32p(at_o + 32, reinterpret_cast<uint32_t*>(o) + 32);
                tmem_wait_ld();
            }
        }
        if (valid && ok) {
            int row = row0 + r;
            asm volatile("" : "+r"(row));  // worked out again, not kept in registers all the while
            if (a.whole ? parts > 1 : a.slots > 1) {
                const int64_t at_slot = a.whole ? split * a.slot_rows + (int64_t)(item - a.first_split) * BLOCK + r
                                                : (args.own ? a.splits_p : split) * a.slot_rows + (int64_t)kvh * a.R + row;
                a.ml[at_slot] = make_float2(m, l);
                float4* to = reinterpret_cast<float4*>(a.part + at_slot * 64);
#pragma unroll
                for (int i = 0; i < 16; ++i) to[i] = make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
            } else {
                const float f = l != 0.f ? 1.f / l : 0.f;
                const Where to_row = where(row);
                uint4* to = reinterpret_cast<uint4*>(const_cast<X*>(row_of<X>(a.O, to_row.b, to_row.h, to_row.t)));
                if constexpr (LOW) {
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        to[i] = make_uint4(__float_as_uint(o[4 * i] * f), __float_as_uint(o[4 * i + 1] * f), __float_as_uint(o[4 * i + 2] * f), __float_as_uint(o[4 * i + 3] * f));
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        to[i] = make_uint4(pack<X>(o[8 * i] * f, o[8 * i + 1] * f), pack<X>(o[8 * i + 2] * f, o[8 * i + 3] * f),
                                           pack<X>(o[8 * i + 4] * f, o[8 * i + 5] * f), pack<X>(o[8 * i + 6] * f, o[8 * i + 7] * f));
                }
                a.LSE[to_row.b * a.lse_sB + to_row.h * a.lse_sH + to_row.t] = l != 0.f ? (m + log2f(l)) * LN2 : -INFINITY;
            }
        }
    }
    tc_fence_before_sync();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after_sync();
        tmem_dealloc(tmem, 512);
        if (lane == 0) report_abort(sh.abort, a.status);
    }
    if (args.late && blockIdx.x == gridDim.x - 1) pdl_wait();  // this kernel is complete when the one over the prefix is
}

template <class X>
int launch(const ManyArgs& args, int dtype, int64_t blocks, cudaStream_t stream) {
    typedef Many<X> C;
    static std::once_flag once[HK_MAX_DEVICES];
    static cudaError_t rc[HK_MAX_DEVICES];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= HK_MAX_DEVICES) return HK_ERR_CUDA;
    std::call_once(once[dev], [dev] { rc[dev] = cudaFuncSetAttribute(prefix_many_kernel<X>, cudaFuncAttributeMaxDynamicSharedMemorySize, Many<X>::SMEM); });
    if (rc[dev] != cudaSuccess) return HK_ERR_CUDA;
    if (blocks > 0x7fffffffLL) return HK_ERR_BAD_SHAPE;
    const PrefixArgs& a = args.p;
    CUtensorMap kp, vp, k, v;
    int s;
    if ((s = prefix_tile_map(&kp, a.Kp, dtype, 1, a.Hk, args.prefix ? a.P : 0, C::KEYS, false)) || (s = prefix_tile_map(&vp, a.Vp, dtype, 1, a.Hk, args.prefix ? a.P : 0, C::KEYS, true)) ||
        (s = prefix_tile_map(&k, a.K, dtype, a.B, a.Hk, args.own ? a.S : 0, C::KEYS, false)) || (s = prefix_tile_map(&v, a.V, dtype, a.B, a.Hk, args.own ? a.S : 0, C::KEYS, true)))
        return s;
    LaunchConfig lc((unsigned)blocks, Many<X>::THREADS, Many<X>::SMEM, stream, 1, true);
    if (cudaLaunchKernelEx(&lc.cfg, prefix_many_kernel<X>, kp, vp, k, v, args) != cudaSuccess) return check_launch();
    count_launch();
    return HK_OK;
}
int launch(const ManyArgs& args, int dtype, int64_t blocks, cudaStream_t stream) {
    return dtype == HK_F32 ? launch<float>(args, dtype, blocks, stream) : dtype == HK_BF16 ? launch<__nv_bfloat16>(args, dtype, blocks, stream) : launch<__half>(args, dtype, blocks, stream);
}

}  // namespace

ManyPlan many_plan(int dtype) { return dtype == HK_F32 ? ManyPlan{TILE, 64} : ManyPlan{2 * TILE, 128}; }
int launch_prefix_many(const PrefixArgs& a, int dtype, cudaStream_t stream) {
    return launch(ManyArgs{a, 0, 1, 0, a.tiles_p}, dtype, (int64_t)a.Hk * a.tiles_p * a.splits_p, stream);
}
int launch_own_many(const PrefixArgs& a, int dtype, cudaStream_t stream) {
    const int64_t items = (int64_t)a.B * a.Hk * a.tiles_o;
    return launch(ManyArgs{a, 1, a.whole, !a.whole && a.splits_p > 0, a.tiles_o}, dtype, a.whole ? a.first_split + (items - a.first_split) * a.slots : items, stream);
}

}  // namespace hk
