// Sliding-window attention with first tokens that stay visible, head_dim 64, grouped key / value heads:
//   out_i = sum_j p_ij v_j,  p_i = softmax over { j < kv_len : j < sinks or pos_i - left <= j <= pos_i + right } of scale q_i.k_j + mask_j
// (with causal_sinks of the first tokens, too, only j <= pos_i + right; that matters only where the first tokens and the window touch:
// behind a gap every query of an item is past them).
//
// The keys that a block of 128 queries can see are at most two runs: the first tokens [0, sinks) and the window
// [p_first - left, p_last + right], one run where they touch.  An item (128 queries of one head of one sequence) walks the
// runs in tiles of up to 128 keys that start where the run starts, not at multiples of 128; the last tile of a run is as
// short as the run needs, in steps of 32 keys (QK^T with N = 32 c, PV with K = 32 c, c chunks of softmax).  First tokens that fit
// behind the window's last, short tile share it; otherwise they have a tile of their own, four sinks a quarter of one.
//
// tcgen05 (S = Q K^T, O += P V), one softmax warpgroup, online softmax with lazy maximum; two CTAs per SM, so that one's exp
// pass covers the other's hand-offs.  How long an item takes depends on its sequence's length and on its place in it, so items
// are not dealt in advance: the grid has a CTA per item, and a running CTA takes over the next one that has not started
// (cluster launch control), prefetching its queries and scores while it is still at work on its own.
//
// 16384 causal queries, window 1024, 4 sinks, 16 / 4 heads, bf16: 141 us (67 GFLOP visible; the exp unit's floor is 58), 4 x 4096 queries,
// window 256 to both sides, ragged: 59 to 67 us.  With an additive mask, where every tile takes the edges' path, 190 and 77 (padding
// belongs in kv_len).  First tokens that share a tile: 11 x 1302 queries, window 142 to both sides, 16 sinks
// 69 -> 64 us, 16 x 393, window 6, 28 -> 24.7; windows of whole tiles pay up to 2 % for it (139.6 -> 142).  The exp unit is 56 % busy: the two softmax warps of a scheduler wait for fixed
// latencies and tend to be in the exp pass together.  Exponentials by a polynomial (1/4 of them 153 us), two threads per row
// (140), both passes rolled (155) did not help.
#include "linear_common.cuh"
#include "ptx.cuh"
#include "window.cuh"

namespace b200 {
using namespace win;
namespace {

constexpr int TQ = 128;                      // queries per item
constexpr int TK = 128;                      // keys per tile at most
constexpr int TILE_BYTES = 128 * HD * 2;
constexpr int CHUNK_BYTES = 32 * HD * 2;     // a load: 32 keys
constexpr float kLazyLog2 = 8.0f;            // the running maximum moves only when a tile exceeds it by more than 2^8

struct TileParams : WindowParams {
    uint32_t idesc_qk, idesc_pv;             // idesc_qk without its N field
    int n_qb;
};

// ---------------------------------------------------------------------------------------------------------------
// Roles (256 threads, two CTAs per SM; registers move from the control warpgroup to the softmax warpgroup):
//   warp 0     : producer, TMA loads of Q (two sets: this item's, the next one's) and of K / V tiles through a 2-stage ring,
//                and with a mask the tile's 128 additive values and visible bits;
//   warp 1     : UMMA issuer (one elected lane): S(j + 1) before PV(j), across items;
//   warp 2     : zeroes the V rows of a tile that no query may see (beyond the run, or dropped by the mask): their weight is
//                exactly 0, but 0 x NaN is not;
//   warp 3     : takes over items and hands their numbers to the others through a ring of kIds;
//   warps 4..7 : softmax, thread = query row.
// TMEM: S 128 columns, O 64, P 64 (half precision, the A operand of PV).
struct WCfg {
    static constexpr int THREADS = 256;
    static constexpr int REGS_CONTROL = 72, REGS_SOFTMAX = 184;
    static constexpr int NST = 2;
    static constexpr int OFF_Q = 0;
    static constexpr int OFF_K = 2 * TILE_BYTES;
    static constexpr int OFF_V = OFF_K + NST * TILE_BYTES;
    static constexpr int OFF_MASK = OFF_V + NST * TILE_BYTES;      // NST x 128 floats
    static constexpr int OFF_BITS = OFF_MASK + NST * TK * 4;       // NST x 4 words
    static constexpr int OFF_TAKEN = OFF_BITS + NST * 16;          // 16 bytes: the answer of a take-over
    static constexpr int kIds = 2;                                 // items on their way to the other roles
    static constexpr int OFF_ITEMS = OFF_TAKEN + 16;               // kIds x 48 bytes
    static constexpr int OFF_BAR = OFF_ITEMS + kIds * 48;
    static constexpr int SMEM = OFF_BAR + 384;
    static constexpr int kReaders = 7;                             // producer, issuer, V rows, four softmax warps
    static constexpr int TMEM_COLS = 256, COL_O = 128, COL_P = 192;
};
static_assert(128 * WCfg::REGS_CONTROL + 128 * WCfg::REGS_SOFTMAX <= 65536 / 2, "setmaxnreg moves registers inside the CTA's own share");

struct __align__(16) WItem {
    int b, head, q0;
    int lo, hi;               // the window of the item's first query
    int a_end, b_lo, b_hi;    // the runs
    int there;                // 0: no further item; 1 + the chunks of the first tokens that share the last tile
    __device__ __forceinline__ int shared() const { return there - 1; }
    __device__ __forceinline__ int tiles_a() const { return there > 1 ? 0 : (a_end + TK - 1) / TK; }
    __device__ __forceinline__ int tiles() const { return tiles_a() + (b_hi - b_lo + TK - 1) / TK; }
};
static_assert(sizeof(WItem) == 48, "two of them in WCfg::OFF_ITEMS");

// Asks for the first CTA of the grid that has not started; the answer arrives in shared memory and completes 16 bytes of `bar`.
__device__ __forceinline__ void take_over(void* answer, uint64_t* bar) {
    asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];"
                 ::"r"(smem_u32(answer)), "r"(smem_u32(bar))
                 : "memory");
}
// Its block index, or -1 if every CTA has started.  The slot is read through the generic proxy and written by the next request
// through the async one: the fence keeps that write behind this read (an item would be lost or done twice).
__device__ __forceinline__ int taken_over(const void* answer) {
    uint32_t ok, x;
    asm volatile(
        "{\n\t.reg .b128 h;\n\t.reg .pred p;\n\t"
        "ld.shared.b128 h, [%2];\n\t"
        "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, h;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t"
        "mov.u32 %1, 0;\n\t"
        "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %1, h;\n\t}"
        : "=r"(ok), "=r"(x)
        : "r"(smem_u32(answer))
        : "memory");
    fence_async_proxy_shared();
    return ok ? static_cast<int>(x) : -1;
}
struct WTile {
    int k0, end, own, chunks; // first key, end of its run, 32-key chunks of the run and all (the first tokens' behind them)
    __device__ __forceinline__ int first(int c) const { return c < own ? k0 + c * 32 : (c - own) * 32; }   // key of chunk c
    __device__ __forceinline__ int limit(int c, const WItem& it) const { return c < own ? end : (c < chunks ? it.a_end : 0); }
};

__device__ __forceinline__ WItem load_item(const TileParams& p, int id) {
    WItem it;
    // heads fastest: the heads of a group read the same keys and values
    it.head = id % p.heads;
    const int rest = id / p.heads;
    it.q0 = (rest % p.n_qb) * TQ;
    it.b = rest / p.n_qb;
    const Window w = first_window(p, it.b);
    it.lo = w.lo + it.q0;
    it.hi = w.hi + it.q0;
    const Runs r = visible_runs(p, sequence_keys(p, it.b), it.lo, it.hi + min(TQ, p.Sq - it.q0) - 1);
    it.a_end = r.a_end;
    it.b_lo = r.b_lo;
    it.b_hi = r.b_hi;
    it.there = 1;
    const int tiles_b = (r.b_hi - r.b_lo + TK - 1) / TK, a = (r.a_end + 31) >> 5;
    if (a > 0 && tiles_b > 0 && a + ((r.b_hi - r.b_lo - (tiles_b - 1) * TK + 31) >> 5) <= TK / 32) it.there = 1 + a;
    return it;
}
__device__ __forceinline__ WTile load_tile(const WItem& it, int j) {
    WTile t;
    const int n_a = it.tiles_a();
    t.k0 = j < n_a ? j * TK : it.b_lo + (j - n_a) * TK;
    t.end = j < n_a ? it.a_end : it.b_hi;
    t.own = (min(TK, t.end - t.k0) + 31) >> 5;
    t.chunks = t.own + (j == it.tiles() - 1 ? it.shared() : 0);
    return t;
}

// MASKED: scores are scaled (and given their additive mask, if there is one) before the maximum: with a mask, or a scale that is
// not positive; otherwise the scale is folded into the exponential.
template <int DT, bool MASKED>
__global__ void __launch_bounds__(WCfg::THREADS, 2)
window_attention_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                        const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ CUtensorMap tm_o, const TileParams p) {
    using C = WCfg;
    constexpr int NST = C::NST;
    extern __shared__ __align__(1024) uint8_t smem[];
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR);
    uint64_t* q_full = bars;                 // [2]
    uint64_t* q_free = q_full + 2;           // [2] the item's output, staged in the place of its queries, has been read
    uint64_t* k_full = q_free + 2;           // [NST]
    uint64_t* v_full = k_full + NST;
    uint64_t* v_ready = v_full + NST;        // the rows that nobody may see are zero
    uint64_t* k_empty = v_ready + NST;
    uint64_t* v_empty = k_empty + NST;
    uint64_t* m_full = v_empty + NST;        // mask values and bits written (32 arrivals)
    uint64_t* s_full = m_full + NST;
    uint64_t* s_free = s_full + 1;           // the scores are in registers (4 arrivals)
    uint64_t* p_full = s_free + 1;           // 4 arrivals
    uint64_t* o_full = p_full + 1;
    uint64_t* taken = o_full + 1;
    uint64_t* id_full = taken + 1;           // [kIds]
    uint64_t* id_free = id_full + C::kIds;   // [kIds], a reader's arrival each
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(id_free + C::kIds);
    volatile uint32_t* abort_flag = tmem_slot + 1;
    WItem* items = reinterpret_cast<WItem*>(smem + C::OFF_ITEMS);   // [kIds]
    float* mask_s = reinterpret_cast<float*>(smem + C::OFF_MASK);
    uint32_t* bits_s = reinterpret_cast<uint32_t*>(smem + C::OFF_BITS);

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if ((smem_u32(smem) & 1023u) != 0) {
        if (tid == 0 && p.status) atomicOr(p.status, 4u);
        return;
    }
    if (tid == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(&q_full[i], 1);
            mbar_init(&q_free[i], 4);
        }
        for (int i = 0; i < NST; ++i) {
            mbar_init(&k_full[i], 1);
            mbar_init(&v_full[i], 1);
            mbar_init(&v_ready[i], 32);
            mbar_init(&k_empty[i], 1);
            mbar_init(&v_empty[i], 1);
            mbar_init(&m_full[i], 32);
        }
        mbar_init(s_full, 1);
        mbar_init(s_free, 4);
        mbar_init(p_full, 4);
        mbar_init(o_full, 1);
        mbar_init(taken, 1);
        for (int i = 0; i < C::kIds; ++i) {
            mbar_init(&id_full[i], 1);
            mbar_init(&id_free[i], C::kReaders);
        }
        *abort_flag = 0;
        mbar_fence_init();
        prefetch_tmap(&tm_q);
        prefetch_tmap(&tm_k);
        prefetch_tmap(&tm_v);
    }
    if (warp == 1) {
        tmem_alloc(tmem_slot, C::TMEM_COLS);
        tmem_relinquish();
    }
    tcgen05_fence_before();
    __syncthreads();
    tcgen05_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    pdl_launch_dependents();
    pdl_wait();   // q, k, v, kv_len and q_start come from earlier kernels; the output may still be read by one

    constexpr bool masked = MASKED;
    // The CTA's next item; `n` counts the caller's reads.  A warp reads as one (lane 0 arrives), the issuer is a single thread.
    auto next_item = [&](uint32_t& n, WItem& it) -> bool {
        const uint32_t slot = n % C::kIds;
        if (!mbar_wait_small(&id_full[slot], (n / C::kIds) & 1u, abort_flag)) return false;
        it = items[slot];
        mbar_arrive(&id_free[slot]);
        ++n;
        return it.there != 0;
    };
    auto next_item_warp = [&](uint32_t& n, WItem& it) -> bool {
        const uint32_t slot = n % C::kIds;
        const bool ok = mbar_wait_small(&id_full[slot], (n / C::kIds) & 1u, abort_flag);
        if (!__all_sync(0xffffffffu, ok)) return false;
        it = items[slot];
        __syncwarp();
        if (lane == 0) mbar_arrive(&id_free[slot]);
        ++n;
        return it.there != 0;
    };
    // Items without a visible key have no tiles: only the softmax warpgroup, which writes their zeros, stops at them.  `k`
    // counts the others (query set and phase), `t` tiles (ring stage and phase).
    if (warp < 4) {
        setmaxnreg_dec<C::REGS_CONTROL>();
        if (warp == 0) {
            // ------------------------------------------------------------ producer
            bool ok = true;
            uint32_t k = 0, t = 0, n = 0;
            WItem it;
            while (ok && next_item_warp(n, it)) {
                const int n_tiles = it.tiles();
                if (n_tiles == 0) continue;
                const int kv_col = it.head / p.group * HD;
                const uint32_t set = k & 1u;
                if (!mbar_wait_small(&q_free[set], ((k >> 1) & 1u) ^ 1u, abort_flag)) { ok = false; break; }
                if (lane == 0) {
                    mbar_expect_tx(&q_full[set], TILE_BYTES);
                    tma_load_3d(smem + C::OFF_Q + set * TILE_BYTES, &tm_q, &q_full[set], it.head * HD, it.q0, it.b);
                }
                ++k;
#pragma unroll 1
                for (int j = 0; j < n_tiles; ++j, ++t) {
                    const WTile tl = load_tile(it, j);
                    const int st = static_cast<int>(t % NST);
                    const uint32_t ph = ((t / NST) & 1u) ^ 1u;
                    if (!mbar_wait_small(&k_empty[st], ph, abort_flag)) { ok = false; break; }
                    if (lane == 0) mbar_expect_tx(&k_full[st], tl.chunks * CHUNK_BYTES);
                    __syncwarp();
                    if (lane < tl.chunks)
                        tma_load_3d(smem + C::OFF_K + st * TILE_BYTES + lane * CHUNK_BYTES, &tm_k, &k_full[st], kv_col, tl.first(lane), it.b);
                    if (!mbar_wait_small(&v_empty[st], ph, abort_flag)) { ok = false; break; }   // also: the stage's mask is done with
                    if (lane == 0) mbar_expect_tx(&v_full[st], tl.chunks * CHUNK_BYTES);
                    __syncwarp();
                    if (lane < tl.chunks)
                        tma_load_3d(smem + C::OFF_V + st * TILE_BYTES + lane * CHUNK_BYTES, &tm_v, &v_full[st], kv_col, tl.first(lane), it.b);
                    if (masked) {
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            const int key = tl.first(c) + lane;
                            float m = 0.f;
                            bool seen = false;
                            if (key < tl.limit(c, it) && p.mask_add != nullptr) {
                                m = p.mask_add[static_cast<long long>(it.b) * p.Sk + key];
                                seen = m > p.mask_below;
                            }
                            mask_s[st * TK + c * 32 + lane] = seen ? m * kLog2e : 0.f;
                            const uint32_t word = __ballot_sync(0xffffffffu, seen);
                            if (lane == 0) bits_s[st * 4 + c] = p.mask_add != nullptr ? word : 0xFFFFFFFFu;
                        }
                        mbar_arrive(&m_full[st]);
                    }
                }
            }
            __syncwarp();
        } else if (warp == 1) {
            // ------------------------------------------------------------ UMMA issuer
            if (elect_one()) {
                const uint64_t dq0 = make_smem_desc_sw128(smem_u32(smem + C::OFF_Q));
                const uint64_t dk0 = make_smem_desc_sw128(smem_u32(smem + C::OFF_K));
                const uint64_t dv0 = make_smem_desc_sw128(smem_u32(smem + C::OFF_V));
                uint32_t n_s = 0, n_pv = 0;   // QK^T and PV issued so far
                // S of tile j of the CTA's k-th item, once the softmax has taken the scores in front of it
                auto issue_s = [&](const WItem& it, int j, uint32_t k) -> bool {
                    const int st = static_cast<int>(n_s % NST);
                    if (j == 0 && !mbar_wait_small(&q_full[k & 1u], (k >> 1) & 1u, abort_flag)) return false;
                    if (!mbar_wait_small(&k_full[st], (n_s / NST) & 1u, abort_flag)) return false;
                    if (!mbar_wait_small(s_free, (n_s & 1u) ^ 1u, abort_flag)) return false;
                    tcgen05_fence_after();
                    const uint32_t idesc = p.idesc_qk | (static_cast<uint32_t>(load_tile(it, j).chunks * 4) << 17);
                    const uint64_t a = dq0 + static_cast<uint64_t>((k & 1u) * (TILE_BYTES >> 4));
                    const uint64_t b = dk0 + static_cast<uint64_t>(st * (TILE_BYTES >> 4));
#pragma unroll
                    for (int e = 0; e < HD / 16; ++e) umma_f16_ss(tmem_base, a + 2u * e, b + 2u * e, idesc, e != 0 ? 1u : 0u);
                    umma_commit(s_full);
                    umma_commit(&k_empty[st]);
                    ++n_s;
                    return true;
                };
                auto issue_pv = [&](const WItem& it, int j) -> bool {
                    const int st = static_cast<int>(n_pv % NST);
                    if (!mbar_wait_small(&v_ready[st], (n_pv / NST) & 1u, abort_flag)) return false;
                    if (!mbar_wait_small(p_full, n_pv & 1u, abort_flag)) return false;
                    tcgen05_fence_after();
                    const int steps = load_tile(it, j).chunks * 2;
                    const uint64_t b = dv0 + static_cast<uint64_t>(st * (TILE_BYTES >> 4));
#pragma unroll 2
                    for (int e = 0; e < steps; ++e)   // P: 8 columns per 16 keys, V: 2 KB per 16 keys
                        umma_f16_ts(tmem_base + C::COL_O, tmem_base + C::COL_P + e * 8, b + static_cast<uint64_t>(e * (2048 >> 4)),
                                    p.idesc_pv, (j | e) != 0 ? 1u : 0u);
                    umma_commit(o_full);
                    umma_commit(&v_empty[st]);
                    ++n_pv;
                    return true;
                };
                uint32_t n = 0;
                // The next item that has tiles: 1 found, 0 there is none, and, unless `wait`, -1: not known yet.  It must not be
                // waited for with a tile's PV outstanding: the softmax warps read on in the ring only when their item is done.
                auto next = [&](WItem& it, bool wait) -> int {
                    for (;;) {
                        const uint32_t slot = n % C::kIds;
                        if (!wait && !mbar_try_wait(&id_full[slot], (n / C::kIds) & 1u)) return -1;
                        if (!next_item(n, it)) return 0;
                        if (it.tiles() != 0) return 1;
                    }
                };
                WItem it, it_n;
                uint32_t k = 0;
                int there = next(it, true);
                bool ok = there != 1 || issue_s(it, 0, k);
                while (ok && there == 1) {
                    const int n_tiles = it.tiles();
                    for (int j = 0; ok && j < n_tiles; ++j) {
                        if (j + 1 < n_tiles) {   // the following scores before this tile's PV
                            ok = issue_s(it, j + 1, k);
                        } else {
                            there = next(it_n, false);
                            if (there == 1) ok = issue_s(it_n, 0, k + 1);
                        }
                        ok = ok && issue_pv(it, j);
                        if (ok && there == -1) {
                            there = next(it_n, true);
                            if (there == 1) ok = issue_s(it_n, 0, k + 1);
                        }
                    }
                    it = it_n;
                    ++k;
                }
            }
            __syncwarp();
        } else if (warp == 2) {
            // ------------------------------------------------------------ V rows that nobody may see
            bool ok = true;
            uint32_t t = 0, n = 0;
            WItem it;
            while (ok && next_item_warp(n, it)) {
                const int n_tiles = it.tiles();
                for (int j = 0; j < n_tiles; ++j, ++t) {
                    const WTile tl = load_tile(it, j);
                    const int st = static_cast<int>(t % NST);
                    const uint32_t ph = (t / NST) & 1u;
                    if (!mbar_wait_small(&v_full[st], ph, abort_flag)) { ok = false; break; }
                    if (masked && !mbar_wait_small(&m_full[st], ph, abort_flag)) { ok = false; break; }
                    __syncwarp();
                    if (masked || tl.end - tl.k0 < tl.own * 32 || tl.own < tl.chunks) {
                        uint8_t* v = smem + C::OFF_V + st * TILE_BYTES;
#pragma unroll 1
                        for (int c = 0; c < tl.chunks; ++c) {
                            uint32_t hide = ~low_bits(tl.limit(c, it) - tl.first(c));
                            if (masked) hide |= ~bits_s[st * 4 + c];
                            while (hide != 0) {   // four rows of 128 bytes at a time, 8 lanes each (zeros need no swizzle)
                                uint32_t rest = hide;
                                int row = -1;
                                for (int i = 0; i < 4 && rest != 0; ++i) {
                                    if (i == (lane >> 3)) row = __ffs(rest) - 1;
                                    rest &= rest - 1u;
                                }
                                if (row >= 0)
                                    *reinterpret_cast<uint4*>(v + (c * 32 + row) * 128 + (lane & 7) * 16) = make_uint4(0, 0, 0, 0);
                                hide = rest;
                            }
                        }
                        fence_async_proxy_shared();   // the UMMA reads shared memory through the async proxy
                    }
                    mbar_arrive(&v_ready[st]);
                }
            }
            __syncwarp();
        } else {
            // ------------------------------------------------------------ items: this CTA's own, then those it takes over
            if (elect_one()) {
                int id = blockIdx.x;
                for (uint32_t n = 0;; ++n) {
                    const uint32_t slot = n % C::kIds;
                    // the next one is asked for while this one is looked up
                    if (id >= 0) {
                        mbar_expect_tx(taken, 16);
                        take_over(smem + C::OFF_TAKEN, taken);
                    }
                    if (!mbar_wait_small(&id_free[slot], ((n / C::kIds) & 1u) ^ 1u, abort_flag)) break;
                    WItem it = {};
                    if (id >= 0) it = load_item(p, id);
                    items[slot] = it;
                    mbar_arrive(&id_full[slot]);
                    if (id < 0) break;   // every CTA has started: not asked again
                    if (!mbar_wait_small(taken, n & 1u, abort_flag)) break;
                    id = taken_over(smem + C::OFF_TAKEN);
                }
            }
            __syncwarp();
        }
    } else {
        setmaxnreg_inc<C::REGS_SOFTMAX>();
        // ------------------------------------------------------------ softmax
        const int r_in_tile = tid - 128;
        const uint32_t t_s = tmem_base + (static_cast<uint32_t>((warp & 3) * 32) << 16);
        const uint32_t t_o = t_s + C::COL_O, t_p = t_s + C::COL_P;
        uint32_t t = 0, n = 0, k = 0;
        bool ok = true, staged = false;   // staged: item k - 1's output is on its way out of query set (k - 1) & 1
        WItem it;
        while (ok && next_item_warp(n, it)) {
            const int n_tiles = it.tiles();
            if (n_tiles == 0) {   // no key: zeros
                const int q = it.q0 + r_in_tile;
                uint16_t* dst = static_cast<uint16_t*>(p.out) + it.b * p.o_batch + q * p.ldo + it.head * HD;
                if (q < p.Sq)
#pragma unroll 1
                    for (int g = 0; g < HD / 8; ++g) *reinterpret_cast<uint4*>(dst + g * 8) = make_uint4(0, 0, 0, 0);
                continue;
            }
            // what every row of the item sees: keys [all_lo, all_hi] (and the first tokens); what this row does
            const int all_lo = it.lo + min(TQ, p.Sq - it.q0) - 1, all_hi = it.hi;
            // tiles [0, plain_a) and [plain_lo, plain_hi): every key visible to every row
            const int n_a = it.tiles_a(), plain_a = masked ? 0 : it.a_end / TK;
            const int plain_lo = n_a + (max(all_lo - it.b_lo, 0) + TK - 1) / TK;
            const int plain_hi = masked ? 0 : n_a + max(min(it.b_hi, all_hi + 1) - it.b_lo, 0) / TK;
            int k0 = n_a > 0 ? 0 : it.b_lo, end = n_a > 0 ? it.a_end : it.b_hi;
            const int row_lo = it.lo + r_in_tile, row_hi = it.hi + r_in_tile, row_first = first_tokens(p, row_hi);
            float m_run = -INFINITY, l_run = 0.f;
            for (int j = 0; j < n_tiles; ++j, ++t) {
                const int own = (min(TK, end - k0) + 31) >> 5, with = j + 1 == n_tiles ? it.shared() : 0, chunks = own + with;
                int first = k0, limit = end;   // of the chunk at hand, behind the run's own the first tokens'
                const int st = static_cast<int>(t % NST);
                const bool plain = j < plain_a || (j >= plain_lo && j < plain_hi);
                k0 += TK;
                if (j + 1 == n_a) {
                    k0 = it.b_lo;
                    end = it.b_hi;
                }
                if (masked && !mbar_wait_small(&m_full[st], (t / NST) & 1u, abort_flag)) { ok = false; break; }
                if (!mbar_wait_small(s_full, t & 1u, abort_flag)) { ok = false; break; }
                __syncwarp();
                tcgen05_fence_after();
                // Hidden keys become -inf in TMEM, and so does what lies behind a short tile's last chunk; from there on all kinds
                // of tiles share one path.  What bounds this kernel first is fetching instructions: with the edges' code in the
                // passes below, unrolled four times over, and unrolled waits it was 69 KB long and took 150 us for 16384 causal
                // queries of 16 heads, window 1024; 49 KB took 139.6.
                if (!plain) {
#pragma unroll 1
                    for (int c = 0; c < 4; ++c) {
                        uint32_t s[32];
                        uint32_t bits = (low_bits(row_hi + 1 - first) & ~low_bits(row_lo - first)) | low_bits(row_first - first);
                        bits &= low_bits(limit - first);
                        first += 32;
                        if (c + 1 == own) {
                            first = 0;
                            limit = with != 0 ? it.a_end : 0;
                        }
                        tmem_ld_32x32b_x32(t_s + c * 32, s);
                        tmem_ld_wait(s);
                        if (masked) {
                            if (p.mask_add != nullptr) {
                                bits &= bits_s[st * 4 + c];
#pragma unroll
                                for (int e = 0; e < 32; ++e)
                                    s[e] = __float_as_uint(fmaf(__uint_as_float(s[e]), p.scale_log2, mask_s[st * TK + c * 32 + e]));
                            } else {
#pragma unroll
                                for (int e = 0; e < 32; ++e) s[e] = __float_as_uint(__uint_as_float(s[e]) * p.scale_log2);
                            }
                        }
#pragma unroll
                        for (int e = 0; e < 32; ++e)
                            if ((bits & (1u << e)) == 0) s[e] = 0xFF800000u;
                        tmem_st_32x32b_x32(t_s + c * 32, s);
                    }
                    tmem_st_wait();
                }
                uint32_t s[TK];
#pragma unroll
                for (int c = 0; c < 4; ++c) tmem_ld_32x32b_x32(t_s + c * 32, reinterpret_cast<uint32_t(&)[32]>(s[c * 32]));
#pragma unroll
                for (int c = 0; c < 4; ++c) tmem_ld_wait(reinterpret_cast<uint32_t(&)[32]>(s[c * 32]));
                tcgen05_fence_before();
                __syncwarp();
                mbar_arrive_if(s_free, lane == 0);
                float tmx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int e = 0; e < TK; e += 2)
                    tmx[(e >> 1) & 3] = fmax3(tmx[(e >> 1) & 3], __uint_as_float(s[e]), __uint_as_float(s[e + 1]));
                float tmax = fmaxf(fmaxf(tmx[0], tmx[1]), fmaxf(tmx[2], tmx[3]));
                if (!masked) tmax *= p.scale_log2;   // (positive: other scales take the masked form)
                const bool move = tmax > m_run + kLazyLog2;
                const float m_new = move ? tmax : m_run;
                const float m_use = (m_new == -INFINITY) ? 0.f : m_new;
                const float alpha = move ? fast_exp2(m_run - m_use) : 1.f;
                // PV of the item's previous tile is complete: it read the P columns and wrote the accumulator
                if (j > 0 && !mbar_wait_small(o_full, (t - 1u) & 1u, abort_flag)) { ok = false; break; }
                __syncwarp();
                if (j > 0 && __any_sync(0xffffffffu, move)) {
                    tcgen05_fence_after();
#pragma unroll
                    for (int c = 0; c < HD / 16; ++c) {   // 16 columns at a time: the scores occupy most registers
                        uint32_t ro[16];
                        tmem_ld_32x32b_x16(t_o + c * 16, ro);
                        tmem_ld_wait(ro);
#pragma unroll
                        for (int e = 0; e < 16; ++e) ro[e] = __float_as_uint(__uint_as_float(ro[e]) * alpha);
                        tmem_st_32x32b_x16(t_o + c * 16, ro);
                    }
                }
                const float mul = masked ? 1.f : p.scale_log2;
                const uint64_t mul2 = pack_f32x2(mul, mul), neg2 = pack_f32x2(-m_use, -m_use);
                uint64_t ps2[2] = {0ull, 0ull};
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    if (c < chunks) {
                        // The weights are rounded to the operands' type for PV, half a step of it each (2^-11, 2^-8) and independent
                        // of one another: 2.3e-3 of the result's norm in bf16 where its own rounding is 1.7e-3.  A second product
                        // with what the rounding left would double PV and its conversions.  Their sum is kept unrounded.
                        uint32_t pk[16];
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            const int i = c * 32 + e * 2;
                            float x0, x1;
                            unpack_f32x2(fma_f32x2(pack_f32x2(__uint_as_float(s[i]), __uint_as_float(s[i + 1])), mul2, neg2), x0, x1);
                            x0 = fast_exp2(x0);
                            x1 = fast_exp2(x1);
                            ps2[e & 1] = add_f32x2(ps2[e & 1], pack_f32x2(x0, x1));
                            pk[e] = pack2t<DT>(x0, x1);
                        }
                        tmem_st_32x32b_x16(t_p + c * 16, pk);
                    }
                }
                float a0, a1, a2, a3;
                unpack_f32x2(ps2[0], a0, a1);
                unpack_f32x2(ps2[1], a2, a3);
                l_run = l_run * alpha + ((a0 + a1) + (a2 + a3));
                m_run = m_new;
                tmem_st_wait();
                tcgen05_fence_before();
                __syncwarp();
                mbar_arrive_if(p_full, lane == 0);
                if (j == 0 && staged) {   // the previous item's output has had this tile's time to leave
                    if (lane == 0) {
                        tma_store_wait_read<0>();
                        mbar_arrive(&q_free[(k - 1) & 1u]);
                    }
                    __syncwarp();
                    staged = false;
                }
            }
            if (!ok) break;
            if (!mbar_wait_small(o_full, (t - 1u) & 1u, abort_flag)) { ok = false; break; }
            __syncwarp();
            tcgen05_fence_after();
            // The output takes the place of the item's queries (its last QK^T is long done) and leaves by TMA, 32 rows of a warp at
            // a time, clipped at row Sq.  (Stored from registers, 16 bytes of 32 rows per instruction, it held the warps up for
            // 1600 to 3700 clocks an item.)
            // l_run is 0 where no key was visible (a sum of weights is at least the maximum's 2^-8), NaN where a score was
            const float inv = l_run == 0.f ? 0.f : 1.0f / l_run;
            uint8_t* strip = smem + C::OFF_Q + (k & 1u) * TILE_BYTES + (warp & 3) * 32 * 128;
#pragma unroll
            for (int c = 0; c < HD / 32; ++c) {
                uint32_t r[32];
                tmem_ld_32x32b_x32(t_o + c * 32, r);
                tmem_ld_wait(r);
                const bool none = l_run == 0.f;
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    uint4 qv;
                    qv.x = none ? 0u : pack2t<DT>(__uint_as_float(r[g * 8 + 0]) * inv, __uint_as_float(r[g * 8 + 1]) * inv);
                    qv.y = none ? 0u : pack2t<DT>(__uint_as_float(r[g * 8 + 2]) * inv, __uint_as_float(r[g * 8 + 3]) * inv);
                    qv.z = none ? 0u : pack2t<DT>(__uint_as_float(r[g * 8 + 4]) * inv, __uint_as_float(r[g * 8 + 5]) * inv);
                    qv.w = none ? 0u : pack2t<DT>(__uint_as_float(r[g * 8 + 6]) * inv, __uint_as_float(r[g * 8 + 7]) * inv);
                    *reinterpret_cast<uint4*>(strip + lane * 128 + (((c * 4 + g) ^ (lane & 7)) << 4)) = qv;
                }
            }
            fence_async_proxy_shared();
            __syncwarp();
            if (lane == 0 && it.q0 + (warp & 3) * 32 < p.Sq) {
                tma_store_3d(&tm_o, strip, it.head * HD, it.q0 + (warp & 3) * 32, it.b);
                tma_store_commit();
            }
            staged = true;
            ++k;
            tcgen05_fence_before();
        }
        if (lane == 0) tma_store_wait_read<0>();
        __syncwarp();
    }

    tcgen05_fence_before();
    __syncthreads();
    if (warp == 1) {
        if (*abort_flag != 0) let_copies_land();
        tcgen05_fence_after();
        tmem_dealloc(tmem_base, C::TMEM_COLS);
    }
    if (tid == 0 && *abort_flag != 0 && p.status != nullptr) atomicOr(p.status, 2u);
}

bool set_window_attributes(int dev) {
    static PerDeviceOnce once;
    return once.ensure(dev, []() {
        auto set = [](const void* f) {
            return cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, WCfg::SMEM) == cudaSuccess;
        };
        return set(reinterpret_cast<const void*>(window_attention_kernel<B200_F16, false>)) &&
               set(reinterpret_cast<const void*>(window_attention_kernel<B200_F16, true>)) &&
               set(reinterpret_cast<const void*>(window_attention_kernel<B200_BF16, false>)) &&
               set(reinterpret_cast<const void*>(window_attention_kernel<B200_BF16, true>));
    });
}

}  // namespace
}  // namespace b200

extern "C" int b200_window_attention_fwd(const B200WindowAttentionDesc* d, b200_stream_t stream_) {
    using namespace b200;
    if (!d || !d->q || !d->k || !d->v || !d->out) return B200_ERR_PARAM;
    if (d->B < 0 || d->Sq < 0 || d->Sk <= 0 || d->heads <= 0 || d->kv_heads <= 0 || d->heads % d->kv_heads || d->sinks < 0 ||
        (d->causal_sinks != 0 && d->causal_sinks != 1))
        return B200_ERR_PARAM;
    if (d->head_dim != HD) return B200_ERR_UNSUPPORTED;
    if (!is_half_dtype(d->dtype)) return B200_ERR_PARAM;
    const int64_t wq = static_cast<int64_t>(d->heads) * HD, wk = static_cast<int64_t>(d->kv_heads) * HD;
    if ((d->ldq % 8) || (d->ldk % 8) || (d->ldv % 8) || (d->ldo % 8)) return B200_ERR_PARAM;
    if ((d->q_batch % 8) || (d->k_batch % 8) || (d->v_batch % 8) || (d->o_batch % 8)) return B200_ERR_PARAM;
    if (d->ldq < wq || d->ldk < wk || d->ldv < wk || d->ldo < wq) return B200_ERR_PARAM;
    if (d->B > 1 && (d->q_batch <= 0 || d->k_batch <= 0 || d->v_batch <= 0)) return B200_ERR_PARAM;
    // no row of the output in two places: sequences behind one another, or their rows interleaved ([Sq, B, width])
    if (d->B > 1 && d->Sq > 0 && !(d->o_batch >= wq && (d->o_batch - wq) / d->ldo >= d->Sq - 1) &&
        !(d->o_batch >= wq && (d->ldo - wq) / d->o_batch >= d->B - 1))
        return B200_ERR_PARAM;
    if (!aligned16(d->q) || !aligned16(d->k) || !aligned16(d->v) || !aligned16(d->out)) return B200_ERR_PARAM;
    if (d->mask_add && d->mask_exclude_below != d->mask_exclude_below) return B200_ERR_PARAM;
    if (d->B > 65535 || d->heads > 65535 || d->Sq > (1 << 24) || d->Sk > (1 << 24)) return B200_ERR_UNSUPPORTED;
    if (d->B == 0 || d->Sq == 0) return B200_OK;
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return B200_ERR_LAUNCH;
    const int sms = lin::device_sm_count();
    if (sms <= 0) return B200_ERR_NOT_SM100;
    cudaStream_t stream = static_cast<cudaStream_t>(stream_);

    TileParams p;
    p.mask_add = d->mask_add;
    p.kv_len = d->kv_len;
    p.q_start = d->q_start;
    p.out = d->out;
    p.q = d->q;
    p.k = d->k;
    p.v = d->v;
    p.B = static_cast<int>(d->B);
    p.Sq = static_cast<int>(d->Sq);
    p.Sk = static_cast<int>(d->Sk);
    p.heads = d->heads;
    p.group = d->heads / d->kv_heads;
    p.ldq = d->ldq;
    p.ldk = d->ldk;
    p.ldv = d->ldv;
    p.ldo = d->ldo;
    const bool many = d->B > 1;   // one sequence: the batch strides mean nothing
    p.q_batch = many ? d->q_batch : d->Sq * d->ldq;
    p.k_batch = many ? d->k_batch : d->Sk * d->ldk;
    p.v_batch = many ? d->v_batch : d->Sk * d->ldv;
    p.o_batch = many ? d->o_batch : d->Sq * d->ldo;
    auto side = [](int64_t w) { return w < 0 || w > kUnlimited ? kUnlimited : static_cast<long long>(w); };
    p.left = side(d->left);
    p.right = side(d->right);
    p.sinks = d->sinks > d->Sk ? p.Sk : static_cast<int>(d->sinks);
    p.causal_sinks = d->causal_sinks;
    p.scale_log2 = d->scale * kLog2e;
    p.mask_below = d->mask_exclude_below > kLeastMask ? d->mask_exclude_below : kLeastMask;
    p.status = device_status_ptr();

    if (token_kernel_takes(p)) return launch_window_token(p, d->dtype, sms, stream);

    const long long n_qb = (d->Sq + TQ - 1) / TQ;
    const long long items = n_qb * d->heads * d->B;
    if (items > 0x7fff0000ll) return B200_ERR_UNSUPPORTED;
    p.n_qb = static_cast<int>(n_qb);
    const int fmt = d->dtype == B200_BF16 ? 1 : 0;
    p.idesc_qk = make_idesc_f16(TQ, 0, fmt, 0, 0);
    p.idesc_pv = make_idesc_f16(TQ, HD, fmt, 0, 1);   // V is MN-major
    const uint32_t box[3] = {HD, 128, 1};
    const uint64_t B = static_cast<uint64_t>(d->B);
    const uint64_t qd[3] = {static_cast<uint64_t>(wq), static_cast<uint64_t>(d->Sq), B};
    const uint64_t kd[3] = {static_cast<uint64_t>(wk), static_cast<uint64_t>(d->Sk), B};
    const uint64_t qs[2] = {static_cast<uint64_t>(d->ldq) * 2, static_cast<uint64_t>(p.q_batch) * 2};
    const uint64_t ks[2] = {static_cast<uint64_t>(d->ldk) * 2, static_cast<uint64_t>(p.k_batch) * 2};
    const uint64_t vs[2] = {static_cast<uint64_t>(d->ldv) * 2, static_cast<uint64_t>(p.v_batch) * 2};
    const uint64_t os[2] = {static_cast<uint64_t>(d->ldo) * 2, static_cast<uint64_t>(p.o_batch) * 2};
    const uint32_t strip[3] = {HD, 32, 1};
    CUtensorMap tq, tk, tv, to;
    if (!get_tensor_map(&tq, d->q, 3, qd, qs, box) || !get_tensor_map(&tk, d->k, 3, kd, ks, strip) ||
        !get_tensor_map(&tv, d->v, 3, kd, vs, strip) || !get_tensor_map(&to, d->out, 3, qd, os, strip))
        return B200_ERR_DRIVER;
    if (!set_window_attributes(dev)) return B200_ERR_LAUNCH;
    const dim3 grid(static_cast<unsigned>(items));
    const bool masked = d->mask_add != nullptr || !(d->scale > 0.f);
    auto kernel = d->dtype == B200_F16 ? (masked ? window_attention_kernel<B200_F16, true> : window_attention_kernel<B200_F16, false>)
                                       : (masked ? window_attention_kernel<B200_BF16, true> : window_attention_kernel<B200_BF16, false>);
    launch_kernel(kernel, grid, dim3(WCfg::THREADS), WCfg::SMEM, stream, tq, tk, tv, to, p);
    count_launch();
    return check_launch();
}
