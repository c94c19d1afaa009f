// Attention of up to 256 query rows against 128-token tiles on the 5th-generation tensor cores, for rows that see a
// window with sinks or a draft tree: two row streams per CTA, keys split over CTAs when there are few rows.
//
// Work item: one entry of the work list (a unit's tiles, or a part of them) and one KV head.  Per tile and stream
//     S[128 rows x 128 tokens] = Q . K^T      tcgen05.mma, both operands K-major in shared memory, fp32 in TMEM
//     P = 2^(scale S - m)                     one TMEM lane (= one row) per thread, 128 keys; P overwrites its S as 16-bit
//     O[128 rows x D] += P . V                tcgen05.mma, A from TMEM, V in place as an MN-major operand
// A unit of more than 128 rows runs its two row blocks as the two streams over the same tiles, so a K/V tile is loaded
// once for 256 rows; a smaller one deals its tiles to the streams alternately and joins the two states at the end.
// Either way the tensor pipe works on one stream while the other stream's warps make exponentials: two 128 x 128 x 128
// tiles, one per stream, cost the tensor pipe 1024 cycles and the special-function unit another 1024, and a single stream
// would spend them one after the other.  What bounds it: the two steps take 1700 cycles, 0.6 of the tensor pipe's rate (46 %
// of it and 50 % of the special-function unit's over a whole prefill chunk, masked and uneven tiles included),
// of which S alone, with both operands from shared memory, is at what shared memory delivers.  Steps of 64 keys were 13 %
// slower, streams that take no turns 15 %.  Measured: a prefill chunk of 2 x 2041 rows, 32 heads of 128, window 4096 and 16
// sinks, 275 GFLOP, in 304 us with its work list (0.90 PFLOP/s); a step with 48 trees of 27 rows at contexts to 8192, where
// the pool's bytes bound it, 886 MB in 184 us (4.8 TB/s).
//
// A row's running maximum is followed lazily: O in TMEM is rescaled only when the maximum has grown by more than 2^8, so
// the stored weights stay below 2^15 and the row sum carries the same factor, which cancels in O / l.
// Sums and states are 32-bit; weights are rounded to the pool's 16-bit type, as the tensor core takes its operands in one.
//
// Masks are 64-bit words: for a tile that is not visible as a whole, each thread forms the visibility of its row's 128
// keys as two words (window, sinks, shifted tree mask) and tests constant bits.  A masked weight is zero, but 0 * NaN would
// reach the rows: in tiles that some row sees in part only, one warp clears values that no row of the unit sees, and those
// that are not finite; a row that sees one of these gets NaN.
//
// Warp roles: 0-3 stream 0, 4-7 stream 1, 8 TMA producer, 9 and 10 MMA issuers of the two streams (9 owns the TMEM), 11
// looks values over.  An issuing warp is held up until the tensor pipe has room for its instructions; with a warp of its
// own, a stream's products are in the queue as soon as its weights are there.  All waits are bounded.
#include "tcgen05.cuh"
#include "tensor_maps.cuh"
#include "visible_plan.cuh"

namespace emlx {

constexpr int kWdSoftThreads = 256;
constexpr int kWdProducer = 8, kWdMma = 9;  // warps 9 and 10 issue the products of stream 0 and 1
constexpr int kWdThreads = kWdSoftThreads + 128;  // whole warpgroups, since registers are moved between them
// A softmax thread holds a row's 128 scores: it gets the registers that the copying and issuing warps do not need.
// Together they stay inside what the block is launched with, 168 x 384.
constexpr int kWdSoftRegs = 216, kWdOtherRegs = 72;
static_assert(kWdSoftThreads * kWdSoftRegs + 128 * kWdOtherRegs <= 168 * kWdThreads, "the warpgroups' shares exceed the block's registers");
constexpr int kRowBlock = 128;

struct WideParams {
    void* out;
    float* slots;  // partial states: [slot][kWideRows * (D + 2)]
    const int32_t* bt;
    const int32_t* kv_lens;
    const int32_t* qsl;
    int32_t* plan;
    int32_t* status;
    const uint64_t* bits;  // tree masks, windowed ones when there is a window
    Visibility vis;
    VisibleLayout L;
    long long num_blocks;
    int Hq, Hkv, G, MB;
    int bs, ppt_log;
    float scale_log2e;
};

template <int D>
struct WdCfg {
    static constexpr int HALVES = D / 64;
    static constexpr int QBLOCK = kRowBlock * D * 2;      // one row block of Q
    static constexpr int TILE = kTile * D * 2;            // one K or V tile
    static constexpr int OFF_RING = 2 * QBLOCK;
    // Ring of tile places, each a K and a V slot: tile t of an item lies in place t % PLACES.  PLACES is even, so that where the
    // streams take alternate tiles a place belongs to one of them, and whoever waits for a place has seen its every use.
    static constexpr int PLACES = D == 128 ? 2 : 4;
    static constexpr int OFF_BAR = OFF_RING + 2 * PLACES * TILE;
    static constexpr int SMEM = OFF_BAR + 512 + 1024;
    static constexpr size_t SLOT_FLOATS = (size_t)kWideRows * (D + 2);
};

struct WdBarriers {
    uint64_t full[8], empty[8];     // ring slots: 2 j = K of place j, 2 j + 1 = V
    uint64_t q_full, q_free;        // Q loaded; every QK of the item has read it
    uint64_t s_full[2];             // per stream: S complete (and with it every earlier product)
    uint64_t p_half[2], p_ready[2]; // per stream: P of the tile's first 64 keys written, all of P written
    uint64_t o_full[2];             // per stream: the item's last PV is complete
    uint64_t item_full[4];
    uint64_t item_done[2];          // the rows of an item of this parity are stored
    uint64_t xch;                   // exchange steps between the streams
    uint64_t v_seen[4];             // per ring place: its values have been looked over, and `odd` is that of its tile
    uint64_t turn[2];               // the tensor pipe is stream s's
    uint64_t drain;                 // every product of the CTA is complete
    int item_ring[4];
    alignas(16) uint32_t odd[4][4]; // per ring place: tokens of the tile whose values are not all finite
    uint32_t tmem_base;
    int abort_word;
};
static_assert(sizeof(WdBarriers) <= 512, "the barrier block has 512 bytes of shared memory");

struct WideItem : WideEntry {
    int head;
};
__device__ __forceinline__ WideItem wide_item(const WideParams& p, int idx) {
    WideItem it;
    const int e = idx / p.Hkv;
    (WideEntry&)it = ((const WideEntry*)(p.plan + p.L.entry))[e];
    it.head = idx - e * p.Hkv;
    it.slot += it.head * it.parts;
    return it;
}
// Which tiles hold values that some row of the unit must not meet: a masked weight is an exact zero, but 0 * NaN is not.
// `clear(tok)`: no row of the unit sees the token.  `mixed`: some rows may see a token of the tile and others not.
struct UnitValues {
    int kv_len, sinks, lo, lo_max, hi;
    bool rows;
    __device__ __forceinline__ UnitValues(const WideParams& p, const WideItem& it) {
        const int ctx = it.kv_len - it.q_len, R = it.q_len * p.G;
        kv_len = it.kv_len;
        sinks = p.vis.sinks;
        rows = it.q_len > 1 || it.tree != 0;  // (one token's rows agree, but a tree's bounds are not exact)
        lo = unit_lo(p.vis, it.tree != 0, it.row0, p.G, ctx, kv_len);
        lo_max = window_lo(p.vis, ctx, it.tree ? it.q_len : (min(it.row0 + kWideRows, R) - 1) / p.G + 1);
        hi = it.tree ? ctx : min(kv_len, ctx + it.row0 / p.G + 1);
    }
    __device__ __forceinline__ bool clear(int tok) const { return tok >= kv_len || (tok < lo && tok >= sinks); }
    __device__ __forceinline__ bool mixed(int t0) const {
        return rows && ((t0 < lo_max && t0 + kTile > max(lo, sinks) && lo_max > sinks) || (t0 + kTile > hi && t0 < kv_len));
    }
    __device__ __forceinline__ bool touched(int t0) const {
        return t0 + kTile > kv_len || (t0 < lo && t0 + kTile > sinks) || mixed(t0);
    }
};
// Uses of the ring's places so far: every role counts them the same way, item by item.
template <int PLACES>
struct RingCount {
    uint32_t used[PLACES];
    __device__ __forceinline__ RingCount() {
#pragma unroll
        for (int j = 0; j < PLACES; ++j) used[j] = 0;
    }
    __device__ __forceinline__ uint32_t use_of(int t) const {  // which use of its place tile t of the current item is
        uint32_t u = used[0];
#pragma unroll
        for (int j = 1; j < PLACES; ++j) u = (t % PLACES) == j ? used[j] : u;
        return u + (uint32_t)(t / PLACES);
    }
    __device__ __forceinline__ void finish(int count) {
#pragma unroll
        for (int j = 0; j < PLACES; ++j) used[j] += (uint32_t)((count - j + PLACES - 1) / PLACES);
    }
};

// Bits [from, to) of the 64 keys that start at `base`.
__device__ __forceinline__ uint64_t key_range(int from, int to, int base) {
    const int a = max(from - base, 0), b = min(to - base, 64);
    if (b <= a) return 0;
    return (b >= 64 ? ~0ull : (1ull << b) - 1) & ~((1ull << a) - 1);
}

// 2^x on the special-function unit; ex2(-inf) = 0
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// sm_100's packed and three-operand forms: two 32-bit elements per instruction
__device__ __forceinline__ uint64_t pack2u(uint32_t lo, uint32_t hi) { return (uint64_t)lo | ((uint64_t)hi << 32); }
__device__ __forceinline__ uint64_t pack2f(float lo, float hi) { return pack2u(__float_as_uint(lo), __float_as_uint(hi)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
// Waits, with a limit, until a barrier has no copy in flight: until the phase that is open completes, if bytes are
// expected in it.
__device__ __forceinline__ void drain_copies(uint64_t* bar) {
    int never = 0;
    for (uint32_t parity = 0; parity < 2; ++parity) {
        if (ptx::mbar_try_wait(bar, parity)) continue;      // the open phase has the other parity
        ptx::mbar_wait(bar, parity, &never, 1u << 14);      // no copy: the wait runs out
    }
}
// Two 16-bit values: acc + 0 * v, which is NaN once a value is infinite or NaN, and the pair with zeros in place of such values.
template <bool BF16>
__device__ __forceinline__ uint32_t times_zero(uint32_t v, uint32_t acc) {
    if constexpr (BF16) asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(acc) : "r"(v), "r"(0u), "r"(acc));
    else asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(acc) : "r"(v), "r"(0u), "r"(acc));
    return acc;
}
template <bool BF16>
__device__ __forceinline__ uint32_t finite_only(uint32_t v) {
    constexpr uint32_t kExp = BF16 ? 0x7f80u : 0x7c00u;
    if ((v & kExp) == kExp) v &= 0xffff0000u;
    if (((v >> 16) & kExp) == kExp) v &= 0x0000ffffu;
    return v;
}
// The rare paths stay out of the tile loop's instruction stream: a warp runs through that loop's straight code once per
// tile, and what lies between costs fetches even when it is skipped.
//
// Scores of this thread's row that it does not see become -inf: `seen_at(key)` gives the visibility of the 64 keys from
// `key` on.
template <typename F>
__device__ __forceinline__ void mask_scores(uint32_t s_addr, F seen_at, int t0) {
#pragma unroll 1
    for (int w = 0; w < 2; ++w) {
        const uint64_t seen = seen_at(t0 + 64 * w);
        if (__all_sync(0xffffffffu, seen == ~0ull)) continue;
#pragma unroll 1
        for (int c = 0; c < 2; ++c) {
            const uint32_t bits = c ? (uint32_t)(seen >> 32) : (uint32_t)seen;
            uint32_t v[32];
            tmem_ld32_nowait(s_addr + 64 * w + 32 * c, v);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 32; ++e)
                if (!(bits & (1u << e))) v[e] = 0xff800000u;  // -inf
            tmem_st32_nowait(s_addr + 64 * w + 32 * c, v);
        }
    }
    tmem_wait_st();
}
__device__ __forceinline__ void scale_columns(uint32_t addr, int chunks, float factor) {
#pragma unroll 1
    for (int c = 0; c < chunks; ++c) {
        uint32_t v[32];
        tmem_ld32_nowait(addr + 32 * c, v);
        tmem_wait_ld();
#pragma unroll
        for (int e = 0; e < 32; ++e) v[e] = __float_as_uint(__uint_as_float(v[e]) * factor);
        tmem_st32_nowait(addr + 32 * c, v);
    }
}

template <int D, bool BF16>
__global__ void __launch_bounds__(kWdThreads, 1)
attn_wide_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
                 const __grid_constant__ CUtensorMap vmap, const __grid_constant__ WideParams p) {
    using C = WdCfg<D>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    uint8_t* q_smem = smem;
    uint8_t* ring = smem + C::OFF_RING;
    WdBarriers* bars = (WdBarriers*)(smem + C::OFF_BAR);
    volatile int* abort_word = &bars->abort_word;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    if (tid == 0) {
        for (int s = 0; s < 2 * C::PLACES; ++s) {
            ptx::mbar_init(&bars->full[s], 1);
            ptx::mbar_init(&bars->empty[s], 2);  // two arrivals per use: one per stream, or both from the one that used it
        }
        ptx::mbar_init(&bars->q_full, 1);
        ptx::mbar_init(&bars->q_free, 2);  // one per stream
        for (int s = 0; s < 2; ++s) {
            ptx::mbar_init(&bars->s_full[s], 1);
            ptx::mbar_init(&bars->p_half[s], kRowBlock);
            ptx::mbar_init(&bars->p_ready[s], kRowBlock);
            ptx::mbar_init(&bars->o_full[s], 1);
            ptx::mbar_init(&bars->turn[s], 1);
        }
        for (int s = 0; s < 4; ++s) ptx::mbar_init(&bars->item_full[s], 1);
        for (int s = 0; s < 4; ++s) ptx::mbar_init(&bars->v_seen[s], 1);
        for (int s = 0; s < 2; ++s) ptx::mbar_init(&bars->item_done[s], kWdSoftThreads);
        ptx::mbar_init(&bars->xch, kWdSoftThreads);
        ptx::mbar_init(&bars->drain, 2);
        bars->abort_word = 0;
        ptx::fence_barrier_init();
        ptx::prefetch_tensormap(&qmap);
        ptx::prefetch_tensormap(&kmap);
        ptx::prefetch_tensormap(&vmap);
    }
    if (warp == kWdMma) tmem_alloc(&bars->tmem_base, 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = bars->tmem_base;
    const uint32_t tmem_S = tmem_base, tmem_O = tmem_base + 256;  // stream s: S at + 128 s, O at + 128 s
    // everything above is independent of earlier kernels; the work list, the pool and the queries are not
    grid_dep_wait();
    grid_dep_launch();
    int32_t* queue = p.plan + p.L.queue;
    const int items = p.plan[p.L.queue + 2] * p.Hkv;

    if (warp >= kWdProducer) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kWdOtherRegs));
        if (warp == kWdProducer) {
            // ------------------------------------------------------------------ TMA producer
            const uint64_t keep = ptx::l2_policy_evict_normal();
            RingCount<C::PLACES> uses;
            uint32_t done_seen = 0;
            int next = lane == 0 ? atomicAdd(queue, 1) : 0;
            bool last_pair = false;
            for (uint32_t k = 0;; ++k) {
                int idx = __shfl_sync(0xffffffffu, next, 0);
                if (idx >= items || *abort_word) idx = -1;
                if (lane == 0) {
                    bars->item_ring[k & 3] = idx;
                    ptx::mbar_arrive(&bars->item_full[k & 3]);
                }
                if (idx < 0) break;
                if (lane == 0) next = atomicAdd(queue, 1);  // the following item, drawn while this one is loaded
                const WideItem it = wide_item(p, idx);
                const int seq = it.seq, row0 = it.row0, tile_lo = it.tile_lo, qs = it.qs, q_len = it.q_len, kv_len = it.kv_len;
                const bool pair = q_len * p.G - row0 > kRowBlock;
                const int sinks_in = sink_tiles(p.vis.sinks, tile_lo);
                const int lo = unit_lo(p.vis, it.tree != 0, row0, p.G, kv_len - q_len, kv_len);
                // The item's Q replaces the last one's: every QK of that item must have read it, and where its streams joined
                // their states through the same memory, its rows must be stored.  (The done phases are waited for in turn, and
                // alternate between two barriers, since the last item may be done as well: a wait two phases behind never ends.)
                if (k > 0) {
                    const uint32_t need = last_pair ? k - 1 : k;
                    for (; done_seen < need; ++done_seen) ptx::mbar_wait(&bars->item_done[done_seen & 1], (done_seen >> 1) & 1, abort_word);
                    ptx::mbar_wait(&bars->q_free, (k - 1) & 1, abort_word);
                }
                last_pair = pair;
                if (lane == 0 && !*abort_word) {
                    ptx::mbar_arrive_expect_tx(&bars->q_full, (uint32_t)((pair ? 2 : 1) * C::QBLOCK));
                    for (int b = 0; b < (pair ? 2 : 1); ++b)
    #pragma unroll
                        for (int h = 0; h < C::HALVES; ++h)
                            ptx::tma_load_3d(q_smem + b * C::QBLOCK + h * (kRowBlock * 128), &qmap, &bars->q_full, 64 * h,
                                             it.head * p.G, qs + (row0 + b * kRowBlock) / p.G);
                }
                // page ids in batches of 32, two batches kept (K runs ahead of V): lane l holds page l % ppt of tile l / ppt
                const int ppt_log = p.ppt_log, ppt = 1 << ppt_log, per_batch = 32 >> ppt_log;
                auto load_pages = [&](int first) -> int {
                    const int t = first + (lane >> ppt_log);
                    if (t >= it.count) return -1;
                    const long long pidx = ((long long)tile_of(it.j0 + t, sinks_in, tile_lo) << ppt_log) + (lane & (ppt - 1));
                    return pidx < p.MB ? p.bt[(long long)seq * p.MB + pidx] : -1;
                };
                int pg_cur = load_pages(0), pg_next = load_pages(per_batch), pg_base = 0;
                auto issue = [&](int t, bool is_k) {
                    const uint32_t slot = 2 * (t % C::PLACES) + (is_k ? 0 : 1), use = uses.use_of(t);
                    if (use > 0) ptx::mbar_wait(&bars->empty[slot], (use - 1) & 1, abort_word);
                    const bool go = !*abort_word;
                    if (go && lane == 0) ptx::mbar_arrive_expect_tx(&bars->full[slot], C::TILE);
                    __syncwarp();
                    uint8_t* tile = ring + (size_t)slot * C::TILE;
                    const long long tok = (long long)tile_of(it.j0 + t, sinks_in, tile_lo) * kTile;
                    for (int sub = 0; sub < ppt; ++sub) {
                        const int at = ((t - pg_base) << ppt_log) + sub;
                        const int a = __shfl_sync(0xffffffffu, pg_cur, at & 31), b = __shfl_sync(0xffffffffu, pg_next, at & 31);
                        const int pg = at < 32 ? a : b;
                        if (go && elect_one()) {
                            const bool bad = pg < 0 || pg >= p.num_blocks;
                            const long long key = tok + (long long)sub * p.bs;
                            // a page that no row of the unit sees may be gone; a missing one reads as zero rows
                            if (is_k && bad && key < kv_len && (key < p.vis.sinks || key + p.bs > lo)) flag_error(p.status, EMLX_DEV_BAD_PAGE);
                            const int tok0 = bad ? -p.bs : pg * p.bs;
    #pragma unroll
                            for (int h = 0; h < C::HALVES; ++h)
                                ptx::tma_load_3d(tile + h * (kTile * 128) + (size_t)sub * p.bs * 128, is_k ? &kmap : &vmap, &bars->full[slot],
                                                 64 * h, it.head, tok0, keep);
                        }
                    }
                    __syncwarp();
                };
                // K runs a ring ahead of V: its slot is free behind QK, V's only behind PV
                for (int t = 0; t < min(C::PLACES, it.count); ++t) issue(t, true);
                for (int t = 0; t < it.count; ++t) {
                    issue(t, false);
                    if (t + C::PLACES < it.count) issue(t + C::PLACES, true);
                    if (t + 1 == pg_base + per_batch) {  // V below is all issued, and K at most PLACES <= per_batch tiles above
                        pg_base += per_batch;
                        pg_cur = pg_next;
                        pg_next = load_pages(pg_base + per_batch);
                    }
                }
                uses.finish(it.count);
            }
            if (*abort_word) {
                // a wait of this CTA gave up: its copies in flight must land before the block may leave
                __threadfence_block();
                for (int t = 0; t < 2 * C::PLACES; ++t) drain_copies(&bars->full[t]);
                drain_copies(&bars->q_full);
            }
        } else if (warp < kWdMma + 2) {
            // ------------------------------------------------------------------ MMA issuer of stream s
            const int s = warp - kWdMma;
            constexpr uint32_t idesc_qk = instr_desc(128, 128, BF16, false);
            constexpr uint32_t idesc_pv = instr_desc(128, D, BF16, true);
            const uint64_t q_desc0 = smem_desc(ptx::smem_u32(q_smem), 16, 1024);
            const uint64_t k_desc0 = smem_desc(ptx::smem_u32(ring), 16, 1024);
            const uint64_t v_desc0 = smem_desc(ptx::smem_u32(ring), kTile * 128, 1024);
            const uint32_t tS = tmem_S + 128 * s, tO = tmem_O + 128 * s;
            uint32_t p_phase = 0, t_phase = 0;
            RingCount<C::PLACES> uses;
            for (uint32_t k = 0;; ++k) {
                if (!ptx::mbar_wait(&bars->item_full[k & 3], (k >> 2) & 1, abort_word)) break;
                const int idx = bars->item_ring[k & 3];
                if (idx < 0) break;
                const WideItem it = wide_item(p, idx);
                const bool pair = it.q_len * p.G - it.row0 > kRowBlock;
                const int steps = pair ? it.count : (it.count - s + 1) / 2, other = pair ? it.count : (it.count - (s ^ 1) + 1) / 2;
                ptx::mbar_wait(&bars->q_full, k & 1, abort_word);
                if (steps == 0 && lane == 0) ptx::mbar_arrive(&bars->q_free);
                // S of step i is overwritten by QK of step i + 1: its softmax has arrived on p_ready by then, and PV of step i,
                // which reads P from the same columns, was issued before (the pipe runs a thread's products in issue order)
                auto issue_qk = [&](int i) {
                    const int t = pair ? i : 2 * i + s;
                    const uint32_t slot = 2 * (t % C::PLACES);
                    const bool ok = ptx::mbar_wait(&bars->full[slot], uses.use_of(t) & 1, abort_word);
                    tc_fence_after();
                    if (ok && elect_one()) {
                        const uint64_t qd = q_desc0 + (uint64_t)((pair ? s : 0) * (C::QBLOCK >> 4));
                        const uint64_t kd = k_desc0 + (uint64_t)(slot * (C::TILE >> 4));
#pragma unroll
                        for (int ks = 0; ks < D / 16; ++ks) {
                            const uint32_t off = (uint32_t)((ks >> 2) * ((kTile * 128) >> 4) + (ks & 3) * 2);
                            tc_mma_f16(tS, qd + off, kd + off, idesc_qk, ks > 0);
                        }
                        tc_commit(&bars->s_full[s]);
                        tc_commit(&bars->empty[slot]);
                        if (!pair) tc_commit(&bars->empty[slot]);
                        if (i == steps - 1) tc_commit(&bars->q_free);
                    }
                    __syncwarp();
                };
                if (steps > 0) issue_qk(0);
                for (int i = 0; i < steps; ++i, ++p_phase) {
                    const int t = pair ? i : 2 * i + s;
                    const uint32_t slot = 2 * (t % C::PLACES) + 1;
                    bool ok = ptx::mbar_wait(&bars->full[slot], uses.use_of(t) & 1, abort_word);
                    ok = ptx::mbar_wait(&bars->v_seen[t % C::PLACES], uses.use_of(t) & 1, abort_word) && ok;
                    const uint64_t vd = v_desc0 + (uint64_t)(slot * (C::TILE >> 4));
                    // The product starts on the first 64 keys while the softmax warps are at the others.  The rest, and QK behind
                    // it, go in turn with the other stream: two streams that are in step would share the pipe and then the
                    // special-function unit, one of the two always idle.
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        if (half == 1 && (s == 1 || i > 0)) {
                            ptx::mbar_wait(&bars->turn[s], t_phase & 1, abort_word);
                            ++t_phase;
                        }
                        ok = ptx::mbar_wait(half ? &bars->p_ready[s] : &bars->p_half[s], p_phase & 1, abort_word) && ok;
                        tc_fence_after();
                        if (ok && elect_one()) {
#pragma unroll
                            for (int kk = 4 * half; kk < 4 * half + 4; ++kk)
                                tc_mma_f16_ts(tO, tS + kk * 8, vd + (uint64_t)(kk * ((16 * 128) >> 4)), idesc_pv, i > 0 || kk > 0);
                            if (half == 1) {
                                tc_commit(&bars->empty[slot]);
                                if (!pair) tc_commit(&bars->empty[slot]);
                                if (i == steps - 1) tc_commit(&bars->o_full[s]);
                            }
                        }
                        __syncwarp();
                    }
                    if (i + 1 < steps) issue_qk(i + 1);
                    // stream 0 goes first and has as many steps or one more: a turn is given only where it will be taken
                    if (lane == 0 && (s == 0 ? i < other : i + 1 < other)) ptx::mbar_arrive(&bars->turn[s ^ 1]);
                }
                uses.finish(it.count);
            }
            if (elect_one()) tc_commit(&bars->drain);
            __syncwarp();
            int never = 0;  // (waited for even when another wait has given up)
            ptx::mbar_wait(&bars->drain, 0, &never);
        } else {
            // ------------------------------------------------------------------ values that are not for every row
            // In a tile that some row sees in part only, the values of tokens that no row sees are cleared, and so are values
            // that are not finite; the softmax threads are told where those were.  (One warp beside the tile loop: done by the
            // softmax threads themselves it cost a prefill chunk 7 to 13 %, and so 1 %; four reads in flight, not eight: 4 % better.)
            RingCount<C::PLACES> uses;
            for (uint32_t k = 0;; ++k) {
                if (!ptx::mbar_wait(&bars->item_full[k & 3], (k >> 2) & 1, abort_word)) break;
                const int idx = bars->item_ring[k & 3];
                if (idx < 0) break;
                const WideItem it = wide_item(p, idx);
                const int sinks_in = sink_tiles(p.vis.sinks, it.tile_lo);
                const UnitValues values(p, it);
                for (int t = 0; t < it.count; ++t) {
                    const int place = t % C::PLACES, t0 = tile_of(it.j0 + t, sinks_in, it.tile_lo) * kTile;
                    const bool mixed = values.mixed(t0);
                    const bool loaded = ptx::mbar_wait(&bars->full[2 * place + 1], uses.use_of(t) & 1, abort_word);
                    if (__all_sync(0xffffffffu, loaded) && values.touched(t0)) {
#pragma unroll 1
                        for (int w = 0; w < kTile / 32; ++w) {  // lane = token; eight neighbours start at different 16-byte pieces
                            uint8_t* row = ring + (size_t)(2 * place + 1) * C::TILE + (32 * w + lane) * 128;
                            const bool clear = values.clear(t0 + 32 * w + lane);
                            uint32_t acc = 0;  // stays zero as long as every value times zero is
                            if (mixed && !clear) {
#pragma unroll 4
                                for (int c = 0; c < 8 * C::HALVES; ++c) {
                                    const uint4 v = *(const uint4*)(row + (c >> 3) * (kTile * 128) + ((c ^ lane) & 7) * 16);
                                    acc = times_zero<BF16>(v.w, times_zero<BF16>(v.z, times_zero<BF16>(v.y, times_zero<BF16>(v.x, acc))));
                                }
                            }
                            const bool bad = (acc & 0x7fff7fffu) != 0;
                            const uint32_t word = __ballot_sync(0xffffffffu, bad);
                            if (lane == 0) bars->odd[place][w] = word;
                            if (clear || bad) {
#pragma unroll 1
                                for (int c = 0; c < 8 * C::HALVES; ++c) {
                                    uint4* at = (uint4*)(row + (c >> 3) * (kTile * 128) + ((c ^ lane) & 7) * 16);
                                    const uint4 v = *at;
                                    *at = clear ? make_uint4(0u, 0u, 0u, 0u)
                                                : make_uint4(finite_only<BF16>(v.x), finite_only<BF16>(v.y), finite_only<BF16>(v.z), finite_only<BF16>(v.w));
                                }
                            }
                        }
                        ptx::fence_proxy_async();  // the tensor core reads V through the async proxy
                    }
                    __syncwarp();
                    if (lane == 0) ptx::mbar_arrive(&bars->v_seen[place]);
                }
                uses.finish(it.count);
            }
        }
    } else {
        // ------------------------------------------------------------------ softmax: thread = row of stream g
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kWdSoftRegs));
        const int g = warp >> 2, r = tid & 127;
        const uint32_t lane_addr = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t s_addr = tmem_S + 128 * g + lane_addr, o_addr = tmem_O + 128 * g + lane_addr;
        uint32_t s_phase = 0, o_phase[2] = {0, 0}, x_phase = 0;
        RingCount<C::PLACES> uses;
        auto exchange = [&]() {  // every softmax thread: what was written before is visible behind it
            ptx::mbar_arrive(&bars->xch);
            ptx::mbar_wait(&bars->xch, x_phase & 1, abort_word);
            ++x_phase;
        };
        for (uint32_t k = 0;; ++k) {
            if (!ptx::mbar_wait(&bars->item_full[k & 3], (k >> 2) & 1, abort_word)) break;
            const int idx = bars->item_ring[k & 3];
            if (idx < 0) break;
            const WideItem it = wide_item(p, idx);
            const int row0 = it.row0, tile_lo = it.tile_lo, qs = it.qs, q_len = it.q_len, kv_len = it.kv_len;
            const int R = q_len * p.G, ctx = kv_len - q_len;
            const bool pair = R - row0 > kRowBlock, tree = it.tree != 0;
            const int sinks_in = sink_tiles(p.vis.sinks, tile_lo);
            const int block0 = row0 + (pair ? kRowBlock * g : 0);     // first row of this stream
            const int rows_here = min(kRowBlock, R - block0);
            // a warp whose 32 rows all lie past the unit keeps its appointments only; its lanes of S, P and O hold
            // garbage that nobody reads
            const bool dead = (warp & 3) * 32 >= rows_here;
            const int ti = min(block0 + r, R - 1) / p.G;              // this row's token
            const uint64_t* bits = tree ? p.bits + (long long)(qs + ti) * p.vis.words : nullptr;
            const uint64_t word0 = tree ? tree_word(p.vis, bits, 0, q_len) : 0;  // all of the mask up to 64 tokens
            const int n_new = tree ? tree_count(p.vis, p.vis.tree + (long long)(qs + ti) * p.vis.words, q_len) : ti + 1;
            const int hi = max(0, tree ? min(ctx, kv_len) : min(kv_len, ctx + ti + 1));  // end of the plain range
            const int lo = window_lo(p.vis, ctx, n_new), sinks = p.vis.sinks;
            // bounds over the stream's rows, for tiles that need no mask
            const int hi_min = tree ? ctx : min(kv_len, ctx + block0 / p.G + 1);
            const int lo_max = window_lo(p.vis, ctx, tree ? q_len : (block0 + rows_here - 1) / p.G + 1);
            const UnitValues values(p, it);
            const int steps = pair ? it.count : (it.count - g + 1) / 2;

            float m_ref = -INFINITY, l = 0.f;
            for (int i = 0; i < steps; ++i) {
                const int t = pair ? i : 2 * i + g;
                const int t0 = tile_of(it.j0 + t, sinks_in, tile_lo) * kTile;
                const bool whole = t0 + kTile <= hi_min && (t0 >= lo_max || t0 + kTile <= sinks);
                ptx::mbar_wait(&bars->s_full[g], s_phase & 1, abort_word);
                ++s_phase;
                tc_fence_after();
                // the keys [b, b + 64) that this row sees
                auto seen_at = [&](int b) {
                    uint64_t seen = key_range(lo, hi, b) | key_range(0, min(sinks, hi), b);
                    if (tree && b + 64 > ctx && b < kv_len) {
                        const int j = b - ctx;  // new token that key b is
                        if (j >= 0) {
                            seen |= (j < 64 ? word0 : tree_word(p.vis, bits, j >> 6, q_len)) >> (j & 63);
                            if ((j & 63) && p.vis.words > (j >> 6) + 1) seen |= tree_word(p.vis, bits, (j >> 6) + 1, q_len) << (64 - (j & 63));
                        } else if (j > -64) {
                            seen |= word0 << (-j);
                        }
                    }
                    return seen;
                };
                if (!dead) {
                    if (!whole) mask_scores(s_addr, seen_at, t0);
                    uint32_t sv[kTile];
                    uint64_t sum2[2] = {0, 0}, neg2 = 0;
                    const uint64_t scale2 = pack2f(p.scale_log2e, p.scale_log2e);
                    auto weights = [&](int c) {  // 32 keys
                        uint32_t packed[16];
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            const uint64_t x = fma2(pack2u(sv[32 * c + 2 * e], sv[32 * c + 2 * e + 1]), scale2, neg2);
                            // (A polynomial on the FMA pipe for every 2nd, 4th, 8th or 16th pair was measured: -15 %, -4 %, 0, 0 on
                            // a prefill chunk.  The unit is not what a tile waits for.)
                            const float p0 = ex2(__uint_as_float((uint32_t)x)), p1 = ex2(__uint_as_float((uint32_t)(x >> 32)));
                            sum2[e & 1] = add2(sum2[e & 1], pack2f(p0, p1));
                            if constexpr (BF16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(packed[e]) : "f"(p1), "f"(p0));
                            else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(packed[e]) : "f"(p1), "f"(p0));
                        }
                        tmem_st16_nowait(s_addr + 16 * c, packed);
                    };
#pragma unroll
                    for (int c = 0; c < kTile / 32; ++c) tmem_ld32_nowait(s_addr + 32 * c, sv + 32 * c);
                    tmem_wait_ld();
                    // The first half's weights are made with the reference the row has, and the tile's maximum is taken beside
                    // them, in issue slots the special-function unit leaves; only when it has outgrown the reference (the
                    // first tile, rarely a later one) are they made again.
                    // fp16 weights are stored as 2^(s - m_ref + 7): a key rounds to zero below 2^-32 of the reference only
                    constexpr float kShift = BF16 ? 0.0f : 7.0f;
#pragma unroll 1
                    for (;;) {
                        const float neg_m = kShift - (m_ref == -INFINITY ? 0.f : m_ref);
                        neg2 = pack2f(neg_m, neg_m);
                        sum2[0] = sum2[1] = 0;
                        weights(0);
                        weights(1);
                        float mx4[4];  // independent chains
#pragma unroll
                        for (int e = 0; e < 4; ++e) mx4[e] = __uint_as_float(sv[e]);
#pragma unroll
                        for (int e = 4; e + 1 < kTile; e += 2) mx4[(e >> 1) & 3] = max3(mx4[(e >> 1) & 3], __uint_as_float(sv[e]), __uint_as_float(sv[e + 1]));
                        const float m_new = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) * p.scale_log2e;
                        const bool grow = m_new > m_ref + 8.0f || (m_ref == -INFINITY && m_new > m_ref);
                        if (!__any_sync(0xffffffffu, grow)) break;
                        // (the S waited for was committed behind this stream's last PV, so O is complete)
                        float corr = 1.0f;
                        if (grow) {
                            corr = ex2(m_ref - m_new);
                            m_ref = m_new;
                        }
                        if (i > 0) {
                            scale_columns(o_addr, D / 32, corr);
                            l *= corr;
                        }
                    }
                    tmem_wait_st();
                    tc_fence_before();
                    ptx::mbar_arrive(&bars->p_half[g]);
                    weights(2);
                    weights(3);
                    const uint64_t both = add2(sum2[0], sum2[1]);
                    l += __uint_as_float((uint32_t)both) + __uint_as_float((uint32_t)(both >> 32));
                    tmem_wait_st();
                } else {
                    ptx::mbar_arrive(&bars->p_half[g]);
                }
                if (values.mixed(t0)) {  // a row that sees a value that is not finite gets NaN for its sum
                    const int place = t % C::PLACES;
                    ptx::mbar_wait(&bars->v_seen[place], uses.use_of(t) & 1, abort_word);
                    const uint4 odd = *(const uint4*)bars->odd[place];
                    if (odd.x | odd.y | odd.z | odd.w) {
                        const uint64_t seen = (seen_at(t0) & pack2u(odd.x, odd.y)) | (seen_at(t0 + 64) & pack2u(odd.z, odd.w));
                        if (seen) l = __int_as_float(0x7fffffff);
                    }
                }
                tc_fence_before();
                ptx::mbar_arrive(&bars->p_ready[g]);
            }
            uses.finish(it.count);

            // ---------------------------------------------------------------- the item's rows
            const bool other_ran = pair || it.count > 1;
            if (steps > 0) ptx::mbar_wait(&bars->o_full[g], o_phase[g] & 1, abort_word);
            int c_begin = 0, c_end = D / 32;  // 32-column chunks of O that this thread stores
            float l_tot = l, mine = 1.f, theirs = 0.f;
            float* xch = (float*)q_smem;
            if (!pair && other_ran) {
                // both streams hold the same rows over other tiles: each takes one half of the columns from the other,
                // through the memory of Q (all QK are complete behind both o_full)
                ptx::mbar_wait(&bars->o_full[g ^ 1], o_phase[g ^ 1] & 1, abort_word);
                xch[(2 * g) * kRowBlock + r] = m_ref;
                xch[(2 * g + 1) * kRowBlock + r] = l;
                exchange();
                const float m_o = xch[(2 * (g ^ 1)) * kRowBlock + r], l_o = xch[(2 * (g ^ 1) + 1) * kRowBlock + r];
                exchange();
                const float M = fmaxf(m_ref, m_o), M_safe = M == -INFINITY ? 0.f : M;
                mine = ex2(m_ref - M_safe);
                theirs = ex2(m_o - M_safe);
                // both add in the same order and get the same sum
                l_tot = g == 0 ? fmaf(l, mine, l_o * theirs) : fmaf(l_o, theirs, l * mine);
                m_ref = M;
                tc_fence_after();
                constexpr int HC = D / 64;  // chunks per half
                if (!dead) {
#pragma unroll 1
                    for (int c = 0; c < HC; ++c) {
                        uint32_t ov[32];
                        tmem_ld32_nowait(o_addr + 32 * ((g ^ 1) * HC + c), ov);
                        tmem_wait_ld();
#pragma unroll
                        for (int e = 0; e < 32; ++e) xch[((g ^ 1) * (D / 2) + 32 * c + e) * kRowBlock + r] = __uint_as_float(ov[e]);
                    }
                }
                exchange();
                c_begin = g * HC;
                c_end = c_begin + HC;
            } else {
                tc_fence_after();
                if (!pair && g == 1) c_end = 0;  // stream 0 had the only tile
            }
            const bool store = block0 + r < R && !dead;
            const float inv = l_tot != 0.f ? 1.0f / l_tot : 0.f;  // (a sum that is not a number stays one)
            const int oi = (block0 + r) / p.G, ohh = (block0 + r) - oi * p.G;
            uint4* dst = (uint4*)((uint16_t*)p.out + ((long long)(qs + oi) * p.Hq + it.head * p.G + ohh) * D);
            float* slot = p.slots + (size_t)(it.slot) * C::SLOT_FLOATS;
            const int srow = block0 - row0 + r;
            if (it.parts > 1 && store && c_begin == 0 && c_end > 0) {
                slot[kWideRows * D + srow] = m_ref;
                slot[kWideRows * (D + 1) + srow] = l_tot;
            }
#pragma unroll 1
            for (int c = c_begin; c < c_end && !dead; ++c) {
                uint32_t ov[32];
                tmem_ld32_nowait(o_addr + 32 * c, ov);
                tmem_wait_ld();
                if (!store) continue;
                float x[32];
#pragma unroll
                for (int e = 0; e < 32; ++e) {
                    x[e] = __uint_as_float(ov[e]);
                    // a weight of zero must not meet what an empty stream left in TMEM
                    if (!pair && other_ran)
                        x[e] = (mine > 0.f ? x[e] * mine : 0.f) + (theirs > 0.f ? xch[(32 * c + e) * kRowBlock + r] * theirs : 0.f);
                }
                if (it.parts > 1) {
                    float4* to = (float4*)(slot + (size_t)srow * D + 32 * c);
#pragma unroll
                    for (int e = 0; e < 8; ++e) to[e] = make_float4(x[4 * e], x[4 * e + 1], x[4 * e + 2], x[4 * e + 3]);
                } else {
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        uint32_t w[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float x0 = x[8 * q + 2 * e] * inv, x1 = x[8 * q + 2 * e + 1] * inv;
                            if constexpr (BF16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w[e]) : "f"(x1), "f"(x0));
                            else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(w[e]) : "f"(x1), "f"(x0));
                        }
                        dst[4 * c + q] = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                }
            }
            // the other stream's phase is seen through as well, so that no wait falls two phases behind it
            if (pair) ptx::mbar_wait(&bars->o_full[g ^ 1], o_phase[g ^ 1] & 1, abort_word);
            o_phase[0] += 1;
            o_phase[1] += other_ran ? 1 : 0;
            tc_fence_before();
            ptx::fence_proxy_async();  // the next item's Q arrives by TMA over the memory of the exchange
            ptx::mbar_arrive(&bars->item_done[k & 1]);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == kWdMma) tmem_dealloc(tmem_base, 512);
    if (*abort_word && tid == 0) flag_error(p.status, EMLX_DEV_WAIT_TIMEOUT);
    if (tid == 0) {
        // every draw of this CTA is behind us; the last CTA to get here puts the item counter back to zero
        __threadfence();
        if (atomicInc((unsigned int*)&queue[1], gridDim.x - 1) == gridDim.x - 1) queue[0] = 0;
    }
}

// Units that were split along their keys: one warp per row joins the parts' states (in part order) and stores the row.
// Bound by L2: every state is read once.  The work list comes from before the attention kernel, whose CTAs had all seen it
// complete when they let this grid start, so a row's whereabouts are looked up ahead of the wait; behind it a row takes
// two round trips, the parts' rows on their way together with their maxima and sums.
template <int D, bool BF16>
__global__ void __launch_bounds__(256, 4) wide_combine_kernel(const __grid_constant__ WideParams p) {
    grid_dep_launch();
    const int lane = threadIdx.x & 31;
    const int split = p.plan[p.L.queue + 3];
    constexpr size_t kSlot = WdCfg<D>::SLOT_FLOATS;
    constexpr int V = D / 32, kDeep = 8;
    const int total = split * p.Hkv * kWideRows;
    bool waited = false;
    for (int row = blockIdx.x * 8 + (threadIdx.x >> 5); row < total; row += gridDim.x * 8) {
        const int sr = row % kWideRows, rest = row / kWideRows, head = rest % p.Hkv, k = rest / p.Hkv;
        const WideSplit sp = ((const WideSplit*)(p.plan + p.L.split))[k];
        if (sr >= sp.rows) continue;
        const int parts = sp.parts, qs = sp.qs, r = sp.row0 + sr;
        const float* base = p.slots + (size_t)(sp.slot + head * parts) * kSlot;
        if (!waited) grid_dep_wait();
        waited = true;
        float v[kDeep][V];
        auto load = [&](int j0) {
#pragma unroll
            for (int q = 0; q < kDeep; ++q) {
                const float* src = base + (size_t)min(j0 + q, parts - 1) * kSlot + (size_t)sr * D + V * lane;
                if constexpr (V == 4) {
                    const float4 x = __ldcg((const float4*)src);
                    v[q][0] = x.x; v[q][1] = x.y; v[q][2] = x.z; v[q][3] = x.w;
                } else {
                    const float2 x = __ldcg((const float2*)src);
                    v[q][0] = x.x; v[q][1] = x.y;
                }
            }
        };
        load(0);
        float M = -INFINITY;
        for (int j = lane; j < parts; j += 32)
            if (__ldcg(base + j * kSlot + kWideRows * (D + 1) + sr) != 0.f) M = fmaxf(M, __ldcg(base + j * kSlot + kWideRows * D + sr));
        M = warp_max(M);
        float acc[V], den = 0.f;
#pragma unroll
        for (int e = 0; e < V; ++e) acc[e] = 0.f;
        for (int j0 = 0; j0 < parts; j0 += 32) {
            const int jl = j0 + lane, n = min(32, parts - j0);
            const float lp = jl < parts ? __ldcg(base + jl * kSlot + kWideRows * (D + 1) + sr) : 0.f;
            const float mp = jl < parts ? __ldcg(base + jl * kSlot + kWideRows * D + sr) : -INFINITY;
            const float w = lp != 0.f ? ex2(mp - M) : 0.f;
            den += warp_sum(w * lp);
            for (int j = 0; j < n; j += kDeep) {
                if (j0 + j > 0) load(j0 + j);
#pragma unroll
                for (int q = 0; q < kDeep; ++q) {
                    const float wj = __shfl_sync(0xffffffffu, w, (j + q) & 31);
                    if (j + q < n && wj > 0.f) {  // a part in which the row sees nothing holds no numbers
#pragma unroll
                        for (int e = 0; e < V; ++e) acc[e] = fmaf(wj, v[q][e], acc[e]);
                    }
                }
            }
        }
        const float inv = den != 0.f ? 1.0f / den : 0.f;
        const int oi = r / p.G, ohh = r - oi * p.G;
        uint32_t* dst = (uint32_t*)((uint16_t*)p.out + ((long long)(qs + oi) * p.Hq + head * p.G + ohh) * D + V * lane);
#pragma unroll
        for (int e = 0; e < V / 2; ++e) {
            uint32_t w;
            if constexpr (BF16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(acc[2 * e + 1] * inv), "f"(acc[2 * e] * inv));
            else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(acc[2 * e + 1] * inv), "f"(acc[2 * e] * inv));
            dst[e] = w;
        }
    }
    if (!waited) grid_dep_wait();  // what follows in the stream relies on this grid for the one before it as well
}

// ------------------------------------------------------------------------------------------ host
// A unit of more tiles than an SM's share is cut into at most twice as many parts as shares, so the split parts of a batch
// are at most two per CTA.
size_t wide_slot_bytes(int D) {
    const int sms = num_sms();
    return (size_t)2 * (sms > 0 && sms < kMaxGrid ? sms : kMaxGrid) * kWideRows * (D + 2) * sizeof(float);
}

// Q is [T, Hq, D]; a box of {64 columns, G heads, 128/G tokens} lands in shared memory as 128 rows in the unit's row
// order (token-major, then head), 128 bytes per row and swizzled like the K/V tiles.
static int encode_q_map(const emlx_attn_args* a, int D, int G, CUtensorMap* out) {
    EncodeTiledFn enc = encode_fn();
    if (!enc) return fail(EMLX_ERR_CUDA, "cuTensorMapEncodeTiled is not available from this driver");
    const cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)a->num_q_heads, (cuuint64_t)a->total_tokens};
    const cuuint64_t strides[2] = {(cuuint64_t)D * 2, (cuuint64_t)a->num_q_heads * D * 2};
    const cuuint32_t box[3] = {64, (cuuint32_t)G, (cuuint32_t)(kRowBlock / G)};
    const cuuint32_t ones[3] = {1, 1, 1};
    const CUtensorMapDataType dt = a->q_dtype == EMLX_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    const CUresult r = enc(out, dt, 3, const_cast<void*>(a->queries), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                           CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(EMLX_ERR_CUDA, "cuTensorMapEncodeTiled failed for the query tensor (%d)", (int)r);
    return EMLX_OK;
}

template <int D, bool BF16>
static int launch_wd(const CUtensorMap& qmap, const MapPair& maps, const WideParams& p, int grid, cudaStream_t stream) {
    using C = WdCfg<D>;
    auto kernel = attn_wide_kernel<D, BF16>;
    static DeviceOnce configured;
    EMLX_CUDA_OK(allow_dynamic_smem(kernel, C::SMEM, configured));
    EMLX_CUDA_OK(launch_pdl(kernel, grid, kWdThreads, C::SMEM, stream, qmap, maps.k, maps.v, p));
    EMLX_LAUNCHED();
    EMLX_CUDA_OK(launch_pdl(wide_combine_kernel<D, BF16>, 4 * num_sms(), 256, 0, stream, p));
    EMLX_LAUNCHED();
    return EMLX_OK;
}

int launch_wide(const emlx_attn_args* a, const emlx_pool* pool, const Visibility& vis, const VisibleLayout& L, float* slots,
                const MapPair& maps, cudaStream_t stream) {
    const int D = pool->head_dim, Hq = a->num_q_heads, Hkv = pool->num_kv_heads, G = Hq / Hkv;
    if (!prefill_supported(pool->kv_format, Hq, Hkv, D))
        return fail(EMLX_ERR_UNSUPPORTED, "256-row units need an fp16/bf16 pool, head_dim 64/128 and 128 %% (Hq/Hkv) == 0");
    CUtensorMap qmap;
    if (int rc = encode_q_map(a, D, G, &qmap)) return rc;
    WideParams p{};
    p.out = a->out; p.slots = slots; p.bt = a->block_tables; p.kv_lens = a->kv_lens; p.qsl = a->query_start_loc;
    p.plan = (int32_t*)a->plan; p.status = a->status; p.vis = vis; p.L = L;
    p.bits = vis.window > 0 ? (const uint64_t*)((int32_t*)a->plan + L.eff) : vis.tree;
    p.num_blocks = pool->num_blocks;
    p.Hq = Hq; p.Hkv = Hkv; p.G = G; p.MB = a->max_blocks_per_seq;
    p.bs = pool->block_size; p.ppt_log = pages_per_tile_log2(pool->block_size);
    p.scale_log2e = a->softmax_scale * 1.4426950408889634f;
    const int grid = num_sms() < kMaxGrid ? num_sms() : kMaxGrid;
    const bool bf16 = a->q_dtype == EMLX_BF16;
    if (D == 128) return bf16 ? launch_wd<128, true>(qmap, maps, p, grid, stream) : launch_wd<128, false>(qmap, maps, p, grid, stream);
    return bf16 ? launch_wd<64, true>(qmap, maps, p, grid, stream) : launch_wd<64, false>(qmap, maps, p, grid, stream);
}

}  // namespace emlx
