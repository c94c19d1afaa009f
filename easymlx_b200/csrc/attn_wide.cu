// Attention of up to 256 query rows against 128-token tiles on the 5th-generation tensor cores, for rows that see a
// window with sinks or a draft tree: two row streams per CTA, keys split over CTAs when there are few rows.
//
// Work item: one entry of the work list (a unit's tiles, or a part of them) and one KV head.  Per tile and stream
//     S[128 rows x 128 tokens] = Q . K^T      tcgen05.mma, both operands K-major in shared memory, fp32 in TMEM
//     P = 2^(scale S - m)                     one TMEM lane (= one row) per thread, 128 keys; P overwrites its S as 16-bit
//     O[128 rows x D] += P . V                tcgen05.mma, A from TMEM, V in place as an MN-major operand
// A unit of more than 128 rows runs its two row blocks as the two streams over the same tiles, so a K/V tile is loaded
// once for 256 rows; a smaller one deals its tiles to the streams alternately and joins the two states at the end.
// Either way the tensor pipe works on one stream while the other stream's warps make exponentials: a 128 x 128 x 128
// tile costs the tensor pipe 1024 cycles and the special-function unit (16 a clock) another 1024, and a single stream
// would spend them one after the other.
//
// A row's running maximum is followed lazily: O in TMEM is rescaled only when the maximum has grown by more than 2^8, so
// the stored weights stay below 2^15 and the row sum carries the same factor, which cancels in O / l.
//
// Masks are 64-bit words: for a tile that is not visible as a whole, each thread forms the visibility of its row's 128
// keys as two words (window, sinks, shifted tree mask) and tests constant bits.  Values at tokens that no row of the
// unit sees are cleared in shared memory first, since 0 * NaN would reach the rows.
//
// Warp roles: 0-3 stream 0, 4-7 stream 1, 8 TMA producer, 9 MMA issuer (and TMEM owner), 10-11 idle.  All waits are bounded.
#include "tcgen05.cuh"
#include "tensor_maps.cuh"
#include "visible_plan.cuh"

namespace emlx {

constexpr int kWdSoftThreads = 256;
constexpr int kWdProducer = 8, kWdMma = 9;
constexpr int kWdThreads = kWdSoftThreads + 128;  // whole warpgroups, since registers are moved between them (two warps idle)
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
    static constexpr int SLOTS = D == 128 ? 5 : 8;
    static constexpr int OFF_BAR = OFF_RING + SLOTS * TILE;
    static constexpr int SMEM = OFF_BAR + 512 + 1024;
    static constexpr size_t SLOT_FLOATS = (size_t)kWideRows * (D + 2);
};

struct WdBarriers {
    uint64_t full[8], empty[8];     // ring slots
    uint64_t q_full, q_free;        // Q loaded; every QK of the item has read it
    uint64_t s_full[2], p_ready[2]; // per stream: S complete (and with it every earlier product), P written
    uint64_t o_full[2];             // per stream: the item's last PV is complete
    uint64_t item_full[4];
    uint64_t item_done;             // the item's rows are stored
    uint64_t xch;                   // exchange steps between the streams
    int item_ring[4];
    uint32_t tmem_base;
    int abort_word;
};
static_assert(sizeof(WdBarriers) <= 512, "the barrier block has 512 bytes of shared memory");

struct WideItem {
    int u, head, j0, count, part, parts, slot;
};
__device__ __forceinline__ WideItem wide_item(const WideParams& p, int idx) {
    WideItem it;
    const int e = idx / p.Hkv;
    it.head = idx - e * p.Hkv;
    it.u = p.plan[p.L.entry_unit + e];
    it.j0 = p.plan[p.L.entry_tile + e];
    it.count = p.plan[p.L.entry_count + e];
    const int pp = p.plan[p.L.entry_part + e];
    it.part = pp & 0xffff;
    it.parts = pp >> 16;
    it.slot = p.plan[p.L.entry_slot + e] + it.head * it.parts;
    return it;
}
// Place of tile t's K and V in the item's load order: the order in which the products use them up.
__device__ __forceinline__ int k_place(int t, bool pair) { return pair ? 2 * t : (t == 0 ? 0 : 2 * t - 1); }
__device__ __forceinline__ int v_place(int t, bool pair, int count) { return pair ? 2 * t + 1 : min(2 * t + 2, 2 * count - 1); }

// Bits [from, to) of the 64 keys that start at `base`.
__device__ __forceinline__ uint64_t key_range(int from, int to, int base) {
    const int a = max(from - base, 0), b = min(to - base, 64);
    if (b <= a) return 0;
    return (b >= 64 ? ~0ull : (1ull << b) - 1) & ~((1ull << a) - 1);
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
        for (int s = 0; s < C::SLOTS; ++s) {
            ptx::mbar_init(&bars->full[s], 1);
            ptx::mbar_init(&bars->empty[s], 1);
        }
        ptx::mbar_init(&bars->q_full, 1);
        ptx::mbar_init(&bars->q_free, 1);
        for (int s = 0; s < 2; ++s) {
            ptx::mbar_init(&bars->s_full[s], 1);
            ptx::mbar_init(&bars->p_ready[s], kRowBlock);
            ptx::mbar_init(&bars->o_full[s], 1);
        }
        for (int s = 0; s < 4; ++s) ptx::mbar_init(&bars->item_full[s], 1);
        ptx::mbar_init(&bars->item_done, kWdSoftThreads);
        ptx::mbar_init(&bars->xch, kWdSoftThreads);
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
    const PlanLayout& PL = p.L.base;
    const int32_t *unit_seq = p.plan + PL.unit_seq[3], *unit_row0 = p.plan + PL.unit_row0[3], *unit_tile_lo = p.plan + PL.unit_tile_lo[3];

    if (warp >= kWdProducer) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kWdOtherRegs));
        if (warp == kWdProducer) {
            // ------------------------------------------------------------------ TMA producer
            const uint64_t keep = ptx::l2_policy_evict_normal();
            uint32_t base = 0;  // ring places handed out so far
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
                const int seq = unit_seq[it.u], row0 = unit_row0[it.u], tile_lo = unit_tile_lo[it.u];
                const int qs = p.qsl[seq], q_len = p.qsl[seq + 1] - qs, kv_len = p.kv_lens[seq];
                const bool pair = q_len * p.G - row0 > kRowBlock;
                const int sinks_in = sink_tiles(p.vis.sinks, tile_lo);
                const int lo = unit_lo(p.vis, is_tree(p.vis, seq), row0, p.G, kv_len - q_len, kv_len);
                // The item's Q replaces the last one's: every QK of that item must have read it, and where its streams joined
                // their states through the same memory, its rows must be stored.  (The done phases are waited for in turn, so
                // that none is two phases behind.)
                if (k > 0) {
                    const uint32_t need = last_pair ? k - 1 : k;
                    for (; done_seen < need; ++done_seen) ptx::mbar_wait(&bars->item_done, done_seen & 1, abort_word);
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
                    const uint32_t place = base + (uint32_t)(is_k ? k_place(t, pair) : v_place(t, pair, it.count));
                    const uint32_t slot = place % C::SLOTS, use = place / C::SLOTS;
                    if (use > 0) ptx::mbar_wait(&bars->empty[slot], (use - 1) & 1, abort_word);
                    const bool go = lane == 0 && !*abort_word;
                    if (go) ptx::mbar_arrive_expect_tx(&bars->full[slot], C::TILE);
                    uint8_t* tile = ring + (size_t)slot * C::TILE;
                    const long long tok = (long long)tile_of(it.j0 + t, sinks_in, tile_lo) * kTile;
                    for (int sub = 0; sub < ppt; ++sub) {
                        const int at = ((t - pg_base) << ppt_log) + sub;
                        const int a = __shfl_sync(0xffffffffu, pg_cur, at & 31), b = __shfl_sync(0xffffffffu, pg_next, at & 31);
                        const int pg = at < 32 ? a : b;
                        if (go) {
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
                // in the order of k_place / v_place
                if (!pair) issue(0, true);
                for (int t = 0; t < it.count; ++t) {
                    if (pair) issue(t, true);
                    else if (t + 1 < it.count) issue(t + 1, true);
                    issue(t, false);
                    if (t + 1 == pg_base + per_batch) {  // tiles below are all issued; at most one tile above is looked up
                        pg_base += per_batch;
                        pg_cur = pg_next;
                        pg_next = load_pages(pg_base + per_batch);
                    }
                }
                base += 2u * (uint32_t)it.count;
            }
        } else if (warp == kWdMma) {
            // ------------------------------------------------------------------ MMA issuer
            constexpr uint32_t idesc_qk = instr_desc(128, 128, BF16, false);
            constexpr uint32_t idesc_pv = instr_desc(128, D, BF16, true);
            const uint64_t q_desc0 = smem_desc(ptx::smem_u32(q_smem), 16, 1024);
            const uint64_t k_desc0 = smem_desc(ptx::smem_u32(ring), 16, 1024);
            const uint64_t v_desc0 = smem_desc(ptx::smem_u32(ring), kTile * 128, 1024);
            uint32_t base = 0, p_phase[2] = {0, 0};
            for (uint32_t k = 0;; ++k) {
                if (!ptx::mbar_wait(&bars->item_full[k & 3], (k >> 2) & 1, abort_word)) break;
                const int idx = bars->item_ring[k & 3];
                if (idx < 0) break;
                const WideItem it = wide_item(p, idx);
                const int seq = unit_seq[it.u], row0 = unit_row0[it.u];
                const bool pair = (p.qsl[seq + 1] - p.qsl[seq]) * p.G - row0 > kRowBlock;
                const int steps = pair ? 2 * it.count : it.count;
                ptx::mbar_wait(&bars->q_full, k & 1, abort_word);
                // S of step n is overwritten by QK of step n + 2 of the same stream: its softmax has arrived on p_ready by then,
                // and PV of step n, which reads P from the same columns, was issued before (the pipe runs in issue order)
                auto issue_qk = [&](int n) {
                    const int s = n & 1, t = pair ? n >> 1 : n;
                    const uint32_t place = base + (uint32_t)k_place(t, pair), slot = place % C::SLOTS;
                    const bool ok = ptx::mbar_wait(&bars->full[slot], (place / C::SLOTS) & 1, abort_word);
                    tc_fence_after();
                    if (lane == 0 && ok) {
                        const uint64_t qd = q_desc0 + (uint64_t)((pair ? s : 0) * (C::QBLOCK >> 4));
                        const uint64_t kd = k_desc0 + (uint64_t)(slot * (C::TILE >> 4));
    #pragma unroll
                        for (int ks = 0; ks < D / 16; ++ks) {
                            const uint32_t off = (uint32_t)((ks >> 2) * ((kTile * 128) >> 4) + (ks & 3) * 2);
                            tc_mma_f16(tmem_S + 128 * s, qd + off, kd + off, idesc_qk, ks > 0);
                        }
                        tc_commit(&bars->s_full[s]);
                        if (!pair || s == 1) tc_commit(&bars->empty[slot]);
                        if (n == steps - 1) tc_commit(&bars->q_free);
                    }
                    __syncwarp();
                };
                issue_qk(0);
                if (steps > 1) issue_qk(1);
                for (int n = 0; n < steps; ++n) {
                    const int s = n & 1, t = pair ? n >> 1 : n;
                    const uint32_t place = base + (uint32_t)v_place(t, pair, it.count), slot = place % C::SLOTS;
                    bool ok = ptx::mbar_wait(&bars->full[slot], (place / C::SLOTS) & 1, abort_word);
                    ok = ptx::mbar_wait(&bars->p_ready[s], p_phase[s] & 1, abort_word) && ok;
                    ++p_phase[s];
                    tc_fence_after();
                    if (lane == 0 && ok) {
                        const uint64_t vd = v_desc0 + (uint64_t)(slot * (C::TILE >> 4));
    #pragma unroll
                        for (int kk = 0; kk < kTile / 16; ++kk)
                            tc_mma_f16_ts(tmem_O + 128 * s, tmem_S + 128 * s + kk * 8, vd + (uint64_t)(kk * ((16 * 128) >> 4)), idesc_pv,
                                          n > 1 || kk > 0);
                        if (!pair || s == 1) tc_commit(&bars->empty[slot]);
                        if (n + 2 >= steps) tc_commit(&bars->o_full[s]);
                    }
                    __syncwarp();
                    if (n + 2 < steps) issue_qk(n + 2);
                }
                base += 2u * (uint32_t)it.count;
            }
        }
    } else {
        // ------------------------------------------------------------------ softmax: thread = row of stream g
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kWdSoftRegs));
        const int g = warp >> 2, r = tid & 127;
        const uint32_t lane_addr = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t s_addr = tmem_S + 128 * g + lane_addr, o_addr = tmem_O + 128 * g + lane_addr;
        uint32_t base = 0, s_phase = 0, o_phase[2] = {0, 0}, x_phase = 0;
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
            const int seq = unit_seq[it.u], row0 = unit_row0[it.u], tile_lo = unit_tile_lo[it.u];
            const int qs = p.qsl[seq], q_len = p.qsl[seq + 1] - qs, kv_len = p.kv_lens[seq];
            const int R = q_len * p.G, ctx = kv_len - q_len;
            const bool pair = R - row0 > kRowBlock, tree = is_tree(p.vis, seq);
            const int sinks_in = sink_tiles(p.vis.sinks, tile_lo);
            const int block0 = row0 + (pair ? kRowBlock * g : 0);     // first row of this stream
            const int rows_here = min(kRowBlock, R - block0);
            // a warp whose 32 rows all lie past the unit keeps its appointments only; its lanes of S, P and O hold
            // garbage that nobody reads
            const bool dead = (warp & 3) * 32 >= rows_here;
            const int ti = min(block0 + r, R - 1) / p.G;              // this row's token
            const uint64_t* bits = tree ? p.bits + (long long)(qs + ti) * p.vis.words : nullptr;
            const int n_new = tree ? tree_count(p.vis, p.vis.tree + (long long)(qs + ti) * p.vis.words, q_len) : ti + 1;
            const int hi = max(0, tree ? min(ctx, kv_len) : min(kv_len, ctx + ti + 1));  // end of the plain range
            const int lo = window_lo(p.vis, ctx, n_new), sinks = p.vis.sinks;
            // bounds over the stream's rows, for tiles that need no mask
            const int hi_min = tree ? ctx : min(kv_len, ctx + block0 / p.G + 1);
            const int lo_max = window_lo(p.vis, ctx, tree ? q_len : (block0 + rows_here - 1) / p.G + 1);
            const int lo_unit = unit_lo(p.vis, tree, row0, p.G, ctx, kv_len);
            const int steps = pair ? it.count : (it.count - g + 1) / 2;

            float m_ref = -INFINITY, l = 0.f;
            for (int i = 0; i < steps; ++i) {
                const int t = pair ? i : 2 * i + g;
                const int t0 = tile_of(it.j0 + t, sinks_in, tile_lo) * kTile;
                const bool whole = t0 + kTile <= hi_min && (t0 >= lo_max || t0 + kTile <= sinks);
                ptx::mbar_wait(&bars->s_full[g], s_phase & 1, abort_word);
                ++s_phase;
                tc_fence_after();
                if (!dead) {
                    uint32_t sv[kTile];
#pragma unroll
                    for (int c = 0; c < kTile / 32; ++c) tmem_ld32_nowait(s_addr + 32 * c, sv + 32 * c);
                    tmem_wait_ld();
                    if (!whole) {
#pragma unroll
                        for (int w = 0; w < 2; ++w) {
                            const int b = t0 + 64 * w;
                            uint64_t seen = key_range(lo, hi, b) | key_range(0, min(sinks, hi), b);
                            if (tree && b + 64 > ctx && b < kv_len) {
                                const int j = b - ctx;  // new token that key b is
                                if (j >= 0) {
                                    seen |= tree_word(p.vis, bits, j >> 6, q_len) >> (j & 63);
                                    if (j & 63) seen |= tree_word(p.vis, bits, (j >> 6) + 1, q_len) << (64 - (j & 63));
                                } else if (j > -64) {
                                    seen |= tree_word(p.vis, bits, 0, q_len) << (-j);
                                }
                            }
                            const uint32_t s0 = (uint32_t)seen, s1 = (uint32_t)(seen >> 32);
#pragma unroll
                            for (int e = 0; e < 32; ++e) {
                                if (!(s0 & (1u << e))) sv[64 * w + e] = 0xff800000u;  // -inf
                                if (!(s1 & (1u << e))) sv[64 * w + 32 + e] = 0xff800000u;
                            }
                        }
                    }
                    float mx8[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) mx8[e] = __uint_as_float(sv[e]);
#pragma unroll
                    for (int e = 8; e < kTile; ++e) mx8[e & 7] = fmaxf(mx8[e & 7], __uint_as_float(sv[e]));
                    const float mx = fmaxf(fmaxf(fmaxf(mx8[0], mx8[1]), fmaxf(mx8[2], mx8[3])), fmaxf(fmaxf(mx8[4], mx8[5]), fmaxf(mx8[6], mx8[7])));
                    const float m_new = mx * p.scale_log2e;
                    const bool grow = i == 0 || m_new > m_ref + 8.0f;
                    float corr = 1.0f;
                    if (grow) {
                        const float m_tgt = fmaxf(m_ref, m_new);
                        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(corr) : "f"(m_ref - (m_tgt == -INFINITY ? 0.f : m_tgt)));
                        m_ref = m_tgt;
                    }
                    // the S just waited for was committed behind this stream's last PV, so O is complete
                    if (i > 0 && __any_sync(0xffffffffu, grow)) {
#pragma unroll 1
                        for (int c = 0; c < D / 32; ++c) {
                            uint32_t ov[32];
                            tmem_ld32_nowait(o_addr + 32 * c, ov);
                            tmem_wait_ld();
#pragma unroll
                            for (int e = 0; e < 32; ++e) ov[e] = __float_as_uint(__uint_as_float(ov[e]) * corr);
                            tmem_st32_nowait(o_addr + 32 * c, ov);
                        }
                        l *= corr;
                    }
                    // fp16 weights are stored as 2^(s - m_ref + 7): a key rounds to zero below 2^-32 of the reference only
                    constexpr float kShift = BF16 ? 0.0f : 7.0f;
                    const float neg_m = kShift - (m_ref == -INFINITY ? 0.f : m_ref);
                    float ls0 = 0.f, ls1 = 0.f, ls2 = 0.f, ls3 = 0.f;
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        uint32_t packed[32];
#pragma unroll
                        for (int e = 0; e < 32; ++e) {
                            float p0, p1;
                            asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(p0) : "f"(fmaf(__uint_as_float(sv[64 * c + 2 * e]), p.scale_log2e, neg_m)));
                            asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(p1) : "f"(fmaf(__uint_as_float(sv[64 * c + 2 * e + 1]), p.scale_log2e, neg_m)));
                            if (e & 1) { ls2 += p0; ls3 += p1; } else { ls0 += p0; ls1 += p1; }
                            if constexpr (BF16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(packed[e]) : "f"(p1), "f"(p0));
                            else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(packed[e]) : "f"(p1), "f"(p0));
                        }
                        tmem_st32_nowait(s_addr + 32 * c, packed);
                    }
                    l += (ls0 + ls1) + (ls2 + ls3);
                    tmem_wait_st();
                }
                // tokens of the tile that no row of the unit sees: their values are cleared (thread r owns token r); the two
                // streams of a pair share the tile and stream 0, whose product reads it first, does it
                if ((!pair || g == 0) && (t0 + kTile > kv_len || (t0 < lo_unit && t0 + kTile > sinks))) {
                    const uint32_t place = base + (uint32_t)v_place(t, pair, it.count), slot = place % C::SLOTS;
                    ptx::mbar_wait(&bars->full[slot], (place / C::SLOTS) & 1, abort_word);
                    const int tok = t0 + r;
                    if (tok >= kv_len || (tok < lo_unit && tok >= sinks)) {
#pragma unroll
                        for (int h = 0; h < C::HALVES; ++h) {
                            uint8_t* vrow = ring + (size_t)slot * C::TILE + h * (kTile * 128) + r * 128;
#pragma unroll
                            for (int c = 0; c < 8; ++c) *(uint4*)(vrow + c * 16) = make_uint4(0u, 0u, 0u, 0u);
                        }
                    }
                    ptx::fence_proxy_async();  // the tensor core reads V through the async proxy
                }
                tc_fence_before();
                ptx::mbar_arrive(&bars->p_ready[g]);
            }
            base += 2u * (uint32_t)it.count;

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
                asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(mine) : "f"(m_ref - M_safe));
                asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(theirs) : "f"(m_o - M_safe));
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
            // (both phases move on with the item, waited for here or not: the other stream's last product of an earlier item is
            // complete when a later one of this stream is, so a wait is never two phases behind)
            o_phase[0] += 1;
            o_phase[1] += other_ran ? 1 : 0;
            const bool store = block0 + r < R && !dead;
            const float inv = l_tot > 0.f ? 1.0f / l_tot : 0.f;
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
            tc_fence_before();
            ptx::fence_proxy_async();  // the next item's Q arrives by TMA over the memory of the exchange
            ptx::mbar_arrive(&bars->item_done);
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
// Bound by L2: every state is read once.
template <int D, bool BF16>
__global__ void __launch_bounds__(256) wide_combine_kernel(const __grid_constant__ WideParams p) {
    grid_dep_wait();
    grid_dep_launch();
    const int lane = threadIdx.x & 31;
    const int split = p.plan[p.L.queue + 3];
    const PlanLayout& PL = p.L.base;
    constexpr size_t kSlot = WdCfg<D>::SLOT_FLOATS;
    constexpr int V = D / 32;
    const int total = split * p.Hkv * kWideRows;
    for (int row = blockIdx.x * 8 + (threadIdx.x >> 5); row < total; row += gridDim.x * 8) {
        const int sr = row % kWideRows, rest = row / kWideRows, head = rest % p.Hkv, k = rest / p.Hkv;
        const int u = p.plan[p.L.split_unit + 3 * k], parts = p.plan[p.L.split_unit + 3 * k + 1];
        const int seq = p.plan[PL.unit_seq[3] + u], qs = p.qsl[seq], R = (p.qsl[seq + 1] - qs) * p.G;
        const int r = p.plan[PL.unit_row0[3] + u] + sr;
        if (r >= R) continue;
        const float* base = p.slots + (size_t)(p.plan[p.L.split_unit + 3 * k + 2] + head * parts) * kSlot;
        float M = -INFINITY;
        for (int j = lane; j < parts; j += 32)
            if (__ldcg(base + j * kSlot + kWideRows * (D + 1) + sr) > 0.f) M = fmaxf(M, __ldcg(base + j * kSlot + kWideRows * D + sr));
        M = warp_max(M);
        float acc[V], den = 0.f;
#pragma unroll
        for (int e = 0; e < V; ++e) acc[e] = 0.f;
        for (int j0 = 0; j0 < parts; j0 += 32) {
            const int jl = j0 + lane;
            const float lp = jl < parts ? __ldcg(base + jl * kSlot + kWideRows * (D + 1) + sr) : 0.f;
            const float mp = jl < parts ? __ldcg(base + jl * kSlot + kWideRows * D + sr) : -INFINITY;
            float w = 0.f;
            if (lp > 0.f) asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(w) : "f"(mp - M));
            den += warp_sum(w * lp);
            const int n = min(32, parts - j0);
            constexpr int kDeep = 8;
            for (int j = 0; j < n; j += kDeep) {
                float v[kDeep][V], wj[kDeep];
#pragma unroll
                for (int q = 0; q < kDeep; ++q) {
                    wj[q] = __shfl_sync(0xffffffffu, w, (j + q) & 31);
                    if (j + q >= n) wj[q] = 0.f;
                    const float* src = base + (size_t)(j0 + min(j + q, n - 1)) * kSlot + (size_t)sr * D + V * lane;
                    if constexpr (V == 4) {
                        const float4 x = __ldcg((const float4*)src);
                        v[q][0] = x.x; v[q][1] = x.y; v[q][2] = x.z; v[q][3] = x.w;
                    } else {
                        const float2 x = __ldcg((const float2*)src);
                        v[q][0] = x.x; v[q][1] = x.y;
                    }
                }
#pragma unroll
                for (int q = 0; q < kDeep; ++q)
                    if (wj[q] > 0.f) {  // a part in which the row sees nothing holds no numbers
#pragma unroll
                        for (int e = 0; e < V; ++e) acc[e] = fmaf(wj[q], v[q][e], acc[e]);
                    }
            }
        }
        const float inv = den > 0.f ? 1.0f / den : 0.f;
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
    EMLX_CUDA_OK(launch_pdl(wide_combine_kernel<D, BF16>, 2 * num_sms(), 256, 0, stream, p));
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
