// Work list of an attention call with sinks or a draft tree.
//
// The short-row classes 0-2 are those of the causal work list (attn_tiled.cuh): units of up to 8 / 16 / 32 rows, cut into
// one slice of the flat (unit, head, tile) order per CTA.  A unit's tiles are the tiles that hold sinks, followed by
// the tiles from the window's first key on; tile_of() maps the running index back.
//
// Rows beyond 16 per sequence form units of up to 256 rows for the tcgen05 kernel (class 3).  A unit whose tiles exceed an
// SM's share of the batch is split along its keys: the list holds *entries* (unit, first tile, tiles, part), one item per
// entry and KV head, longest first, and the parts' states are combined by a second kernel.
//
// The arrival counters of the split short rows, the item queue and the windowed masks live in the plan buffer and are
// set up here, so an attention call needs no zeroed workspace and nothing is carried from one call to the next.
#pragma once
#include "plan_device.cuh"
#include "visible.cuh"

namespace emlx {

constexpr int kVpThreads = 256;      // CTA width of everything that builds this list
constexpr int kWideRows = 256;       // rows of a class-3 unit
constexpr int kMinSplitTiles = 4;    // a unit is never cut into parts shorter than this
constexpr int kVpBins = kVpThreads;
constexpr int kVpSeqs = 2048;        // offsets and tile prefixes up to these counts stay in shared memory: a search in global
constexpr int kVpUnits = 2304;       // memory is a chain of L2 round trips, half a microsecond each
constexpr int kMinSliceTiles = 2;    // a CTA of the short-row classes gets at least so many tiles: more parts than that only
                                     // lengthen the join of a unit's states
constexpr int kPlanAbsentShift = 16; // plan flag bits 16-19: row classes that the caller knows do not occur

// All that an item needs to know, so that it starts with one round of loads instead of a chain entry -> unit -> sequence.
struct alignas(16) WideEntry {
    int j0, count;              // first tile (index inside the unit) and tiles
    int part, parts;
    int slot;                   // partial slot of head 0; slot of head h: + h * parts
    int seq, row0, tile_lo;
    int qs, q_len, kv_len, tree;
};
struct alignas(16) WideSplit {
    int parts, slot, row0, rows, qs, pad[3];
};

struct VisibleLayout {
    PlanLayout base;            // class 3: unit_seq, unit_row0, unit_tile_lo, unit_cum
    int counters[3];            // arrival counters of the short-row classes, cap * Hkv words each
    int queue;                  // class 3: [0] next item, [1] CTAs done, [2] entries, [3] split units
    int entry;                  // class 3: WideEntry records, longest first (16-byte aligned)
    int split;                  // WideSplit records of the units that were split
    int max_entries, max_split;
    int eff;                    // windowed masks, T * words 64-bit words (8-byte aligned), only under a window
    int words;                  // 32-bit words in all
};

__host__ __device__ inline VisibleLayout visible_layout(int S, int T, int Hq, int Hkv, int tree_words) {
    VisibleLayout V;
    V.base = plan_layout(S, T, Hq, Hkv);
    int w = V.base.words;
    for (int c = 0; c < 3; ++c) { V.counters[c] = w; w += V.base.cap[c] * Hkv; }
    V.queue = w; w += 8;
    V.max_split = 2 * kMaxGrid;
    V.max_entries = V.base.cap[3] + V.max_split;
    w = (w + 3) & ~3;
    V.entry = w; w += V.max_entries * (int)(sizeof(WideEntry) / 4);
    V.split = w; w += V.max_split * (int)(sizeof(WideSplit) / 4);
    w = (w + 1) & ~1;
    V.eff = w; w += 2 * T * tree_words;
    V.words = w;
    return V;
}

struct VisiblePlanArgs {
    int32_t* plan;
    VisibleLayout L;
    int G, Hkv, num_ctas, class_lo, class_hi, wide, two_per_sm, absent;
};

// Exclusive prefix of one value per thread over a CTA of THREADS threads; smem: THREADS / 32 + 1 words.
template <int THREADS>
__device__ __forceinline__ int scan_value(int v, int32_t* smem, int& total) {
    constexpr int kW = THREADS / 32;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int incl = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += up;
    }
    __syncthreads();  // smem free from the previous use
    if (lane == 31) smem[warp] = incl;
    __syncthreads();
    if (warp == 0) {
        const int wsum = lane < kW ? smem[lane] : 0;
        int wi = wsum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int up = __shfl_up_sync(0xffffffffu, wi, o);
            if (lane >= o) wi += up;
        }
        __syncwarp();
        if (lane < kW) smem[lane] = wi - wsum;
        if (lane == kW - 1) smem[kW] = wi;
    }
    __syncthreads();
    total = smem[kW];
    return smem[warp] + incl - v;
}

// Tiles in front of the window that hold sinks.
__device__ __forceinline__ int sink_tiles(int sinks, int tile_lo) { return min((sinks + kTile - 1) / kTile, tile_lo); }
// Tile of running index j of a unit.
__device__ __forceinline__ int tile_of(int j, int sink_count, int tile_lo) { return j < sink_count ? j : tile_lo + j - sink_count; }

// Lower bound of the context keys that rows [row0, ..) of a sequence see beside the sinks.  A tree row sees at least the
// context (n >= 0), a causal one itself as well.
__device__ __forceinline__ int unit_lo(const Visibility& vis, bool tree, int row0, int G, int ctx, int kv_len) {
    return min(window_lo(vis, ctx, tree ? 0 : row0 / G + 1), max(kv_len - 1, 0));
}

__device__ __forceinline__ void visible_unit_tiles(const Visibility& vis, int seq, int row0, int row1, int G, int q_len, int kv_len,
                                                   int& tile_lo, int& ntiles) {
    const int ctx = kv_len - q_len;
    const bool tree = is_tree(vis, seq);
    const int hi = tree ? kv_len : min(kv_len, ctx + (row1 - 1) / G + 1);
    tile_lo = 0;
    ntiles = 1;  // a unit without keys keeps one masked tile, so that its rows are written as zeros
    if (hi > 0) {
        tile_lo = min(unit_lo(vis, tree, row0, G, ctx, kv_len), hi - 1) / kTile;
        ntiles = sink_tiles(vis.sinks, tile_lo) + (hi + kTile - 1) / kTile - tile_lo;
    }
}

// Mask row of a token as the kernels read it under a window: the entries that the window drops are cleared.
__device__ __forceinline__ void write_effective_mask(const Visibility& vis, int64_t t, int ctx, int q_len, uint64_t* eff) {
    const uint64_t* row = vis.tree + t * vis.words;
    const int n = tree_count(vis, row, q_len), first = vis.sinks - ctx, last = n - vis.window;
    int rank = 0;
    for (int w = 0; w < vis.words; ++w) {
        uint64_t x = tree_word(vis, row, w, q_len);
        const int in_word = __popcll(x);
        if (rank < last) x = drop_ranks(x, rank, first, last);
        rank += in_word;
        eff[t * vis.words + w] = x;
    }
}

// Called by one CTA of kVpThreads threads.  qsl [S + 1] and kv_lens [S] may lie in shared memory.
__device__ __forceinline__ void build_visible_plan(const VisiblePlanArgs& a, const Visibility& vis, const int32_t* qsl,
                                                   const int32_t* kv_lens, int S, int32_t* scan_smem, int32_t* status) {
    __shared__ int32_t bins[kVpBins];
    __shared__ int32_t s_off[kVpSeqs], s_cum[kVpUnits + 1];
    __shared__ int s_chunk, s_max;
    const int tid = threadIdx.x;
    const PlanLayout& L = a.L.base;
    int32_t* plan = a.plan;
    if (vis.tree != nullptr) {
        for (int s = tid; s < S; s += kVpThreads)
            if (is_tree(vis, s) && qsl[s + 1] - qsl[s] > 64 * vis.words) flag_error(status, EMLX_DEV_BAD_TREE);
    }
    for (int c = 0; c < kNumClasses; ++c) {
        const int num_ctas = class_ctas(c, a.num_ctas, a.two_per_sm != 0);
        bool mine = false;
        if (c >= a.class_lo && c <= a.class_hi && !((a.absent >> c) & 1))
            for (int s = tid; s < S; s += kVpThreads) {
                const int q_len = qsl[s + 1] - qsl[s];
                mine |= q_len > 0 && unit_class(q_len * a.G, a.wide != 0) == c;
            }
        if (!__syncthreads_or(mine)) {
            if (tid == 0) { plan[4 * c] = 0; plan[4 * c + 1] = 0; }
            if (c == 3) { if (tid < 4) plan[a.L.queue + tid] = 0; }
            else for (int i = tid; i <= num_ctas; i += kVpThreads) { plan[L.cta_start[c] + i] = 0; plan[L.cta_unit[c] + i] = 0; }
            continue;
        }
        const int rows_c = c == 3 ? kWideRows : class_rows(c);
        int32_t *unit_seq = plan + L.unit_seq[c], *unit_row0 = plan + L.unit_row0[c];
        int32_t *unit_tile_lo = plan + L.unit_tile_lo[c], *unit_cum = plan + L.unit_cum[c];
        int32_t* seq_off = S <= kVpSeqs ? s_off : plan + L.tmp;
        int num_units = 0;
        for (int s0 = 0; s0 < S; s0 += kVpThreads) {
            const int s = s0 + tid;
            int n = 0;
            if (s < S) {
                const int q_len = qsl[s + 1] - qsl[s], rows = q_len * a.G;
                if (q_len > 0 && unit_class(rows, a.wide != 0) == c) n = (rows + rows_c - 1) / rows_c;
            }
            int n_total;
            const int off = num_units + scan_value<kVpThreads>(n, scan_smem, n_total);
            if (s < S) seq_off[s] = off;
            num_units += n_total;
        }
        __syncthreads();
        int tile_base = 0;
        for (int i0 = 0; i0 < num_units; i0 += kVpThreads) {
            const int idx = i0 + tid;
            int nt = 0;
            if (idx < num_units) {
                int lo = 0, hi = S;  // largest s with seq_off[s] <= idx
                while (hi - lo > 1) {
                    const int mid = (lo + hi) >> 1;
                    if (seq_off[mid] <= idx) lo = mid; else hi = mid;
                }
                const int s = lo, u = idx - seq_off[s], q_len = qsl[s + 1] - qsl[s], rows = q_len * a.G;
                int tile_lo;
                visible_unit_tiles(vis, s, u * rows_c, min(rows, (u + 1) * rows_c), a.G, q_len, kv_lens[s], tile_lo, nt);
                unit_seq[idx] = s;
                unit_row0[idx] = u * rows_c;
                unit_tile_lo[idx] = tile_lo;
            }
            int t_total;
            const int t_off = tile_base + scan_value<kVpThreads>(nt, scan_smem, t_total);
            if (idx < num_units) {
                unit_cum[idx] = t_off;
                if (num_units <= kVpUnits) s_cum[idx] = t_off;
            }
            tile_base += t_total;
        }
        const int32_t* cum = num_units <= kVpUnits ? s_cum : unit_cum;
        if (tid == 0) {
            if (num_units <= kVpUnits) s_cum[num_units] = tile_base;
            unit_cum[num_units] = tile_base;
            plan[4 * c] = num_units;
            plan[4 * c + 1] = tile_base;
        }
        if (c < 3)
            for (int i = tid; i < num_units * a.Hkv; i += kVpThreads) plan[a.L.counters[c] + i] = 0;
        __syncthreads();
        if (c < 3) {
            const long long tiles = (long long)tile_base * a.Hkv;
            cut_slices<kVpThreads>(c, cum, num_units, tile_base, a.Hkv, num_ctas, plan, L,
                                   (int)min((long long)num_ctas, (tiles + kMinSliceTiles - 1) / kMinSliceTiles));
            __syncthreads();
            continue;
        }
        // ---- parts: the smallest part length for which the items fit one round of CTAs, or, when there are more units
        // than CTAs already, an SM's share of the tiles
        if (tid == 0) { s_chunk = 0x7fffffff; s_max = 1; }
        bins[tid] = 0;
        __syncthreads();
        for (int u = tid; u < num_units; u += kVpThreads) atomicMax(&s_max, cum[u + 1] - cum[u]);
        __syncthreads();
        const long long total = (long long)tile_base * a.Hkv;
        const int share = max(kMinSplitTiles, (int)((total + a.num_ctas - 1) / a.num_ctas));
        const int longest = s_max;
        if ((long long)num_units * a.Hkv < a.num_ctas && longest > share) {
            const int step = (longest - share + kVpThreads - 2) / (kVpThreads - 1);
            const int cand = share + tid * step;
            long long items = 0;
            for (int u = 0; u < num_units; ++u) items += (cum[u + 1] - cum[u] + cand - 1) / cand;
            if (items * a.Hkv <= a.num_ctas) atomicMin(&s_chunk, cand);
            __syncthreads();
        }
        const int chunk = s_chunk == 0x7fffffff ? share : s_chunk;
        // Units of about one length that fill some rounds of CTAs and then a part of one: the units of that last round are
        // split over all CTAs.  (Units of mixed lengths fill the last round by themselves, the shortest come last.)
        const int items = num_units * a.Hkv, last = items % a.num_ctas;
        int tail_from = num_units, tail_parts = 1;
        if (items > a.num_ctas && last > 0 && 2 * last <= a.num_ctas && (long long)longest * num_units * 4 <= (long long)tile_base * 5) {
            tail_from = num_units - (last + a.Hkv - 1) / a.Hkv;
            tail_parts = max(1, min(a.num_ctas / last, longest / kMinSplitTiles));
        }
        // entries: counting sort by decreasing length (longer ones than the last bin share it)
        auto parts_of = [&](int u) {
            const int nt = cum[u + 1] - cum[u];
            return u >= tail_from ? min(tail_parts, nt) : (nt + chunk - 1) / chunk;
        };
        for (int u = tid; u < num_units; u += kVpThreads) {
            const int nt = cum[u + 1] - cum[u], parts = parts_of(u);
            const int small = nt / parts, big = nt - small * parts;  // `big` parts of small + 1 tiles
            if (big) atomicAdd(&bins[kVpBins - 1 - min(small + 1, kVpBins - 1)], big);
            atomicAdd(&bins[kVpBins - 1 - min(small, kVpBins - 1)], parts - big);
        }
        __syncthreads();
        int n_entries;
        const int first = scan_value<kVpThreads>(bins[tid], scan_smem, n_entries);
        __syncthreads();
        bins[tid] = first;
        __syncthreads();
        int split_base = 0, slot_base = 0;
        for (int u0 = 0; u0 < num_units; u0 += kVpThreads) {
            const int u = u0 + tid;
            int nt = 0, parts = 0;
            if (u < num_units) { nt = cum[u + 1] - cum[u]; parts = parts_of(u); }
            int split_total, slot_total;
            const int split_idx = split_base + scan_value<kVpThreads>(parts > 1 ? 1 : 0, scan_smem, split_total);
            const int slot = slot_base + scan_value<kVpThreads>(parts > 1 ? parts * a.Hkv : 0, scan_smem, slot_total);
            WideEntry rec{};
            if (parts > 0) {
                rec.parts = parts; rec.seq = unit_seq[u]; rec.row0 = unit_row0[u]; rec.tile_lo = unit_tile_lo[u];
                rec.qs = qsl[rec.seq]; rec.q_len = qsl[rec.seq + 1] - rec.qs; rec.kv_len = kv_lens[rec.seq];
                rec.tree = is_tree(vis, rec.seq) ? 1 : 0;
            }
            if (parts > 1) {
                WideSplit sp{};
                sp.parts = parts; sp.slot = slot; sp.row0 = rec.row0; sp.rows = min(kWideRows, rec.q_len * a.G - rec.row0); sp.qs = rec.qs;
                ((WideSplit*)(plan + a.L.split))[split_idx] = sp;
            }
            const int small = parts ? nt / parts : 0, big = nt - small * parts;
            for (int k = 0, at = 0; k < parts; ++k) {
                const int count = small + (k < big ? 1 : 0);
                const int e = atomicAdd(&bins[kVpBins - 1 - min(count, kVpBins - 1)], 1);
                rec.j0 = at; rec.count = count; rec.part = k; rec.slot = slot + k;
                ((WideEntry*)(plan + a.L.entry))[e] = rec;
                at += count;
            }
            split_base += split_total;
            slot_base += slot_total;
        }
        if (tid == 0) {
            plan[a.L.queue] = 0;
            plan[a.L.queue + 1] = 0;
            plan[a.L.queue + 2] = n_entries;
            plan[a.L.queue + 3] = split_base;
        }
        __syncthreads();
    }
}

inline size_t visible_plan_bytes(int S, int T, int Hq, int Hkv, int tree_words) {
    return (size_t)visible_layout(S, T, Hq, Hkv, tree_words).words * sizeof(int32_t);
}

inline int visible_plan_args(VisiblePlanArgs* a, int S, int T, int Hq, int Hkv, int block_size, int max_query_len, int plan_flags,
                             const Visibility& vis, void* plan, size_t plan_bytes) {
    if (Hkv <= 0 || Hq <= 0 || Hq % Hkv) return fail(EMLX_ERR_INVALID, "num_q_heads must be divisible by num_kv_heads (GQA)");
    if (!tiled_page_size_ok(block_size, 0)) return fail(EMLX_ERR_UNSUPPORTED, "the attention work list needs page size 16, 32, 64 or 128");
    const int words = vis.tree ? vis.words : 0;
    if (!plan || plan_bytes < visible_plan_bytes(S, T, Hq, Hkv, words))
        return fail(EMLX_ERR_WORKSPACE, "plan buffer missing or smaller than emlx_visible_plan_bytes()");
    if ((uintptr_t)plan & 15) return fail(EMLX_ERR_INVALID, "plan must be 16-byte aligned");
    a->plan = (int32_t*)plan;
    a->L = visible_layout(S, T, Hq, Hkv, words);
    a->G = Hq / Hkv; a->Hkv = Hkv;
    a->num_ctas = num_sms() < kMaxGrid ? num_sms() : kMaxGrid;
    a->wide = (plan_flags & kPlanWideUnits) != 0;
    a->two_per_sm = (plan_flags & kPlanTwoCtas) != 0;
    a->absent = (plan_flags >> kPlanAbsentShift) & 15;
    class_range(a->G, max_query_len, a->wide != 0, a->class_lo, a->class_hi);
    return EMLX_OK;
}

}  // namespace emlx
