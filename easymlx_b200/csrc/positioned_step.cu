// One step of the paged cache whose rotary positions are not the slots of the rows: positions given per token and axis
// (time, height, width of a picture or video), or the depth of a token in a tree of drafts.
//
// Pair i of a head turns by the angle  position[axis(i)] * inv_freq[i].  A position of 10^5 times a frequency near 1 needs 41 bits
// to be known to 2^-24, so the product and its reduction to [-pi, pi] are done in 64 bits and only the reduced angle
// goes to sinf / cosf.  The angles of a token are the same for all of its heads: a CTA makes a table of cosines and sines
// for its tokens once (two per thread and token at head size 128) and applies it to every query and key head.
//
// Bound by HBM: every row is read once and written once.  A row of D 16-bit elements is handled by D / 16 lanes, each
// with the 16 bytes of the first half and the matching 16 bytes of the second half, so that a pair never leaves its
// lane (the table then sits in registers for all heads of a token).  Other layouts (adjacent pairs, partly rotated heads,
// quantised pools, 32-bit rows) take one warp per row and read the partner of each element again, from L1.  Measured: 4 x 2047
// rows of 64 and 8 heads of 128 in 74 us (4.5 TB/s), 64 rows in 6.2 us.
//
// CTA 0 of the fused step does the metadata and the attention work list; the stored lengths are advanced by the CTA that
// draws the last ticket, after every CTA has read them (no CTA waits for another).
#include "kv_write_device.cuh"
#include "visible_plan.cuh"

namespace emlx {

constexpr int kPosMaxSeqs = 2048;
constexpr int kPosThreads = kVpThreads;
constexpr int kPosMaxTokens = 8;  // tokens of a write CTA's table

struct Axes {
    const int32_t* positions;  // [axes, T], nullptr: slot positions, or depths under a tree
    const uint8_t* pair_axis;  // [dims / 2], nullptr: axis 0 everywhere
    const double* inv_freq;    // [dims / 2], position scale included
    int64_t stride;            // elements between two axes
    int count;
};

struct PosParams {
    WriteParams w;  // rows, pool, rotation layout; slot_mapping only in the separate write
    Axes axes;
    Visibility vis;
    const int32_t* query_lens;  // nullptr: one token per sequence
    const int32_t* slot_ids;
    const int32_t* bt_all;
    int32_t* kv_lens_all;
    int32_t* qsl;
    int32_t* bt_out;
    int32_t* kv_out;
    int32_t* ticket;
    VisiblePlanArgs plan;
    int S, T, num_slots, MB, advance;
    int tokens_per_cta, chunks;  // chunks: CTAs that share the rows of the same tokens
    int fast;                    // rows of the paired 16-byte layout
};

// Angle of pair i of token t; `fallback` stands in for the position when none are given.
__device__ __forceinline__ float2 pair_turn(const Axes& a, int i, int t, int fallback) {
    int pos = fallback;
    if (a.positions != nullptr) {
        const int axis = a.pair_axis != nullptr ? min((int)a.pair_axis[i], a.count - 1) : 0;
        pos = a.positions[axis * a.stride + t];
    }
    const double angle = (double)pos * a.inv_freq[i];
    const double turns = rint(angle * 0.15915494309189533577);  // 1 / (2 pi)
    float sn, cs;
    sincosf((float)fma(turns, -6.28318530717958647692, angle), &sn, &cs);
    return make_float2(cs, sn);
}

// Element d of a row after the rotation, from the token's table; rounded to the input type like a separate rotation.
template <typename TIn>
__device__ __forceinline__ float turned_elem(const TIn* row, int d, const float2* table, const WriteParams& w) {
    const float x = to_f32<TIn>(row[d]);
    if (d >= w.rope_dims) return x;
    const int half = w.rope_dims >> 1;
    const bool first = w.traditional ? ((d & 1) == 0) : (d < half);
    const int i = w.traditional ? (d >> 1) : (first ? d : d - half);
    const float y = to_f32<TIn>(row[w.traditional ? (d ^ 1) : (first ? d + half : d - half)]);
    const float a = (first ? x : y) * w.mscale, b = (first ? y : x) * w.mscale;
    const float2 cs = table[i];
    const float r = first ? a * cs.x - b * cs.y : a * cs.y + b * cs.x;
    return to_f32<TIn>(from_f32<TIn>(r));
}

template <typename TIn>
__device__ __forceinline__ uint32_t pack_pair(float a, float b) {
    if constexpr (sizeof(TIn) == 2) {
        const TIn x = from_f32<TIn>(a), y = from_f32<TIn>(b);
        return (uint32_t)*reinterpret_cast<const uint16_t*>(&x) | ((uint32_t)*reinterpret_cast<const uint16_t*>(&y) << 16);
    } else return 0u;
}
template <typename TIn>
__device__ __forceinline__ float2 unpack_pair(uint32_t v) {
    if constexpr (sizeof(TIn) == 2) {
        const uint16_t a = (uint16_t)v, b = (uint16_t)(v >> 16);
        return make_float2(to_f32<TIn>(*reinterpret_cast<const TIn*>(&a)), to_f32<TIn>(*reinterpret_cast<const TIn*>(&b)));
    } else return make_float2(0.f, 0.f);
}

// The rows of `count` tokens from `t0` on: s_slot = pool row of each (negative: none), s_turn = their tables.  Row r of a
// token: q heads, then k heads, then v heads; CTA `chunk` of `chunks` takes every chunks-th group of rows.
template <typename TIn>
__device__ __forceinline__ void write_rows(const PosParams& p, int t0, int count, const int64_t* s_slot,
                                           const float2* s_turn, int chunk) {
    const WriteParams& w = p.w;
    const emlx_pool& pool = w.pool;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    constexpr int kWarps = kPosThreads / 32;
    const int D = pool.head_dim, Hkv = w.has_pool ? pool.num_kv_heads : 0, Hq = w.q_out != nullptr ? w.Hq : 0;
    const int rows = Hq + 2 * Hkv, half = w.rope_dims >> 1;
    const int64_t pool_rows = w.has_pool ? pool.num_blocks * pool.block_size : 0;
    if (p.fast) {
        // kWarps / count warps per token (count is 1, 2, 4 or 8 up to the batch's tail)
        const int lanes = D >> 4, per_warp = 32 / lanes, sub = lane / lanes, l = lane - sub * lanes;
        const int share = max(1, kWarps / count);
        const int ti = warp / share;
        if (ti >= count || warp >= share * count) return;
        const int64_t slot = s_slot[ti];
        const bool stored = slot >= 0 && slot < pool_rows;
        if (slot >= pool_rows && w.has_pool && lane == 0) flag_error(w.status, EMLX_DEV_BAD_PAGE);
        float cs[8], sn[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float2 v = w.rope_dims > 0 ? s_turn[ti * half + 8 * l + e] : make_float2(1.f, 0.f);
            cs[e] = v.x; sn[e] = v.y;
        }
        const int64_t t = t0 + ti;
        const int step = share * per_warp * p.chunks;
        constexpr int kDeep = 4;  // rows in flight per lane
        for (int r0 = (chunk * share + warp % share) * per_warp + sub; r0 < rows; r0 += kDeep * step) {
            uint4 a[kDeep], b[kDeep];
#pragma unroll
            for (int k = 0; k < kDeep; ++k) {
                const int r = r0 + k * step;
                if (r < rows) {
                    const uint16_t* src = r < Hq ? (const uint16_t*)w.q_in + (t * Hq + r) * D
                                        : r < Hq + Hkv ? (const uint16_t*)w.keys + (t * Hkv + (r - Hq)) * D
                                                       : (const uint16_t*)w.values + (t * Hkv + (r - Hq - Hkv)) * D;
                    a[k] = *(const uint4*)(src + 8 * l);
                    b[k] = *(const uint4*)(src + (D >> 1) + 8 * l);
                }
            }
#pragma unroll
            for (int k = 0; k < kDeep; ++k) {
                const int r = r0 + k * step;
                if (r >= rows || (r >= Hq && !stored)) continue;
                uint16_t* dst = r < Hq ? (uint16_t*)w.q_out + (t * Hq + r) * D
                              : r < Hq + Hkv ? (uint16_t*)pool.key_cache + (slot * Hkv + (r - Hq)) * D
                                             : (uint16_t*)pool.value_cache + (slot * Hkv + (r - Hq - Hkv)) * D;
                if (r < Hq + Hkv && w.rope_dims > 0) {
                    uint32_t* x = (uint32_t*)&a[k];
                    uint32_t* y = (uint32_t*)&b[k];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float2 u = unpack_pair<TIn>(x[e]), v = unpack_pair<TIn>(y[e]);
                        const float u0 = u.x * w.mscale, u1 = u.y * w.mscale, v0 = v.x * w.mscale, v1 = v.y * w.mscale;
                        x[e] = pack_pair<TIn>(u0 * cs[2 * e] - v0 * sn[2 * e], u1 * cs[2 * e + 1] - v1 * sn[2 * e + 1]);
                        y[e] = pack_pair<TIn>(u0 * sn[2 * e] + v0 * cs[2 * e], u1 * sn[2 * e + 1] + v1 * cs[2 * e + 1]);
                    }
                }
                *(uint4*)(dst + 8 * l) = a[k];
                *(uint4*)(dst + (D >> 1) + 8 * l) = b[k];
            }
        }
        return;
    }
    // one warp per (token, query head) or (token, kv head)
    for (int item = chunk * kWarps + warp; item < count * (Hq + Hkv); item += kWarps * p.chunks) {
        const int ti = item / (Hq + Hkv), h = item - ti * (Hq + Hkv);
        const int64_t t = t0 + ti;
        const float2* table = s_turn + ti * half;
        if (h < Hq) {
            const TIn* src = (const TIn*)w.q_in + (t * Hq + h) * D;
            TIn* dst = (TIn*)w.q_out + (t * Hq + h) * D;
            for (int d = lane; d < D; d += 32) dst[d] = from_f32<TIn>(turned_elem<TIn>(src, d, table, w));
            continue;
        }
        const int kvh = h - Hq;
        const TIn* krow = (const TIn*)w.keys + (t * Hkv + kvh) * D;
        const TIn* vrow = (const TIn*)w.values + (t * Hkv + kvh) * D;
        RowRegs r;
        if (pool.kv_format != EMLX_KV_FLOAT) {
#pragma unroll
            for (int g = 0; g < kMaxGroups; ++g) {
                const int d0 = g * kQuantGroup + 2 * lane;
                if (d0 < D) {
                    r.k[2 * g] = turned_elem<TIn>(krow, d0, table, w); r.k[2 * g + 1] = turned_elem<TIn>(krow, d0 + 1, table, w);
                    r.v[2 * g] = to_f32<TIn>(vrow[d0]); r.v[2 * g + 1] = to_f32<TIn>(vrow[d0 + 1]);
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < 2 * kMaxGroups; ++i) {
                const int d = lane + 32 * i;
                if (d < D) { r.k[i] = turned_elem<TIn>(krow, d, table, w); r.v[i] = to_f32<TIn>(vrow[d]); }
            }
        }
        store_token_head<TIn>(w, kvh, lane, s_slot[ti], r);
    }
}

// Tables of the CTA's tokens; s_pos = the position used when none are given.
__device__ __forceinline__ void make_tables(const PosParams& p, int t0, int count, const int* s_pos, float2* s_turn) {
    const int half = p.w.rope_dims >> 1;
    for (int e = threadIdx.x; e < count * half; e += kPosThreads) {
        const int ti = e / half, i = e - ti * half;
        s_turn[e] = pair_turn(p.axes, i, t0 + ti, s_pos[ti]);
    }
}

// The fused step.
template <typename TIn>
__global__ void __launch_bounds__(kPosThreads) positioned_step_kernel(const PosParams p) {
    __shared__ int32_t scan_smem[kPosThreads / 32 + 1];
    __shared__ int32_t s_q[kPosMaxSeqs + 1], s_kv[kPosMaxSeqs];
    __shared__ float2 s_turn[kPosMaxTokens * 128];
    __shared__ int64_t s_slot[kPosMaxTokens];
    __shared__ int s_pos[kPosMaxTokens];
    __shared__ int s_last;
    grid_dep_wait();
    grid_dep_launch();
    const int tid = threadIdx.x;
    const emlx_pool& pool = p.w.pool;
    const int S = p.S, MB = p.MB, bs = pool.block_size;
    const int64_t capacity = (int64_t)MB * bs;
    const bool ragged = p.query_lens != nullptr;
    int total = S;
    if (ragged) {
        int carry = 0;
        for (int i0 = 0; i0 < S; i0 += kPosThreads) {
            const int i = i0 + tid;
            const int q_len = i < S ? max(p.query_lens[i], 0) : 0;
            int chunk_total;
            const int excl = carry + scan_value<kPosThreads>(q_len, scan_smem, chunk_total);
            if (i < S) s_q[i] = excl;
            carry += chunk_total;
        }
        total = carry;
        if (tid == 0) s_q[S] = total;
        __syncthreads();
    }
    auto q_start = [&](int s) { return ragged ? s_q[s] : s; };

    if (blockIdx.x == 0) {
        for (int i = tid; i < S; i += kPosThreads) {
            const int slot = p.slot_ids[i], q_len = q_start(i + 1) - q_start(i);
            bool ok = slot >= 0 && slot < p.num_slots;
            int base = 0;
            if (ok) base = p.kv_lens_all[slot];
            else flag_error(p.w.status, EMLX_DEV_BAD_SLOT);
            if (ok && (int64_t)base + q_len > capacity) {
                flag_error(p.w.status, EMLX_DEV_OVERFLOW);
                ok = false;
            }
            const int after = ok ? base + q_len : 0;
            s_kv[i] = after;
            if (!ragged) s_q[i] = i;
            p.qsl[i] = q_start(i);
            p.kv_out[i] = after;
        }
        if (tid == 0) {
            s_q[S] = total;
            p.qsl[S] = total;
            if (total != p.T) flag_error(p.w.status, EMLX_DEV_TOKEN_MISMATCH);
        }
        __syncthreads();
        if (p.plan.plan != nullptr) build_visible_plan(p.plan, p.vis, s_q, s_kv, S, scan_smem, p.w.status);
    } else {
        const int n_tok = min(p.T, total), writers = (int)gridDim.x - 1;
        const int groups = (n_tok + p.tokens_per_cta - 1) / p.tokens_per_cta * p.chunks;
        for (int g = (int)blockIdx.x - 1; g < groups; g += writers) {
            const int t0 = g / p.chunks * p.tokens_per_cta, count = min(p.tokens_per_cta, n_tok - t0);
            if (tid < count) {
                const int t = t0 + tid;
                const int s = ragged ? find_sequence(s_q, S, t) : t;
                const int slot = s >= 0 ? p.slot_ids[s] : -1;
                int64_t row = -1;
                int turn_pos = 0;
                if (slot >= 0 && slot < p.num_slots) {
                    const int base = p.kv_lens_all[slot], q_len = q_start(s + 1) - q_start(s);
                    const int pos = base + (t - q_start(s)), page_idx = pos / bs;
                    turn_pos = pos;
                    if (is_tree(p.vis, s))  // a drafted token stands behind its ancestors, wherever its slot is
                        turn_pos = base + tree_count(p.vis, p.vis.tree + (int64_t)t * p.vis.words, q_len) - 1;
                    if (base >= 0 && (int64_t)base + q_len <= capacity && page_idx < MB) {
                        const int page = p.bt_all[(int64_t)slot * MB + page_idx];
                        if (page >= 0 && page < pool.num_blocks) row = (int64_t)page * bs + (pos - page_idx * bs);
                        else flag_error(p.w.status, EMLX_DEV_BAD_PAGE);
                    }
                }
                s_slot[tid] = row;
                s_pos[tid] = turn_pos;
                if (p.plan.plan != nullptr && p.vis.window > 0 && s >= 0 && is_tree(p.vis, s))
                    write_effective_mask(p.vis, t, slot >= 0 && slot < p.num_slots ? p.kv_lens_all[slot] : 0,
                                         q_start(s + 1) - q_start(s), (uint64_t*)(p.plan.plan + p.plan.L.eff));
            }
            __syncthreads();
            if (p.w.rope_dims > 0) {
                make_tables(p, t0, count, s_pos, s_turn);
                __syncthreads();
            }
            write_rows<TIn>(p, t0, count, s_slot, s_turn, g % p.chunks);
            __syncthreads();
        }
        const int64_t cells = (int64_t)S * MB, stride = (int64_t)writers * kPosThreads;
        for (int64_t c = (int64_t)(blockIdx.x - 1) * kPosThreads + tid; c < cells; c += stride) {
            const int row = (int)(c / MB), col = (int)(c - (int64_t)row * MB);
            const int slot = p.slot_ids[row];
            p.bt_out[c] = (slot >= 0 && slot < p.num_slots) ? p.bt_all[(int64_t)slot * MB + col] : -1;
        }
    }
    if (!p.advance) return;
    __syncthreads();
    if (tid == 0) {
        __threadfence();
        s_last = atomicAdd(p.ticket, 1) == (int)gridDim.x - 1 ? 1 : 0;
    }
    __syncthreads();
    if (!s_last) return;
    __threadfence();
    for (int i = tid; i < S; i += kPosThreads) {
        const int slot = p.slot_ids[i];
        if (slot < 0 || slot >= p.num_slots) continue;
        const int q_len = q_start(i + 1) - q_start(i), base = p.kv_lens_all[slot];
        if ((int64_t)base + q_len <= capacity) p.kv_lens_all[slot] = base + q_len;
    }
    if (tid == 0) *p.ticket = 0;
}

// Rows whose pool rows and positions are known already: batches above kPosMaxSeqs sequences (behind
// emlx_build_metadata) and the rotation of a tensor on its own.
template <typename TIn>
__global__ void __launch_bounds__(kPosThreads) positioned_write_kernel(const PosParams p) {
    __shared__ float2 s_turn[kPosMaxTokens * 128];
    __shared__ int64_t s_slot[kPosMaxTokens];
    __shared__ int s_pos[kPosMaxTokens];
    grid_dep_wait();
    grid_dep_launch();
    const int tid = threadIdx.x;
    const int groups = (p.T + p.tokens_per_cta - 1) / p.tokens_per_cta * p.chunks;
    for (int g = (int)blockIdx.x; g < groups; g += (int)gridDim.x) {
        const int t0 = g / p.chunks * p.tokens_per_cta, count = min(p.tokens_per_cta, p.T - t0);
        if (tid < count) {
            const int t = t0 + tid;
            s_slot[tid] = p.w.slot_mapping != nullptr ? p.w.slot_mapping[t] : -1;
            int pos = p.w.positions != nullptr ? p.w.positions[t] : 0;
            if (p.vis.tree != nullptr && p.qsl != nullptr) {
                const int s = find_sequence(p.qsl, p.S, t);
                if (s >= 0 && is_tree(p.vis, s)) {
                    const int q0 = p.qsl[s], q_len = p.qsl[s + 1] - q0;
                    pos += tree_count(p.vis, p.vis.tree + (int64_t)t * p.vis.words, q_len) - 1 - (t - q0);
                }
            }
            s_pos[tid] = pos;
        }
        __syncthreads();
        if (p.w.rope_dims > 0) {
            make_tables(p, t0, count, s_pos, s_turn);
            __syncthreads();
        }
        write_rows<TIn>(p, t0, count, s_slot, s_turn, g % p.chunks);
        __syncthreads();
    }
}

static int set_rows(PosParams& p, const emlx_pool* pool, const emlx_rope* rope, const emlx_axes* axes, const void* queries,
                    void* queries_out, int num_q_heads, const void* keys, const void* values, int in_dtype, int head_dim) {
    WriteParams& w = p.w;
    if (in_dtype < EMLX_F16 || in_dtype > EMLX_F32) return fail(EMLX_ERR_INVALID, "unknown in_dtype %d", in_dtype);
    w.keys = keys; w.values = values; w.T = p.T;
    w.mscale = 1.0f;
    if (pool) { w.pool = *pool; w.has_pool = 1; }
    else { w.pool.head_dim = head_dim; w.pool.num_kv_heads = 1; w.pool.block_size = 1; }
    if (rope) {
        if (rope->dims <= 0 || (rope->dims & 1) || rope->dims > head_dim)
            return fail(EMLX_ERR_INVALID, "rope dims must be positive, even and at most head_dim");
        if (!axes || !axes->inv_freq) return fail(EMLX_ERR_INVALID, "a rotated step needs emlx_axes with inv_freq");
        if (axes->positions && (axes->num_axes <= 0 || axes->num_axes > 255 || (axes->num_axes > 1 && axes->axis_stride < p.T)))
            return fail(EMLX_ERR_INVALID, "rope positions must be [num_axes, total_tokens] with 1 to 255 axes");
        w.rope_dims = rope->dims; w.traditional = rope->traditional; w.mscale = rope->mscale;
        p.axes.positions = axes->positions; p.axes.pair_axis = axes->pair_axis; p.axes.inv_freq = axes->inv_freq;
        p.axes.stride = axes->axis_stride; p.axes.count = axes->num_axes;
        if (queries_out) {
            if (!queries || num_q_heads <= 0) return fail(EMLX_ERR_INVALID, "queries / num_q_heads missing");
            w.q_in = queries; w.q_out = queries_out; w.Hq = num_q_heads;
        }
    }
    const bool pow2 = head_dim == 64 || head_dim == 128 || head_dim == 256;
    const bool turned = w.rope_dims == 0 || (w.rope_dims == head_dim && !w.traditional);
    uintptr_t at = (uintptr_t)w.q_in | (uintptr_t)w.q_out;
    if (pool) at |= (uintptr_t)keys | (uintptr_t)values | (uintptr_t)pool->key_cache | (uintptr_t)pool->value_cache;
    p.fast = pow2 && turned && in_dtype != EMLX_F32 && (at & 15) == 0 &&
             (!pool || (pool->kv_format == EMLX_KV_FLOAT && pool->kv_dtype == in_dtype));
    // A CTA makes the table of its tokens before their rows, so a large batch takes as many tokens as the table holds; a
    // small one takes one token per CTA, and splits that token's rows over CTAs while the GPU has idle SMs (the
    // table is then made again in each: a few hundred cycles against the latency of another round of rows).
    const int rows = (w.q_out ? w.Hq : 0) + (pool ? 2 * pool->num_kv_heads : 0);
    const int sms = num_sms();
    p.tokens_per_cta = kPosMaxTokens;
    while (p.tokens_per_cta > 1 && p.T < 2 * sms * p.tokens_per_cta) p.tokens_per_cta /= 2;
    const int rows_per_pass = p.fast ? kPosThreads * 16 / head_dim : kPosThreads / 32;
    p.chunks = 1;
    while (p.tokens_per_cta == 1 && (int64_t)p.T * p.chunks < sms && p.chunks * rows_per_pass * 2 <= rows) p.chunks *= 2;
    return EMLX_OK;
}

static unsigned row_ctas(const PosParams& p, int per_sm) {
    const int64_t groups = ((int64_t)p.T + p.tokens_per_cta - 1) / p.tokens_per_cta * p.chunks;
    const int64_t most = (int64_t)per_sm * num_sms();
    return (unsigned)(groups < 1 ? 1 : groups < most ? groups : most);
}

static int launch_rows(PosParams& p, int in_dtype, cudaStream_t s) {
    const unsigned grid = row_ctas(p, 8);
    switch (in_dtype) {
        case EMLX_F16: EMLX_CUDA_OK(launch_pdl(positioned_write_kernel<__half>, grid, kPosThreads, 0, s, p)); break;
        case EMLX_BF16: EMLX_CUDA_OK(launch_pdl(positioned_write_kernel<__nv_bfloat16>, grid, kPosThreads, 0, s, p)); break;
        default: EMLX_CUDA_OK(launch_pdl(positioned_write_kernel<float>, grid, kPosThreads, 0, s, p)); break;
    }
    EMLX_LAUNCHED();
    return EMLX_OK;
}

}  // namespace emlx

extern "C" int emlx_positioned_step(const emlx_step_args* a, const emlx_pool* pool, const emlx_rope* rope,
                                    const emlx_axes* axes, const emlx_visibility* visibility, void* stream) {
    using namespace emlx;
    if (!a) return fail(EMLX_ERR_INVALID, "step arguments are NULL");
    if (int rc = validate_pool(pool)) return rc;
    if (visibility)
        if (int rc = validate_visibility(visibility, a->sliding_window)) return rc;
    if (a->num_seqs < 0 || a->total_tokens < 0) return fail(EMLX_ERR_INVALID, "num_seqs/total_tokens must be non-negative");
    if (a->num_seqs == 0) return EMLX_OK;
    if (a->num_seqs > kPosMaxSeqs)
        return fail(EMLX_ERR_UNSUPPORTED, "the single-launch step takes up to %d sequences; use emlx_build_metadata + emlx_positioned_write",
                    kPosMaxSeqs);
    if (!a->query_lens && a->total_tokens != a->num_seqs)
        return fail(EMLX_ERR_INVALID, "without query_lens every sequence has one token: total_tokens must equal num_seqs");
    if (a->max_blocks_per_seq <= 0 || a->num_slots <= 0) return fail(EMLX_ERR_INVALID, "max_blocks_per_seq and num_slots must be positive");
    if (!a->slot_ids || !a->block_tables_all || !a->kv_lens_all || !a->query_start_loc || !a->block_tables || !a->kv_lens || !a->ticket)
        return fail(EMLX_ERR_INVALID, "positioned_step: NULL argument");
    if (a->total_tokens > 0 && (!a->keys || !a->values)) return fail(EMLX_ERR_INVALID, "positioned_step: NULL key/value input");
    PosParams p{};
    p.S = a->num_seqs; p.T = a->total_tokens; p.num_slots = a->num_slots; p.MB = a->max_blocks_per_seq; p.advance = a->advance_kv_lens;
    p.w.status = a->status;
    if (int rc = set_rows(p, pool, rope, axes, a->queries, a->queries_out, a->num_q_heads, a->keys, a->values, a->in_dtype, pool->head_dim))
        return rc;
    p.vis = make_visibility(visibility, a->sliding_window);
    p.query_lens = a->query_lens; p.slot_ids = a->slot_ids; p.bt_all = a->block_tables_all; p.kv_lens_all = a->kv_lens_all;
    p.qsl = a->query_start_loc; p.bt_out = a->block_tables; p.kv_out = a->kv_lens; p.ticket = a->ticket;
    if (a->plan && a->total_tokens > 0)
        if (int rc = visible_plan_args(&p.plan, a->num_seqs, a->total_tokens, a->num_q_heads, pool->num_kv_heads, pool->block_size,
                                       a->query_lens ? a->max_query_len : 1, a->plan_flags, p.vis, a->plan, a->plan_bytes))
            return rc;
    // every CTA scans the query lengths: with many sequences fewer CTAs loop, with few the scheduler deals out single groups
    const unsigned grid = 1u + row_ctas(p, p.S <= kPosThreads ? 16 : 3);
    cudaStream_t s = (cudaStream_t)stream;
    switch (a->in_dtype) {
        case EMLX_F16: EMLX_CUDA_OK(launch_pdl(positioned_step_kernel<__half>, grid, kPosThreads, 0, s, p)); break;
        case EMLX_BF16: EMLX_CUDA_OK(launch_pdl(positioned_step_kernel<__nv_bfloat16>, grid, kPosThreads, 0, s, p)); break;
        default: EMLX_CUDA_OK(launch_pdl(positioned_step_kernel<float>, grid, kPosThreads, 0, s, p)); break;
    }
    EMLX_LAUNCHED();
    return EMLX_OK;
}

extern "C" int emlx_positioned_write(const void* queries, void* queries_out, int32_t num_q_heads, const void* keys,
                                     const void* values, int32_t in_dtype, int32_t total_tokens, const int64_t* slot_mapping,
                                     const int32_t* token_positions, const int32_t* query_start_loc, int32_t num_seqs,
                                     const emlx_rope* rope, const emlx_axes* axes, const emlx_visibility* visibility,
                                     const emlx_pool* pool, int32_t* status, void* stream) {
    using namespace emlx;
    if (total_tokens < 0 || num_seqs < 0) return fail(EMLX_ERR_INVALID, "total_tokens/num_seqs must be non-negative");
    if (visibility)
        if (int rc = validate_visibility(visibility, 0)) return rc;
    if (total_tokens == 0) return EMLX_OK;
    PosParams p{};
    p.T = total_tokens; p.S = num_seqs; p.w.status = status;
    int head_dim = 0;
    if (pool) {
        if (int rc = validate_pool(pool)) return rc;
        if (!keys || !values || !slot_mapping) return fail(EMLX_ERR_INVALID, "positioned_write: NULL key/value input");
        head_dim = pool->head_dim;
    } else {
        if (!rope || !queries_out) return fail(EMLX_ERR_INVALID, "without a pool there must be queries to rotate");
        head_dim = rope->head_dim_if_no_pool;
        if (head_dim <= 0 || head_dim > 256) return fail(EMLX_ERR_INVALID, "rope->head_dim_if_no_pool must lie in [1, 256]");
    }
    if (rope && axes && !axes->positions && !token_positions) return fail(EMLX_ERR_INVALID, "no positions given");
    if (int rc = set_rows(p, pool, rope, axes, queries, queries_out, num_q_heads, keys, values, in_dtype, head_dim)) return rc;
    p.w.slot_mapping = slot_mapping; p.w.positions = token_positions;
    p.qsl = const_cast<int32_t*>(query_start_loc);
    p.vis = make_visibility(visibility, 0);
    if (!query_start_loc) p.vis.tree = nullptr;
    return launch_rows(p, in_dtype, (cudaStream_t)stream);
}
