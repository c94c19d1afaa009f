// Coverage kernel of the attention calls with sinks or a draft tree: any head_dim <= 256, any page size, fp16 / bf16 /
// fp32 queries and pools, affine pools.  Eight warps walk the visible keys of one (packed token, q head) row, every
// eighth key each, with an fp32 online softmax, and their states are folded in warp order.  A key that a row does not
// see is never read, so nothing that lies there (infinities, NaN, pages handed to another sequence) can reach the row.
// Bound by the latency of one key after the other (one tree of 16 rows at 2045 keys, 32 heads of 128: 1.3 ms against 0.06 of
// the tensor-core kernel, both with their host call; 8 trees of 16 at 2048 keys, heads of 256: 15.6 ms); the tiled kernels
// serve the geometries that matter.
#include "pool_view.cuh"
#include "visible.cuh"

namespace emlx {

int validate_attn(const emlx_attn_args* a, const emlx_pool* pool, bool need_plan);

int validate_visibility(const emlx_visibility* v, int window) {
    if (!v) return fail(EMLX_ERR_INVALID, "visibility is NULL");
    if (window < 0) return fail(EMLX_ERR_INVALID, "sliding_window must be non-negative");
    if (v->sink_tokens < 0) return fail(EMLX_ERR_INVALID, "sink_tokens must be non-negative");
    if (v->tree_mask && (v->tree_words <= 0 || v->tree_words > kMaxTreeWords))
        return fail(EMLX_ERR_INVALID, "tree_words must lie in [1, %d]", kMaxTreeWords);
    if (((uintptr_t)v->tree_mask & 7) || ((uintptr_t)v->tree_seqs & 3))
        return fail(EMLX_ERR_INVALID, "tree_mask / tree_seqs are misaligned");
    return EMLX_OK;
}

constexpr int kVgWarps = 8;

template <typename TQ>
__global__ void __launch_bounds__(32 * kVgWarps) attn_visible_generic_kernel(emlx_attn_args a, PoolView pv, Visibility vis) {
    __shared__ float part_acc[kVgWarps][kMaxHeadDim];
    __shared__ float part_ml[kVgWarps][2];
    grid_dep_wait();
    grid_dep_launch();
    const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
    const int Hq = a.num_q_heads, D = pv.p.head_dim, bs = pv.p.block_size;
    const int token = (int)(blockIdx.x / Hq), head = (int)(blockIdx.x - (int64_t)token * Hq);
    const int kvh = head / (Hq / pv.p.num_kv_heads);

    float acc[kPerLane], q[kPerLane];
    const TQ* qrow = (const TQ*)a.queries + ((int64_t)token * Hq + head) * D;
#pragma unroll
    for (int j = 0; j < kPerLane; ++j) {
        const int d = lane + 32 * j;
        acc[j] = 0.f;
        q[j] = d < D ? __fmul_rn(to_f32<TQ>(qrow[d]), a.softmax_scale) : 0.f;
    }

    const int s = find_sequence(a.query_start_loc, a.num_seqs, token);
    int ctx = 0, q_len = 0, kv_len = 0, lo = 0, hi = 0, sinks = 0, n = 0;
    const uint64_t* row = nullptr;
    if (s >= 0) {
        const int q0 = a.query_start_loc[s];
        q_len = a.query_start_loc[s + 1] - q0;
        kv_len = a.kv_lens[s];
        ctx = kv_len - q_len;
        if (is_tree(vis, s)) {
            row = vis.tree + (int64_t)token * vis.words;
            n = tree_count(vis, row, q_len);
            hi = max(0, min(ctx, kv_len));
            if (q_len > 64 * vis.words && threadIdx.x == 0) flag_error(a.status, EMLX_DEV_BAD_TREE);
        } else {
            n = token - q0 + 1;
            hi = max(0, min(kv_len, ctx + n));
        }
        lo = min(window_lo(vis, ctx, n), hi);
        sinks = min(vis.sinks, lo);
    }
    // keys [0, sinks), [lo, hi), then the visible new keys of a tree row
    const int plain = sinks + (hi - lo);
    float m = -INFINITY, l = 0.f;
    const int32_t* table = a.block_tables + (int64_t)max(s, 0) * a.max_blocks_per_seq;
    auto take = [&](int k) {
        const int page_idx = k / bs, off = k - page_idx * bs;
        const int64_t page = page_idx < a.max_blocks_per_seq ? table[page_idx] : -1;
        const bool live = page >= 0 && page < pv.p.num_blocks;  // an unassigned page reads as zero rows
        if (!live && lane == 0) flag_error(a.status, EMLX_DEV_BAD_PAGE);
        float dot = 0.f;
        if (live) {
#pragma unroll
            for (int j = 0; j < kPerLane; ++j) {
                const int d = lane + 32 * j;
                if (d < D) dot = fmaf(q[j], pv.key(page, off, kvh, d), dot);
            }
        }
        dot = warp_sum(dot);
        const float m_new = fmaxf(m, dot);
        if (m_new == -INFINITY && dot == dot) return;  // a score of -inf carries no weight
        const float corr = expf(m - m_new), p = expf(dot - m_new);
        l = fmaf(l, corr, p);
#pragma unroll
        for (int j = 0; j < kPerLane; ++j) {
            const int d = lane + 32 * j;
            const float v = (live && d < D) ? pv.value(page, off, kvh, d) : 0.f;
            acc[j] = fmaf(acc[j], corr, p * v);
        }
        m = m_new;
    };
    for (int i = wid; i < plain; i += kVgWarps) take(i < sinks ? i : lo + (i - sinks));
    if (row != nullptr) {
        // new key j has rank ctx + (set bits below j); the window and the sinks go by rank
        const int first = vis.sinks - ctx, last = vis.window > 0 ? n - vis.window : 0;
        int rank = 0, turn = 0;
        for (int w = 0; w < vis.words; ++w) {
            uint64_t x = tree_word(vis, row, w, q_len);
            const int in_word = __popcll(x);
            if (rank < last) x = drop_ranks(x, rank, first, last);
            rank += in_word;
            while (x) {
                const int k = ctx + 64 * w + __ffsll((long long)x) - 1;
                x &= x - 1;
                if (turn++ % kVgWarps == wid && k >= 0 && k < kv_len) take(k);
            }
        }
    }
    part_ml[wid][0] = m;
    part_ml[wid][1] = l;
#pragma unroll
    for (int j = 0; j < kPerLane; ++j) {
        const int d = lane + 32 * j;
        if (d < D) part_acc[wid][d] = acc[j];
    }
    __syncthreads();
    float M = -INFINITY;
    for (int w = 0; w < kVgWarps; ++w) M = fmaxf(M, part_ml[w][0]);
    TQ* out = (TQ*)a.out + ((int64_t)token * Hq + head) * D;
    float weight[kVgWarps], den = 0.f;
    for (int w = 0; w < kVgWarps; ++w) {
        weight[w] = part_ml[w][0] == -INFINITY ? 0.f : expf(part_ml[w][0] - M);
        den += weight[w] * part_ml[w][1];
    }
    for (int d = threadIdx.x; d < D; d += 32 * kVgWarps) {
        float x = 0.f;
        for (int w = 0; w < kVgWarps; ++w)
            if (weight[w] != 0.f) x = fmaf(weight[w], part_acc[w][d], x);
        out[d] = from_f32<TQ>(den != 0.f ? x / den : 0.f);
    }
}

}  // namespace emlx

extern "C" int emlx_attn_visible_generic(const emlx_attn_args* args, const emlx_pool* pool, const emlx_visibility* visibility,
                                         void* stream) {
    using namespace emlx;
    if (int rc = validate_attn(args, pool, false)) return rc;
    if (int rc = validate_visibility(visibility, args->sliding_window)) return rc;
    if (pool->head_dim > kMaxHeadDim) return fail(EMLX_ERR_UNSUPPORTED, "head_dim %d > %d", pool->head_dim, kMaxHeadDim);
    if (args->total_tokens == 0) return EMLX_OK;
    const int64_t rows = (int64_t)args->total_tokens * args->num_q_heads;
    if (rows > 0x7fffffff) return fail(EMLX_ERR_UNSUPPORTED, "more than 2^31 - 1 (token, head) rows");
    const PoolView pv{*pool};
    const Visibility vis = make_visibility(visibility, args->sliding_window);
    cudaStream_t s = (cudaStream_t)stream;
    const dim3 grid((unsigned)rows), block(32 * kVgWarps);
    switch (args->q_dtype) {
        case EMLX_F16: EMLX_CUDA_OK(launch_pdl(attn_visible_generic_kernel<__half>, grid, block, 0, s, *args, pv, vis)); break;
        case EMLX_BF16: EMLX_CUDA_OK(launch_pdl(attn_visible_generic_kernel<__nv_bfloat16>, grid, block, 0, s, *args, pv, vis)); break;
        default: EMLX_CUDA_OK(launch_pdl(attn_visible_generic_kernel<float>, grid, block, 0, s, *args, pv, vis)); break;
    }
    EMLX_LAUNCHED();
    return EMLX_OK;
}
