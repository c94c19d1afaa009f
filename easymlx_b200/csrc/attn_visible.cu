// Attention calls with sinks or a draft tree: the short-row classes on the tiled kernels' VIS builds, the others on the
// 256-row kernel.
#include "attn_tiled_kernel.cuh"

namespace emlx {

int validate_attn(const emlx_attn_args* a, const emlx_pool* pool, bool need_plan);
size_t wide_slot_bytes(int D);
int launch_wide(const emlx_attn_args* a, const emlx_pool* pool, const Visibility& vis, const VisibleLayout& L, float* slots,
                const MapPair& maps, cudaStream_t stream);

namespace {

template <int D, int NT, int FMT, bool BF16>
int launch_one(const MapPair& maps, const TiledParams& p, int grid, cudaStream_t stream) {
    using C = Cfg<D, NT, FMT>;
    auto go = [&](auto kernel, DeviceOnce& configured) -> int {
        EMLX_CUDA_OK(allow_dynamic_smem(kernel, C::SMEM, configured));
        EMLX_CUDA_OK(launch_pdl(kernel, grid, kThreads, C::SMEM, stream, maps.k, maps.v, p));
        return EMLX_OK;
    };
    static DeviceOnce once_plain, once_help;
    const int rc = p.few_units ? go(attn_tiled_kernel<D, NT, FMT, BF16, false, true, true>, once_help)
                               : go(attn_tiled_kernel<D, NT, FMT, BF16, false, false, true>, once_plain);
    if (rc) return rc;
    EMLX_LAUNCHED();
    return EMLX_OK;
}
template <int D, int NT>
int launch_fmt(int fmt, bool bf16, const MapPair& maps, const TiledParams& p, int grid, cudaStream_t stream) {
    if (fmt == EMLX_KV_AFFINE8) return bf16 ? launch_one<D, NT, 8, true>(maps, p, grid, stream) : launch_one<D, NT, 8, false>(maps, p, grid, stream);
    if (fmt == EMLX_KV_AFFINE4) return bf16 ? launch_one<D, NT, 4, true>(maps, p, grid, stream) : launch_one<D, NT, 4, false>(maps, p, grid, stream);
    return bf16 ? launch_one<D, NT, 0, true>(maps, p, grid, stream) : launch_one<D, NT, 0, false>(maps, p, grid, stream);
}
template <int D>
int launch_class(int cls, int fmt, bool bf16, const MapPair& maps, const TiledParams& p, int grid, cudaStream_t s) {
    if (cls == 0) return launch_fmt<D, 1>(fmt, bf16, maps, p, grid, s);
    if (cls == 1) return launch_fmt<D, 2>(fmt, bf16, maps, p, grid, s);
    return launch_fmt<D, 4>(fmt, bf16, maps, p, grid, s);
}

// Workspace: [partial rows of the short classes] [partial states of the wide units] [expanded pages].
constexpr size_t kShortSlotBytes = ((size_t)kMaxGrid * 2 * kSlotFloats * sizeof(float) + 255) & ~(size_t)255;
struct Parts {
    size_t wide_off, end;
};
Parts workspace_parts(int Hq, int Hkv, int D, int max_query_len, int flags) {
    int lo, hi;
    class_range(Hq / Hkv, max_query_len, (flags & kPlanWideUnits) != 0, lo, hi);
    Parts w;
    w.wide_off = lo < 3 ? kShortSlotBytes : 0;
    w.end = w.wide_off + (hi == 3 ? (wide_slot_bytes(D) + 255) & ~(size_t)255 : 0);
    return w;
}

}  // namespace

int run_visible(const emlx_attn_args* a, const emlx_pool* pool, const emlx_visibility* visibility, void* stream) {
    if (int rc = validate_attn(a, pool, true)) return rc;
    if (int rc = validate_visibility(visibility, a->sliding_window)) return rc;
    if (a->total_tokens == 0) return EMLX_OK;
    const int D = pool->head_dim, Hq = a->num_q_heads, Hkv = pool->num_kv_heads, G = Hq / Hkv;
    if (!tiled_page_size_ok(pool->block_size, pool->kv_format))
        return fail(EMLX_ERR_UNSUPPORTED, "the tiled kernels need page size 128 (16, 32 or 64 also for fp16/bf16 pools)");
    if (D != 64 && D != 128) return fail(EMLX_ERR_UNSUPPORTED, "the tiled kernels need head_dim 64 or 128");
    if (a->q_dtype == EMLX_F32) return fail(EMLX_ERR_UNSUPPORTED, "the tiled kernels need fp16 or bf16 queries");
    if (pool->kv_format == EMLX_KV_FLOAT && pool->kv_dtype != a->q_dtype)
        return fail(EMLX_ERR_UNSUPPORTED, "the tiled kernels need the pool dtype to equal the query dtype");
    if (((uintptr_t)a->queries | (uintptr_t)a->out) & 15) return fail(EMLX_ERR_INVALID, "queries/out must be 16-byte aligned");
    if ((uintptr_t)a->plan & 15) return fail(EMLX_ERR_INVALID, "plan must be 16-byte aligned");
    if ((uintptr_t)a->workspace & 15) return fail(EMLX_ERR_INVALID, "workspace must be 16-byte aligned");
    const Visibility vis = make_visibility(visibility, a->sliding_window);
    const int words = vis.tree ? vis.words : 0;
    const VisibleLayout V = visible_layout(a->num_seqs, a->total_tokens, Hq, Hkv, words);
    const PlanLayout& L = V.base;
    const bool wide = (a->plan_flags & kPlanWideUnits) != 0, expand = wide && pool->kv_format != EMLX_KV_FLOAT;
    const Parts W = workspace_parts(Hq, Hkv, D, a->max_query_len, a->plan_flags);
    if (a->plan_bytes < (size_t)V.words * 4 || a->workspace_bytes < W.end)
        return fail(EMLX_ERR_WORKSPACE, "plan/workspace smaller than emlx_visible_plan_bytes()/emlx_visible_workspace_bytes()");
    if (wide && !prefill_geometry_ok(Hq, Hkv, D))
        return fail(EMLX_ERR_INVALID, "plan_flags ask for units that this head geometry cannot run");
    int lo, hi;
    class_range(G, a->max_query_len, wide, lo, hi);
    auto skipped = [&](int c) { return a->row_class_mask != 0 && !((a->row_class_mask >> c) & 1); };
    bool any = false;
    for (int c = lo; c <= hi; ++c) any |= !skipped(c);
    if (!any) return fail(EMLX_ERR_UNSUPPORTED, "row_class_mask names no row class that this call can launch");
    MapPair maps;
    if (int rc = encode_maps(*pool, &maps)) return rc;
    DequantScratch scratch{};
    cudaStream_t s = (cudaStream_t)stream;
    if (expand && hi == 3 && !skipped(3)) {
        if (!dequant_scratch_layout(pool, a, (uint8_t*)a->workspace + W.end, a->workspace_bytes - W.end, &scratch))
            return fail(EMLX_ERR_WORKSPACE, "wide units over an affine pool need emlx_attn_dequant_bytes() of memory behind the workspace");
        // (a tree row may see one context key more than a causal first token: the window is taken one wider)
        if (int rc = launch_dequant_pages(a, pool, scratch, s, vis.window > 0 ? vis.window + 1 : 0, vis.sinks)) return rc;
    }
    const int32_t* plan = (const int32_t*)a->plan;
    for (int c = lo; c <= hi; ++c) {
        if (skipped(c)) continue;
        if (c == 3) {
            emlx_attn_args a3 = *a;
            emlx_pool pool3 = *pool;
            MapPair maps3 = maps;
            if (expand) {  // the scratch pool stands in for the pool, in fp16 (also under bf16 queries)
                pool3.key_cache = scratch.k; pool3.value_cache = scratch.v;
                pool3.k_scale = pool3.k_bias = pool3.v_scale = pool3.v_bias = nullptr;
                pool3.num_blocks = scratch.cap; pool3.block_size = kTile;
                pool3.kv_format = EMLX_KV_FLOAT; pool3.kv_dtype = EMLX_F16;
                a3.block_tables = scratch.sbt;
                if (a->q_dtype == EMLX_BF16) { a3.queries = scratch.q16; a3.out = scratch.out16; a3.q_dtype = EMLX_F16; }
                if (int rc = encode_maps(pool3, &maps3)) return rc;
            }
            if (int rc = launch_wide(&a3, &pool3, vis, V, (float*)((uint8_t*)a->workspace + W.wide_off), maps3, s)) return rc;
            if (expand && a->q_dtype == EMLX_BF16)
                if (int rc = launch_convert_out_rows(a, pool, scratch, s)) return rc;
            continue;
        }
        TiledParams p{};
        p.q = a->queries; p.out = a->out; p.bt = a->block_tables; p.kv_lens = a->kv_lens; p.qsl = a->query_start_loc;
        p.hdr = plan + 4 * c;
        p.unit_seq = plan + L.unit_seq[c]; p.unit_row0 = plan + L.unit_row0[c];
        p.unit_tile_lo = plan + L.unit_tile_lo[c]; p.unit_cum = plan + L.unit_cum[c];
        p.cta_start = plan + L.cta_start[c]; p.cta_unit = plan + L.cta_unit[c];
        p.counters = (int32_t*)a->plan + V.counters[c];
        p.slots = (float*)a->workspace;
        p.status = a->status;
        p.k_scale = (const __half*)pool->k_scale; p.k_bias = (const __half*)pool->k_bias;
        p.v_scale = (const __half*)pool->v_scale; p.v_bias = (const __half*)pool->v_bias;
        p.num_blocks = pool->num_blocks;
        p.Hq = Hq; p.Hkv = Hkv; p.G = G; p.MB = a->max_blocks_per_seq; p.window = a->sliding_window;
        p.bs = pool->block_size; p.ppt_log = pages_per_tile_log2(pool->block_size);
        p.scale_log2e = a->softmax_scale * 1.4426950408889634f;
        p.out_Hq = Hq;
        p.vis = vis;
        p.tree_bits = vis.window > 0 ? (const uint64_t*)((const int32_t*)a->plan + V.eff) : vis.tree;
        const int grid = class_ctas(c, min(num_sms(), kMaxGrid), (a->plan_flags & kPlanTwoCtas) != 0);
        p.few_units = (long long)a->num_seqs * Hkv * (kHelpMinParts - 1) <= grid;
        const bool bf16 = a->q_dtype == EMLX_BF16;
        if (int rc = D == 128 ? launch_class<128>(c, pool->kv_format, bf16, maps, p, grid, s) : launch_class<64>(c, pool->kv_format, bf16, maps, p, grid, s))
            return rc;
    }
    return EMLX_OK;
}

}  // namespace emlx

extern "C" {
size_t emlx_visible_workspace_bytes(int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim, int32_t max_query_len, int32_t plan_flags) {
    if (num_kv_heads <= 0 || num_q_heads <= 0 || head_dim <= 0) return 0;
    return emlx::workspace_parts(num_q_heads, num_kv_heads, head_dim, max_query_len, plan_flags).end;
}
int emlx_attn_visible(const emlx_attn_args* args, const emlx_pool* pool, const emlx_visibility* visibility, void* stream) {
    return emlx::run_visible(args, pool, visibility, stream);
}
}
