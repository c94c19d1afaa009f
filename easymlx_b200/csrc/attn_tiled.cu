// Host side of the tiled attention kernels (attn_tiled_kernel.cuh): tensor maps, launches, and the entry points that run
// a work list's row classes.
#include "attn_tiled_kernel.cuh"

#include <map>
#include <mutex>
#include <tuple>

namespace emlx {

int validate_attn(const emlx_attn_args* a, const emlx_pool* pool, bool need_plan);

// ------------------------------------------------------------------------------------------ host
EncodeTiledFn encode_fn() {
    static EncodeTiledFn fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void* ptr = nullptr;
        cudaDriverEntryPointQueryResult qres;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &qres) == cudaSuccess &&
            qres == cudaDriverEntryPointSuccess)
            fn = (EncodeTiledFn)ptr;
    });
    return fn;
}

static CUtensorMapSwizzle swizzle_of(int row_bytes) {
    return row_bytes == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : (row_bytes == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_32B);
}

int encode_maps(const emlx_pool& pool, MapPair* out) {
    EncodeTiledFn enc = encode_fn();
    if (!enc) return fail(EMLX_ERR_CUDA, "cuTensorMapEncodeTiled is not available from this driver");
    if (((uintptr_t)pool.key_cache | (uintptr_t)pool.value_cache) & 15)
        return fail(EMLX_ERR_INVALID, "key_cache/value_cache must be 16-byte aligned");
    MapPair& mp = *out;
    const cuuint64_t NB = (cuuint64_t)pool.num_blocks, Hkv = (cuuint64_t)pool.num_kv_heads, D = (cuuint64_t)pool.head_dim;
    const cuuint32_t ones[3] = {1, 1, 1};
    CUresult r1, r2;
    if (pool.kv_format == EMLX_KV_FLOAT) {
        const CUtensorMapDataType dt = pool.kv_dtype == EMLX_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
        const cuuint64_t bs = (cuuint64_t)pool.block_size;  // a box is one page (128 tokens, or a part of a tile)
        const cuuint64_t dims[3] = {D, Hkv, NB * bs};
        const cuuint64_t strides[2] = {D * 2, Hkv * D * 2};
        const cuuint32_t box[3] = {64, 1, (cuuint32_t)bs};
        // a tile row is D*2 contiguous bytes: do not let L2 promotion pull in the neighbouring head's row
        const CUtensorMapL2promotion promo = D * 2 >= 256 ? CU_TENSOR_MAP_L2_PROMOTION_L2_256B : CU_TENSOR_MAP_L2_PROMOTION_L2_128B;
        r1 = enc(&mp.k, dt, 3, pool.key_cache, dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                 CU_TENSOR_MAP_SWIZZLE_128B, promo, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
        r2 = enc(&mp.v, dt, 3, pool.value_cache, dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                 CU_TENSOR_MAP_SWIZZLE_128B, promo, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    } else {
        const cuuint64_t bits = (cuuint64_t)pool.kv_format;
        const cuuint64_t krow = D * bits / 8, vrow = (cuuint64_t)kTile * bits / 8;
        const cuuint64_t kdims[3] = {krow, Hkv, NB * kTile};
        const cuuint64_t kstrides[2] = {krow, Hkv * krow};
        const cuuint32_t kbox[3] = {(cuuint32_t)krow, 1, kTile};
        const CUtensorMapL2promotion kpromo = krow >= 128 ? CU_TENSOR_MAP_L2_PROMOTION_L2_128B
                                                          : (krow >= 64 ? CU_TENSOR_MAP_L2_PROMOTION_L2_64B : CU_TENSOR_MAP_L2_PROMOTION_NONE);
        r1 = enc(&mp.k, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, pool.key_cache, kdims, kstrides, kbox, ones,
                 CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle_of((int)krow), kpromo, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
        const cuuint64_t vdims[2] = {vrow, NB * Hkv * D};
        const cuuint64_t vstrides[1] = {vrow};
        const cuuint32_t vbox[2] = {(cuuint32_t)vrow, (cuuint32_t)D};
        r2 = enc(&mp.v, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, pool.value_cache, vdims, vstrides, vbox, ones,
                 CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle_of((int)vrow), CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                 CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    }
    if (r1 != CUDA_SUCCESS || r2 != CUDA_SUCCESS)
        return fail(EMLX_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d, %d)", (int)r1, (int)r2);
    return EMLX_OK;
}

// Tensor maps depend only on the pool's address and geometry; they are encoded once and cached.  The pair is
// copied out while the lock is held, so a concurrent call that evicts the cache cannot invalidate it.
int get_maps(const emlx_pool& pool, MapPair* out) {
    static std::mutex mu;
    static std::map<std::tuple<void*, void*, long long, int, int, int, int, int>, MapPair> cache;
    auto key = std::make_tuple(pool.key_cache, pool.value_cache, (long long)pool.num_blocks, pool.num_kv_heads,
                               pool.head_dim, pool.kv_format, pool.kv_dtype, pool.block_size);
    std::lock_guard<std::mutex> lock(mu);
    auto it = cache.find(key);
    if (it != cache.end()) {
        *out = it->second;
        return EMLX_OK;
    }
    MapPair mp;
    if (int rc = encode_maps(pool, &mp)) return rc;
    if (cache.size() > 256) cache.clear();
    cache[key] = mp;
    *out = mp;
    return EMLX_OK;
}

template <int D, int NT, int FMT, bool BF16>
static int launch_one(const MapPair& maps, const TiledParams& p, int grid, cudaStream_t stream) {
    using C = Cfg<D, NT, FMT>;
    // Three builds of the kernel.  Codes paths that an ordinary batch never takes still cost it a per cent or two
    // when they sit in the same kernel (measured; the tile loop is the same, its scheduling is not): the final merge
    // shared by the consumer warps is only built in for batches of few, long units, the gather only for gathering calls.
    auto go = [&](auto kernel, DeviceOnce& configured) -> int {
        EMLX_CUDA_OK(allow_dynamic_smem(kernel, C::SMEM, configured));
        EMLX_CUDA_OK(launch_pdl(kernel, grid, kThreads, C::SMEM, stream, maps.k, maps.v, p));
        return EMLX_OK;
    };
    static DeviceOnce once_plain, once_help, once_gather;
    int rc;
    if (p.peer) rc = go(attn_tiled_kernel<D, NT, FMT, BF16, true, true, false>, once_gather);
    else if (p.few_units) rc = go(attn_tiled_kernel<D, NT, FMT, BF16, false, true, false>, once_help);
    else rc = go(attn_tiled_kernel<D, NT, FMT, BF16, false, false, false>, once_plain);
    if (rc) return rc;
    EMLX_LAUNCHED();
    return EMLX_OK;
}

template <int D, int NT>
static int launch_fmt(int fmt, bool bf16, const MapPair& maps, const TiledParams& p, int grid, cudaStream_t stream) {
    if (fmt == EMLX_KV_AFFINE8) return bf16 ? launch_one<D, NT, 8, true>(maps, p, grid, stream) : launch_one<D, NT, 8, false>(maps, p, grid, stream);
    if (fmt == EMLX_KV_AFFINE4) return bf16 ? launch_one<D, NT, 4, true>(maps, p, grid, stream) : launch_one<D, NT, 4, false>(maps, p, grid, stream);
    return bf16 ? launch_one<D, NT, 0, true>(maps, p, grid, stream) : launch_one<D, NT, 0, false>(maps, p, grid, stream);
}

static int launch_class(int cls, int D, int fmt, bool bf16, const MapPair& maps, const TiledParams& p, int grid, cudaStream_t s) {
    if (D == 128) {
        if (cls == 0) return launch_fmt<128, 1>(fmt, bf16, maps, p, grid, s);
        if (cls == 1) return launch_fmt<128, 2>(fmt, bf16, maps, p, grid, s);
        return launch_fmt<128, 4>(fmt, bf16, maps, p, grid, s);
    }
    if (cls == 0) return launch_fmt<64, 1>(fmt, bf16, maps, p, grid, s);
    if (cls == 1) return launch_fmt<64, 2>(fmt, bf16, maps, p, grid, s);
    return launch_fmt<64, 4>(fmt, bf16, maps, p, grid, s);
}

// Measurement aid, only in builds with -DEMLX_TRACE: a device buffer of at least 4 * 256 int64 into which every CTA
// of the tiled kernel writes {start ns, end ns, tiles processed, SM id}; -DEMLX_TRACE_PARTS / -DEMLX_TRACE_PREFILL
// add per-part and per-tile records behind those (the buffer must then hold 1024 + 256 * 16 * 4 int64).
#ifdef EMLX_TRACE
static long long* g_trace = nullptr;
#ifdef EMLX_TRACE_TIMELINE
// every launch that asks gets the next of 16 regions of 8192 int64, so that the kernels of consecutive steps captured
// into one CUDA graph leave separate records
static int g_trace_launch = 0;
long long* trace_buffer() { return g_trace ? g_trace + (size_t)(g_trace_launch++ % 16) * 8192 : nullptr; }
#else
long long* trace_buffer() { return g_trace; }
#endif
#else
long long* trace_buffer() { return nullptr; }
#endif

// A gathering call: the flag block of this rank and where its heads sit in the full output.
struct GatherTarget {
    void* flag_block;
    int total_q_heads, head_offset;
};

static int run_tiled(const emlx_attn_args* a, const emlx_pool* pool, void* stream, int class_lo, int class_hi,
                     const GatherTarget* gather = nullptr) {
    if (int rc = validate_attn(a, pool, true)) return rc;
    if (a->total_tokens == 0) return EMLX_OK;
    const int D = pool->head_dim, Hq = a->num_q_heads, Hkv = pool->num_kv_heads, G = Hq / Hkv;
    if (!tiled_page_size_ok(pool->block_size, pool->kv_format))
        return fail(EMLX_ERR_UNSUPPORTED, "the tiled kernels need page size 128 (16, 32 or 64 also for fp16/bf16 pools)");
    if (D != 64 && D != 128) return fail(EMLX_ERR_UNSUPPORTED, "the tiled kernels need head_dim 64 or 128");
    if (a->q_dtype == EMLX_F32) return fail(EMLX_ERR_UNSUPPORTED, "the tiled kernels need fp16 or bf16 queries");
    const bool bf16 = a->q_dtype == EMLX_BF16;
    if (pool->kv_format == EMLX_KV_FLOAT && pool->kv_dtype != a->q_dtype)
        return fail(EMLX_ERR_UNSUPPORTED, "the tiled kernels need the pool dtype to equal the query dtype");
    const PlanLayout L = plan_layout(a->num_seqs, a->total_tokens, Hq, Hkv);
    const WorkspaceLayout W = workspace_layout(a->num_seqs, a->total_tokens, Hq, Hkv, D);
    if (a->plan_bytes < (size_t)L.words * 4 || a->workspace_bytes < W.bytes)
        return fail(EMLX_ERR_WORKSPACE, "plan/workspace smaller than emlx_attn_plan_bytes()/emlx_attn_workspace_bytes()");
    if (((uintptr_t)a->queries | (uintptr_t)a->out) & 15) return fail(EMLX_ERR_INVALID, "queries/out must be 16-byte aligned");
    MapPair maps;
    if (int rc = get_maps(*pool, &maps)) return rc;

    // the row classes a plan holds depend on the flags it was built with, not on what this pool could support
    const bool wide = (a->plan_flags & kPlanWideUnits) != 0;
    // 128-row units over an affine pool: the pages of the sequences that own them are expanded into scratch memory that
    // the caller appended to the workspace (emlx_attn_dequant_bytes), and the 128-row kernel reads that
    const bool expand = wide && pool->kv_format != EMLX_KV_FLOAT;
    DequantScratch scratch{};
    if (expand) {
        if (!prefill_geometry_ok(Hq, Hkv, D))
            return fail(EMLX_ERR_INVALID, "plan_flags ask for 128-row units, which this head geometry cannot run");
        if (!dequant_scratch_layout(pool, a, (uint8_t*)a->workspace + W.bytes, a->workspace_bytes - W.bytes, &scratch))
            return fail(EMLX_ERR_WORKSPACE, "128-row units over an affine pool need emlx_attn_dequant_bytes() of memory "
                                            "behind the workspace");
    } else if (wide && !prefill_supported(pool->kv_format, Hq, Hkv, D)) {
        return fail(EMLX_ERR_INVALID, "plan_flags ask for 128-row units, which this pool / head geometry cannot run");
    }
    int lo, hi;
    class_range(G, a->max_query_len, wide, lo, hi);
    if (max(lo, class_lo) > min(hi, class_hi))
        return fail(EMLX_ERR_UNSUPPORTED,
                    "this plan holds row classes %d..%d and the entry point serves %d..%d: nothing to launch (build "
                    "the plan with other plan_flags or call emlx_attn_unified)", lo, hi, class_lo, class_hi);
    lo = max(lo, class_lo);
    hi = min(hi, class_hi);
    const int32_t* plan = (const int32_t*)a->plan;
    bool short_rows_launched = false;
    int first_launched = -1, last_launched = -1;
    for (int c = lo; c <= hi; ++c) {
        if (a->row_class_mask != 0 && !((a->row_class_mask >> c) & 1)) continue;
        if (first_launched < 0) first_launched = c;
        last_launched = c;
    }
    if (first_launched < 0) return fail(EMLX_ERR_UNSUPPORTED, "row_class_mask names no row class that this call can launch");
    const bool class3 = hi == 3 && (a->row_class_mask == 0 || ((a->row_class_mask >> 3) & 1));
    // the expansion comes first: the short-row kernels wait for it at their start, and the 128-row kernel, which may
    // run beside them, starts only after all their CTAs have passed that wait
    if (expand && class3)
        if (int rc = launch_dequant_pages(a, pool, scratch, (cudaStream_t)stream, a->sliding_window, 0)) return rc;
    for (int c = lo; c <= hi; ++c) {
        if (a->row_class_mask != 0 && !((a->row_class_mask >> c) & 1)) continue;  // the caller knows this class is empty
        if (c == 3) {
            // the 128-row kernel comes last; behind a short-row kernel of this call it runs beside that kernel
            emlx_attn_args a3 = *a;
            emlx_pool pool3 = *pool;
            MapPair maps3 = maps;
            if (expand) {  // the scratch pool stands in for the pool: fp16 rows (also under bf16 queries), its own page table
                pool3.key_cache = scratch.k; pool3.value_cache = scratch.v;
                pool3.k_scale = pool3.k_bias = pool3.v_scale = pool3.v_bias = nullptr;
                pool3.num_blocks = scratch.cap; pool3.block_size = kTile;
                pool3.kv_format = EMLX_KV_FLOAT; pool3.kv_dtype = EMLX_F16;
                a3.block_tables = scratch.sbt;
                if (a->q_dtype == EMLX_BF16) {
                    // the tensor core takes both operands of a product in one type: fp16 copies of these sequences'
                    // queries (made by the expansion kernel) go in, fp16 rows come out and are converted below
                    a3.queries = scratch.q16; a3.out = scratch.out16; a3.q_dtype = EMLX_F16;
                }
                if (int rc = get_maps(pool3, &maps3)) return rc;
            }
            if (int rc = launch_prefill(&a3, &pool3, plan + 4 * c, plan + L.unit_seq[c], plan + L.unit_row0[c],
                                        plan + L.unit_tile_lo[c], plan + L.unit_cum[c], plan + L.unit_order,
                                        (int32_t*)((uint8_t*)a->workspace + W.counter_off[3]), short_rows_launched, maps3,
                                        (cudaStream_t)stream))
                return rc;
            if (expand && a->q_dtype == EMLX_BF16)
                if (int rc = launch_convert_out_rows(a, pool, scratch, (cudaStream_t)stream)) return rc;
            continue;
        }
        short_rows_launched = true;
        TiledParams p;
        p.q = a->queries; p.out = a->out; p.bt = a->block_tables; p.kv_lens = a->kv_lens; p.qsl = a->query_start_loc;
        p.hdr = plan + 4 * c;
        p.unit_seq = plan + L.unit_seq[c]; p.unit_row0 = plan + L.unit_row0[c];
        p.unit_tile_lo = plan + L.unit_tile_lo[c]; p.unit_cum = plan + L.unit_cum[c];
        p.cta_start = plan + L.cta_start[c];
        p.cta_unit = plan + L.cta_unit[c];
        p.counters = (int32_t*)((uint8_t*)a->workspace + W.counter_off[c]);
        p.slots = (float*)((uint8_t*)a->workspace + W.slots_off);
        p.status = a->status;
        p.trace = trace_buffer();
        p.k_scale = (const __half*)pool->k_scale; p.k_bias = (const __half*)pool->k_bias;
        p.v_scale = (const __half*)pool->v_scale; p.v_bias = (const __half*)pool->v_bias;
        p.num_blocks = pool->num_blocks;
        p.Hq = Hq; p.Hkv = Hkv; p.G = G; p.MB = a->max_blocks_per_seq; p.window = a->sliding_window;
        p.bs = pool->block_size; p.ppt_log = pages_per_tile_log2(pool->block_size);
        p.scale_log2e = a->softmax_scale * 1.4426950408889634f;
        p.out_Hq = gather ? gather->total_q_heads : Hq;
        p.out_head0 = gather ? gather->head_offset : 0;
        p.peer = gather ? (const PeerTable*)((const uint8_t*)gather->flag_block + kPeerTableOffset) : nullptr;
        p.peer_flags = gather ? (int32_t*)gather->flag_block : nullptr;
        p.peer_phase = (c == first_launched ? kPeerFirstLaunch : 0) | (c == last_launched ? kPeerLastLaunch : 0);
        // a (sequence, KV head) unit is shared by about grid / units CTAs
        p.few_units = (long long)a->num_seqs * Hkv * (kHelpMinParts - 1) <=
                      class_ctas(c, min(num_sms(), kMaxGrid), (a->plan_flags & kPlanTwoCtas) != 0);
        // the grid a class is launched with is the one its slices were cut for
        const int grid = class_ctas(c, min(num_sms(), kMaxGrid), (a->plan_flags & kPlanTwoCtas) != 0);
        if (int rc = launch_class(c, D, pool->kv_format, bf16, maps, p, grid, (cudaStream_t)stream)) return rc;
    }
    return EMLX_OK;
}

}  // namespace emlx

#ifdef EMLX_TRACE
extern "C" __attribute__((visibility("default"))) void emlx_set_trace_buffer(int64_t* records) {
    emlx::g_trace = (long long*)records;
#ifdef EMLX_TRACE_TIMELINE
    emlx::g_trace_launch = 0;
#endif
}
#endif
extern "C" {
int emlx_attn_unified(const emlx_attn_args* a, const emlx_pool* p, void* s) { return emlx::run_tiled(a, p, s, 0, emlx::kNumClasses - 1); }
int emlx_attn_decode(const emlx_attn_args* a, const emlx_pool* p, void* s) { return emlx::run_tiled(a, p, s, 0, 2); }
int emlx_attn_prefill(const emlx_attn_args* a, const emlx_pool* p, void* s) { return emlx::run_tiled(a, p, s, 3, 3); }
int emlx_attn_decode_gather(const emlx_attn_args* a, const emlx_pool* p, void* flag_block, int32_t total_q_heads,
                            int32_t head_offset, void* s) {
    if (!a || !flag_block) return emlx::fail(EMLX_ERR_INVALID, "gather: null argument");
    if (head_offset < 0 || total_q_heads < head_offset + a->num_q_heads)
        return emlx::fail(EMLX_ERR_INVALID, "gather: heads [%d, %d) do not fit %d output heads", head_offset,
                          head_offset + a->num_q_heads, total_q_heads);
    if (a->plan_flags & emlx::kPlanWideUnits)
        return emlx::fail(EMLX_ERR_UNSUPPORTED, "gather: build the work list without 128-row units (plan_flags bit 0)");
    const emlx::GatherTarget g{flag_block, total_q_heads, head_offset};
    return emlx::run_tiled(a, p, s, 0, 2, &g);
}
int emlx_attn_plan_flags(int32_t kv_format, int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim) {
    return (emlx::prefill_supported(kv_format, num_q_heads, num_kv_heads, head_dim) ? emlx::kPlanWideUnits : 0) |
           (kv_format == EMLX_KV_AFFINE4 ? emlx::kPlanTwoCtas : 0);
}
int emlx_attn_row_class(int32_t kv_format, int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim, int32_t query_len) {
    if (query_len <= 0 || num_kv_heads <= 0 || num_q_heads <= 0 || num_q_heads % num_kv_heads) return -1;
    const long long rows = (long long)query_len * (num_q_heads / num_kv_heads);
    return emlx::unit_class(rows > (1 << 20) ? (1 << 20) : (int)rows,
                            emlx::prefill_supported(kv_format, num_q_heads, num_kv_heads, head_dim));
}
}
