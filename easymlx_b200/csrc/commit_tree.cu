// Keeping the accepted path of a draft tree: the K/V rows of the accepted tokens move to the front of the tree's rows, in
// every layer's pool, and the stored lengths grow by the path.
//
// The accepted indices increase, so row j of the path never lies before its destination and a destination is never the
// source of a later row: whoever owns a column of the rows (16 bytes of a key row; one element of the transposed value
// codes) moves it for one token after the other, four loads in flight, and needs no staging.
//
// One CTA serves one (layer, sequence); all layers go in one launch (32 descriptors fit the kernel's parameters), since
// a row is a few KB and a launch per layer would cost more than the move.  Bound by launch latency and by the chain length ->
// page id -> row -> store; a large batch by HBM (24 layers and 64 paths of up to 8 rows of 2 KB: 18 us; 16 layers and
// one path: 4.3 us).  The lengths are advanced by the CTA that draws the last ticket, after
// every CTA has read them: layers may share their tables.
#include "common.cuh"

namespace emlx {

int validate_pool(const emlx_pool* pool);

namespace {

constexpr int kCommitThreads = 256;
constexpr int kCommitLayers = 32;
constexpr int kPathChunk = 64;  // path rows whose addresses are in shared memory at a time

struct CommitParams {
    emlx_commit_layer layer[kCommitLayers];
    const int32_t* slot_ids;
    const int32_t* accepted;
    int32_t* committed;
    int32_t* ticket;
    int32_t* status;
    int S, M, num_slots, MB, bs, Hkv, D, format, row_bytes, write_lens, any_advance;
};

// `unit` bytes per thread and step; rows are `bytes` long and start at base + row * bytes.
template <typename V>
__device__ __forceinline__ void move_rows(uint8_t* base, int64_t bytes, const int64_t* src, const int64_t* dst, int n) {
    constexpr int kDeep = 4;
    for (int64_t c = threadIdx.x; c < bytes / (int64_t)sizeof(V); c += kCommitThreads) {
        for (int j0 = 0; j0 < n; j0 += kDeep) {
            V v[kDeep];
#pragma unroll
            for (int k = 0; k < kDeep; ++k)
                if (j0 + k < n) v[k] = ((const V*)(base + src[j0 + k] * bytes))[c];
#pragma unroll
            for (int k = 0; k < kDeep; ++k)
                if (j0 + k < n && src[j0 + k] != dst[j0 + k]) ((V*)(base + dst[j0 + k] * bytes))[c] = v[k];
        }
    }
}
__device__ __forceinline__ void move_rows_any(void* base, int64_t bytes, const int64_t* src, const int64_t* dst, int n) {
    if (((bytes | (int64_t)(uintptr_t)base) & 15) == 0) move_rows<uint4>((uint8_t*)base, bytes, src, dst, n);
    else if (((bytes | (int64_t)(uintptr_t)base) & 3) == 0) move_rows<uint32_t>((uint8_t*)base, bytes, src, dst, n);
    else move_rows<uint8_t>((uint8_t*)base, bytes, src, dst, n);
}

__global__ void __launch_bounds__(kCommitThreads) commit_tree_kernel(const __grid_constant__ CommitParams p) {
    __shared__ int64_t s_src[kPathChunk], s_dst[kPathChunk];
    __shared__ int s_len, s_bad, s_last;
    grid_dep_wait();
    grid_dep_launch();
    const int tid = threadIdx.x, i = blockIdx.x;
    const emlx_commit_layer& layer = p.layer[blockIdx.y];
    const int slot = p.slot_ids[i];
    const int32_t* path = p.accepted + (int64_t)i * p.M;
    if (tid == 0) { s_len = p.M; s_bad = 0; }
    __syncthreads();
    const bool known = slot >= 0 && slot < p.num_slots;
    const int ctx = known ? layer.kv_lens[slot] : 0;
    if (!known) { if (tid == 0) s_bad = EMLX_DEV_BAD_SLOT; }
    else {
        for (int j = tid; j < i; j += kCommitThreads)
            if (p.slot_ids[j] == slot) atomicOr(&s_bad, EMLX_DEV_BAD_SLOT);
        for (int j = tid; j < p.M; j += kCommitThreads)
            if (path[j] < 0) atomicMin(&s_len, j);
    }
    __syncthreads();
    const int n = s_len;
    if (known) {
        const int32_t* table = layer.block_tables + (int64_t)slot * p.MB;
        for (int j = tid; j < n; j += kCommitThreads) {
            int bad = 0;
            if (path[j] < j || (j > 0 && path[j] <= path[j - 1])) bad = EMLX_DEV_BAD_TREE;
            else {
                const int64_t from = (int64_t)ctx + path[j], to = (int64_t)ctx + j;
                if (ctx < 0 || from >= (int64_t)p.MB * p.bs) bad = EMLX_DEV_OVERFLOW;
                else {
                    const int a = table[from / p.bs], b = table[to / p.bs];
                    if (a < 0 || a >= layer.num_blocks || b < 0 || b >= layer.num_blocks) bad = EMLX_DEV_BAD_PAGE;
                }
            }
            if (bad) atomicOr(&s_bad, bad);
        }
    }
    __syncthreads();
    const int bad = s_bad;
    if (bad && tid == 0) flag_error(p.status, bad);
    if (p.write_lens && blockIdx.y == 0 && tid == 0) p.committed[i] = ctx + (bad ? 0 : n);
    if (!bad) {
        const int32_t* table = layer.block_tables + (int64_t)slot * p.MB;
        for (int j0 = 0; j0 < n; j0 += kPathChunk) {
            const int m = min(kPathChunk, n - j0);
            if (tid < m) {
                const int from = ctx + path[j0 + tid], to = ctx + j0 + tid;
                s_src[tid] = (int64_t)table[from / p.bs] * p.bs + from % p.bs;
                s_dst[tid] = (int64_t)table[to / p.bs] * p.bs + to % p.bs;
            }
            __syncthreads();
            move_rows_any(layer.key_cache, p.row_bytes, s_src, s_dst, m);
            if (p.format == EMLX_KV_FLOAT) {
                move_rows_any(layer.value_cache, p.row_bytes, s_src, s_dst, m);
            } else {
                // value codes [NB, Hkv, D, bs]: a thread owns one (head, element) and all tokens of the path in it
                uint8_t* v = (uint8_t*)layer.value_cache;
                const int col_bytes = p.bs * p.format / 8;
                for (int c = tid; c < p.Hkv * p.D; c += kCommitThreads)
                    for (int j = 0; j < m; ++j) {
                        const int64_t sp = s_src[j] / p.bs, dp = s_dst[j] / p.bs;
                        const int so = (int)(s_src[j] - sp * p.bs), to = (int)(s_dst[j] - dp * p.bs);
                        const uint8_t* src = v + (sp * p.Hkv * p.D + c) * col_bytes;
                        uint8_t* dst = v + (dp * p.Hkv * p.D + c) * col_bytes;
                        if (p.format == EMLX_KV_AFFINE8) dst[to] = src[so];
                        else {
                            const int code = (src[so >> 1] >> ((so & 1) * 4)) & 15, shift = (to & 1) * 4;
                            dst[to >> 1] = (uint8_t)((dst[to >> 1] & ~(15 << shift)) | (code << shift));
                        }
                    }
                // scales and biases [NB, Hkv, bs, D / 64]
                const int groups = p.D / kQuantGroup;
                for (int c = tid; c < 4 * p.Hkv * groups; c += kCommitThreads) {
                    const int which = c / (p.Hkv * groups), h = c / groups % p.Hkv, g = c % groups;
                    uint16_t* a = (uint16_t*)(which == 0 ? layer.k_scale : which == 1 ? layer.k_bias : which == 2 ? layer.v_scale : layer.v_bias);
                    for (int j = 0; j < m; ++j) {
                        const int64_t sp = s_src[j] / p.bs, dp = s_dst[j] / p.bs;
                        const int64_t so = s_src[j] - sp * p.bs, to = s_dst[j] - dp * p.bs;
                        a[((dp * p.Hkv + h) * p.bs + to) * groups + g] = a[((sp * p.Hkv + h) * p.bs + so) * groups + g];
                    }
                }
            }
            __syncthreads();
        }
    }
    if (!p.any_advance) return;
    // every CTA of the launch has read the lengths when the last ticket is drawn
    __syncthreads();
    if (tid == 0) {
        __threadfence();
        s_last = atomicAdd(p.ticket, 1) == (int)(gridDim.x * gridDim.y) - 1 ? 1 : 0;
    }
    __syncthreads();
    if (!s_last) return;
    __threadfence();
    for (int k = tid; k < p.S; k += kCommitThreads) {
        // committed holds layer 0's result; a sequence that was left alone keeps its length, a slot named twice has the
        // first one's
        const int sl = p.slot_ids[k];
        bool first = sl >= 0 && sl < p.num_slots;
#pragma unroll 8
        for (int j = 0; j < k; ++j) first = first && p.slot_ids[j] != sl;
        if (!first) continue;
        const int len = __ldcg(p.committed + k);
        for (int y = 0; y < (int)gridDim.y; ++y)
            if (p.layer[y].advance) p.layer[y].kv_lens[sl] = len;
    }
    if (tid == 0) *p.ticket = 0;
}

}  // namespace
}  // namespace emlx

extern "C" int emlx_commit_tree(const emlx_commit_layer* layers, int32_t num_layers, const emlx_pool* pool,
                                const int32_t* slot_ids, int32_t num_seqs, const int32_t* accepted, int32_t max_path,
                                int32_t num_slots, int32_t max_blocks_per_seq, int32_t* committed, int32_t* ticket,
                                int32_t* status, void* stream) {
    using namespace emlx;
    if (!layers || num_layers <= 0) return fail(EMLX_ERR_INVALID, "commit_tree: no layers");
    if (!pool) return fail(EMLX_ERR_INVALID, "pool is NULL");
    if (num_seqs < 0 || max_path < 0) return fail(EMLX_ERR_INVALID, "num_seqs/max_path must be non-negative");
    if (num_slots <= 0 || max_blocks_per_seq <= 0) return fail(EMLX_ERR_INVALID, "max_blocks_per_seq and num_slots must be positive");
    for (int y = 0; y < num_layers; ++y) {
        emlx_pool one = *pool;
        one.key_cache = layers[y].key_cache; one.value_cache = layers[y].value_cache;
        one.k_scale = layers[y].k_scale; one.k_bias = layers[y].k_bias;
        one.v_scale = layers[y].v_scale; one.v_bias = layers[y].v_bias;
        one.num_blocks = layers[y].num_blocks;
        if (int rc = validate_pool(&one)) return rc;
        if (!layers[y].block_tables || !layers[y].kv_lens) return fail(EMLX_ERR_INVALID, "commit_tree: layer without tables");
    }
    if (num_seqs == 0) return EMLX_OK;
    if (!slot_ids || !committed || !ticket || (max_path > 0 && !accepted)) return fail(EMLX_ERR_INVALID, "commit_tree: NULL argument");
    CommitParams p;
    p.slot_ids = slot_ids; p.accepted = accepted; p.committed = committed; p.ticket = ticket; p.status = status;
    p.S = num_seqs; p.M = max_path; p.num_slots = num_slots; p.MB = max_blocks_per_seq;
    p.bs = pool->block_size; p.Hkv = pool->num_kv_heads; p.D = pool->head_dim; p.format = pool->kv_format;
    const int64_t bits = pool->kv_format == EMLX_KV_FLOAT ? (pool->kv_dtype == EMLX_F32 ? 32 : 16) : pool->kv_format;
    p.row_bytes = (int)(pool->num_kv_heads * (int64_t)pool->head_dim * bits / 8);
    for (int y0 = 0; y0 < num_layers; y0 += kCommitLayers) {
        const int n = num_layers - y0 < kCommitLayers ? num_layers - y0 : kCommitLayers;
        for (int y = 0; y < kCommitLayers; ++y) p.layer[y] = layers[y0 + (y < n ? y : 0)];
        // lengths that several layers share advance once, behind the last of those layers (it may be in a later launch)
        for (int y = 0; y < n; ++y) {
            int wanted = 0, last = 1;
            for (int k = 0; k < num_layers; ++k)
                if (layers[k].kv_lens == layers[y0 + y].kv_lens) {
                    wanted |= layers[k].advance;
                    if (k > y0 + y) last = 0;
                }
            p.layer[y].advance = wanted && last;
        }
        p.write_lens = y0 == 0;
        p.any_advance = 0;
        for (int y = 0; y < n; ++y) p.any_advance |= p.layer[y].advance;
        EMLX_CUDA_OK(launch_pdl(commit_tree_kernel, dim3((unsigned)num_seqs, (unsigned)n), kCommitThreads, 0, (cudaStream_t)stream, p));
        EMLX_LAUNCHED();
    }
    return EMLX_OK;
}
