// Stand-alone work list of an attention call with sinks or a draft tree, for callers that bring their own
// query_start_loc / kv_lens.  CTA 0 builds the list, the others the masks of windowed trees.
#include "visible_plan.cuh"

namespace emlx {

__global__ void __launch_bounds__(kVpThreads) visible_plan_kernel(const VisiblePlanArgs a, const Visibility vis,
                                                                  const int32_t* qsl, const int32_t* kv_lens, int S, int T,
                                                                  int32_t* status) {
    __shared__ int32_t scan_smem[kVpThreads / 32 + 1];
    grid_dep_wait();
    grid_dep_launch();
    if (blockIdx.x == 0) {
        __shared__ int32_t s_q[kVpSeqs + 1], s_kv[kVpSeqs];
        if (S <= kVpSeqs) {
            for (int s = threadIdx.x; s <= S; s += kVpThreads) {
                s_q[s] = qsl[s];
                if (s < S) s_kv[s] = kv_lens[s];
            }
            __syncthreads();
            qsl = s_q;
            kv_lens = s_kv;
        }
        build_visible_plan(a, vis, qsl, kv_lens, S, scan_smem, status);
        return;
    }
    for (int t = (blockIdx.x - 1) * kVpThreads + threadIdx.x; t < T; t += (gridDim.x - 1) * kVpThreads) {
        const int s = find_sequence(qsl, S, t);
        if (s < 0 || !is_tree(vis, s)) continue;
        const int q_len = qsl[s + 1] - qsl[s];
        write_effective_mask(vis, t, kv_lens[s] - q_len, q_len, (uint64_t*)(a.plan + a.L.eff));
    }
}

}  // namespace emlx

extern "C" {

size_t emlx_visible_plan_bytes(int32_t num_seqs, int32_t total_tokens, int32_t num_q_heads, int32_t num_kv_heads, int32_t tree_words) {
    if (num_kv_heads <= 0 || num_q_heads <= 0 || num_seqs < 0 || total_tokens < 0 || tree_words < 0) return 0;
    return emlx::visible_plan_bytes(num_seqs, total_tokens, num_q_heads, num_kv_heads, tree_words);
}

int emlx_visible_plan(const int32_t* query_start_loc, const int32_t* kv_lens, int32_t num_seqs, int32_t total_tokens,
                      int32_t num_q_heads, int32_t num_kv_heads, int32_t block_size, int32_t sliding_window,
                      const emlx_visibility* visibility, int32_t max_query_len, int32_t plan_flags, void* plan,
                      size_t plan_bytes, int32_t* status, void* stream) {
    using namespace emlx;
    if (int rc = validate_visibility(visibility, sliding_window)) return rc;
    if (num_seqs < 0 || total_tokens < 0) return fail(EMLX_ERR_INVALID, "num_seqs/total_tokens must be non-negative");
    if (num_seqs > 0 && (!query_start_loc || !kv_lens)) return fail(EMLX_ERR_INVALID, "visible_plan: NULL input");
    const Visibility vis = make_visibility(visibility, sliding_window);
    VisiblePlanArgs a;
    if (int rc = visible_plan_args(&a, num_seqs, total_tokens, num_q_heads, num_kv_heads, block_size, max_query_len, plan_flags,
                                   vis, plan, plan_bytes))
        return rc;
    const int masks = vis.tree && vis.window > 0 ? min((total_tokens + kVpThreads - 1) / kVpThreads, 64) : 0;
    EMLX_CUDA_OK(launch_pdl(visible_plan_kernel, dim3(1u + (unsigned)masks), kVpThreads, 0, (cudaStream_t)stream, a, vis,
                            query_start_loc, kv_lens, num_seqs, total_tokens, status));
    EMLX_LAUNCHED();
    return EMLX_OK;
}

}  // extern "C"
