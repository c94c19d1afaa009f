// Which keys a row sees beyond a plain causal sequence: sliding windows whose first tokens stay visible, and trees of
// drafted tokens.
//
// A sequence has ctx = kv_len - q_len keys from earlier steps and q_len new ones.  The *visible sequence* of row i is
// the context followed by the new keys j whose mask bit is set, in slot order (a causal row: every j <= i); n_i is the
// number of those.  A window W keeps the entries of rank >= ctx + n_i - W, sinks N keep the entries of rank < N on top.
// For a causal row the rank of a key is its position, so this is the usual window; for a tree it is the position the
// key has on the row's own path.
#pragma once
#include "common.cuh"

namespace emlx {

constexpr int kMaxTreeWords = 64;  // 4096 drafted tokens per sequence

struct Visibility {
    const uint64_t* tree;      // [T, words], nullptr: every row is causal
    const int32_t* tree_seqs;  // [S] nonzero: rows of the sequence follow the mask; nullptr: all sequences do
    int words, sinks, window;
};

inline Visibility make_visibility(const emlx_visibility* v, int window) {
    Visibility r{};
    r.window = window;
    if (v) {
        r.tree = v->tree_mask;
        r.tree_seqs = v->tree_seqs;
        r.words = v->tree_words;
        r.sinks = window > 0 ? v->sink_tokens : 0;  // without a window every key is visible anyway
    }
    return r;
}
int validate_visibility(const emlx_visibility* v, int window);

__device__ __forceinline__ bool is_tree(const Visibility& v, int seq) {
    return v.tree != nullptr && (v.tree_seqs == nullptr || v.tree_seqs[seq] != 0);
}

// Word w of a row's mask without the bits past the sequence's q_len tokens.
__device__ __forceinline__ uint64_t tree_word(const Visibility& v, const uint64_t* row, int w, int q_len) {
    const int left = q_len - 64 * w;
    if (w >= v.words || left <= 0) return 0;
    const uint64_t x = row[w];
    return left >= 64 ? x : x & ((1ull << left) - 1);
}

// Entries of a row's visible sequence that are new keys: n_i.
__device__ __forceinline__ int tree_count(const Visibility& v, const uint64_t* row, int q_len) {
    int n = 0;
    for (int w = 0; w < v.words; ++w) n += __popcll(tree_word(v, row, w, q_len));
    return n;
}

// First context key inside the window of a row with n visible new keys (0 without a window).
__device__ __forceinline__ int window_lo(const Visibility& v, int ctx, int n) {
    return v.window > 0 ? max(0, ctx + n - v.window) : 0;
}

// Bits of `x` without those whose rank among its set bits (starting at `rank`) lies in [first, last).
__device__ __forceinline__ uint64_t drop_ranks(uint64_t x, int rank, int first, int last) {
    uint64_t kept = 0;
    while (x) {
        const uint64_t low = x & (0 - x);
        if (rank < first || rank >= last) kept |= low;
        x ^= low;
        ++rank;
    }
    return kept;
}

}  // namespace emlx
