// What the two kernels of attention over trees of drafted tokens share.
//
// A request of the step brings n tokens that form a tree (or several): node i is cached at place len + i behind the request's len
// settled tokens, but sits at position len + depth.  It sees the settled tokens that its window lets its position see, and of the
// step's own tokens those whose bit is set in its row of `ancestors` (itself among them), as far as its window reaches back to
// their positions.  A node whose own bit is not set is padding: nobody sees it, whatever other rows say, and its row of the cache
// may hold anything; it sees the settled tokens and the ancestors it names.
#pragma once
#include "attention.cuh"

struct TreeStep {
    const int* cu_seqlens;       // [n_segments + 1]
    const unsigned* ancestors;   // [tokens, n_words]
    int n_segments;
    int n_words;
};

// Is node `i` of the segment that starts at token `first` a token of its own (its own bit is set)?
__device__ __forceinline__ bool tree_node_is_real(const TreeStep& x, int first, int i) {
    return i < 32 * x.n_words && (x.ancestors[(size_t)(first + i) * x.n_words + i / 32] >> (i % 32) & 1u);
}

// The sink folded into a row's finished state (as fold_sink); one of minus infinity adds nothing, also to a row that sees no key.
__device__ __forceinline__ float tree_fold_sink(const AttentionParams& p, int head, float m, float& l) {
    return p.has_sink && sink_of(p, head) > -INFINITY ? fold_sink(p, head, m, l) : 1.f;
}
