// What the two kernels of attention over trees of drafted tokens share.
//
// A request of the step brings n tokens that form a tree (or several): node i is cached at place len + i behind the request's len
// settled tokens, but sits at position len + depth.  It sees the settled tokens that its window lets its position see, and of the
// step's own tokens those whose bit is set in its row of `ancestors` (itself among them), as far as its window reaches back to
// their positions.  A node whose own bit is not set is padding: nobody sees it, whatever other rows say, and its row of the cache
// may hold anything; it sees the settled tokens and the ancestors it names.
#pragma once
#include "attention.cuh"

#include <atomic>

struct TreeStep {
    const int* cu_seqlens;       // [n_segments + 1]
    const unsigned* ancestors;   // [tokens, n_words]
    int n_segments;
    int n_words;
};

// What a call is given.
struct TreeCall {
    AttentionParams p;
    StepTokens b;
    PagedCache c;
    TreeStep x;
};
static inline bool tree_call_ok(const TreeCall& a) {
    if (!a.p.q || !a.p.out || !a.c.kv || !a.b.positions || !a.b.seg_of_token || !a.b.block_table || !a.x.cu_seqlens || !a.x.ancestors) return false;
    if (a.b.n_tokens < 0 || a.b.table_width < 1 || a.c.n_pages < 1 || a.c.page_size < 1 || a.x.n_segments < 1 || a.x.n_words < 1) return false;
    if (a.p.num_heads < 1 || a.c.num_kv_heads < 1 || a.p.num_heads % a.c.num_kv_heads || a.c.head_dim < 1) return false;
    return a.p.window_kind >= 0 && a.p.window_kind <= 2 && (a.p.window_kind == SPITE_WINDOW_FULL || a.p.window_size >= 1) && distance_bias_ok(&a.p);
}

// Lets a kernel take `most` bytes of dynamic shared memory, the most that any call of it needs: once a device (`done` has a bit each), since the limit
// is the process's, and a call that set it to its own size could lower it under another thread's launch.
template <typename K>
static bool allow_shared(K kernel, size_t most, std::atomic<unsigned long long>& done) {
    int device = 0;
    if (cudaGetDevice(&device) != cudaSuccess) return false;
    const unsigned long long bit = device < 64 ? 1ull << device : 0;
    if (done.load(std::memory_order_acquire) & bit) return true;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most) != cudaSuccess) return false;
    done.fetch_or(bit, std::memory_order_release);
    return true;
}

// Is node `i` of the segment that starts at token `first` a token of its own (its own bit is set)?
__device__ __forceinline__ bool tree_node_is_real(const TreeStep& x, int first, int i) {
    return i < 32 * x.n_words && (x.ancestors[(size_t)(first + i) * x.n_words + i / 32] >> (i % 32) & 1u);
}

// A row's maximum and sum as others read them: a sum that is NaN makes the maximum NaN (a row whose scores are all NaN has the maximum of a row
// that sees nothing, minus infinity, and would be passed over).
__device__ __forceinline__ float2 tree_state(float m, float l) { return make_float2(l != l ? l : m, l); }
// What a row's values are divided by: its sum, NaN included, or for a row that sees nothing a number that leaves its zeros.
__device__ __forceinline__ float tree_divisor(float l) { return l < 1e-30f ? 1e-30f : l; }

// The sink folded into a row's finished state (as fold_sink); one of minus infinity adds nothing, also to a row that sees no key.
__device__ __forceinline__ float tree_fold_sink(const AttentionParams& p, int head, float m, float& l) {
    return p.has_sink && sink_of(p, head) > -INFINITY ? fold_sink(p, head, m, l) : 1.f;
}
