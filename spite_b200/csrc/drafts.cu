// What stands around a step that verifies drafted tokens, without the host in between: the step's integer inputs from the requests'
// lengths (block tables with pages taken from and given back to a stack of free ones, slot map, positions, ancestor sets), and
// the walk down every request's tree by the target tokens with the accepted tokens' cache rows moved to their places.
//
// Both are bound by latency: a few dependent rounds through L2 and what is launched around them.  us on the device, in a graph of calls (a call
// takes the host 11 to 12): the layout of one request 5.4, of 64 trees with tables of 2,049 pages 8.4 where no page moves and 28 where two ended
// requests give 1,659 pages back and 16 are taken, of 250 portions with a sliding window 7.6, with 221 pages back and 32 taken 13.7; accepted
// paths of one request 4.1, of 8 requests in 48 caches 5.1, of 61 in 24 caches, 25.8 MB read and written, 8.5 (3.0 TB/s, much of it in L2).
// What bounds the layout is the plan, some ten dependent rounds by one block (L2, block barriers, the scan), and the pages that go back, a warp
// a request; what bounds the accepted paths is the
// chain lengths -> tree -> slot map -> rows, four round trips, and the largest only in part the bytes.
#include "common.cuh"

#define SPITE_MAX_DRAFTS 1024            // tokens of one request's tree
#define SPITE_LAYOUT_MAX_REQUESTS 4096   // requests of one step
#define SPITE_LAYOUT_MAX_ROWS (1 << 16)  // rows of the page tables (a bit each in shared memory)

// What `status` says (zero: the step is laid out).
#define SPITE_LAYOUT_OUT_OF_PAGES 1      // the stack holds fewer pages than the step needs
#define SPITE_LAYOUT_MALFORMED 2         // a slot twice or out of range, a length that the table does not cover, too many tokens

struct LayoutParams {
    int* tables;                 // [n_rows, table_width] page of a logical page, -1: none (before a row's first page, behind its last)
    int* held;                   // [n_rows] logical pages that a row reaches to
    int* free_pages;             // [n_pages] a stack, or null: the tables cover every token already and nothing is given back
    int* n_free;                 // [1] its height
    const int* slots;            // [n_requests] rows of the step's requests, -1: padding
    const int* lengths;          // [n_rows] tokens cached
    const int* new_tokens;       // [n_requests] tokens that the step brings, -1: the request has ended
    const int* parents;          // [n_parents] a token's parent within its request (-1: none), or null: every token follows the one before
    int* block_table;            // [n_requests, out_width]
    int* cu_seqlens;             // [n_requests + 1]
    int* positions;              // [n_tokens] (as the two below: rows behind the last request's stay as they are)
    int* seg_of_token;
    long long* slot_map;         // row of the cache, page * page_size + offset, -1: none
    unsigned* ancestors;         // [n_tokens, n_words], or null
    int* status;                 // [1]
    int n_rows, table_width, n_pages, n_requests, out_width, n_tokens, n_parents, n_words, page_size, window_kind, window_size;
};

namespace {

constexpr int PLAN_THREADS = 512, PLAN_WARPS = PLAN_THREADS / 32;
constexpr int FEW_PAGES = 4;             // that a request's own thread takes

__host__ __device__ __forceinline__ int first_needed(const LayoutParams& p, int len) {       // (a later token reads nothing before it)
    if (p.window_kind == 1) return len / p.window_size * p.window_size;
    if (p.window_kind == 2) return max(0, len - p.window_size + 1);
    return 0;
}

// Sums over the block's threads before this one, of three counts; the totals are added to `total`.
__device__ void scan3(const int (&v)[3], int (*scratch)[3], long long (&total)[3], long long (&before)[3]) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int incl[3];
#pragma unroll
    for (int k = 0; k < 3; ++k) {
        int x = v[k];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += u;
        }
        incl[k] = x;
        if (lane == 31) scratch[warp][k] = x;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 3; ++k) {
        int w = lane < PLAN_WARPS ? scratch[lane][k] : 0;
#pragma unroll
        for (int o = 1; o < PLAN_WARPS; o <<= 1) {
            const int u = __shfl_up_sync(0xffffffffu, w, o);
            if (lane >= o) w += u;
        }
        const int mine = warp ? __shfl_sync(0xffffffffu, w, warp - 1) : 0;
        before[k] = total[k] + mine + incl[k] - v[k];
        total[k] += __shfl_sync(0xffffffffu, w, PLAN_WARPS - 1);
    }
    __syncthreads();
}

// What the tokens are laid out by: where every request's begin, its row (-1: it has no pages in the step) and cached tokens.
struct Known { int cu[PLAN_THREADS + 1], row[PLAN_THREADS], len[PLAN_THREADS]; };

struct Request { int row, fresh, len, held, need, goes_to, goes, at; };   // (goes: pages [goes_to - goes, goes_to) go back)

__host__ __device__ constexpr Request nothing() { return Request{-1, 0, 0, 0, 0, 0, 0, 0}; }

// What request s of the step has and wants; nothing where there is nothing to do, or where it cannot be right (`ok` false: none of its numbers
// may index the tables then).
__host__ __device__ __forceinline__ Request request_of(const LayoutParams& p, int s, bool& ok) {
    const int row = p.slots[s], fresh = p.new_tokens[s];
    Request r = nothing();
    ok = row >= -1 && row < p.n_rows && fresh >= -1;
    if (!ok || row < 0) return r;
    r = Request{row, fresh, p.lengths[row], p.held[row], 0, 0, 0, 0};
    ok = r.held >= 0 && r.held <= p.table_width;
    if (fresh < 0) {                                           // it has ended: with a stack all its pages go back
        r.need = p.free_pages ? 0 : r.held;
        r.goes_to = p.free_pages ? r.held : 0;
    } else {
        const unsigned end = (unsigned)r.len + (unsigned)fresh, pages = end / p.page_size + (end % p.page_size != 0);       // (len and fresh are below 2^31)
        ok = ok && r.len >= 0 && (long long)r.held * p.page_size >= r.len && end <= 0x7fffffffu && pages <= (unsigned)min(p.table_width, p.out_width) &&
             (p.free_pages || pages <= (unsigned)r.held) && fresh <= p.n_tokens && (!p.parents || fresh <= SPITE_MAX_DRAFTS) && (!p.ancestors || fresh <= 32 * p.n_words);
        if (!ok) return nothing();
        r.need = max(r.held, (int)pages);
        r.goes_to = p.free_pages ? min(first_needed(p, r.len) / p.page_size, r.held) : 0;
    }
    return ok ? r : nothing();
}

// One block plans the step and changes the persistent state: whose pages go back, who gets which.  A thread a request, a warp a
// request where its pages are looked at.  The requests of a step are few and all it reads lies in L2, so that what counts is the
// number of dependent reads.  `known` (with no more requests than threads): filled in for what follows.
__device__ void plan_step(const LayoutParams& p, Known* known) {
    extern __shared__ unsigned seen[];                         // a bit a row of the tables
    __shared__ Request reqs[PLAN_THREADS];
    __shared__ int scratch[PLAN_WARPS][3];
    __shared__ int bad;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, words = (p.n_rows + 31) / 32;
    for (int i = threadIdx.x; i < words; i += PLAN_THREADS) seen[i] = 0;
    if (threadIdx.x == 0) bad = 0;
    __syncthreads();

    // The requests from s0 on, a thread each, with the number of pages that go back.  Those lie side by side below goes_to: in
    // front of them a row holds -1.  A warp looks at them from above, 32 at a time.
    auto take_up = [&](int s0, bool check) {
        const int s = s0 + threadIdx.x;
        Request r = nothing();
        if (s < p.n_requests) {
            bool ok;
            r = request_of(p, s, ok);
            if (check && ok && r.row >= 0) ok = (atomicOr(&seen[r.row / 32], 1u << (r.row % 32)) >> (r.row % 32) & 1u) == 0;
            if (!ok) { bad = SPITE_LAYOUT_MALFORMED; r = nothing(); }
        }
        if (r.goes_to > 0 && p.tables[(size_t)r.row * p.table_width + r.goes_to - 1] < 0) r.goes_to = 0;     // (they have gone already)
        reqs[threadIdx.x] = r;
        if (!__syncthreads_or(r.goes_to)) return r;
        for (int i = warp; i < min(PLAN_THREADS, p.n_requests - s0); i += PLAN_WARPS) {
            const Request q = reqs[i];
            if (q.row < 0 || q.goes_to == 0) continue;
            const int* table = p.tables + (size_t)q.row * p.table_width;
            int n = 0;
            for (int hi = q.goes_to; hi > 0; hi -= 32) {
                const int at = hi - 1 - lane;
                const unsigned none = __ballot_sync(0xffffffffu, at < 0 || table[at] < 0);
                if (none) { n += __ffs(none) - 1; break; }
                n += 32;
            }
            if (lane == 0) reqs[i].goes = n;
        }
        __syncthreads();
        return reqs[threadIdx.x];
    };

    const int n_free = p.free_pages ? *p.n_free : 0;
    long long total[3] = {0, 0, 0}, before[3];                 // tokens, pages back, pages taken
    const bool one = p.n_requests <= PLAN_THREADS;             // (what is known of the requests then stays in place)
    Request r = nothing();
    for (int s0 = 0; s0 < p.n_requests; s0 += PLAN_THREADS) {
        r = take_up(s0, true);
        int v[3] = {max(r.fresh, 0), r.goes, r.fresh >= 0 ? r.need - r.held : 0};
        scan3(v, scratch, total, before);
    }
    if (threadIdx.x == 0) {
        int status = bad;
        if (total[0] > p.n_tokens || (p.parents && total[0] > p.n_parents)) status = SPITE_LAYOUT_MALFORMED;
        if (p.free_pages && (n_free < 0 || n_free + total[1] > p.n_pages)) status = SPITE_LAYOUT_MALFORMED;
        if (p.free_pages && !status && total[2] > n_free + total[1]) status = SPITE_LAYOUT_OUT_OF_PAGES;
        *p.status = bad = status;
        p.cu_seqlens[p.n_requests] = status ? 0 : (int)total[0];
    }
    __syncthreads();
    if (bad) {                                                 // nothing is changed and the step has no tokens
        for (int s = threadIdx.x; s < p.n_requests; s += PLAN_THREADS) p.cu_seqlens[s] = 0;
        if (known) {
            known->cu[threadIdx.x] = 0;
            known->row[threadIdx.x] = -1;
            if (threadIdx.x == 0) known->cu[PLAN_THREADS] = 0;
        }
        return;
    }
    const int top = n_free + (int)total[1];                    // the stack's height once the pages are back
    long long run[3] = {0, 0, 0};
    for (int s0 = 0; s0 < p.n_requests; s0 += PLAN_THREADS) {
        if (!one) {
            r = take_up(s0, false);
            int v[3] = {max(r.fresh, 0), r.goes, 0};
            scan3(v, scratch, run, before);
        }
        const int s = s0 + threadIdx.x;
        if (s < p.n_requests) p.cu_seqlens[s] = (int)before[0];
        if (known) {
            known->cu[threadIdx.x] = (int)before[0];           // (behind the last request: all tokens)
            known->row[threadIdx.x] = r.fresh >= 0 ? r.row : -1;
            known->len[threadIdx.x] = r.len;
            if (threadIdx.x == 0) known->cu[PLAN_THREADS] = (int)total[0];
        }
        if (total[1] == 0) continue;                           // (the same for all)
        reqs[threadIdx.x].at = n_free + (int)before[1];
        __syncthreads();
        for (int i = warp; i < min(PLAN_THREADS, p.n_requests - s0); i += PLAN_WARPS) {
            const Request q = reqs[i];
            if (q.row < 0 || q.goes == 0) continue;
            int* table = p.tables + (size_t)q.row * p.table_width + q.goes_to - q.goes;
            for (int k = lane; k < q.goes; k += 32) {          // back on the stack, in ascending order
                p.free_pages[q.at + k] = table[k];
                table[k] = -1;
            }
        }
        __syncthreads();
    }
    if (!p.free_pages) return;
    __threadfence_block();
    __syncthreads();                                           // every page is back before the first is taken
    long long taken[3] = {0, 0, 0};
    for (int s0 = 0; s0 < p.n_requests; s0 += PLAN_THREADS) {
        if (!one) {
            bool ok;
            const int s = s0 + threadIdx.x;
            r = nothing();
            if (s < p.n_requests) r = request_of(p, s, ok);
            int v[3] = {0, 0, r.fresh >= 0 ? r.need - r.held : 0};
            scan3(v, scratch, taken, before);
        }
        r.at = top - 1 - (int)before[2];
        const int takes = r.row >= 0 ? r.need - r.held : 0;
        int* mine = p.tables + (size_t)max(r.row, 0) * p.table_width + r.held;
        for (int k = 0; k < min(takes, FEW_PAGES); ++k) mine[k] = p.free_pages[r.at - k];
        if (takes) p.held[r.row] = r.need;                     // (an ended request's, to none)
        reqs[threadIdx.x] = r;
        if (!__syncthreads_or(takes > FEW_PAGES)) continue;    // a prompt's, by a warp each
        for (int i = warp; i < min(PLAN_THREADS, p.n_requests - s0); i += PLAN_WARPS) {
            const Request q = reqs[i];
            if (q.row < 0) continue;
            int* table = p.tables + (size_t)q.row * p.table_width + q.held;
            for (int k = FEW_PAGES + lane; k < q.need - q.held; k += 32) table[k] = p.free_pages[q.at - k];
        }
        __syncthreads();
    }
    if (threadIdx.x == 0) *p.n_free = top - (int)total[2];
}

// Everything that follows from the plan, a thread a number, by `n` threads of which this is number `i`; `known` or, without it, what lies in global
// memory, where the search through cu_seqlens is a chain of reads from L2.  (With a bad status the requests have no tokens and no pages.)
__device__ void fill_step(const LayoutParams& p, const Known* known, bool bad, long long i, long long n) {
    auto cu = [&](int s) { return known ? known->cu[s] : p.cu_seqlens[s]; };
    auto row_of = [&](int s) { return known ? known->row[s] : !bad && p.slots[s] >= 0 && p.new_tokens[s] >= 0 ? p.slots[s] : -1; };
    const long long total = bad ? 0 : cu(p.n_requests);
    for (long long t = i; t < total; t += n) {
        int lo = 0, hi = p.n_requests;                         // cu[lo] <= t < cu[hi]
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (cu(mid) <= t) lo = mid; else hi = mid;
        }
        const int row = row_of(lo), first = cu(lo), node = (int)t - first, len = known ? known->len[lo] : p.lengths[row], place = len + node;
        bool real = true;
        int depth = node;
        if (p.parents) {
            // A token's ancestors, from itself upward: the parents' numbers fall, so the words of its set are finished one by one.  (A parent
            // that is not in front of its child ends the walk; one below -1 marks padding, which has no row in the cache.)
            depth = 0;
            real = p.parents[t] >= -1;
            unsigned* set = p.ancestors ? p.ancestors + t * p.n_words : nullptr;
            int word = p.n_words - 1, at = real ? node : -1;
            unsigned bits = 0;
            while (at >= 0) {
                if (set) {
                    for (; word > at / 32; --word) { set[word] = bits; bits = 0; }
                    bits |= 1u << (at % 32);
                }
                const int up = p.parents[first + at];
                if (up >= at || up < 0) break;
                at = up;
                ++depth;
            }
            if (set)
                for (; word >= 0; --word) { set[word] = bits; bits = 0; }
        } else if (p.ancestors) {
            for (int w = 0; w < p.n_words; ++w)
                p.ancestors[t * p.n_words + w] = w < node / 32 ? 0xffffffffu : w > node / 32 ? 0u : 0xffffffffu >> (31 - node % 32);
        }
        p.positions[t] = len + depth;
        p.seg_of_token[t] = lo;
        const int page = p.tables[(size_t)row * p.table_width + place / p.page_size];
        p.slot_map[t] = real && page >= 0 ? (long long)page * p.page_size + place % p.page_size : -1;
    }
    // the block table, a warp a row (or several a row): the rows' addresses are then the same for its lanes
    constexpr int AHEAD = 8;                                   // numbers of a lane asked for together
    const int lane = (int)(i & 31), per = (p.out_width + 32 * AHEAD - 1) / (32 * AHEAD);
    for (long long piece = i >> 5; piece < (long long)p.n_requests * per; piece += n >> 5) {
        const int s = (int)((unsigned)piece / (unsigned)per), c0 = ((int)piece - s * per) * 32 * AHEAD + lane, row = row_of(s);
        const bool has = row >= 0;
        const int* from = p.tables + (size_t)(has ? row : 0) * p.table_width;
        int* to = p.block_table + (size_t)s * p.out_width;
        int v[AHEAD];
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) v[k] = has && c0 + 32 * k < min(p.table_width, p.out_width) ? from[c0 + 32 * k] : -1;
#pragma unroll
        for (int k = 0; k < AHEAD; ++k)
            if (c0 + 32 * k < p.out_width) to[c0 + 32 * k] = v[k];
    }
}

// The whole in one launch, for up to PLAN_THREADS requests: one block, or a cluster of which the first block plans while the others look up what
// does not depend on the plan and wait at the cluster's barrier.
__global__ void __launch_bounds__(PLAN_THREADS) layout_kernel(const LayoutParams p) {
    __shared__ Known known;
    __shared__ int status;
    pdl_wait();
    pdl_launch_dependents();
    if (blockIdx.x == 0) {
        plan_step(p, &known);
    } else if ((int)threadIdx.x < p.n_requests) {
        const int row = p.slots[threadIdx.x];
        const bool has = row >= 0 && row < p.n_rows && p.new_tokens[threadIdx.x] >= 0;
        known.row[threadIdx.x] = has ? row : -1;
        known.len[threadIdx.x] = has ? p.lengths[row] : 0;
    }
    if (gridDim.x > 1) {
        __threadfence();
        asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;\n" ::: "memory");
        if (blockIdx.x != 0)
            for (int s = threadIdx.x; s <= p.n_requests; s += PLAN_THREADS) known.cu[s] = __ldcg(p.cu_seqlens + s);
    }
    if (threadIdx.x == 0) status = __ldcg(p.status);
    __syncthreads();
    const bool bad = status != 0;
    if (bad && (int)threadIdx.x < p.n_requests) known.row[threadIdx.x] = -1;
    __syncthreads();
    fill_step(p, &known, bad, (long long)blockIdx.x * PLAN_THREADS + threadIdx.x, (long long)gridDim.x * PLAN_THREADS);
}
// In two: the plan, and as many blocks as a large table needs.
__global__ void __launch_bounds__(PLAN_THREADS) layout_plan_kernel(const LayoutParams p) {
    pdl_wait();
    pdl_launch_dependents();
    plan_step(p, nullptr);
}
__global__ void __launch_bounds__(256) layout_fill_kernel(const LayoutParams p) {
    pdl_wait();
    pdl_launch_dependents();
    fill_step(p, nullptr, *p.status != 0, (long long)blockIdx.x * 256 + threadIdx.x, (long long)gridDim.x * 256);
}

// A launch of one cluster (of one block: an ordinary one).
void launch_cluster(const LayoutParams& p, int blocks, size_t smem, cudaStream_t st) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(blocks);
    cfg.blockDim = dim3(PLAN_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    int n = 0;
    if (spite_pdl_enabled()) {
        attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[n++].val.programmaticStreamSerializationAllowed = 1;
    }
    if (blocks > 1) {
        attr[n].id = cudaLaunchAttributeClusterDimension;
        attr[n].val.clusterDim.x = blocks;
        attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
        ++n;
    }
    cfg.attrs = attr;
    cfg.numAttrs = n;
    (void)cudaLaunchKernelEx(&cfg, layout_kernel, p);
}

}  // namespace

// Lays a step out.  `blocks`: one launch of a cluster of so many (1..8), for up to 512 requests, or 0: two launches.
SPITE_API int spite_layout_step(const LayoutParams* p, int blocks, void* stream) {
    if (!p || !p->tables || !p->held || !p->slots || !p->lengths || !p->new_tokens || !p->block_table || !p->cu_seqlens || !p->status) return SPITE_BAD_ARG;
    if (!p->free_pages != !p->n_free || p->n_rows < 1 || p->table_width < 1 || p->out_width < 1 || p->n_requests < 1 || p->page_size < 1) return SPITE_BAD_ARG;
    if (p->n_tokens < 0 || (p->n_tokens > 0 && (!p->positions || !p->seg_of_token || !p->slot_map))) return SPITE_BAD_ARG;
    if (p->window_kind < 0 || p->window_kind > 2 || (p->window_kind && p->window_size < 1)) return SPITE_BAD_ARG;
    if ((p->ancestors && p->n_words < 1) || (p->free_pages && p->n_pages < 1) || (p->parents && p->n_parents < 0) || blocks < 0 || blocks > 8) return SPITE_BAD_ARG;
    if (p->n_tokens > (1 << 20) || p->table_width > (1 << 20) || p->n_requests > SPITE_LAYOUT_MAX_REQUESTS || p->n_rows > SPITE_LAYOUT_MAX_ROWS ||
        p->n_words > SPITE_MAX_DRAFTS / 32 || (blocks && p->n_requests > PLAN_THREADS)) return SPITE_UNSUPPORTED;
    cudaStream_t st = (cudaStream_t)stream;
    const size_t smem = (size_t)(p->n_rows + 31) / 32 * 4;
    if (blocks) {
        launch_cluster(*p, blocks, smem, st);
    } else {
        SPITE_LAUNCH(layout_plan_kernel, 1, PLAN_THREADS, smem, st, *p);
        const long long pieces = (long long)p->n_requests * ((p->out_width + 255) / 256), fill = (pieces + 7) / 8;
        SPITE_LAUNCH(layout_fill_kernel, (unsigned)(fill < 2048 ? fill : 2048), 256, 0, st, *p);
    }
    return spite_launch_status();
}

// ---------------------------------------------------------------- accepted drafts
#define SPITE_ACCEPT_GROUPS 8

// One group of caches that share a slot map: planes (caches x keys, values) of pages [pages][kv heads][page_size][row_bytes], and a
// float per key beside the first plane of every cache, or none.
struct AcceptGroup {
    unsigned char* kv;
    float* key_scales;           // [caches][pages][kv heads][page_size], or null
    const long long* slot_map;   // [tokens]
    long long plane_bytes;       // of one plane
    int planes, caches, n_pages, num_kv_heads, page_size, row_bytes;
};
struct AcceptParams {
    const int* tokens;           // [n_tokens] drafted tokens
    const int* parents;          // [n_tokens] or null: a chain
    const int* targets;          // [n_tokens] what the model says follows each
    const int* cu_seqlens;       // [n_requests + 1]
    int* counts;                 // [n_requests] accepted tokens, the first among them
    int* path;                   // [n_requests, depth] their numbers within the request, -1 behind the last
    int* emitted;                // [n_requests, depth] their targets, -1 behind the last
    const int* slots;            // [n_requests] or null
    const int* lengths;          // [rows] or null
    int* lengths_out;
    int n_tokens, n_requests, depth, n_rows, n_groups;
    AcceptGroup groups[SPITE_ACCEPT_GROUPS];
};

namespace {

constexpr int ACCEPT_THREADS = 256;
constexpr int ACCEPT_BATCH = 8;          // rows that a thread asks for together

// grid (requests, pieces of the caches' columns).  Every block walks its request's tree for itself (the tree is small and lies in
// L2): each token that is its parent's target offers itself to the parent, the lowest number wins, and the path is the chain of winners.
// Then a thread moves its 16 bytes (or 4, or a byte) of a row for all accepted tokens: token d of the path goes from the place of its
// number to place d, which is never behind it, so that in ascending order nothing is read after it was written, and reads may go
// ahead of writes.
template <typename V>
__global__ void __launch_bounds__(ACCEPT_THREADS) accept_kernel(const AcceptParams p) {
    __shared__ int next[SPITE_MAX_DRAFTS];
    __shared__ int path[SPITE_MAX_DRAFTS];
    __shared__ long long from_row[SPITE_MAX_DRAFTS], to_row[SPITE_MAX_DRAFTS];
    __shared__ int n_path;
    pdl_wait();
    pdl_launch_dependents();
    const int s = blockIdx.x;
    const int first = min(max(p.cu_seqlens[s], 0), p.n_tokens), end = min(max(p.cu_seqlens[s + 1], first), p.n_tokens);
    const int n = min(end - first, SPITE_MAX_DRAFTS);
    for (int i = threadIdx.x; i < n; i += ACCEPT_THREADS) next[i] = 0x7fffffff;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += ACCEPT_THREADS) {
        const int up = p.parents ? p.parents[first + i] : i - 1;
        if (up >= 0 && up < i && p.tokens[first + i] == p.targets[first + up]) atomicMin(&next[up], i);
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        int k = 0;
        for (int at = 0; k < p.depth && at < n; at = next[at]) path[k++] = at;
        n_path = k;
    }
    __syncthreads();
    const int count = n_path;
    if (blockIdx.y == 0) {
        for (int d = threadIdx.x; d < p.depth; d += ACCEPT_THREADS) {
            p.path[(size_t)s * p.depth + d] = d < count ? path[d] : -1;
            p.emitted[(size_t)s * p.depth + d] = d < count ? p.targets[first + path[d]] : -1;
        }
        if (threadIdx.x == 0) {
            p.counts[s] = count;
            const int row = p.slots ? p.slots[s] : s;
            if (p.lengths && row >= 0 && row < p.n_rows) p.lengths_out[row] = p.lengths[row] + count;
        }
    }
    for (int g = 0; g < p.n_groups; ++g) {
        const AcceptGroup& c = p.groups[g];
        const long long n_slots = (long long)c.n_pages * c.page_size;
        // where every accepted token's row lies and where it goes (in rows, of head 0); a token that stays, or has no row, from -1
        if (g) __syncthreads();
        for (int d = threadIdx.x; d < count; d += ACCEPT_THREADS) {
            long long a = -1, b = -1;
            if (path[d] != d) { a = c.slot_map[first + path[d]]; b = c.slot_map[first + d]; }
            const bool ok = a >= 0 && a < n_slots && b >= 0 && b < n_slots;
            from_row[d] = ok ? a / c.page_size * c.num_kv_heads * c.page_size + a % c.page_size : -1;
            to_row[d] = ok ? b / c.page_size * c.num_kv_heads * c.page_size + b % c.page_size : -1;
        }
        __syncthreads();
        const int per_row = c.row_bytes / (int)sizeof(V), per_plane = c.num_kv_heads * per_row;
        const long long units = (long long)c.planes * per_plane;
        for (long long u = (long long)blockIdx.y * ACCEPT_THREADS + threadIdx.x; u < units; u += (long long)gridDim.y * ACCEPT_THREADS) {
            const int plane = (int)(u / per_plane), in_plane = (int)(u - (long long)plane * per_plane), head = in_plane / per_row;
            unsigned char* base = c.kv + plane * c.plane_bytes + (long long)head * c.page_size * c.row_bytes + (in_plane - head * per_row) * sizeof(V);
            for (int d0 = 1; d0 < count; d0 += ACCEPT_BATCH) {
                V v[ACCEPT_BATCH];
#pragma unroll
                for (int k = 0; k < ACCEPT_BATCH; ++k)
                    if (d0 + k < count && from_row[d0 + k] >= 0) v[k] = *(const V*)(base + from_row[d0 + k] * c.row_bytes);
#pragma unroll
                for (int k = 0; k < ACCEPT_BATCH; ++k)
                    if (d0 + k < count && from_row[d0 + k] >= 0) *(V*)(base + to_row[d0 + k] * c.row_bytes) = v[k];
            }
        }
        if (c.key_scales && blockIdx.y == 0) {
            for (int u = threadIdx.x; u < c.caches * c.num_kv_heads; u += ACCEPT_THREADS) {
                float* base = c.key_scales + (long long)(u / c.num_kv_heads) * n_slots * c.num_kv_heads + u % c.num_kv_heads * c.page_size;
                for (int d = 1; d < count; ++d)
                    if (from_row[d] >= 0) base[to_row[d]] = base[from_row[d]];
            }
        }
    }
}

}  // namespace

// Follows every request's tree and moves the accepted rows.  `pieces`: blocks a request.
SPITE_API int spite_accept_drafts(const AcceptParams* p, int pieces, void* stream) {
    if (!p || (p->n_tokens > 0 && (!p->tokens || !p->targets)) || !p->cu_seqlens || !p->counts || !p->path || !p->emitted) return SPITE_BAD_ARG;
    if (p->n_tokens < 0 || p->n_requests < 1 || p->depth < 1 || pieces < 1 || p->n_groups < 0) return SPITE_BAD_ARG;
    if (!p->lengths != !p->lengths_out || (p->lengths && p->n_rows < 1)) return SPITE_BAD_ARG;
    if (p->depth > SPITE_MAX_DRAFTS || p->n_groups > SPITE_ACCEPT_GROUPS || pieces > 65535) return SPITE_UNSUPPORTED;
    uintptr_t bits = 0;
    for (int g = 0; g < p->n_groups; ++g) {
        const AcceptGroup& c = p->groups[g];
        if (!c.kv || (p->n_tokens > 0 && !c.slot_map) || c.planes < 1 || c.caches < 1 || c.n_pages < 1 || c.num_kv_heads < 1 || c.page_size < 1 || c.row_bytes < 1)
            return SPITE_BAD_ARG;
        bits |= (uintptr_t)c.kv | (uintptr_t)c.plane_bytes | (uintptr_t)c.row_bytes;
    }
    if (bits & 1) return SPITE_UNSUPPORTED;
    const dim3 grid(p->n_requests, pieces);
    cudaStream_t st = (cudaStream_t)stream;
    if (bits % 16 == 0) SPITE_LAUNCH(accept_kernel<uint4>, grid, ACCEPT_THREADS, 0, st, *p);
    else if (bits % 4 == 0) SPITE_LAUNCH(accept_kernel<unsigned>, grid, ACCEPT_THREADS, 0, st, *p);
    else SPITE_LAUNCH(accept_kernel<unsigned short>, grid, ACCEPT_THREADS, 0, st, *p);
    return spite_launch_status();
}
