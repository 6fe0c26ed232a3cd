// Attention over trees of drafted tokens on the fifth-generation tensor cores (bfloat16, heads of 64 or 128 elements, pages of a multiple
// of 64 keys, up to 128 query heads per kv head).
//
// The rows of a row tile are the (node, query head of one kv group) pairs of consecutive nodes of one request, 128 of them at most, and
// all see nearly the same keys: the request's settled tokens.  What has to be read is the cache, once a kv head, and that bounds the kernel up
// to some 128 rows a request and kv head; beyond, the products and the exponentials do.  So a block works on
//   a pair    two row tiles of a request, each on every key tile (64 keys, a TMA box, never across a page), which is fetched once for both, or
//   a single  one row tile (a small tree, or the odd one of a large), whose key tiles the block's two halves share out, one the even tiles and one
//             the odd ones, each with a softmax state and an output of its own; the two are added up in the end.
// Either way one half's exponentials run beside the other half's products.  The lengths are on the device only, so the launch has one block a
// multiprocessor and the blocks find their work themselves: all (pair or single, kv head) items end to end are one line, each as
// long as its key tiles cost, every block takes an equal stretch of it, and what a stretch holds of an item that it shares with others leaves
// its output before the division, its maximum and its sum to a second kernel, which adds them up in the order of the keys.
// Nothing stops between items: the rings and all barriers go on counting, and the loaders fetch the next item's keys while this one's end.
//
// Roles (12 warps):
//   0        one lane loads K and V tiles into a ring               3        one lane loads the items' rows of q
//   1, 2     one lane each issues S = Q K^T and O += P V of its half, scores two tiles ahead; P is read from tensor memory
//   4 - 11   four softmax warps a half, one thread a row: scores by tcgen05.ld, scale, mask, running maximum (which moves only
//            when it grows by more than 2^8) and sum in float32, P as bfloat16 over the scores it came from
// P is rounded to bfloat16 because the tensor cores take both operands in one type; the sum is taken of the unrounded weights.
//
// Masks matter in the tiles at a window's end and in those with the step's own nodes; there a row makes 64 bits of what it sees.  A value row
// that is no node's (padding, what lies behind the last node) may hold anything, and 0 x NaN is NaN: the softmax warps clear
// these rows of the tile in shared memory before the product.  Settled rows are finite as everywhere in the cache; a value of a node or of a settled
// row that is not reaches the other rows of its request, and a row whose sum is NaN is NaN.
//
// Measured (40 query heads on 8 of 128 elements, device time with both kernels): one request of 131,072 keys, up to 25 nodes (singles) 97 to 103 us,
// 5.2 to 5.6 TB/s: memory; 50 nodes (pairs) 162 us, 826 TFLOP/s, and 100 nodes 884: a pair's key tile takes 1.25 us, the chain scores -> softmax
// -> product of a half, whose gaps the other half fills only in part (tensor pipe 43 % busy, special functions 42 %); heads of 64 elements have
// the same chain for half the bytes, 0.75 us a key tile for a single (3.2 TB/s) and 1.3 for a pair.  8 requests of 16 nodes and 8,192 keys: 64 us,
// 4.3 TB/s; one of 8 nodes and 100 keys: 7.5 us, half of it the start.  Measured and not kept: two threads a row (sixteen softmax warps; 405 against
// 381 us for 16 requests of 64 nodes, 8,192 keys, 64 heads), part of the exponentials by a polynomial on the multiply-add units (390 against 355:
// the loop outgrows the instruction cache), no turns at the exponentials or turns passed on after a half or seven eighths of a tile (within 3 %),
// registers moved to the softmax warps (no change), a half's state handed over before its last product (168 against 163), other costs of a tile
// and an item within a factor of 1.5 (within 5 %).
//
// Score, mask and softmax: crates/spite-compute/src/flash_attn.rs:111-156, with the mask of attention_tree.cuh.  Every wait is bounded
// (see tcgen05.cuh); codes: 1 a loader, 2 tensor-core issue, 3 softmax.
#include "attention_tree.cuh"
#include "packed.cuh"
#include "tcgen05.cuh"

namespace {
using namespace tc;
using namespace packed;

constexpr int BM = 128;                 // rows of a row tile
constexpr int BN = 64;                  // keys of a tile
constexpr int THREADS = 12 * 32;
constexpr int TMEM_COLS = 512;
constexpr int GROUP_COLS = 256;         // tensor-memory columns of a half: S0, S1 (64 each), O
constexpr float RESCALE_STEP = 8.f;     // log2 units
constexpr float LOG2E = 1.4426950408889634f;
constexpr int MAX_SEGMENTS = 640;       // requests of one launch (the line lies in shared memory); more take several

// The line: what a key tile of a pair and of a single costs, what an item costs besides, the shortest part.
constexpr int COST_PAIR = 3, COST_SINGLE = 2, COST_ITEM = 6;
constexpr int PIECE = 3;                // key tiles: a cut closer to an item's end moves there
constexpr int SHARE = 14;               // the shortest stretch, while there are blocks for every item

__device__ int g_attn_tree_error = 0;
}  // namespace
SPITE_WAIT_CONTROLS(attention_tree_tc, g_attn_tree_error)
namespace {

struct TreeCut {
    float* partial;                     // [blocks][2: a block's first part, its last][2 row tiles x (HD + 2) x 128]
    int4* items;                        // [blocks]: where block i's beginning is the first cut within an item: (the item's first token, tokens, kv head,
};                                      // parts); no parts: none

// A block's part of the line, and the item that it begins in.
struct Stretch {
    unsigned line_end, sharers, each, rest, begin, end, at;
    int seg, kvh, idx;
    __device__ __forceinline__ unsigned cut(unsigned i) const { return i >= sharers ? line_end : each * i + rest * i / sharers; }     // line_end * i / sharers
};
__host__ __device__ constexpr size_t slot_floats(int head_dim) { return 2 * (size_t)(head_dim + 2) * BM; }

constexpr int MAX_STAGES = 18;
__host__ __device__ constexpr int stages(int nkb) { return nkb == 1 ? MAX_STAGES : MAX_STAGES / 2; }      // 144 KB of keys and values
struct HalfBarriers { unsigned long long s_full[2], p_ready, pv_done, exp_done; };
struct Barriers {
    unsigned long long q_full, q_empty, full[MAX_STAGES], empty[MAX_STAGES], state_ready, state_read;
    HalfBarriers g[2];
    unsigned tmem_base;
    int abort_flag;
};

// An item, or the part of it that a block works on: key tiles [from, to) of `tiles`.
struct Item { int seg, first, n, len, kvh, node0, nodes, k_begin, tiles, from, to; bool pair; };

// The order in which an item's tiles go through the ring, which is the order in which they are used: a half issues the scores of its first two
// tiles and then, tile by tile, the product with the values and the scores of the tile after next.  So the keys are `ahead` by 2 tiles
// (4 where the halves share the tiles out), and then values and keys alternate.
struct Order {
    int n, ahead;
    __device__ __forceinline__ Order(const Item& it) : n(it.to - it.from), ahead(min(n, it.pair ? 2 : 4)) {}
    __device__ __forceinline__ int keys(int t) const { return t < ahead ? t : 2 * t - ahead + 1; }
    __device__ __forceinline__ int values(int t) const { return ahead + t + min(t, n - ahead); }
};

__device__ __forceinline__ float row_scale_of(const AttentionParams& p, int tok, int head, float m, float l) {
    float shrink = 1.f;
    if (p.has_sink && sink_of(p, head) > -INFINITY) {           // the sink joins the sum, in powers of two
        const float sink2 = sink_of(p, head) * LOG2E, m2 = fmaxf(m, sink2);
        shrink = m == -INFINITY ? 0.f : exp2f(m - m2);
        l = l * shrink + exp2f(sink2 - m2);
    }
    return shrink * gate_of(p, tok, head) / tree_divisor(l);
}

// The n lowest of 64 bits.
__device__ __forceinline__ unsigned long long low_bits(int n) { return n <= 0 ? 0ull : n >= 64 ? ~0ull : (1ull << n) - 1; }

// NKB = head_dim / 64.  One block a multiprocessor.
template <int NKB, int FORM>
__global__ void __launch_bounds__(THREADS, 1)
attn_tree_tc_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                    const AttentionParams p, const StepTokens b, const PagedCache c, const TreeStep x, const int tpt, const int q_box_tokens, const TreeCut cut,
                    const WaitControl waits) {
    constexpr int HD = 64 * NKB, ST = stages(NKB);
    constexpr bool CAP = FORM != FORM_PLAIN, BIAS = FORM == FORM_ANY;      // (with a bias, a cap is chosen at run time)
    constexpr int Q_BYTES = NKB * BM * 128, KT_BYTES = NKB * BN * 128;
    extern __shared__ __align__(1024) unsigned char smem[];     // [Q0][Q1][ring], 1024-byte aligned, then the line
    __shared__ Barriers bars;
    __shared__ float2 state_s[2][BM];                            // a single's two softmax states
    __shared__ Stretch stretch;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int nq = p.num_heads, nkv = c.num_kv_heads, G = nq / nkv, S = x.n_segments;
    unsigned char* q_s = smem;
    unsigned char* ring = q_s + 2 * Q_BYTES;
    int4* const known = (int4*)(ring + ST * KT_BYTES);           // [S] a request's first node, nodes, settled tokens, key tiles
    unsigned* line = (unsigned*)(known + S);                     // [S + 1] what the requests before cost (for one kv head)
    volatile int* abort_flag = &bars.abort_flag;
    int* const err = waits.error_word ? waits.error_word : &g_attn_tree_error;
    const long long limit = waits.limit_cycles;

    if (threadIdx.x == 0) {
        bars.abort_flag = 0;
        mbar_init(smem_u32(&bars.q_full), 1);
        mbar_init(smem_u32(&bars.q_empty), 2);
        for (int s = 0; s < ST; ++s) {
            mbar_init(smem_u32(&bars.full[s]), 1); mbar_init(smem_u32(&bars.empty[s]), 2);      // both halves release a stage
        }
        for (int g = 0; g < 2; ++g) {
            mbar_init(smem_u32(&bars.g[g].s_full[0]), 1); mbar_init(smem_u32(&bars.g[g].s_full[1]), 1);
            mbar_init(smem_u32(&bars.g[g].p_ready), 4);
            mbar_init(smem_u32(&bars.g[g].pv_done), 1);
            mbar_init(smem_u32(&bars.g[g].exp_done), 4);
        }
        mbar_init(smem_u32(&bars.state_ready), 8);
        mbar_init(smem_u32(&bars.state_read), 8);
        mbar_init_fence();
    }
    if (warp == 1) tmem_alloc(&bars.tmem_base, TMEM_COLS);
    if (threadIdx.x == 3 * 32) {                                 // the tensor maps are needed first thing
        asm volatile("prefetch.tensormap [%0];\n" ::"l"((unsigned long long)&map_q) : "memory");
        asm volatile("prefetch.tensormap [%0];\n" ::"l"((unsigned long long)&map_k) : "memory");
        asm volatile("prefetch.tensormap [%0];\n" ::"l"((unsigned long long)&map_v) : "memory");
    }
    pdl_wait();
    pdl_launch_dependents();

    // ---- the line
    struct Request { int first, n, len, tiles, pairs, single; unsigned pair_len, single_len; };
    auto request_of = [&](int s) {
        const int4 v = known[s];
        const int row_tiles = v.w ? (v.y + tpt - 1) / tpt : 0;
        return Request{v.x, v.y, v.z, v.w, row_tiles / 2, row_tiles & 1, (unsigned)(COST_ITEM + v.w * COST_PAIR), (unsigned)(COST_ITEM + v.w * COST_SINGLE)};
    };
    auto begin_of = [&](int len) { return window_lowest(p.window_kind, p.window_size, len) / BN * BN; };      // of the first key tile
    for (int s = threadIdx.x; s < S; s += THREADS) {
        const int first = min(max(x.cu_seqlens[s], 0), b.n_tokens), n = min(max(x.cu_seqlens[s + 1], first), b.n_tokens) - first;
        const int len = n ? max(b.positions[first], 0) : 0, k_begin = begin_of(len);
        const int places = (int)min((long long)len + n, (long long)b.table_width * c.page_size);
        known[s] = make_int4(first, n, len, n && places > k_begin ? (places - k_begin + BN - 1) / BN : 0);
        const Request r = request_of(s);
        line[s + 1] = r.pairs * r.pair_len + (r.single ? r.single_len : 0);
    }
    fence_before();
    __syncthreads();
    fence_after();
    const unsigned tmem = bars.tmem_base;
    // the key tile where a cut `off` behind an item's beginning falls
    auto tile_at = [](unsigned off, bool pair, int tiles) {
        const int o = off <= COST_ITEM ? 0 : (int)off - COST_ITEM, t = pair ? (o + COST_PAIR / 2) / COST_PAIR : (o + COST_SINGLE / 2) / COST_SINGLE;
        return t < PIECE ? 0 : tiles - t < PIECE ? tiles : t;
    };
    if (warp == 0) {
        unsigned sum = 0, sets = 0;
        for (int s0 = 0; s0 < S; s0 += 32) {
            const bool there = s0 + lane < S;
            unsigned v = there ? line[s0 + lane + 1] : 0;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const unsigned u = __shfl_up_sync(0xffffffffu, v, o);
                if (lane >= o) v += u;
            }
            if (there) {
                line[s0 + lane + 1] = sum + v;
                const Request r = request_of(s0 + lane);
                sets += r.pairs + r.single;
            }
            sum += __shfl_sync(0xffffffffu, v, 31);
        }
        sets = __reduce_add_sync(0xffffffffu, sets);
        if (lane == 0) line[0] = 0;
        __syncwarp();
        if (lane == 0) {
            // this block's stretch: of as many as there are items, or as shares of the shortest length; and the item that it begins in
            Stretch t;
            t.line_end = sum * nkv;
            t.sharers = min(gridDim.x, max(sets * nkv, t.line_end / SHARE));
            t.each = t.sharers ? t.line_end / t.sharers : 0;
            t.rest = t.line_end - t.each * t.sharers;
            t.begin = t.end = t.at = 0;
            t.seg = t.kvh = t.idx = 0;
            if (blockIdx.x < t.sharers && t.line_end) {
                t.begin = t.cut(blockIdx.x);
                t.end = t.cut(blockIdx.x + 1);
                int lo = 0, hi = S;                              // nkv * line[lo] <= begin < nkv * line[hi]
                while (hi - lo > 1) {
                    const int mid = (lo + hi) >> 1;
                    if (nkv * line[mid] <= t.begin) lo = mid; else hi = mid;
                }
                const Request r = request_of(lo);
                const unsigned per_head = line[lo + 1] - line[lo];
                unsigned rest = t.begin - nkv * line[lo];
                t.seg = lo;
                t.kvh = rest / per_head;
                rest -= t.kvh * per_head;
                t.idx = min((unsigned)r.pairs, rest / r.pair_len);
                t.at = t.begin - (rest - t.idx * r.pair_len);
            }
            stretch = t;
        }
    }
    __syncthreads();
    // every role goes over the block's items alike; f returns false to give up
    auto for_items = [&](auto f) {
        const unsigned begin = stretch.begin, end = stretch.end;
        if (begin >= end) return;
        int seg = stretch.seg, kvh = stretch.kvh, idx = stretch.idx;
        unsigned at = stretch.at;
        Request r = request_of(seg);
        while (true) {
            Item it;
            it.pair = idx < r.pairs;
            const unsigned len = it.pair ? r.pair_len : r.single_len;
            it.seg = seg; it.kvh = kvh; it.first = r.first; it.n = r.n; it.len = r.len; it.k_begin = begin_of(r.len); it.tiles = r.tiles;
            it.node0 = 2 * idx * tpt;
            it.nodes = min((it.pair ? 2 : 1) * tpt, r.n - it.node0);
            it.from = at < begin ? tile_at(begin - at, it.pair, r.tiles) : 0;
            it.to = at + len > end ? tile_at(end - at, it.pair, r.tiles) : r.tiles;
            if (it.from < it.to && !f(it)) return;
            at += len;
            if (at >= end) return;
            if (++idx == r.pairs + r.single) {                   // the next kv head, the next request that has anything
                idx = 0;
                if (++kvh == nkv) {
                    kvh = 0;
                    do ++seg; while (line[seg + 1] == line[seg]);
                    r = request_of(seg);
                }
            }
        }
    };
    if (warp == 11) {
        // for the second kernel, ahead of this warp's rows: is this block's beginning the first cut within an item?
        int4 a = make_int4(0, 0, 0, 0);
        if (stretch.begin < stretch.end) {
            const Request r = request_of(stretch.seg);
            const bool pair = stretch.idx < r.pairs;
            const unsigned at = stretch.at, len = pair ? r.pair_len : r.single_len;
            auto within = [&](unsigned i) {
                const unsigned t = stretch.cut(i);
                if (t <= at || t >= at + len) return false;
                const int tile = tile_at(t - at, pair, r.tiles);
                return tile > 0 && tile < r.tiles;
            };
            if (within(blockIdx.x)) {
                int cuts = 0, before = 0;
                for (unsigned i = lane; i < stretch.sharers; i += 32)
                    if (within(i)) { ++cuts; before += i < blockIdx.x; }
                cuts = __reduce_add_sync(0xffffffffu, cuts);
                before = __reduce_add_sync(0xffffffffu, before);
                const int node0 = 2 * stretch.idx * tpt;
                if (before == 0) a = make_int4(r.first + node0, min((pair ? 2 : 1) * tpt, r.n - node0), stretch.kvh, cuts + 1);
            }
        }
        if (lane == 0) cut.items[blockIdx.x] = a;
    }
    auto wait = [&](unsigned long long& bar, unsigned parity, int code) { return mbar_wait(smem_u32(&bar), parity & 1, abort_flag, err, code, limit); };

    if (warp == 0) {
        if (lane == 0) {
            // ---- keys and values
            unsigned at = 0;                                     // tiles put into the ring so far
            for_items([&](const Item& it) {
                const Order order(it);
                const int* table = b.block_table + (size_t)it.seg * b.table_width;
                auto load = [&](const CUtensorMap* map, int t) {
                    const int j0 = it.k_begin + (it.from + t) * BN, s = at % ST;
                    int page = table[j0 / c.page_size];
                    if (page < 0 || page >= c.n_pages) page = 0;           // (no page: nothing there is visible to a row)
                    const int y = (page * nkv + it.kvh) * c.page_size + j0 % c.page_size;
                    if (!wait(bars.empty[s], at / ST + 1, 1)) return false;
                    mbar_expect_tx(smem_u32(&bars.full[s]), KT_BYTES);
#pragma unroll
                    for (int kb = 0; kb < NKB; ++kb) tma_load_2d(smem_u32(ring + s * KT_BYTES + kb * BN * 128), map, kb * 64, y, smem_u32(&bars.full[s]));
                    ++at;
                    return true;
                };
                for (int t = 0; t < order.ahead; ++t)
                    if (!load(&map_k, t)) return false;
                for (int t = 0; t < order.n; ++t) {
                    if (!load(&map_v, t)) return false;
                    if (t + order.ahead < order.n && !load(&map_k, t + order.ahead)) return false;
                }
                return true;
            });
            // the last releases must have arrived, or (where the block gives up) the copies in flight have landed, before it leaves
            for (unsigned j = at > ST ? at - ST : 0; j < at && !*abort_flag; ++j)
                if (!wait(bars.empty[j % ST], j / ST, 1)) break;
            if (*abort_flag)
                for (unsigned j = at > ST ? at - ST : 0; j < at; ++j) mbar_drain(smem_u32(&bars.full[j % ST]), (j / ST) & 1, limit);
        }
    } else if (warp == 3) {
        if (lane == 0) {
            // ---- the rows of q
            unsigned n = 0;
            for_items([&](const Item& it) {
                if (n > 0 && !wait(bars.q_empty, n - 1, 1)) return false;
                const int tiles = it.pair ? 2 : 1;
                mbar_expect_tx(smem_u32(&bars.q_full), (unsigned)(tiles * NKB * q_box_tokens * G * 128));
                for (int g = 0; g < tiles; ++g)
#pragma unroll
                    for (int kb = 0; kb < NKB; ++kb)
                        tma_load_3d(smem_u32(q_s + g * Q_BYTES + kb * BM * 128), &map_q, kb * 64, it.kvh * G, it.first + it.node0 + g * tpt, smem_u32(&bars.q_full));
                ++n;
                return true;
            });
            if (n > 0 && !*abort_flag) wait(bars.q_empty, n - 1, 1);
            if (n > 0 && *abort_flag) mbar_drain(smem_u32(&bars.q_full), (n - 1) & 1, limit);
        }
    } else if (warp < 3) {
        if (lane == 0) {
            // ---- tensor-core issue for one half
            const int g = warp - 1;
            HalfBarriers& gb = bars.g[g];
            const unsigned tmem_g = tmem + g * GROUP_COLS;
            const unsigned idesc_s = make_idesc(BM, BN), idesc_pv = make_idesc(BM, HD, true);
            unsigned n_items = 0, at = 0;                        // items; tiles of the ring released so far
            unsigned scored = 0, added = 0;                      // own tiles whose scores, whose products with the values are issued
            for_items([&](const Item& it) {
                const Order order(it);
                const int n = order.n, step = it.pair ? 1 : 2, first = it.pair ? 0 : g, own = n > first ? (n - first + step - 1) / step : 0;
                const unsigned base = at;
                unsigned char* q_g = q_s + (it.pair ? g : 0) * Q_BYTES;
                // tiles of the other half's: wait until they have landed (so that the halves drift apart by no more than the ring) and hand them back
                auto pass_to = [&](unsigned to) {
                    for (; at < to; ++at) {
                        if (!wait(bars.full[at % ST], at / ST, 2)) return false;
                        mbar_arrive(smem_u32(&bars.empty[at % ST]));
                    }
                    return true;
                };
                auto issue_scores = [&](int li) {
                    if (!pass_to(base + order.keys(first + li * step))) return false;
                    const int s = at % ST, sb = scored & 1;
                    // P of two tiles before lay where the scores go; the product issued last is waited for (by parity only that can be)
                    if (added > 0 && !wait(gb.pv_done, added - 1, 2)) return false;
                    if (!wait(bars.full[s], at / ST, 2)) return false;
                    fence_after();
                    const unsigned qa = smem_u32(q_g), ka = smem_u32(ring + s * KT_BYTES);
#pragma unroll
                    for (int ks = 0; ks < HD / 16; ++ks)
                        mma(tmem_g + sb * BN, smem_desc_k_major(qa + (ks / 4) * BM * 128 + (ks % 4) * 32),
                            smem_desc_k_major(ka + (ks / 4) * BN * 128 + (ks % 4) * 32), idesc_s, ks > 0 ? 1u : 0u);
                    commit(smem_u32(&gb.s_full[sb]));
                    commit(smem_u32(&bars.empty[s]));
                    if (li == own - 1) commit(smem_u32(&bars.q_empty));
                    ++at;
                    ++scored;
                    return true;
                };
                if (!wait(bars.q_full, n_items, 2)) return false;
                if (own == 0) mbar_arrive(smem_u32(&bars.q_empty));
                if (own > 0 && !issue_scores(0)) return false;
                if (own > 1 && !issue_scores(1)) return false;
                for (int li = 0; li < own; ++li) {
                    if (!pass_to(base + order.values(first + li * step))) return false;
                    const int s = at % ST;
                    if (!wait(gb.p_ready, added, 2) || !wait(bars.full[s], at / ST, 2)) return false;
                    fence_after();
                    const unsigned va = smem_u32(ring + s * KT_BYTES);
#pragma unroll
                    for (int ks = 0; ks < BN / 16; ++ks)
                        mma_a_tmem(tmem_g + 2 * BN, tmem_g + (added & 1) * BN + ks * 8, smem_desc(va + ks * 16 * 128, BN * 128, 1024), idesc_pv,
                                   (li > 0 || ks > 0) ? 1u : 0u);
                    commit(smem_u32(&gb.pv_done));
                    commit(smem_u32(&bars.empty[s]));
                    ++at;
                    ++added;
                    if (li + 2 < own && !issue_scores(li + 2)) return false;
                }
                ++n_items;
                return pass_to(base + 2 * n);
            });
        }
    } else {
        // ---- softmax: one thread a row; warp w may read tensor-memory lanes [32 (w % 4), + 32)
        const int g = (warp - 4) >> 2, quarter = warp & 3, r = quarter * 32 + lane;
        HalfBarriers& gb = bars.g[g];
        const unsigned lane_base = tmem + g * GROUP_COLS + ((unsigned)(quarter * 32) << 16);
        const float scale = p.softmax_scale * LOG2E;
        // cap and slope in units of the raw scores (see the prompts' kernel)
        const bool capped = CAP && p.score_softcap > 0.f, biased = BIAS && p.head_slopes != nullptr;
        const float cap_raw = capped ? p.score_softcap / p.softmax_scale : 0.f, inv_cap_raw = capped ? p.softmax_scale / p.score_softcap : 0.f;
        const float cap_arg = capped ? 2.f * LOG2E * p.softmax_scale / p.score_softcap : 0.f;
        unsigned ring0 = 0, seen = 0, singles = 0, turns = 0;    // tiles of the ring before this item; own tiles so far; singles, a pair's tiles so far
        auto all_wait = [&](unsigned long long& bar, unsigned parity) { return (bool)__all_sync(0xffffffffu, wait(bar, parity, 3)); };
        for_items([&](const Item& it) {
            const Order order(it);
            const int n = order.n, step = it.pair ? 1 : 2, first = it.pair ? 0 : g, own = n > first ? (n - first + step - 1) / step : 0;
            const bool part = it.from > 0 || it.to < it.tiles;
            const int node_base = it.node0 + (it.pair ? g * tpt : 0), nodes = max(0, min(tpt, it.node0 + it.nodes - node_base));
            const int n_rows = nodes * G;
            const bool warp_rows = quarter * 32 < n_rows, row_ok = r < n_rows;
            const int node = node_base + (row_ok ? r / G : 0), tok = it.first + node, head = it.kvh * G + (row_ok ? r % G : 0);
            const int pos = row_ok ? b.positions[tok] : 0;
            const int lo = window_lowest(p.window_kind, p.window_size, pos);
            const int lo_all = window_lowest(p.window_kind, p.window_size, it.len + it.n - 1);      // (no node is deeper)
            const float slope_raw = biased ? slope_of(p, head) / p.softmax_scale : 0.f;
            const unsigned* set = x.ancestors + (size_t)tok * x.n_words;
            float m_ref = -INFINITY, l = 0.f;
            for (int li = 0; li < own; ++li, ++seen) {
                const int i = first + li * step, sb = seen & 1, j0 = it.k_begin + (it.from + i) * BN;
                unsigned long long live = ~0ull;                 // places of the tile whose rows hold a key
                if (j0 + BN > it.len) {                          // a tile with nodes
                    const int b0 = j0 - it.len;
                    auto holds = [&](int a) { return a < 0 || (a < it.n && tree_node_is_real(x, it.first, a)); };
                    live = (unsigned long long)__ballot_sync(0xffffffffu, holds(b0 + lane)) |
                           (unsigned long long)__ballot_sync(0xffffffffu, holds(b0 + 32 + lane)) << 32;
                    if (live != ~0ull) {
                        const unsigned at = ring0 + order.values(i);
                        if (!all_wait(bars.full[at % ST], at / ST)) return false;
                        unsigned char* v_t = ring + (at % ST) * KT_BYTES;
                        for (int e = r; e < BN * 8 * NKB; e += BM) {
                            const int row = e / (8 * NKB), ch = e % (8 * NKB);
                            if (!(live >> row & 1)) *(uint4*)(v_t + (ch / 8) * BN * 128 + row * 128 + (ch % 8) * 16) = make_uint4(0, 0, 0, 0);
                        }
                        fence_proxy_async();
                    }
                }
                if (!all_wait(gb.s_full[sb], seen >> 1)) return false;
                const int turn = turns + i;
                if (!warp_rows) {                                // nothing to compute, but the barriers count every warp
                    if (li > 0 && !all_wait(gb.pv_done, seen - 1)) return false;      // (first: no arrival may run ahead of the other warps' last)
                    __syncwarp();
                    if (it.pair && lane == 0) mbar_arrive(smem_u32(&gb.exp_done));
                    if (lane == 0) mbar_arrive(smem_u32(&gb.p_ready));
                    continue;
                }
                fence_after();
                float s[BN];
                ld64(s, lane_base + sb * BN);
                const bool open = j0 >= lo_all && j0 + BN <= it.len;      // every key visible to every row
                // 64 bits of what this row sees: settled tokens from its window's end on, then nodes
                auto seen_bits = [&]() {
                    unsigned long long vis = low_bits(it.len - j0) & ~low_bits(lo - j0);
                    if (j0 + BN > it.len) {
                        const int b0 = j0 - it.len;
                        auto word = [&](int k) { return row_ok && k < x.n_words ? set[k] : 0u; };
                        unsigned long long bits;
                        if (b0 >= 0) {
                            const int w = b0 >> 5, sh = b0 & 31;
                            const unsigned mid = word(w + 1);
                            bits = (unsigned long long)__funnelshift_r(mid, word(w + 2), sh) << 32 | __funnelshift_r(word(w), mid, sh);
                        } else {
                            bits = ((unsigned long long)word(1) << 32 | word(0)) << -b0;
                        }
                        bits &= live & low_bits(node + 1 - b0);  // (no node behind itself)
                        if (lo > it.len)                         // the window ends within the tree: by the ancestors' positions
                            for (unsigned long long rest = bits; rest; rest &= rest - 1) {
                                const int e = __ffsll((long long)rest) - 1;
                                if (b.positions[it.first + b0 + e] < lo) bits &= ~(1ull << e);
                            }
                        vis |= bits;
                    }
                    return row_ok ? vis : 0ull;
                };
                auto keep_seen = [&](unsigned long long vis, float other) {
#pragma unroll
                    for (int e = 0; e < BN; ++e) s[e] = ((e < 32 ? (unsigned)vis : (unsigned)(vis >> 32)) >> (e & 31) & 1u) ? s[e] : other;
                };
                unsigned long long vis = 0;
                if (CAP && !open) vis = seen_bits();
                if (capped) {
                    // cap tanh(s scale / cap): the series where every score that the row sees in the tile is small against the cap, else by 2^x.  Every
                    // row chooses for itself, so that its bits do not depend on the rows beside it or on keys that it does not see; a warp whose
                    // rows differ makes both one after the other.  (us, against a choice of the warp: 8 requests of 16 nodes, 8,192 keys, 82.9 / 79.2 with
                    // a cap of 50, 116 / 95 with one of 3, that about half of the tiles' largest scores reach; all in one loop with a choice by element spills: 92 / 155.)
                    if (!open) keep_seen(vis, 0.f);
                    float big[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int e = 0; e < BN; ++e) big[e & 3] = fmaxf(big[e & 3], fabsf(s[e]));
                    const bool small = !row_ok || fmaxf(fmaxf(big[0], big[1]), fmaxf(big[2], big[3])) <= CAP_SERIES * cap_raw;
                    if (small) {
                        const f2 inv = pack2(inv_cap_raw, inv_cap_raw), one = pack2(1.f, 1.f), c1 = pack2(CAP_C1, CAP_C1), c2 = pack2(CAP_C2, CAP_C2),
                                 c3 = pack2(CAP_C3, CAP_C3), c4 = pack2(CAP_C4, CAP_C4), c5 = pack2(CAP_C5, CAP_C5);
#pragma unroll
                        for (int e = 0; e < BN; e += 2) {
                            const f2 v = pack2(s[e], s[e + 1]), t = mul2(v, inv), y = mul2(t, t);
                            unpack2(mul2(v, fma2(y, fma2(y, fma2(y, fma2(y, fma2(y, c5, c4), c3), c2), c1), one)), s[e], s[e + 1]);
                        }
                    } else {
#pragma unroll
                        for (int e = 0; e < BN; ++e) s[e] = fmaf(-2.f * cap_raw, reciprocal_approx(ex2(s[e] * cap_arg) + 1.f), cap_raw);
                    }
                    __syncwarp();
                }
                float tile_bias = 0.f;                           // what the tile's keys have in common of a bias by distance
                if (biased) {
                    if (j0 + BN <= it.len) {
                        tile_bias = slope_raw * (float)(j0 - pos);
#pragma unroll
                        for (int e = 0; e < BN; ++e) s[e] = fmaf(slope_raw, (float)e, s[e]);
                    } else {
#pragma unroll
                        for (int e = 0; e < BN; ++e) {
                            const int a = j0 + e - it.len;       // (a node sits at its depth, not at its place)
                            s[e] = fmaf(slope_raw, (float)((a < 0 ? j0 + e : a < it.n ? b.positions[it.first + a] : 0) - pos), s[e]);
                        }
                    }
                }
                if (!open) keep_seen(CAP ? vis : seen_bits(), -INFINITY);
                float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int e = 0; e < BN; ++e) mx4[e & 3] = fmaxf(mx4[e & 3], s[e]);
                const float mx = (fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) + tile_bias) * scale;
                const bool need = mx > m_ref + RESCALE_STEP;
                float corr = 1.f;
                if (need) { corr = exp2f(m_ref - mx); l *= corr; m_ref = mx; }
                const float neg_m = m_ref == -INFINITY ? 0.f : fmaf(tile_bias, scale, -m_ref);
                // a pair's halves take turns at the exponentials: the units serve one while the tensor cores work for the other
                if (it.pair && (g == 1 || turn > 0) && !all_wait(bars.g[g ^ 1].exp_done, g == 0 ? turn - 1 : turn)) return false;
                unsigned packed[BN / 2];
                f2 sum2[4] = {0ull, 0ull, 0ull, 0ull};
                const f2 scale2 = pack2(scale, scale), neg_m2 = pack2(neg_m, neg_m);
#pragma unroll
                for (int e = 0; e < BN; e += 2) {
                    if (e == BN * 3 / 4) {
                        __syncwarp();
                        if (it.pair && lane == 0) mbar_arrive(smem_u32(&gb.exp_done));
                    }
                    float a, d;
                    unpack2(fma2(pack2(s[e], s[e + 1]), scale2, neg_m2), a, d);
                    a = ex2(a);
                    d = ex2(d);
                    sum2[(e >> 1) & 3] = add2(sum2[(e >> 1) & 3], pack2(a, d));
                    packed[e / 2] = pack_bf16(a, d);
                }
                float sum_a, sum_b;
                unpack2(add2(add2(sum2[0], sum2[1]), add2(sum2[2], sum2[3])), sum_a, sum_b);
                l += sum_a + sum_b;
                if (li > 0) {
                    // the product of the tile before must have left O before its rows are rescaled (waited for in every tile: a wait by
                    // parity is only right while the waiter is at most one phase behind)
                    if (!all_wait(gb.pv_done, seen - 1)) return false;
                    if (__any_sync(0xffffffffu, need)) {
                        fence_after();
#pragma unroll 1
                        for (int c0 = 0; c0 < HD; c0 += 32) {
                            float o[32];
                            ld32(o, lane_base + 2 * BN + c0);
#pragma unroll
                            for (int e = 0; e < 32; ++e) o[e] *= corr;
                            st32(lane_base + 2 * BN + c0, o);
                        }
                    }
                }
                st32(lane_base + sb * BN, packed);
                fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&gb.p_ready));
            }
            if (own > 0 && !all_wait(gb.pv_done, seen - 1)) return false;
            fence_after();
            float* slot = cut.partial + (size_t)(2 * blockIdx.x + (it.from == 0)) * slot_floats(HD);
            __nv_bfloat16* dst = (__nv_bfloat16*)p.out + out_row_of(p, tok, head) * HD;
            auto leave = [&](const float (&o)[32], int c0, float inv) {
                if (!row_ok) return;
                if (part) {
                    float* to = slot + (it.pair ? g : 0) * HD * BM + r;
#pragma unroll
                    for (int e = 0; e < 32; ++e) __stcg(to + (c0 + e) * BM, o[e]);        // a column's rows side by side
                    return;
                }
#pragma unroll
                for (int e = 0; e < 32; e += 8)
                    *(uint4*)(dst + c0 + e) = make_uint4(pack_bf16(o[e] * inv, o[e + 1] * inv), pack_bf16(o[e + 2] * inv, o[e + 3] * inv),
                                                         pack_bf16(o[e + 4] * inv, o[e + 5] * inv), pack_bf16(o[e + 6] * inv, o[e + 7] * inv));
            };
            if (it.pair) {
                if (warp_rows) {
                    const float inv = part ? 0.f : row_scale_of(p, tok, head, m_ref, l);
#pragma unroll 1
                    for (int c0 = 0; c0 < HD; c0 += 32) {
                        float o[32];
                        ld32(o, lane_base + 2 * BN + c0);
                        leave(o, c0, inv);
                    }
                    if (part) __stcg((float2*)(slot + 2 * HD * BM) + g * BM + r, tree_state(m_ref, l));
                }
                turns += n;
            } else {
                // the halves' states and outputs are added up: each half takes half of the head, and reads the other's out of tensor memory
                state_s[g][r] = tree_state(m_ref, l);
                fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&bars.state_ready));
                if (!all_wait(bars.state_ready, singles)) return false;
                fence_after();
                if (warp_rows) {
                    const float2 a = state_s[0][r], d = state_s[1][r];
                    const float m = fmaxf(a.x, d.x), fa = a.x == -INFINITY ? 0.f : exp2f(a.x - m), fd = d.x == -INFINITY ? 0.f : exp2f(d.x - m);
                    const float sum = fmaf(a.y, fa, d.y * fd);
                    const float inv = part ? 0.f : row_scale_of(p, tok, head, m, sum);
                    const unsigned row_base = tmem + ((unsigned)(quarter * 32) << 16) + 2 * BN;
#pragma unroll 1
                    for (int c0 = g * (HD / 2); c0 < (g + 1) * (HD / 2); c0 += 32) {
                        float o[32], o1[32];
                        ld32(o, row_base + c0);
                        ld32(o1, row_base + GROUP_COLS + c0);
#pragma unroll
                        for (int e = 0; e < 32; ++e)             // (a half without a key of this row has left anything)
                            o[e] = (fa != 0.f ? o[e] * fa : 0.f) + (fd != 0.f ? o1[e] * fd : 0.f);
                        leave(o, c0, inv);
                    }
                    if (part && g == 0) __stcg((float2*)(slot + 2 * HD * BM) + r, tree_state(m, sum));
                }
                fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&bars.state_read));
                if (!all_wait(bars.state_read, singles)) return false;       // before either output is written again
                ++singles;
            }
            ring0 += 2 * n;
            return true;
        });
    }
    fence_before();
    __syncthreads();
    if (warp == 1) {
        fence_after();
        tmem_free(tmem, TMEM_COLS);
    }
}

// Adds up the parts of the items that were cut, in the order of the keys.  grid (blocks, head_dim / JOIN_COLS, row tiles of a pair), a thread a row;
// part 0 of an item is the last of the block before its first cut, part k the first of the block behind its cut k.  What it costs is the latency of
// its loads, so as many as there are registers for are asked for at once.  (As many blocks as fit beside each other, with a list of the items that
// were cut, were no faster: 8 x 16 nodes, 8,192 keys 63.7 against 62.9 to 67.6 us in all, 16 nodes and 1,000 keys 20 against 17, 16 x 64 nodes 333 against 341.)
constexpr int JOIN_COLS = 8;
__global__ void __launch_bounds__(BM) attn_tree_tc_join_kernel(const AttentionParams p, const TreeCut cut, int nkv, int tpt, int hd) {
    pdl_wait();
    pdl_launch_dependents();
    const int4 item = __ldcg(cut.items + blockIdx.x);
    if (item.w < 2) return;
    const int G = p.num_heads / nkv, g = blockIdx.z, r = threadIdx.x, c0 = blockIdx.y * JOIN_COLS;
    if (r >= min(tpt, item.y - g * tpt) * G) return;             // (a single's second row tile has no rows)
    const int tok = item.x + g * tpt + r / G, head = item.z * G + r % G;
    const float* parts = cut.partial + (size_t)(2 * blockIdx.x) * slot_floats(hd);
    auto slot = [&](int k) { return parts + (k ? 2 * (long long)k - 2 : -1ll) * (long long)slot_floats(hd); };
    float m = -INFINITY, l = 0.f, o[JOIN_COLS];
#pragma unroll
    for (int e = 0; e < JOIN_COLS; ++e) o[e] = 0.f;
    constexpr int N = 12;                                        // parts whose loads are asked for together
    for (int k0 = 0; k0 < item.w; k0 += N) {
        float2 ml[N];
        float v[N][JOIN_COLS];
#pragma unroll
        for (int k = 0; k < N; ++k) {
            if (k0 + k >= item.w) { ml[k] = make_float2(-INFINITY, 0.f); continue; }
            const float* from = slot(k0 + k);
            ml[k] = __ldcg((const float2*)(from + 2 * hd * BM) + g * BM + r);
#pragma unroll
            for (int e = 0; e < JOIN_COLS; ++e) v[k][e] = __ldcg(from + (size_t)(g * hd + c0 + e) * BM + r);
        }
        float top = m;
#pragma unroll
        for (int k = 0; k < N; ++k) top = fmaxf(top, ml[k].x);
        const float keep = m == -INFINITY ? 0.f : exp2f(m - top);
        m = top;
        l *= keep;
#pragma unroll
        for (int e = 0; e < JOIN_COLS; ++e) o[e] *= keep;
#pragma unroll
        for (int k = 0; k < N; ++k) {
            if (ml[k].x == -INFINITY) continue;                  // (no part, or one without a key of this row)
            const float w = exp2f(ml[k].x - m);
            l = fmaf(w, ml[k].y, l);
#pragma unroll
            for (int e = 0; e < JOIN_COLS; ++e) o[e] = fmaf(w, v[k][e], o[e]);
        }
    }
    const float inv = row_scale_of(p, tok, head, m, l);
    *(uint4*)((__nv_bfloat16*)p.out + out_row_of(p, tok, head) * hd + c0) =
        make_uint4(pack_bf16(o[0] * inv, o[1] * inv), pack_bf16(o[2] * inv, o[3] * inv), pack_bf16(o[4] * inv, o[5] * inv), pack_bf16(o[6] * inv, o[7] * inv));
}

template <int NKB>
int launch(const AttentionParams& p, const StepTokens& b, const PagedCache& c, const TreeStep& x, const TreeCut& cut, int n_sm, cudaStream_t st) {
    const int hd = 64 * NKB, nq = p.num_heads, nkv = c.num_kv_heads, G = nq / nkv, tpt = BM / G;
    const int box_tokens = tpt < b.n_tokens ? tpt : b.n_tokens;
    CUtensorMap mq, mk, mv;
    {
        cuuint64_t dims[3] = {(cuuint64_t)hd, (cuuint64_t)nq, (cuuint64_t)b.n_tokens};
        cuuint64_t strides[2] = {(cuuint64_t)hd * 2, (cuuint64_t)nq * hd * 2};
        cuuint32_t box[3] = {64, (cuuint32_t)G, (cuuint32_t)box_tokens};
        if (!make_map(&mq, p.q, 3, dims, strides, box)) return SPITE_LAUNCH_FAILED;
    }
    {
        cuuint64_t dims[2] = {(cuuint64_t)hd, (cuuint64_t)c.n_pages * nkv * c.page_size};
        cuuint64_t strides[1] = {(cuuint64_t)hd * 2};
        cuuint32_t box[2] = {64, (cuuint32_t)BN};
        if (!make_map(&mk, c.kv, 2, dims, strides, box)) return SPITE_LAUNCH_FAILED;
        if (!make_map(&mv, (const __nv_bfloat16*)c.kv + c.v_offset, 2, dims, strides, box)) return SPITE_LAUNCH_FAILED;
    }
    auto smem_for = [](int segments) { return (2 * (size_t)NKB * BM + stages(NKB) * (size_t)NKB * BN) * 128 + (size_t)segments * 20 + 4; };
    const size_t smem = smem_for(x.n_segments < MAX_SEGMENTS ? x.n_segments : MAX_SEGMENTS);
    const int form = p.head_slopes ? FORM_ANY : p.score_softcap > 0.f ? FORM_CAP : FORM_PLAIN;
    auto k = form == FORM_ANY ? attn_tree_tc_kernel<NKB, FORM_ANY> : form == FORM_CAP ? attn_tree_tc_kernel<NKB, FORM_CAP> : attn_tree_tc_kernel<NKB, FORM_PLAIN>;
    static std::atomic<unsigned long long> done[3];
    if (!allow_shared(k, smem_for(MAX_SEGMENTS), done[form])) return SPITE_LAUNCH_FAILED;
    const long long tiles = (long long)b.table_width * c.page_size / BN;
    int launches = 0;
    for (int s0 = 0; s0 < x.n_segments; s0 += MAX_SEGMENTS) {
        TreeStep some = x;
        StepTokens tokens = b;
        some.cu_seqlens += s0;
        some.n_segments = x.n_segments - s0 < MAX_SEGMENTS ? x.n_segments - s0 : MAX_SEGMENTS;
        tokens.block_table += (size_t)s0 * b.table_width;
        SPITE_LAUNCH(k, n_sm, THREADS, smem, st, mq, mk, mv, p, tokens, c, some, tpt, box_tokens, cut, s_waits);
        ++launches;
        if (tiles >= 2 * PIECE) {                                // (with fewer no item is cut)
            SPITE_LAUNCH(attn_tree_tc_join_kernel, dim3(n_sm, hd / JOIN_COLS, 2), BM, 0, st, p, cut, nkv, tpt, hd);
            ++launches;
        }
    }
    const int status = spite_launch_status();
    return status == SPITE_OK ? launches : status;
}

}  // namespace

// `n_sm`: number of multiprocessors (a block each).  `scratch`: n_sm * (4 * (head_dim + 2) * 128 + 4) floats.  Returns the number of launches,
// or what is wrong.
SPITE_API int spite_tree_attention_tc(const TreeCall* call, int n_sm, float* scratch, long long n_floats, void* stream) {
    if (!call || !scratch || n_sm < 1 || !tree_call_ok(*call)) return SPITE_BAD_ARG;
    const AttentionParams& p = call->p;
    const PagedCache& c = call->c;
    if ((c.head_dim != 64 && c.head_dim != 128) || p.num_heads / c.num_kv_heads > BM || c.page_size % BN) return SPITE_UNSUPPORTED;
    if (p.distance_bias || c.key_scale || c.v_offset == 0) return SPITE_UNSUPPORTED;
    if ((long long)c.n_pages * c.num_kv_heads * c.page_size > 0x7fffffffll) return SPITE_UNSUPPORTED;       // TMA coordinates are int32
    if ((((uintptr_t)p.q | (uintptr_t)p.out | (uintptr_t)c.kv | (uintptr_t)scratch) & 15) || (c.v_offset & 7)) return SPITE_UNSUPPORTED;
    const long long slots = 2ll * n_sm * (long long)slot_floats(c.head_dim);
    if (slots + 4ll * n_sm > n_floats) return SPITE_BAD_ARG;
    // the line is counted in 32 bits: no request has more key tiles than its table, no more row tiles than nodes
    const long long tiles = (long long)call->b.table_width * c.page_size / BN + 1;
    const double longest = (double)(COST_ITEM + COST_PAIR * tiles) * c.num_kv_heads * (call->b.n_tokens / (BM / (p.num_heads / c.num_kv_heads)) + call->x.n_segments);
    if (longest >= 4e9) return SPITE_UNSUPPORTED;
    if (call->b.n_tokens == 0) return SPITE_OK;
    const TreeCut cut{scratch, (int4*)(scratch + slots)};
    return c.head_dim == 64 ? launch<1>(p, call->b, c, call->x, cut, n_sm, (cudaStream_t)stream) : launch<2>(p, call->b, c, call->x, cut, n_sm, (cudaStream_t)stream);
}
