// Attention over trees of drafted tokens on the fifth-generation tensor cores (bfloat16, heads of 64 or 128 elements, pages of a multiple
// of 64 keys, up to 128 query heads per kv head, up to 2,048 requests).
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
//   0        one lane loads K and V tiles into two rings            3        one lane loads the items' rows of q
//   1, 2     one lane each issues S = Q K^T and O += P V of its half, scores two tiles ahead; P is read from tensor memory
//   4 - 11   four softmax warps a half, one thread a row: scores by tcgen05.ld, scale, mask, running maximum (which moves only
//            when it grows by more than 2^8) and sum in float32, P as bfloat16 over the scores it came from
// P is rounded to bfloat16 because the tensor cores take both operands in one type; the sum is taken of the unrounded weights.
//
// Masks matter in the tiles at a window's end and in those with the step's own nodes; there a row makes 64 bits of what it sees.  A value row
// that is no node's (padding, what lies behind the last node) may hold anything, and 0 x NaN is NaN: the softmax warps clear
// these rows of the tile in shared memory before the product.  Settled rows are finite as everywhere in the cache.
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
constexpr int MAX_SEGMENTS = 2048;

// The line: what a key tile of a pair and of a single costs, what an item costs besides, the shortest part.
constexpr int COST_PAIR = 3, COST_SINGLE = 2, COST_ITEM = 6;
constexpr int PIECE = 3;                // key tiles: a cut closer to an item's end moves there
constexpr int SHARE = 24;               // the shortest stretch, while there are blocks for every item

__device__ int g_attn_tree_error = 0;
}  // namespace
SPITE_WAIT_CONTROLS(attention_tree_tc, g_attn_tree_error)
namespace {

struct TreeCut {
    float* partial;                     // [blocks][2: a block's first part, its last][2 row tiles x (HD + 2) x 128]
    int4* items;                        // [blocks][2]: where block i's first cut is the first within an item: (segment's first node of the item, nodes,
};                                      // kv head, parts), (pair, -, -, -); no parts: none
__host__ __device__ constexpr size_t slot_floats(int head_dim) { return 2 * (size_t)(head_dim + 2) * BM; }

__host__ __device__ constexpr int stages(int nkb) { return nkb == 1 ? 8 : 4; }
template <bool B> struct Flag { static constexpr bool value = B; };
struct HalfBarriers { unsigned long long s_full[2], p_ready, pv_done, exp_done; };
struct Barriers {
    unsigned long long q_full, q_empty, k_full[8], k_empty[8], v_full[8], v_empty[8], state_ready, state_read;
    HalfBarriers g[2];
    unsigned tmem_base;
    int abort_flag;
};

// An item, or the part of it that a block works on: key tiles [from, to) of `tiles`.
struct Item { int seg, first, n, len, kvh, node0, nodes, k_begin, tiles, from, to; bool pair; };

__device__ __forceinline__ float row_scale_of(const AttentionParams& p, int tok, int head, float m, float l) {
    float shrink = 1.f;
    if (p.has_sink && sink_of(p, head) > -INFINITY) {           // the sink joins the sum, in powers of two
        const float sink2 = sink_of(p, head) * LOG2E, m2 = fmaxf(m, sink2);
        shrink = m == -INFINITY ? 0.f : exp2f(m - m2);
        l = l * shrink + exp2f(sink2 - m2);
    }
    return shrink * gate_of(p, tok, head) / fmaxf(l, 1e-30f);
}

__device__ __forceinline__ unsigned pack_bf16(float a, float b) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *(const unsigned*)&v;
}

// Element e of 64 bits in two words.
__device__ __forceinline__ unsigned long long low_bits(int n) { return n <= 0 ? 0ull : n >= 64 ? ~0ull : (1ull << n) - 1; }

// NKB = head_dim / 64.  One block a multiprocessor.
template <int NKB, bool CAP>
__global__ void __launch_bounds__(THREADS, 1)
attn_tree_tc_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                    const AttentionParams p, const StepTokens b, const PagedCache c, const TreeStep x, const int tpt, const int q_box_tokens, const TreeCut cut,
                    const WaitControl waits) {
    constexpr int HD = 64 * NKB, ST = stages(NKB);
    constexpr int Q_BYTES = NKB * BM * 128, KT_BYTES = NKB * BN * 128;
    extern __shared__ __align__(1024) unsigned char smem[];     // [Q0][Q1][K ring][V ring], 1024-byte aligned, then the line
    __shared__ Barriers bars;
    __shared__ float2 state_s[2][BM];                            // a single's two softmax states
    __shared__ long long n_sets_s;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int nq = p.num_heads, nkv = c.num_kv_heads, G = nq / nkv, S = x.n_segments;
    unsigned char* q_s = smem;
    unsigned char* k_s = q_s + 2 * Q_BYTES;
    unsigned char* v_s = k_s + ST * KT_BYTES;
    long long* line = (long long*)(v_s + ST * KT_BYTES);         // [S + 1] what the requests before cost (for one kv head)
    volatile int* abort_flag = &bars.abort_flag;
    int* const err = waits.error_word ? waits.error_word : &g_attn_tree_error;
    const long long limit = waits.limit_cycles;

    if (threadIdx.x == 0) {
        bars.abort_flag = 0;
        mbar_init(smem_u32(&bars.q_full), 1);
        mbar_init(smem_u32(&bars.q_empty), 2);
        for (int s = 0; s < ST; ++s) {
            mbar_init(smem_u32(&bars.k_full[s]), 1); mbar_init(smem_u32(&bars.k_empty[s]), 2);      // both halves release a stage
            mbar_init(smem_u32(&bars.v_full[s]), 1); mbar_init(smem_u32(&bars.v_empty[s]), 2);
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
    pdl_wait();
    pdl_launch_dependents();

    // ---- the line
    struct Request { int first, n, len, k_begin, tiles, pairs, single; };
    auto request_of = [&](int s) {
        Request r;
        r.first = min(max(x.cu_seqlens[s], 0), b.n_tokens);
        r.n = min(max(x.cu_seqlens[s + 1], r.first), b.n_tokens) - r.first;
        r.len = r.n ? max(b.positions[r.first], 0) : 0;
        const int places = (int)min((long long)r.len + r.n, (long long)b.table_width * c.page_size);
        r.k_begin = window_lowest(p.window_kind, p.window_size, r.len) / BN * BN;
        r.tiles = r.n && places > r.k_begin ? (places - r.k_begin + BN - 1) / BN : 0;
        const int row_tiles = r.tiles ? (r.n + tpt - 1) / tpt : 0;
        r.pairs = row_tiles / 2;
        r.single = row_tiles & 1;
        return r;
    };
    for (int s = threadIdx.x; s < S; s += THREADS) {
        const Request r = request_of(s);
        line[s + 1] = (long long)r.pairs * (COST_ITEM + (long long)r.tiles * COST_PAIR) + r.single * (COST_ITEM + (long long)r.tiles * COST_SINGLE);
    }
    fence_before();
    __syncthreads();
    fence_after();
    const unsigned tmem = bars.tmem_base;
    if (warp == 0) {
        long long sum = 0, sets = 0;
        for (int s0 = 0; s0 < S; s0 += 32) {
            long long v = s0 + lane < S ? line[s0 + lane + 1] : 0;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const long long u = __shfl_up_sync(0xffffffffu, v, o);
                if (lane >= o) v += u;
            }
            if (s0 + lane < S) {
                line[s0 + lane + 1] = sum + v;
                const Request r = request_of(s0 + lane);
                sets += r.pairs + r.single;
            }
            sum += __shfl_sync(0xffffffffu, v, 31);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sets += __shfl_xor_sync(0xffffffffu, sets, o);
        if (lane == 0) { line[0] = 0; n_sets_s = sets; }
    }
    __syncthreads();
    const long long line_end = line[S] * nkv;
    // as many blocks as there are items, or as shares of the shortest length
    const int sharers = (int)min((long long)gridDim.x, max(n_sets_s * nkv, line_end / SHARE));
    struct Place { Item item; long long at; int len; };          // the item's beginning on the line and its length
    auto place_of = [&](long long t) {                           // 0 <= t < line_end
        int lo = 0, hi = S;                                      // nkv * line[lo] <= t < nkv * line[hi]
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (nkv * line[mid] <= t) lo = mid; else hi = mid;
        }
        const Request r = request_of(lo);
        const long long per_head = line[lo + 1] - line[lo];
        long long rest = t - nkv * line[lo];
        Place q;
        q.item.kvh = (int)(rest / per_head);
        q.at = nkv * line[lo] + q.item.kvh * per_head;
        rest -= q.item.kvh * per_head;
        const int pair_len = COST_ITEM + r.tiles * COST_PAIR, idx = (int)min((long long)r.pairs, rest / pair_len);
        q.item.pair = idx < r.pairs;
        q.at += (long long)idx * pair_len;
        q.len = q.item.pair ? pair_len : COST_ITEM + r.tiles * COST_SINGLE;
        q.item.seg = lo; q.item.first = r.first; q.item.n = r.n; q.item.len = r.len; q.item.k_begin = r.k_begin; q.item.tiles = r.tiles;
        q.item.node0 = 2 * idx * tpt;
        q.item.nodes = min((q.item.pair ? 2 : 1) * tpt, r.n - q.item.node0);
        q.item.from = 0; q.item.to = r.tiles;
        return q;
    };
    // the key tile where a cut `off` behind an item's beginning falls
    auto tile_at = [&](long long off, const Item& it) {
        const int w = it.pair ? COST_PAIR : COST_SINGLE;
        const int t = off <= COST_ITEM ? 0 : (int)((off - COST_ITEM + w / 2) / w);
        return t < PIECE ? 0 : it.tiles - t < PIECE ? it.tiles : t;
    };
    auto cut_at = [&](int i) { return i >= sharers ? line_end : line_end * i / sharers; };
    const long long begin = (int)blockIdx.x < sharers && line_end > 0 ? cut_at(blockIdx.x) : 0;
    const long long end = (int)blockIdx.x < sharers && line_end > 0 ? cut_at(blockIdx.x + 1) : 0;
    if (threadIdx.x == 0) {
        int4 a = make_int4(0, 0, 0, 0), d = make_int4(0, 0, 0, 0);
        if (begin < end) {
            const Place q = place_of(begin);
            const int mine = tile_at(begin - q.at, q.item);
            if (mine > 0 && mine < q.item.tiles) {               // the cuts within the item
                int first = -1, n = 0;
                for (int i = (int)(q.at * sharers / line_end); i < sharers; ++i) {
                    const long long t = cut_at(i);
                    if (t >= q.at + q.len) break;
                    if (t <= q.at) continue;
                    const int at = tile_at(t - q.at, q.item);
                    if (at == 0 || at == q.item.tiles) continue;
                    if (n++ == 0) first = i;
                }
                if (first == (int)blockIdx.x) {
                    a = make_int4(q.item.first + q.item.node0, q.item.nodes, q.item.kvh, n + 1);
                    d.x = q.item.pair;
                }
            }
        }
        cut.items[2 * blockIdx.x] = a;
        cut.items[2 * blockIdx.x + 1] = d;
    }
    // every role goes over the block's items alike; f returns false to give up
    auto for_items = [&](auto f) {
        for (long long t = begin; t < end;) {
            Place q = place_of(t);
            if (t == begin) q.item.from = tile_at(t - q.at, q.item);
            if (q.at + q.len > end) q.item.to = tile_at(end - q.at, q.item);
            t = q.at + q.len;
            if (q.item.from < q.item.to && !f(q.item)) return;
        }
    };
    auto wait = [&](unsigned long long& bar, unsigned parity, int code) { return mbar_wait(smem_u32(&bar), parity & 1, abort_flag, err, code, limit); };

    if (warp == 0) {
        if (lane == 0) {
            // ---- keys and values
            unsigned kc = 0;                                     // tiles of the block so far
            unsigned issued_k = 0, issued_v = 0;
            for_items([&](const Item& it) {
                const int* table = b.block_table + (size_t)it.seg * b.table_width;
                for (int i = it.from; i < it.to; ++i, ++kc) {
                    const int j0 = it.k_begin + i * BN, s = kc % ST;
                    int page = table[j0 / c.page_size];
                    if (page < 0 || page >= c.n_pages) page = 0;           // (no page: nothing there is visible to a row)
                    const int y = (page * nkv + it.kvh) * c.page_size + j0 % c.page_size;
                    if (!wait(bars.k_empty[s], kc / ST + 1, 1)) return false;
                    mbar_expect_tx(smem_u32(&bars.k_full[s]), KT_BYTES);
#pragma unroll
                    for (int kb = 0; kb < NKB; ++kb) tma_load_2d(smem_u32(k_s + s * KT_BYTES + kb * BN * 128), &map_k, kb * 64, y, smem_u32(&bars.k_full[s]));
                    ++issued_k;
                    if (!wait(bars.v_empty[s], kc / ST + 1, 1)) return false;
                    mbar_expect_tx(smem_u32(&bars.v_full[s]), KT_BYTES);
#pragma unroll
                    for (int kb = 0; kb < NKB; ++kb) tma_load_2d(smem_u32(v_s + s * KT_BYTES + kb * BN * 128), &map_v, kb * 64, y, smem_u32(&bars.v_full[s]));
                    ++issued_v;
                }
                return true;
            });
            // the last releases must have arrived, or (where the block gives up) the copies in flight have landed, before it leaves
            for (unsigned j = kc > ST ? kc - ST : 0; j < kc && !*abort_flag; ++j)
                if (!wait(bars.k_empty[j % ST], j / ST, 1) || !wait(bars.v_empty[j % ST], j / ST, 1)) break;
            if (*abort_flag) {
                for (unsigned j = issued_k > ST ? issued_k - ST : 0; j < issued_k; ++j) mbar_drain(smem_u32(&bars.k_full[j % ST]), (j / ST) & 1, limit);
                for (unsigned j = issued_v > ST ? issued_v - ST : 0; j < issued_v; ++j) mbar_drain(smem_u32(&bars.v_full[j % ST]), (j / ST) & 1, limit);
            }
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
            unsigned n_items = 0, kp = 0, vp = 0;                // items; key and value tiles of the block released so far
            unsigned scored = 0, added = 0;                      // own tiles whose scores, whose products with the values are issued
            for_items([&](const Item& it) {
                const int n = it.to - it.from, step = it.pair ? 1 : 2, first = it.pair ? 0 : g, own = n > first ? (n - first + step - 1) / step : 0;
                const unsigned base = kp;
                unsigned char* q_g = q_s + (it.pair ? g : 0) * Q_BYTES;
                // a tile of the other half's: wait until it has landed (so that the halves drift apart by no more than the ring) and hand it back
                auto pass = [&](unsigned long long* full, unsigned long long* empty, unsigned& at, unsigned to) {
                    for (; at < to; ++at) {
                        if (!wait(full[at % ST], at / ST, 2)) return false;
                        mbar_arrive(smem_u32(&empty[at % ST]));
                    }
                    return true;
                };
                auto issue_scores = [&](int li) {
                    if (!pass(bars.k_full, bars.k_empty, kp, base + first + li * step)) return false;
                    const int s = kp % ST, sb = scored & 1;
                    if (!wait(bars.k_full[s], kp / ST, 2)) return false;
                    // P of two tiles before lay where the scores go; the product issued last is waited for (by parity only that can be)
                    if (added > 0 && !wait(gb.pv_done, added - 1, 2)) return false;
                    fence_after();
                    const unsigned qa = smem_u32(q_g), ka = smem_u32(k_s + s * KT_BYTES);
#pragma unroll
                    for (int ks = 0; ks < HD / 16; ++ks)
                        mma(tmem_g + sb * BN, smem_desc_k_major(qa + (ks / 4) * BM * 128 + (ks % 4) * 32),
                            smem_desc_k_major(ka + (ks / 4) * BN * 128 + (ks % 4) * 32), idesc_s, ks > 0 ? 1u : 0u);
                    commit(smem_u32(&gb.s_full[sb]));
                    commit(smem_u32(&bars.k_empty[s]));
                    if (li == own - 1) commit(smem_u32(&bars.q_empty));
                    ++kp;
                    ++scored;
                    return true;
                };
                if (!wait(bars.q_full, n_items, 2)) return false;
                if (own == 0) mbar_arrive(smem_u32(&bars.q_empty));
                if (own > 0 && !issue_scores(0)) return false;
                if (own > 1 && !issue_scores(1)) return false;
                for (int li = 0; li < own; ++li) {
                    if (!pass(bars.v_full, bars.v_empty, vp, base + first + li * step)) return false;
                    const int s = vp % ST;
                    if (!wait(gb.p_ready, added, 2) || !wait(bars.v_full[s], vp / ST, 2)) return false;
                    fence_after();
                    const unsigned va = smem_u32(v_s + s * KT_BYTES);
#pragma unroll
                    for (int ks = 0; ks < BN / 16; ++ks)
                        mma_a_tmem(tmem_g + 2 * BN, tmem_g + (added & 1) * BN + ks * 8, smem_desc(va + ks * 16 * 128, BN * 128, 1024), idesc_pv,
                                   (li > 0 || ks > 0) ? 1u : 0u);
                    commit(smem_u32(&gb.pv_done));
                    commit(smem_u32(&bars.v_empty[s]));
                    ++vp;
                    ++added;
                    if (li + 2 < own && !issue_scores(li + 2)) return false;
                }
                ++n_items;
                return pass(bars.k_full, bars.k_empty, kp, base + n) && pass(bars.v_full, bars.v_empty, vp, base + n);
            });
        }
    } else {
        // ---- softmax: one thread a row; warp w may read tensor-memory lanes [32 (w % 4), + 32)
        const int g = (warp - 4) >> 2, quarter = warp & 3, r = quarter * 32 + lane;
        HalfBarriers& gb = bars.g[g];
        const unsigned lane_base = tmem + g * GROUP_COLS + ((unsigned)(quarter * 32) << 16);
        const float scale = p.softmax_scale * LOG2E;
        // cap and slope in units of the raw scores (see the prompts' kernel)
        const float cap_raw = CAP ? p.score_softcap / p.softmax_scale : 0.f, inv_cap_raw = CAP ? p.softmax_scale / p.score_softcap : 0.f;
        const float cap_arg = CAP ? 2.f * LOG2E * p.softmax_scale / p.score_softcap : 0.f;
        const bool biased = p.head_slopes != nullptr;
        unsigned tile0 = 0, seen = 0, singles = 0, turns = 0;    // tiles of the block before this item; own tiles so far; singles, a pair's tiles so far
        auto all_wait = [&](unsigned long long& bar, unsigned parity) { return (bool)__all_sync(0xffffffffu, wait(bar, parity, 3)); };
        for_items([&](const Item& it) {
            const int n = it.to - it.from, step = it.pair ? 1 : 2, first = it.pair ? 0 : g, own = n > first ? (n - first + step - 1) / step : 0;
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
                        const unsigned kt = tile0 + i;
                        if (!all_wait(bars.v_full[kt % ST], kt / ST)) return false;
                        unsigned char* v_t = v_s + (kt % ST) * KT_BYTES;
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
                if (CAP) {
                    // cap tanh(s scale / cap): the series where every score of the warp's rows is small against the cap, else by 2^x
                    float big[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int e = 0; e < BN; ++e) big[e & 3] = fmaxf(big[e & 3], fabsf(s[e]));
                    if (__all_sync(0xffffffffu, fmaxf(fmaxf(big[0], big[1]), fmaxf(big[2], big[3])) <= CAP_SERIES * cap_raw)) {
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
                if (!open) {
                    // 64 bits of what this row sees: settled tokens from its window's end on, then nodes
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
                    if (!row_ok) vis = 0;
#pragma unroll
                    for (int e = 0; e < BN; ++e) s[e] = ((e < 32 ? (unsigned)vis : (unsigned)(vis >> 32)) >> (e & 31) & 1u) ? s[e] : -INFINITY;
                }
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
                auto weights = [&](auto mixed) {
#pragma unroll
                    for (int e = 0; e < BN; e += 2) {
                        if (e == BN * 3 / 4) {
                            __syncwarp();
                            if (it.pair && lane == 0) mbar_arrive(smem_u32(&gb.exp_done));
                        }
                        const f2 y = fma2(pack2(s[e], s[e + 1]), scale2, neg_m2);
                        float a, bb;
                        // three of sixteen pairs on the multiply-add units (not where a masked key must get 0)
                        if (decltype(mixed)::value && ((e / 2) % 16 == 3 || (e / 2) % 16 == 8 || (e / 2) % 16 == 13)) {
                            ex2_pair(y, a, bb);
                        } else {
                            unpack2(y, a, bb);
                            a = ex2(a);
                            bb = ex2(bb);
                        }
                        sum2[(e >> 1) & 3] = add2(sum2[(e >> 1) & 3], pack2(a, bb));
                        packed[e / 2] = pack_bf16(a, bb);
                    }
                };
                if (open) weights(Flag<true>{}); else weights(Flag<false>{});
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
                    if (part) __stcg((float2*)(slot + 2 * HD * BM) + g * BM + r, make_float2(m_ref, l));
                }
                turns += n;
            } else {
                // the halves' states and outputs are added up: each half takes half of the head, and reads the other's out of tensor memory
                state_s[g][r] = make_float2(m_ref, l);
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
                    if (part && g == 0) __stcg((float2*)(slot + 2 * HD * BM) + r, make_float2(m, sum));
                }
                fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&bars.state_read));
                if (!all_wait(bars.state_read, singles)) return false;       // before either output is written again
                ++singles;
            }
            tile0 += n;
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

// Adds up the parts of the items that were cut, in the order of the keys.  grid (blocks, head_dim / JOIN_COLS), a thread a row; part 0 of an item
// is the last of the block before its first cut, part k the first of the block behind its cut k.
constexpr int JOIN_COLS = 16;
__global__ void __launch_bounds__(2 * BM) attn_tree_tc_join_kernel(const AttentionParams p, const TreeCut cut, int nkv, int tpt, int hd) {
    pdl_wait();
    pdl_launch_dependents();
    const int4 item = __ldcg(cut.items + 2 * blockIdx.x);
    if (item.w < 2) return;
    const int G = p.num_heads / nkv, g = threadIdx.x / BM, r = threadIdx.x % BM, c0 = blockIdx.y * JOIN_COLS;
    if (r >= min(tpt, item.y - g * tpt) * G) return;
    const int tok = item.x + g * tpt + r / G, head = item.z * G + r % G;
    auto slot = [&](int k) { return cut.partial + (2 * (size_t)blockIdx.x + 2 * k - (k ? 2 : 1)) * slot_floats(hd); };
    float m = -INFINITY, l = 0.f, o[JOIN_COLS];
#pragma unroll
    for (int e = 0; e < JOIN_COLS; ++e) o[e] = 0.f;
    constexpr int N = 4;                                         // parts whose loads are asked for together
    for (int k0 = 0; k0 < item.w; k0 += N) {
        float2 ml[N];
        float v[N][JOIN_COLS];
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const float* from = slot(min(k0 + k, item.w - 1));
            ml[k] = __ldcg((const float2*)(from + 2 * hd * BM) + threadIdx.x);
#pragma unroll
            for (int e = 0; e < JOIN_COLS; ++e) v[k][e] = __ldcg(from + (size_t)(g * hd + c0 + e) * BM + r);
        }
        float top = m;
#pragma unroll
        for (int k = 0; k < N; ++k) {
            if (k0 + k >= item.w) ml[k].x = -INFINITY;
            top = fmaxf(top, ml[k].x);
        }
        const float keep = m == -INFINITY ? 0.f : exp2f(m - top);
        m = top;
        l *= keep;
#pragma unroll
        for (int e = 0; e < JOIN_COLS; ++e) o[e] *= keep;
#pragma unroll
        for (int k = 0; k < N; ++k) {
            if (ml[k].x == -INFINITY) continue;                  // (a part without a key of this row)
            const float w = exp2f(ml[k].x - m);
            l = fmaf(w, ml[k].y, l);
#pragma unroll
            for (int e = 0; e < JOIN_COLS; ++e) o[e] = fmaf(w, v[k][e], o[e]);
        }
    }
    const float inv = row_scale_of(p, tok, head, m, l);
    __nv_bfloat16* dst = (__nv_bfloat16*)p.out + out_row_of(p, tok, head) * hd + c0;
#pragma unroll
    for (int e = 0; e < JOIN_COLS; e += 8)
        *(uint4*)(dst + e) = make_uint4(pack_bf16(o[e] * inv, o[e + 1] * inv), pack_bf16(o[e + 2] * inv, o[e + 3] * inv),
                                        pack_bf16(o[e + 4] * inv, o[e + 5] * inv), pack_bf16(o[e + 6] * inv, o[e + 7] * inv));
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
    const size_t smem = (2 * (size_t)NKB * BM + 2 * stages(NKB) * (size_t)NKB * BN) * 128 + (size_t)(x.n_segments + 1) * 8;
    auto k = p.score_softcap > 0.f ? attn_tree_tc_kernel<NKB, true> : attn_tree_tc_kernel<NKB, false>;
    if (cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess) return SPITE_LAUNCH_FAILED;
    SPITE_LAUNCH(k, n_sm, THREADS, smem, st, mq, mk, mv, p, b, c, x, tpt, box_tokens, cut, s_waits);
    SPITE_LAUNCH(attn_tree_tc_join_kernel, dim3(n_sm, hd / JOIN_COLS), 2 * BM, 0, st, p, cut, nkv, tpt, hd);
    return spite_launch_status();
}

}  // namespace

// `n_sm`: number of multiprocessors (a block each).  `scratch`: n_sm * (4 * (head_dim + 2) * 128 + 8) floats.
SPITE_API int spite_tree_attention_tc(const AttentionParams* p, const StepTokens* b, const PagedCache* c, const TreeStep* x, int n_sm, float* scratch,
                                      long long n_floats, void* stream) {
    if (!p || !b || !c || !x || !p->q || !p->out || !c->kv || !b->positions || !b->block_table || !x->cu_seqlens || !x->ancestors || !scratch || n_sm < 1)
        return SPITE_BAD_ARG;
    if (b->n_tokens < 0 || b->table_width < 1 || c->n_pages < 1 || c->page_size < 1 || x->n_segments < 1 || x->n_words < 1) return SPITE_BAD_ARG;
    if (p->num_heads < 1 || c->num_kv_heads < 1 || p->num_heads % c->num_kv_heads) return SPITE_BAD_ARG;
    if (p->window_kind < 0 || p->window_kind > 2 || (p->window_kind != SPITE_WINDOW_FULL && p->window_size < 1)) return SPITE_BAD_ARG;
    const int G = p->num_heads / c->num_kv_heads;
    if ((c->head_dim != 64 && c->head_dim != 128) || G > BM || c->page_size % BN || x->n_segments > MAX_SEGMENTS) return SPITE_UNSUPPORTED;
    if (p->distance_bias || c->key_scale || c->v_offset == 0) return SPITE_UNSUPPORTED;
    if ((long long)c->n_pages * c->num_kv_heads * c->page_size > 0x7fffffffll) return SPITE_UNSUPPORTED;       // TMA coordinates are int32
    if ((((uintptr_t)p->q | (uintptr_t)p->out | (uintptr_t)c->kv | (uintptr_t)scratch) & 15) || (c->v_offset & 7)) return SPITE_UNSUPPORTED;
    const long long slots = 2ll * n_sm * (long long)slot_floats(c->head_dim);
    if (slots + 8ll * n_sm > n_floats) return SPITE_BAD_ARG;
    if (b->n_tokens == 0) return SPITE_OK;
    const TreeCut cut{scratch, (int4*)(scratch + slots)};
    return c->head_dim == 64 ? launch<1>(*p, *b, *c, *x, cut, n_sm, (cudaStream_t)stream) : launch<2>(*p, *b, *c, *x, cut, n_sm, (cudaStream_t)stream);
}
