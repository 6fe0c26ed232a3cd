// Attention over trees of drafted tokens, any sizes and both types, in float32 (the fifth-generation tensor cores take bfloat16 with heads of 64
// and 128 elements: attention_tree_tc.cu).
//
// A block of eight warps serves up to 32 rows, (node, query head of one kv group) pairs of consecutive nodes of one request, for one kv head
// and one share of the keys.  Keys and values come in tiles of 64 (32 with heads of more than 128 elements), as they are stored, by asynchronous
// copies: the values while the scores are made, the next tile's keys while the values are added up.  The products are made by mma.sync on numbers
// of 11 bits: a float32 is split into 11 bits, rounded, and the rest, and upper x upper, upper x rest and rest x upper are added up in float32,
// which leaves out 2^-22 of a product at most (rest x rest, and the rest's own rounding), less than float32 sums over a head round off;
// stored bfloat16 has no rest.  On the multiply-add units the reads of shared memory bound the kernel: 16 bytes a lane take four cycles whether
// lanes read the same or not, and 32 rows leave no room for tiles large enough to use a word often (one float32 request of 4 x 13 nodes, 2,047
// keys, 16 heads on 4 of 128: 66 us that way, 37 now, 34 of them this kernel).  What bounds it now is latency, of the few tiles a block works on and of
// finding them (tensor pipe 20 % busy, 0.50 instructions a cycle and scheduler).  The softmax is kept
// as a running maximum and sum; shares of the keys leave their unnormalised results, which a second kernel adds up in the order of the keys.  The rows
// of the cache that are no visible token's are read as zeros, so they may hold anything.
//
// NaN, infinities and numbers next to the largest cannot be split; and the products would carry a value that is not finite into rows that do not see
// it, 0 x NaN being NaN.  Where a warp meets such a number, the results that it goes into are made again one by one in float32, with a row's own
// keys alone; all others keep their bits.  Looking for them takes 2 to 4 % (8 requests of 16 nodes, 2,048 keys, 40 heads on 8 of 128: 273 us, 265 without).
//
// Score, mask and softmax: crates/spite-compute/src/flash_attn.rs:111-156, with the mask of attention_tree.cuh.
#include "attention_tree.cuh"

namespace {

constexpr int ROWS = 32;                 // of a block
constexpr int THREADS = 256;
constexpr int JOIN_THREADS = 128;
constexpr int P_STRIDE = ROWS + 8;       // of a key's weights: four keys x eight rows lie in different banks

// A number as the products take it: rounded to 11 bits, and what that leaves, rounded to 11 bits (the products take the upper bits).  NaN, infinity
// and what rounds up to infinity do not come through that: they make `odd` NaN, which stays zero otherwise.
struct Split { unsigned hi, lo; };
__device__ __forceinline__ Split split(float v) {
    const unsigned hi = (__float_as_uint(v) + 0x1000u) & 0xffffe000u;
    return Split{hi, __float_as_uint(v - __uint_as_float(hi)) + 0x1000u};
}
__device__ __forceinline__ Split split(float v, float& odd) {
    const Split s = split(v);
    odd = fmaf(v - __uint_as_float(s.hi), 0.f, odd);
    return s;
}
__device__ __forceinline__ bool splits(float v) { return fabsf(v) < 0x1.ffep127f; }
// A stored bfloat16 is its own upper bits, and comes through the products whatever it is.
__device__ __forceinline__ Split split(__nv_bfloat16 v, float&) { return Split{__float_as_uint(to_f32(v)), 0u}; }
// d += a b for 16 x 8 and 8 x 8 numbers; lane 4 g + c holds a's rows g, g + 8 of columns c, then of c + 4; b's column g of rows c, c + 4;
// d's rows g (two columns from 2 c on) and g + 8.
__device__ __forceinline__ void mma(float (&d)[4], const unsigned (&a)[4], const unsigned (&b)[2]) {
    asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}
// What a row weighs a key with that it does not see: zero, and by its sign apart from a weight that has become zero.
constexpr float UNSEEN = -0.f;
// A query's product with a key, and a row's sum over a column of the values that it sees (`weights` P_STRIDE apart, `column` `stride`), in float32, where
// a number among them cannot be split; where all can, what the products have `made`.
template <typename T> __device__ __noinline__ float product(const float* q, const T* k, int n, float made) {
    float sum = 0.f;
    bool all = true;
    for (int d = 0; d < n; ++d) {
        const float a = q[d], b = to_f32(k[d]);
        all &= splits(a) && splits(b);
        sum = fmaf(a, b, sum);
    }
    return all ? made : sum;
}
template <typename T> __device__ __noinline__ float seen_values(const float* weights, const T* column, int stride, int n, float made) {
    float sum = 0.f;
    bool all = true;
    for (int j = 0; j < n; ++j) {
        const float w = weights[j * P_STRIDE], v = to_f32(column[j * stride]);
        all &= splits(w) && splits(v);
        if (__float_as_uint(w) != __float_as_uint(UNSEEN)) sum = fmaf(w, v, sum);
    }
    return all ? made : sum;
}
// 16 bytes from global to shared memory, or zeros.
__device__ __forceinline__ void copy16(void* to, const void* from, bool there) {
    const unsigned dst = (unsigned)__cvta_generic_to_shared(to), bytes = there ? 16 : 0;
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst), "l"(from), "r"(bytes) : "memory");
}
__device__ __forceinline__ int padded_head(int hd) { return (hd + 3) & ~3; }
// A share's result of a row: its elements, padded to four, then maximum and sum.
__host__ __device__ constexpr int part_floats(int hd) { return ((hd + 3) & ~3) + 4; }

// Rows of the tiles in shared memory, for a head padded to eight elements: strides by which the lanes of a product read different banks.
__host__ __device__ constexpr int eighths(int hd) { return (hd + 7) & ~7; }
template <typename T> __host__ __device__ constexpr int key_stride(int hd8) { return hd8 + 16 / (int)sizeof(T); }
template <typename T> __host__ __device__ constexpr int value_stride(int hd8) { return sizeof(T) == 4 ? hd8 + (hd8 % 16 ? 0 : 8) : hd8 + 8; }
template <typename T, int BN> constexpr size_t smem_bytes(int hd8) {
    return (size_t)ROWS * (hd8 + 4) * 4 + (size_t)BN * P_STRIDE * 4 + (size_t)BN * (key_stride<T>(hd8) + value_stride<T>(hd8)) * sizeof(T);
}

// grid (chunks of nodes, kv heads x chunks of ROWS heads of a group, shares of the keys).  HD4: 128s of the head; ASYNC: rows are whole 16 bytes.
// partial [tokens, heads, shares, part_floats].
template <typename T, int HD4, bool ASYNC>
__global__ void __launch_bounds__(THREADS, 2) attn_tree_kernel(const AttentionParams p, const StepTokens b, const PagedCache c, const TreeStep x,
                                                            float* partial, const int nodes_per_block, const int n_splits, const int share_tiles) {
    constexpr int BN = 64 / HD4, KT = BN / 32;                // keys of a tile; eights of them of a warp
    constexpr bool REST = sizeof(T) == 4;                      // (bfloat16 has none)
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ long long key_row[2][BN];                       // of two tiles' keys, in elements; -1: no such key
    __shared__ int key_pos[2][BN], key_node[2][BN];            // position; number of the node or -1
    __shared__ float key_factor[2][BN];
    __shared__ float top_s[4][ROWS], l_s[4][ROWS];
    pdl_wait();
    pdl_launch_dependents();

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    // which request and which of its nodes: the blocks' numbers run through the requests, counted 32 at a time
    int seg = -1, first = 0, end = 0, node0 = 0;
    for (int s0 = 0, before = 0; s0 < x.n_segments; s0 += 32) {
        int a = 0, e = 0;
        if (s0 + lane < x.n_segments) {
            a = min(max(x.cu_seqlens[s0 + lane], 0), b.n_tokens);
            e = min(max(x.cu_seqlens[s0 + lane + 1], a), b.n_tokens);
        }
        const int mine = (e - a + nodes_per_block - 1) / nodes_per_block;
        int upto = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += u;
        }
        const int nth = (int)blockIdx.x - before;
        const unsigned holds = __ballot_sync(0xffffffffu, nth < upto);
        if (holds) {
            const int at = __ffs(holds) - 1;
            seg = s0 + at;
            first = __shfl_sync(0xffffffffu, a, at);
            end = __shfl_sync(0xffffffffu, e, at);
            node0 = (nth - __shfl_sync(0xffffffffu, upto - mine, at)) * nodes_per_block;
            break;
        }
        before += __shfl_sync(0xffffffffu, upto, 31);
    }
    if (seg < 0) return;                                       // (the caller counts a block or less too many a request)
    const int t0 = first + node0;
    const int hd = c.head_dim, hdp = padded_head(hd), hd8 = eighths(hd), q_stride = hd8 + 4, k_stride = key_stride<T>(hd8), v_stride = value_stride<T>(hd8);
    float* q_s = (float*)smem;                                 // [ROWS][q_stride]
    float* p_s = q_s + ROWS * q_stride;                        // [BN][P_STRIDE] weights
    T* k_s = (T*)(p_s + BN * P_STRIDE);                        // [BN][k_stride]
    T* v_s = k_s + BN * k_stride;                              // [BN][v_stride]
    const int nq = p.num_heads, nkv = c.num_kv_heads, G = nq / nkv, chunks = (G + ROWS - 1) / ROWS;
    const int kvh = blockIdx.y / chunks, h0 = blockIdx.y % chunks * ROWS, heads = min(ROWS, G - h0);
    const int nt = min(nodes_per_block, end - t0), n_rows = nt * heads;
    const int* table = b.block_table + (size_t)seg * b.table_width;
    const int len = b.positions[first];                        // settled tokens (the first node has no parent)
    const int places = (int)min((long long)len + node0 + nt, (long long)b.table_width * c.page_size);
    const int lo_any = window_lowest(p.window_kind, p.window_size, len);
    const int n_tiles = places > lo_any ? (places - lo_any + BN - 1) / BN : 0, split_no = blockIdx.z;
    // (shares of so many tiles, the last one of the rest: a short request has fewer of them, and their blocks leave at once)
    const int tile0 = min(n_tiles, split_no * share_tiles), tile1 = split_no == n_splits - 1 ? n_tiles : min(n_tiles, tile0 + share_tiles);
    if (tile0 == tile1 && n_splits > 1) {                      // nothing in this share: its rows' maximum says so
        for (int r = threadIdx.x; r < n_rows; r += THREADS)
            __stcg((float2*)(partial + (((size_t)(t0 + r / heads) * nq + kvh * G + h0 + r % heads) * n_splits + split_no) * part_floats(hd) + hdp),
                   make_float2(-INFINITY, 0.f));
        return;
    }

    // where a tile's keys lie: a thread a key, asked for a tile ahead and written down later
    struct Key { long long row; int at, node; float factor; };
    auto find = [&](int ti) {
        const int j = lo_any + ti * BN + (int)threadIdx.x, node = j - len;
        Key k{-1, j, node >= 0 ? node : -1, 1.f};
        if (j < places && (node < 0 || tree_node_is_real(x, first, node))) {
            const int page = table[j / c.page_size];
            if (page >= 0 && page < c.n_pages) {               // (a page that has gone back lies in front of every row's window)
                k.row = (((long long)page * nkv + kvh) * c.page_size + j % c.page_size) * hd;
                if (c.key_scale) k.factor = c.key_scale[k.row / hd];
                if (node >= 0) k.at = b.positions[first + node];
            }
        }
        return k;
    };
    auto note = [&](const Key& k, int slot) {
        key_row[slot][threadIdx.x] = k.row;
        key_pos[slot][threadIdx.x] = k.at;
        key_node[slot][threadIdx.x] = k.node;
        key_factor[slot][threadIdx.x] = k.factor;
    };
    // a warp a row: no division, and a row's 16-byte pieces side by side
    auto fetch = [&](T* to, int stride, const T* plane, int slot) {
        constexpr int E = ASYNC ? 16 / (int)sizeof(T) : 1;
#pragma unroll 4
        for (int r = warp; r < BN; r += THREADS / 32) {
            const long long row = key_row[slot][r];
            const T* from = plane + (row >= 0 ? row : 0);
            for (int d = lane * E; d < hd8; d += 32 * E) {
                if constexpr (ASYNC) copy16(to + r * stride + d, from + (d < hd ? d : 0), row >= 0 && d < hd);
                else to[r * stride + d] = row >= 0 && d < hd ? from[d] : from_f32<T>(0.f);
            }
        }
        if constexpr (ASYNC) asm volatile("cp.async.commit_group;\n" ::: "memory");
    };
    auto landed = [&](bool one_behind) {                       // the copies but the last asked for, or all
        if constexpr (ASYNC) {
            if (one_behind) asm volatile("cp.async.wait_group 1;\n" ::: "memory");
            else asm volatile("cp.async.wait_group 0;\n" ::: "memory");
        }
    };
    const T* keys = (const T*)c.kv;
    const T* values = keys + c.v_offset;
    if (tile0 < tile1 && threadIdx.x < BN) note(find(tile0), 0);
    bool q_odd = false;                                        // some number of q cannot be split
#pragma unroll
    for (int i = 0; i < ROWS / 8; ++i) {
        const int r = warp + 8 * i;
        const T* q = (const T*)p.q + ((size_t)(t0 + (r < n_rows ? r / heads : 0)) * nq + kvh * G + h0 + (r < n_rows ? r % heads : 0)) * hd;
        for (int d = lane; d < hd8; d += 32) {
            const float v = r < n_rows && d < hd ? to_f32(q[d]) : 0.f;
            q_s[r * q_stride + d] = v;
            q_odd |= !splits(v);
        }
    }
    q_odd = __syncthreads_or(q_odd);
    if (tile0 < tile1) fetch(k_s, k_stride, keys, 0);

    // Warps 2 (halves of the rows) x 4 (quarters of the tile's keys, then of the head); a thread's rows are g and g + 8 of the half.
    const int half = warp & 1, quarter = warp >> 1, g = lane >> 2, cc = lane & 3;
    const bool works = 16 * half < n_rows;
    int tok[2], head[2], pos[2], lo[2];
    bool row_ok[2];
    float m[2], l[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int r = 16 * half + g + 8 * i;
        row_ok[i] = r < n_rows;
        tok[i] = t0 + (row_ok[i] ? r / heads : 0);
        head[i] = kvh * G + h0 + (row_ok[i] ? r % heads : 0);
        pos[i] = b.positions[tok[i]];
        lo[i] = window_lowest(p.window_kind, p.window_size, pos[i]);
        m[i] = -INFINITY;
        l[i] = 0.f;
    }
    float acc[4 * HD4][4];                                     // eights of the warp's 32 HD4 elements
#pragma unroll
    for (int e = 0; e < 4 * HD4; ++e) acc[e][0] = acc[e][1] = acc[e][2] = acc[e][3] = 0.f;
    const int lo_all = window_lowest(p.window_kind, p.window_size, len + (x.cu_seqlens[seg + 1] - first) - 1);       // (no node is deeper)
    const bool plain = !c.key_scale && !p.distance_bias && !p.head_slopes && !(p.score_softcap > 0.f);

    for (int ti = tile0; ti < tile1; ++ti) {
        const int slot = (ti - tile0) & 1;
        const bool more = ti + 1 < tile1, finds = more && threadIdx.x < BN;
        fetch(v_s, v_stride, values, slot);
        Key ahead{};
        if (finds) ahead = find(ti + 1);
        landed(true);
        __syncthreads();                                       // the keys are here
        float s[KT][4];                                        // [eight of keys][row g: two keys, row g + 8: two keys]
        unsigned vis = 0;                                      // bit 4 k + e: s[k][e] is a visible key's
        float odd = 0.f;
        if (works) {
#pragma unroll
            for (int k = 0; k < KT; ++k) s[k][0] = s[k][1] = s[k][2] = s[k][3] = 0.f;
            const float* qr = q_s + (16 * half + g) * q_stride + cc;
            const T* kr = k_s + (quarter * 8 * KT + g) * k_stride + cc;
            // (The products' own sums are cut off, not rounded, at every addition: they run over 32 elements and are then added up rounded.)
            for (int d0 = 0; d0 < hd8; d0 += 32) {
                float part[KT][4];
#pragma unroll
                for (int k = 0; k < KT; ++k) part[k][0] = part[k][1] = part[k][2] = part[k][3] = 0.f;
#pragma unroll
                for (int d = d0; d < d0 + 32; d += 8) {
                    if (d >= hd8) break;
                    unsigned hi[4], rest[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const Split v = split(qr[(e & 1) * 8 * q_stride + d + (e >> 1) * 4]);
                        hi[e] = v.hi;
                        rest[e] = v.lo;
                    }
#pragma unroll
                    for (int k = 0; k < KT; ++k) {
                        const Split u = split(kr[8 * k * k_stride + d], odd), w = split(kr[8 * k * k_stride + d + 4], odd);
                        const unsigned b_hi[2] = {u.hi, w.hi}, b_rest[2] = {u.lo, w.lo};
                        if (REST) {
                            mma(part[k], rest, b_hi);
                            mma(part[k], hi, b_rest);
                        }
                        mma(part[k], hi, b_hi);
                    }
                }
#pragma unroll
                for (int k = 0; k < KT; ++k)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[k][e] += part[k][e];
            }
            if (!REST) {                                       // (what bfloat16 keys and queries make that is not finite)
#pragma unroll
                for (int k = 0; k < KT; ++k)
#pragma unroll
                    for (int e = 0; e < 4; ++e) odd = fmaf(s[k][e], 0.f, odd);
            }
            if (__any_sync(0xffffffffu, odd != 0.f) || q_odd) {        // numbers that cannot be split: as the formula has it
#pragma unroll
                for (int k = 0; k < KT; ++k)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        s[k][e] = product(q_s + (16 * half + g + 8 * (e >> 1)) * q_stride, k_s + (quarter * 8 * KT + 8 * k + 2 * cc + (e & 1)) * k_stride, hd, s[k][e]);
            }
            const int j0 = lo_any + ti * BN;
            if (plain && j0 >= lo_all && j0 + BN <= len) {     // settled keys that every row sees
                vis = (row_ok[0] ? 0x33333333u : 0u) | (row_ok[1] ? 0xccccccccu : 0u);
#pragma unroll
                for (int k = 0; k < KT; ++k)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[k][e] = row_ok[e >> 1] ? s[k][e] * p.softmax_scale : -INFINITY;
            } else {
                // scale, cap, bias and mask
#pragma unroll
                for (int k = 0; k < KT; ++k)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int key = quarter * 8 * KT + 8 * k + 2 * cc + (e & 1), i = e >> 1, kp = key_pos[slot][key], kn = key_node[slot][key];
                        bool v = row_ok[i] && key_row[slot][key] >= 0 && kp >= lo[i];
                        if (v && kn >= 0)                      // (a node sees no node behind itself)
                            v = kn <= tok[i] - first && (x.ancestors[(size_t)tok[i] * x.n_words + kn / 32] >> (kn % 32) & 1u);
                        float score = capped(p, s[k][e] * (key_factor[slot][key] * p.softmax_scale));
                        if (p.head_slopes) score -= slope_of(p, head[i]) * (float)(pos[i] - kp);
                        if (p.distance_bias) score += number_at(p, distance_row_of(p, head[i]), pos[i] - kp);
                        s[k][e] = v ? score : -INFINITY;
                        vis |= (unsigned)v << (4 * k + e);
                    }
            }
            // the rows' largest: of a thread's keys, of the four lanes', and below of the four warps'
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                float top = fmaxf(s[0][2 * i], s[0][2 * i + 1]);
#pragma unroll
                for (int k = 1; k < KT; ++k) top = fmaxf(top, fmaxf(s[k][2 * i], s[k][2 * i + 1]));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                if (cc == 0) top_s[quarter][16 * half + g + 8 * i] = top;
            }
        }
        if (finds) note(ahead, slot ^ 1);
        __syncthreads();                                       // the keys have been read, the largest are known
        if (more) fetch(k_s, k_stride, keys, slot ^ 1);
        float shrink[2] = {1.f, 1.f};
        if (works) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int r = 16 * half + g + 8 * i;
                const float m_new = fmaxf(fmaxf(m[i], fmaxf(top_s[0][r], top_s[1][r])), fmaxf(top_s[2][r], top_s[3][r]));
                if (m_new != -INFINITY) shrink[i] = expf(m[i] - m_new);
                const float from = m_new == -INFINITY ? 0.f : m_new;           // (scores of minus infinity weigh nothing)
                m[i] = m_new;
                l[i] *= shrink[i];
#pragma unroll
                for (int k = 0; k < KT; ++k)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const float w = vis >> (4 * k + 2 * i + e) & 1u ? expf(s[k][2 * i + e] - from) : UNSEEN;
                        l[i] += w;                             // (of this thread's keys; the sums meet in the end)
                        p_s[(quarter * 8 * KT + 8 * k + 2 * cc + e) * P_STRIDE + r] = w;
                    }
            }
        }
        landed(more);
        __syncthreads();                                       // weights and values are here
        if (works) {
#pragma unroll
            for (int e = 0; e < 4 * HD4; ++e) { acc[e][0] *= shrink[0]; acc[e][1] *= shrink[0]; acc[e][2] *= shrink[1]; acc[e][3] *= shrink[1]; }
            odd = 0.f;
            float part[4 * HD4][4];
#pragma unroll
            for (int e = 0; e < 4 * HD4; ++e) part[e][0] = part[e][1] = part[e][2] = part[e][3] = 0.f;
            const float* wr = p_s + cc * P_STRIDE + 16 * half + g;
            const T* vr = v_s + cc * v_stride + quarter * 32 * HD4 + g;
#pragma unroll 2
            for (int j = 0; j < BN; j += 8) {
                unsigned hi[4], rest[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const Split v = split(wr[(j + (e >> 1) * 4) * P_STRIDE + (e & 1) * 8], odd);
                    hi[e] = v.hi;
                    rest[e] = v.lo;
                }
#pragma unroll
                for (int e = 0; e < 4 * HD4; ++e) {
                    if (quarter * 32 * HD4 + 8 * e >= hd8) continue;                   // (the head ends before; the same for the warp)
                    const Split u = split(vr[j * v_stride + 8 * e], odd), w = split(vr[(j + 4) * v_stride + 8 * e], odd);
                    const unsigned b_hi[2] = {u.hi, w.hi}, b_rest[2] = {u.lo, w.lo};
                    mma(part[e], rest, b_hi);
                    if (REST) mma(part[e], hi, b_rest);
                    mma(part[e], hi, b_hi);
                }
            }
            if (!REST) {
#pragma unroll
                for (int e = 0; e < 4 * HD4; ++e)
#pragma unroll
                    for (int k = 0; k < 4; ++k) odd = fmaf(part[e][k], 0.f, odd);
            }
            if (__any_sync(0xffffffffu, odd != 0.f)) {
#pragma unroll
                for (int e = 0; e < 4 * HD4; ++e) {
                    if (quarter * 32 * HD4 + 8 * e >= hd8) continue;
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        part[e][k] = seen_values(p_s + 16 * half + g + 8 * (k >> 1), v_s + quarter * 32 * HD4 + 8 * e + 2 * cc + (k & 1), v_stride, BN, part[e][k]);
                }
            }
#pragma unroll
            for (int e = 0; e < 4 * HD4; ++e)
#pragma unroll
                for (int k = 0; k < 4; ++k) acc[e][k] += part[e][k];
        }
        __syncthreads();                                       // values and weights have been read
    }
    if (works) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int r = 16 * half + g + 8 * i;
            l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
            l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
            if (cc == 0) l_s[quarter][r] = l[i];
        }
    }
    __syncthreads();
    if (!works) return;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        if (!row_ok[i]) continue;
        const int r = 16 * half + g + 8 * i, t = tok[i], h = head[i];
        float row_m = m[i], row_l = (l_s[0][r] + l_s[1][r]) + (l_s[2][r] + l_s[3][r]), scale = 1.f;
        if (n_splits == 1) {
            const float fold = tree_fold_sink(p, h, row_m, row_l);
            scale = fold * gate_of(p, t, h) / tree_divisor(row_l);
        }
        T* out = (T*)p.out + out_row_of(p, t, h) * hd;
        float* part = partial + (((size_t)t * nq + h) * n_splits + split_no) * part_floats(hd);
#pragma unroll
        for (int e = 0; e < 4 * HD4; ++e) {
            const int d = quarter * 32 * HD4 + 8 * e + 2 * cc;
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                if (d + k >= hd) continue;
                if (n_splits == 1) out[d + k] = from_f32<T>(acc[e][2 * i + k] * scale); else __stcg(part + d + k, acc[e][2 * i + k]);
            }
        }
        if (n_splits > 1 && quarter == 0 && cc == 0) __stcg((float2*)(part + hdp), tree_state(row_m, row_l));
    }
}

// Adds the shares of a row up, in the order of the keys.  grid (tokens, heads / 4), a warp a row; the loads of eight shares are asked for at once.
template <typename T, int HD4>
__global__ void __launch_bounds__(JOIN_THREADS) attn_tree_join_kernel(const AttentionParams p, const TreeStep x, const float* partial, int hd, int n_splits) {
    pdl_wait();
    pdl_launch_dependents();
    const int t = blockIdx.x, head = blockIdx.y * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31, hdp = padded_head(hd);
    if (head >= p.num_heads || t >= x.cu_seqlens[x.n_segments]) return;     // (rows behind the last request stay as they are)
    const float* part = partial + ((size_t)t * p.num_heads + head) * n_splits * part_floats(hd);
    float2 ml = make_float2(-INFINITY, 0.f);
    if (lane < n_splits) ml = __ldcg((const float2*)(part + lane * part_floats(hd) + hdp));      // (at most 32 shares)
    constexpr int N = 8;
    float4 acc[HD4], v[N][HD4];
#pragma unroll
    for (int e = 0; e < HD4; ++e) acc[e] = make_float4(0.f, 0.f, 0.f, 0.f);
    auto ask = [&](int s0) {
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const float share_m = __shfl_sync(0xffffffffu, ml.x, (s0 + k) & 31);
            const bool there = s0 + k < n_splits && share_m > -INFINITY;       // (a share without a key of this row has left nothing)
#pragma unroll
            for (int e = 0; e < HD4; ++e) {
                const int d = 4 * (lane + 32 * e);
                v[k][e] = there && d < hdp ? __ldcg((const float4*)(part + (s0 + k) * part_floats(hd) + d)) : make_float4(0.f, 0.f, 0.f, 0.f);
            }
        }
    };
    ask(0);
    const float m = warp_max(ml.x);
    const float my_w = ml.x == -INFINITY ? 0.f : expf(ml.x - m);
    float l = warp_sum(ml.y * my_w);
    const float shrink = tree_fold_sink(p, head, m, l);
    const float scale = shrink * gate_of(p, t, head) / tree_divisor(l);
    for (int s0 = 0; s0 < n_splits; s0 += N) {
        if (s0) ask(s0);
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const float w = __shfl_sync(0xffffffffu, my_w, (s0 + k) & 31);
            if (s0 + k >= n_splits) continue;
#pragma unroll
            for (int e = 0; e < HD4; ++e) {
                acc[e].x = fmaf(w, v[k][e].x, acc[e].x); acc[e].y = fmaf(w, v[k][e].y, acc[e].y);
                acc[e].z = fmaf(w, v[k][e].z, acc[e].z); acc[e].w = fmaf(w, v[k][e].w, acc[e].w);
            }
        }
    }
    T* out = (T*)p.out + out_row_of(p, t, head) * hd;
#pragma unroll
    for (int e = 0; e < HD4; ++e) {
        const float o[4] = {acc[e].x, acc[e].y, acc[e].z, acc[e].w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int d = 4 * (lane + 32 * e) + k;
            if (d < hd) out[d] = from_f32<T>(o[k] * scale);
        }
    }
}

template <typename T, int HD4>
int launch(const TreeCall& a, float* partial, int n_splits, int share_keys, cudaStream_t st) {
    const AttentionParams& p = a.p;
    const PagedCache& c = a.c;
    const int hd = c.head_dim, G = p.num_heads / c.num_kv_heads, chunks = (G + ROWS - 1) / ROWS;
    const int nodes = G >= ROWS ? 1 : ROWS / G;
    const size_t smem = smem_bytes<T, 64 / HD4>(eighths(hd));
    const bool async = hd * sizeof(T) % 16 == 0 && !(((uintptr_t)c.kv | (uintptr_t)(c.v_offset * sizeof(T))) & 15);
    if ((long long)c.num_kv_heads * chunks > 65535) return SPITE_UNSUPPORTED;
    const dim3 grid(a.b.n_tokens / nodes + a.x.n_segments, c.num_kv_heads * chunks, n_splits);       // (no request has a chunk more than fill it)
    auto k = async ? attn_tree_kernel<T, HD4, true> : attn_tree_kernel<T, HD4, false>;
    static std::atomic<unsigned long long> done[2];
    if (!allow_shared(k, smem_bytes<T, 64 / HD4>(128 * HD4), done[async])) return SPITE_LAUNCH_FAILED;
    SPITE_LAUNCH(k, grid, THREADS, smem, st, p, a.b, c, a.x, partial, nodes, n_splits, (share_keys + 64 / HD4 - 1) / (64 / HD4));
    if (n_splits > 1)
        SPITE_LAUNCH((attn_tree_join_kernel<T, HD4>), dim3(a.b.n_tokens, (p.num_heads + 3) / 4), JOIN_THREADS, 0, st, p, a.x, (const float*)partial, hd, n_splits);
    return spite_launch_status();
}

}  // namespace

// `n_splits` shares of `share_keys` keys, the last one of the rest.  `partial` (16-byte aligned): tokens * heads * n_splits * (head_dim rounded up to four, + 4) floats where n_splits (1..32) > 1.
SPITE_API int spite_tree_attention(int dtype, const TreeCall* call, float* partial, long long n_partial, int n_splits, int share_keys, void* stream) {
    if (!call || !tree_call_ok(*call)) return SPITE_BAD_ARG;
    const AttentionParams& p = call->p;
    const int hd = call->c.head_dim;
    if (n_splits < 1 || n_splits > 32 || share_keys < 1) return SPITE_BAD_ARG;
    if (n_splits > 1 && (!partial || ((uintptr_t)partial & 15) || n_partial < (long long)call->b.n_tokens * p.num_heads * n_splits * part_floats(hd)))
        return SPITE_BAD_ARG;
    if (hd > 256 || p.num_heads > 4 * 65535) return SPITE_UNSUPPORTED;
    if (call->b.n_tokens == 0) return SPITE_OK;
    cudaStream_t st = (cudaStream_t)stream;
    if (dtype == SPITE_DT_F32) return hd <= 128 ? launch<float, 1>(*call, partial, n_splits, share_keys, st) : launch<float, 2>(*call, partial, n_splits, share_keys, st);
    if (dtype == SPITE_DT_BF16) return hd <= 128 ? launch<__nv_bfloat16, 1>(*call, partial, n_splits, share_keys, st) : launch<__nv_bfloat16, 2>(*call, partial, n_splits, share_keys, st);
    return SPITE_BAD_ARG;
}
