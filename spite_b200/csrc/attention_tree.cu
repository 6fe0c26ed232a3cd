// Attention over trees of drafted tokens, any sizes and both types, on the multiply-add units (the tensor cores take bfloat16 with
// heads of 64 and 128 elements: attention_tree_tc.cu).  Float32 throughout.
//
// A block serves up to 16 rows, (node, query head of one kv group) pairs of consecutive nodes of one request, for one kv head and one
// share of the keys.  Keys and values come in tiles of 32 through shared memory as float32; warp w works on rows 4 w .. 4 w + 3, a
// lane on one key of the tile for the scores and on four neighbouring elements of the head for the values, so that every word it
// reads from shared memory serves four rows.  The softmax is kept as a running maximum and sum; shares of the keys leave
// their unnormalised results, which a second kernel adds up in the order of the keys.  A masked key adds nothing whatever its value
// row holds: its weight is zero and the product is not made.
//
// Score, mask and softmax: crates/spite-compute/src/flash_attn.rs:111-156, with the mask of attention_tree.cuh.
#include "attention_tree.cuh"

namespace {

constexpr int ROWS = 16;                 // of a block
constexpr int BN = 32;                   // keys of a tile
constexpr int THREADS = 128;

// Stored elements, four at a time where rows allow it.
template <typename T> __device__ __forceinline__ float4 load4(const T* p);
template <> __device__ __forceinline__ float4 load4<float>(const float* p) { return *(const float4*)p; }
template <> __device__ __forceinline__ float4 load4<__nv_bfloat16>(const __nv_bfloat16* p) {
    const uint2 w = *(const uint2*)p;
    const float2 a = __bfloat1622float2(*(const __nv_bfloat162*)&w.x), b = __bfloat1622float2(*(const __nv_bfloat162*)&w.y);
    return make_float4(a.x, a.y, b.x, b.y);
}

// grid (tokens, kv heads x chunks of 16 heads of a group, shares of the keys); the block of a token that is not the first of its
// chunk of nodes has nothing to do.  HD4: four-element groups of the head a lane works on (32 lanes), WIDE rows can be read four
// elements at a time.  partial [tokens, heads, shares, head_dim + 2].
template <typename T, int HD4, bool WIDE>
__global__ void __launch_bounds__(THREADS) attn_tree_kernel(const AttentionParams p, const StepTokens b, const PagedCache c, const TreeStep x,
                                                            float* partial, const int nodes_per_block, const int n_splits) {
    extern __shared__ __align__(16) float smem[];
    __shared__ long long key_row[BN];                          // of the tile's keys, in elements; -1: no such key
    __shared__ int key_pos[BN], key_node[BN];                  // position; number of the node or -1
    __shared__ float key_factor[BN];
    __shared__ __align__(16) float weight[ROWS][BN];
    pdl_wait();
    pdl_launch_dependents();

    const int hd = c.head_dim, hdp = (hd + 3) & ~3, stride = hdp + 4;       // a row of a tile; four floats on, so that lanes spread over the banks
    float* q_s = smem;                                         // [ROWS][hdp]
    float* k_s = q_s + ROWS * hdp;                             // [BN][stride]
    float* v_s = k_s + BN * stride;                            // [BN][stride]
    const int t0 = blockIdx.x, seg = b.seg_of_token[t0];
    if (seg < 0 || seg >= x.n_segments) return;
    const int first = x.cu_seqlens[seg], end = min(x.cu_seqlens[seg + 1], b.n_tokens), node0 = t0 - first;
    if (first < 0 || node0 < 0 || t0 >= end || node0 % nodes_per_block) return;
    const int nq = p.num_heads, nkv = c.num_kv_heads, G = nq / nkv, chunks = (G + ROWS - 1) / ROWS;
    const int kvh = blockIdx.y / chunks, h0 = blockIdx.y % chunks * ROWS, heads = min(ROWS, G - h0);
    const int nt = min(nodes_per_block, end - t0), n_rows = nt * heads;
    const int* table = b.block_table + (size_t)seg * b.table_width;
    const int len = b.positions[first];                        // settled tokens (the first node has no parent)
    const int places = min((long long)len + node0 + nt, (long long)b.table_width * c.page_size);
    const int lo_any = window_lowest(p.window_kind, p.window_size, len);
    const int n_tiles = places > lo_any ? (places - lo_any + BN - 1) / BN : 0, split = blockIdx.z;
    const int tile0 = (int)((long long)n_tiles * split / n_splits), tile1 = (int)((long long)n_tiles * (split + 1) / n_splits);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int i = threadIdx.x; i < ROWS * hdp; i += THREADS) {
        const int r = i / hdp, d = i % hdp;
        q_s[i] = r < n_rows && d < hd ? to_f32(((const T*)p.q)[((size_t)(t0 + r / heads) * nq + kvh * G + h0 + r % heads) * hd + d]) : 0.f;
    }
    int tok[4], head[4], pos[4], lo[4];
    float slope[4];
    const float* dist[4];
    bool row_ok[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = 4 * warp + i;
        row_ok[i] = r < n_rows;
        tok[i] = t0 + (row_ok[i] ? r / heads : 0);
        head[i] = kvh * G + h0 + (row_ok[i] ? r % heads : 0);
        pos[i] = b.positions[tok[i]];
        lo[i] = window_lowest(p.window_kind, p.window_size, pos[i]);
        slope[i] = slope_of(p, head[i]);
        dist[i] = distance_row_of(p, head[i]);
    }
    float m[4], l[4];
    float4 acc[4][HD4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        m[i] = -INFINITY;
        l[i] = 0.f;
#pragma unroll
        for (int e = 0; e < HD4; ++e) acc[i][e] = make_float4(0.f, 0.f, 0.f, 0.f);
    }

    for (int ti = tile0; ti < tile1; ++ti) {
        __syncthreads();                                       // the tile before has been read (and q is there)
        if (threadIdx.x < BN) {
            const int j = lo_any + ti * BN + threadIdx.x, node = j - len;
            long long row = -1;
            int at = j;
            float factor = 1.f;
            if (j < places && (node < 0 || tree_node_is_real(x, first, node))) {
                const int page = table[j / c.page_size];
                if (page >= 0 && page < c.n_pages) {           // (a page that has gone back lies in front of every row's window)
                    row = (((long long)page * nkv + kvh) * c.page_size + j % c.page_size) * hd;
                    if (c.key_scale) factor = c.key_scale[row / hd];
                    if (node >= 0) at = b.positions[first + node];
                }
            }
            key_row[threadIdx.x] = row;
            key_pos[threadIdx.x] = at;
            key_node[threadIdx.x] = node >= 0 ? node : -1;
            key_factor[threadIdx.x] = factor;
        }
        __syncthreads();
        if constexpr (WIDE) {
            const int per = hd / 4;
            for (int i = threadIdx.x; i < BN * per; i += THREADS) {
                const int r = i / per, d = i % per * 4;
                const long long row = key_row[r];
                *(float4*)(k_s + r * stride + d) = row >= 0 ? load4((const T*)c.kv + row + d) : make_float4(0.f, 0.f, 0.f, 0.f);
                *(float4*)(v_s + r * stride + d) = row >= 0 ? load4((const T*)c.kv + c.v_offset + row + d) : make_float4(0.f, 0.f, 0.f, 0.f);
            }
        } else {
            for (int i = threadIdx.x; i < BN * hdp; i += THREADS) {
                const int r = i / hdp, d = i % hdp;
                const long long row = key_row[r];
                const bool there = row >= 0 && d < hd;
                k_s[r * stride + d] = there ? to_f32(((const T*)c.kv)[row + d]) : 0.f;
                v_s[r * stride + d] = there ? to_f32(((const T*)c.kv)[c.v_offset + row + d]) : 0.f;
            }
        }
        __syncthreads();
        if (4 * warp >= n_rows) continue;
        // scores: four rows and this lane's key
        float s[4] = {0.f, 0.f, 0.f, 0.f};
        const float* kr = k_s + lane * stride;
        const float* qr = q_s + 4 * warp * hdp;
        for (int d = 0; d < hdp; d += 4) {
            const float4 kv = *(const float4*)(kr + d);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float4 qv = *(const float4*)(qr + i * hdp + d);
                s[i] = fmaf(qv.x, kv.x, s[i]); s[i] = fmaf(qv.y, kv.y, s[i]); s[i] = fmaf(qv.z, kv.z, s[i]); s[i] = fmaf(qv.w, kv.w, s[i]);
            }
        }
        const int kp = key_pos[lane], kn = key_node[lane];
        const bool there = key_row[lane] >= 0;
        const float factor = key_factor[lane];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            bool vis = row_ok[i] && there && kp >= lo[i];
            if (vis && kn >= 0)                                // (a node sees no node behind itself)
                vis = kn <= tok[i] - first && (x.ancestors[(size_t)tok[i] * x.n_words + kn / 32] >> (kn % 32) & 1u);
            float v = -INFINITY;
            if (vis) {
                v = capped(p, s[i] * p.softmax_scale * factor) - slope[i] * (float)(pos[i] - kp);
                if (dist[i]) v += number_at(p, dist[i], pos[i] - kp);
            }
            const float m_new = fmaxf(m[i], warp_max(v));
            const float corr = m_new == -INFINITY ? 1.f : expf(m[i] - m_new);
            const float w = vis ? expf(v - m_new) : 0.f;
            l[i] = l[i] * corr + warp_sum(w);
            m[i] = m_new;
            weight[4 * warp + i][lane] = w;
#pragma unroll
            for (int e = 0; e < HD4; ++e) { acc[i][e].x *= corr; acc[i][e].y *= corr; acc[i][e].z *= corr; acc[i][e].w *= corr; }
        }
        __syncwarp();
        // values: four rows and this lane's elements of the head
        for (int j = 0; j < BN; j += 4) {
            float wj[4][4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float4 four = *(const float4*)&weight[4 * warp + i][j];
                wj[i][0] = four.x; wj[i][1] = four.y; wj[i][2] = four.z; wj[i][3] = four.w;
            }
#pragma unroll
            for (int jj = 0; jj < 4; ++jj)
#pragma unroll
                for (int e = 0; e < HD4; ++e) {
                    const int d = 4 * (lane + 32 * e);
                    if (d >= hdp) continue;
                    const float4 v = *(const float4*)(v_s + (j + jj) * stride + d);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        if (wj[i][jj] == 0.f) continue;        // a masked key's value may be anything
                        acc[i][e].x = fmaf(wj[i][jj], v.x, acc[i][e].x); acc[i][e].y = fmaf(wj[i][jj], v.y, acc[i][e].y);
                        acc[i][e].z = fmaf(wj[i][jj], v.z, acc[i][e].z); acc[i][e].w = fmaf(wj[i][jj], v.w, acc[i][e].w);
                    }
                }
        }
        __syncwarp();                                          // the weights are written again for the next tile
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (!row_ok[i]) continue;
        float scale = 1.f;
        if (n_splits == 1) {
            const float shrink = tree_fold_sink(p, head[i], m[i], l[i]);
            scale = shrink * gate_of(p, tok[i], head[i]) / fmaxf(l[i], 1e-30f);
        }
        T* out = (T*)p.out + out_row_of(p, tok[i], head[i]) * hd;
        float* part = partial + (((size_t)tok[i] * nq + head[i]) * n_splits + split) * (hd + 2);
#pragma unroll
        for (int e = 0; e < HD4; ++e) {
            const float v[4] = {acc[i][e].x, acc[i][e].y, acc[i][e].z, acc[i][e].w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int d = 4 * (lane + 32 * e) + k;
                if (d >= hd) continue;
                if (n_splits == 1) out[d] = from_f32<T>(v[k] * scale); else __stcg(part + 2 + d, v[k]);
            }
        }
        if (n_splits > 1 && lane == 0) { __stcg(part, m[i]); __stcg(part + 1, l[i]); }
    }
}

// Adds the shares of a row up, in the order of the keys.  grid (tokens, heads / 4), a warp a row.
template <typename T>
__global__ void __launch_bounds__(THREADS) attn_tree_join_kernel(const AttentionParams p, const StepTokens b, const TreeStep x, const float* partial, int hd,
                                                                 int n_splits) {
    pdl_wait();
    pdl_launch_dependents();
    const int t = blockIdx.x, head = blockIdx.y * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (head >= p.num_heads || t >= x.cu_seqlens[x.n_segments]) return;     // (rows behind the last request stay as they are)
    const float* part = partial + ((size_t)t * p.num_heads + head) * n_splits * (hd + 2);
    const float my_m = lane < n_splits ? __ldcg(part + lane * (hd + 2)) : -INFINITY;       // (at most 32 shares)
    const float my_l = lane < n_splits ? __ldcg(part + lane * (hd + 2) + 1) : 0.f;
    const float m = warp_max(my_m);
    const float my_w = my_m == -INFINITY ? 0.f : expf(my_m - m);
    float l = warp_sum(my_l * my_w);
    const float shrink = tree_fold_sink(p, head, m, l);
    const float scale = shrink * gate_of(p, t, head) / fmaxf(l, 1e-30f);
    T* out = (T*)p.out + out_row_of(p, t, head) * hd;
    for (int d = lane; d - lane < hd; d += 32) {
        float acc = 0.f;
        for (int s = 0; s < n_splits; ++s) {
            const float w = __shfl_sync(0xffffffffu, my_w, s);
            if (w != 0.f && d < hd) acc = fmaf(w, __ldcg(part + s * (hd + 2) + 2 + d), acc);
        }
        if (d < hd) out[d] = from_f32<T>(acc * scale);
    }
}

template <typename T>
int launch(const AttentionParams& p, const StepTokens& b, const PagedCache& c, const TreeStep& x, float* partial, int n_splits, cudaStream_t st) {
    const int hd = c.head_dim, hdp = (hd + 3) & ~3, G = p.num_heads / c.num_kv_heads, chunks = (G + ROWS - 1) / ROWS;
    const int nodes = G >= ROWS ? 1 : ROWS / G;
    const size_t smem = ((size_t)ROWS * hdp + 2 * BN * (size_t)(hdp + 4)) * 4;
    const bool wide = hd % 4 == 0 && !(((uintptr_t)c.kv | (uintptr_t)(c.v_offset * sizeof(T))) & (4 * sizeof(T) - 1));
    if ((long long)c.num_kv_heads * chunks > 65535) return SPITE_UNSUPPORTED;
    const dim3 grid(b.n_tokens, c.num_kv_heads * chunks, n_splits);
    auto k = hd <= 128 ? (wide ? attn_tree_kernel<T, 1, true> : attn_tree_kernel<T, 1, false>) : (wide ? attn_tree_kernel<T, 2, true> : attn_tree_kernel<T, 2, false>);
    if (smem > 48 * 1024 && cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess) return SPITE_LAUNCH_FAILED;
    SPITE_LAUNCH(k, grid, THREADS, smem, st, p, b, c, x, partial, nodes, n_splits);
    if (n_splits > 1) SPITE_LAUNCH(attn_tree_join_kernel<T>, dim3(b.n_tokens, (p.num_heads + 3) / 4), THREADS, 0, st, p, b, x, (const float*)partial, hd, n_splits);
    return spite_launch_status();
}

}  // namespace

// `partial`: tokens * heads * n_splits * (head_dim + 2) floats where n_splits (1..32) > 1.
SPITE_API int spite_tree_attention(int dtype, const TreeCall* call, float* partial, long long n_partial, int n_splits, void* stream) {
    if (!call || !tree_call_ok(*call)) return SPITE_BAD_ARG;
    const AttentionParams& p = call->p;
    if (n_splits < 1 || n_splits > 32) return SPITE_BAD_ARG;
    if (n_splits > 1 && (!partial || n_partial < (long long)call->b.n_tokens * p.num_heads * n_splits * (call->c.head_dim + 2))) return SPITE_BAD_ARG;
    if (call->c.head_dim > 256 || p.num_heads > 4 * 65535) return SPITE_UNSUPPORTED;
    if (call->b.n_tokens == 0) return SPITE_OK;
    if (dtype == SPITE_DT_F32) return launch<float>(p, call->b, call->c, call->x, partial, n_splits, (cudaStream_t)stream);
    if (dtype == SPITE_DT_BF16) return launch<__nv_bfloat16>(p, call->b, call->c, call->x, partial, n_splits, (cudaStream_t)stream);
    return SPITE_BAD_ARG;
}
