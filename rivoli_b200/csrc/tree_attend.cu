// Attention of a tree of drafted tokens over the paged latent cache: the entry points, and the CUDA-core form for geometries that the
// tensor-core form (tree_mma.cu) does not cover.
//
//     out[node][h] = sum_j softmax_j((q[node][h] . [L_j | R_j]) * scale) * L_j
//
// over the n prefix rows of the node's sequence (a row list, or its first n tokens) and those rows of the tree itself whose bit is up
// in the node's mask; node j's row is the sequence's token tree_pos + j. A node that sees nothing gets zeros and a log-sum-exp of
// minus infinity. Rows on pages that the block table leaves unmapped, and rows whose scale is not above zero, are seen by nobody.
//
// CUDA cores: a block takes 16 (node, head) rows of one sequence, two a warp, and 16 cache rows at a time, dequantised into shared
// memory once for all of them; scores, running maximum and sum, and the output are 32-bit. It is bound by its shuffles and
// shared-memory reads and exists for shapes; the model's shapes do not come here.
#include "codec.cuh"
#include "common.cuh"
#include "tc_common.cuh"
#include "tree_common.cuh"

namespace {

constexpr int TS_WARPS = 8, TS_ROWS = 2 * TS_WARPS, TS_TILE = 16, TS_THREADS = TS_WARPS * 32;
constexpr int TS_W = 640, TS_KVL = 512;    // most columns of a row, and of its latent part

__global__ void __launch_bounds__(TS_THREADS)
tree_simt_kernel(TreeArgs A, int kvl, int rope) {
    extern __shared__ float tile[];        // [TS_TILE][W]
    __shared__ uint32_t s_row[TS_TILE];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, W = kvl + rope;
    rv_grid_dep_wait();
    rv_grid_dep_trigger();
    // the block's sequence and rows: groups of 16 rows are numbered through the sequences
    int b = 0, group = blockIdx.x;
    TreeSeq s;
    for (;; ++b) {
        if (b >= A.B) return;
        s = tree_seq(A, b);
        const int groups = (s.T * A.H + TS_ROWS - 1) / TS_ROWS;
        if (group < groups) break;
        group -= groups;
    }
    float q[2][TS_W / 32], acc[2][TS_KVL / 32], m[2], l[2];
    uint64_t mask[2];
    bool live[2];
    size_t at[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        const int r = group * TS_ROWS + warp * 2 + u, node = r / A.H;
        live[u] = r < s.T * A.H;
        at[u] = (size_t)s.node0 * A.H + r;
        mask[u] = live[u] ? A.node_mask[s.node0 + node] : 0ull;
        m[u] = -INFINITY; l[u] = 0.0f;
#pragma unroll
        for (int k = 0; k < TS_W / 32; ++k) q[u][k] = live[u] && lane + 32 * k < W ? rv_bf16_to_f32(A.q[at[u] * W + lane + 32 * k]) : 0.0f;
#pragma unroll
        for (int k = 0; k < TS_KVL / 32; ++k) acc[u][k] = 0.0f;
    }
    const int total = s.n + s.T;
    for (int j0 = 0; j0 < total; j0 += TS_TILE) {
        __syncthreads();
        if (tid < TS_TILE) {
            const uint32_t r = j0 + tid < total ? tree_pool_row(A, b, tree_token(A, s, b, j0 + tid)) : 0xffffffffu;
            s_row[tid] = r != 0xffffffffu && A.pscale[r] <= 0.0f ? 0xffffffffu : r;
        }
        __syncthreads();
        for (int i = tid; i < TS_TILE * (W / 2); i += TS_THREADS) {
            const int t = i / (W / 2), c = 2 * (i - t * (W / 2));
            float2 v = make_float2(0.0f, 0.0f);
            if (s_row[t] != 0xffffffffu) {
                v = rv_e4m3x2_to_f32x2(*reinterpret_cast<const uint16_t*>(A.pool + (size_t)s_row[t] * W + c));
                const float sc = A.pscale[s_row[t]];
                v.x *= sc; v.y *= sc;
            }
            tile[t * W + c] = v.x; tile[t * W + c + 1] = v.y;
        }
        __syncthreads();
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const uint64_t sees = tree_visible(mask[u], s.T, s.n, j0);
            float mine = -INFINITY;        // lane t: the score of row t
            for (int t = 0; t < TS_TILE; ++t) {
                float d = 0.0f;
#pragma unroll
                for (int k = 0; k < TS_W / 32; ++k)
                    if (lane + 32 * k < W) d = fmaf(q[u][k], tile[t * W + lane + 32 * k], d);
                d = rv_warp_sum(d) * A.softmax_scale;
                if (lane == t && ((sees >> t) & 1) && s_row[t] != 0xffffffffu) mine = d;
            }
            const float top = fmaxf(m[u], rv_warp_max(mine));
            if (top == -INFINITY && !__any_sync(0xffffffffu, mine != mine)) continue;   // nothing seen so far (NaN is something)
            const float fac = expf(m[u] - top), p = expf(mine - top);
            l[u] = l[u] * fac + rv_warp_sum(p);
            m[u] = top;
#pragma unroll
            for (int k = 0; k < TS_KVL / 32; ++k) acc[u][k] *= fac;
            for (int t = 0; t < TS_TILE; ++t) {
                const float w = __shfl_sync(0xffffffffu, p, t);
                if (w == 0.0f) continue;                       // (a hidden row may hold NaN)
#pragma unroll
                for (int k = 0; k < TS_KVL / 32; ++k)
                    if (lane + 32 * k < kvl) acc[u][k] = fmaf(w, tile[t * W + lane + 32 * k], acc[u][k]);
            }
        }
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        if (!live[u]) continue;
        const float inv = l[u] == 0.0f ? 0.0f : 1.0f / l[u];   // (NaN stays NaN)
#pragma unroll
        for (int k = 0; k < TS_KVL / 32; ++k)
            if (lane + 32 * k < kvl) A.out[at[u] * kvl + lane + 32 * k] = rv_f32_to_bf16(acc[u][k] * inv);
        if (A.out_lse && lane == 0) A.out_lse[at[u]] = l[u] == 0.0f ? -INFINITY : m[u] + logf(l[u]);
    }
}

}  // namespace

RIVOLI_API size_t rivoli_mla_tree_attend_scratch_bytes(const DsaGeom* g, int B, int n_nodes) {
    if (!g || B <= 0 || n_nodes <= 0 || rv_check_geom(g)) return 0;
    return rv_tree_mma_supported(g) ? rv_tree_mma_scratch_bytes() : 0;
}

RIVOLI_API int rivoli_mla_tree_attend_paged_bf16(const DsaGeom* g, const uint16_t* q, const uint8_t* latent_pool,
                                                 const float* latent_scale, const int32_t* block_table, const uint32_t* rows,
                                                 int row_stride, const int32_t* n_rows, const int32_t* tree_pos,
                                                 const int32_t* node_start, const uint64_t* node_mask, int B, int n_nodes,
                                                 uint16_t* out, float* out_lse, void* scratch, void* stream) {
    if (int e = rv_check_geom(g)) return e;
    if (B <= 0 || n_nodes <= 0 || !q || !latent_pool || !latent_scale || !block_table || !tree_pos || !node_start || !node_mask || !out)
        return 1001;
    if (rows && (row_stride <= 0 || !n_rows)) return 1001;
    if ((long long)n_nodes * g->n_heads > 0x7fffffffLL / 2 || (long long)g->n_pool_pages * g->page_tokens > 0x7fffffffLL) return 1002;
    if ((((uintptr_t)latent_pool | (uintptr_t)q | (uintptr_t)out | (uintptr_t)scratch) & 15) || ((uintptr_t)node_mask & 7)) return 1005;
    const TreeArgs a{q, latent_pool, latent_scale, block_table, rows, row_stride, n_rows, tree_pos, node_start, node_mask, B, n_nodes,
                     g->n_heads, g->page_tokens, g->max_pages_per_seq, g->n_pool_pages, g->softmax_scale, out, out_lse};
    if (scratch && rv_tree_mma_supported(g)) return rv_tree_mma(a, scratch, (cudaStream_t)stream);
    rv_drain_error();
    const int W = g->kv_lora + g->rope_dim;
    const long long groups = ((long long)n_nodes * g->n_heads) / TS_ROWS + B;
    rv_launch_dependent(tree_simt_kernel, dim3((unsigned)groups), dim3(TS_THREADS), (size_t)TS_TILE * W * 4, (cudaStream_t)stream, a,
                        g->kv_lora, g->rope_dim);
    return rv_launch_status();
}

// Synchronises `stream`; 1008 if a bounded wait of the tensor-core form gave up since the last call on this scratch.
RIVOLI_API int rivoli_mla_tree_attend_status(const DsaGeom* g, void* scratch, void* stream) {
    if (!g || !scratch) return 1001;
    if (!rv_tree_mma_supported(g)) return 0;
    int h = 0;
    cudaError_t e = cudaMemcpyAsync(&h, scratch, sizeof(int), cudaMemcpyDeviceToHost, (cudaStream_t)stream);
    if (e == cudaSuccess) e = cudaStreamSynchronize((cudaStream_t)stream);
    if (e != cudaSuccess) return -(int)e;
    if (h) cudaMemsetAsync(scratch, 0, sizeof(int), (cudaStream_t)stream);
    return h ? 1008 : 0;
}
