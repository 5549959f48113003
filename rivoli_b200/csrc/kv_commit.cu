// The accepted rows of a drafted tree, moved in the paged pools to where the sequence goes on, in all layers with one launch.
//
// Sequence b drafted its nodes into the rows of positions tree_pos[b] + j; path[b][0 .. n_path[b]) (ascending node indices) stays.
// Row tree_pos[b] + path[b][k] becomes row tree_pos[b] + k: codes and scales of the latent row and of the indexer key, bit for bit.
// A row only ever moves down (path[k] >= k), so that no move of a later k reads what an earlier one has written, chunk by chunk: one
// warp moves all rows of a layer, as many chunks at once as it has room for, and reads them before it writes any. Rows that stay where
// they are (a chain that was accepted from its root) are not touched.
// Bound by memory: 712 bytes read and written per moved row and layer of the model geometry. With eight chunks a lane the loads of five
// rows are in flight at once; what stays is the chain path -> page -> layer -> row (64 sequences, 5 rows of 78 layers: 15.0 us with a
// warp per row and one row in flight, 9.2 us so; 4.3 us of traffic).
#include "common.cuh"

namespace {

constexpr int KC_WARPS = 4, KC_MAX_PATH = 64;
constexpr int KC_CHUNKS = 8;            // 16-byte chunks that a lane holds

struct CommitArgs {
    DsaGeom g;
    const CommitLayer* layers; int n_layers;
    const int32_t* block_table; const int32_t* tree_pos; const int32_t* path; const int32_t* n_path;
    int path_stride;
    int32_t* seq_len; int32_t* status;
};

__global__ void __launch_bounds__(KC_WARPS * 32)
kv_commit_kernel(CommitArgs A) {
    __shared__ long long s_src[KC_MAX_PATH], s_dst[KC_MAX_PATH];   // pool rows; -1: nothing to move
    __shared__ int s_bad;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, b = blockIdx.y;
    rv_grid_dep_wait();
    rv_grid_dep_trigger();
    const int pos = A.tree_pos[b], n = min(max(A.n_path[b], 0), A.path_stride);
    if (tid == 0) s_bad = 0;
    __syncthreads();
    if (tid < n) {
        const int node = A.path[(size_t)b * A.path_stride + tid];
        const int before = tid ? A.path[(size_t)b * A.path_stride + tid - 1] : -1;
        auto pool_row = [&](int t) -> long long {
            const int lp = t / A.g.page_tokens;
            const int pg = lp < A.g.max_pages_per_seq ? A.block_table[(size_t)b * A.g.max_pages_per_seq + lp] : -1;
            return pg >= 0 && pg < A.g.n_pool_pages ? (long long)pg * A.g.page_tokens + t % A.g.page_tokens : -1;
        };
        const bool sound = node > before && node >= tid && node < KC_MAX_PATH && pos >= 0 && pos < 0x7fffffff - KC_MAX_PATH;
        long long src = sound ? pool_row(pos + node) : -1, dst = sound ? pool_row(pos + tid) : -1;
        if (src < 0 || dst < 0) s_bad = 1;
        if (node == tid) src = dst = -1;                      // it stays (and so do all before it)
        s_src[tid] = src; s_dst[tid] = dst;
    }
    __syncthreads();
    if (s_bad) {                        // an unsound path or an unmapped page: the sequence is left as it is
        if (A.status && tid == 0 && blockIdx.x == 0) atomicOr(A.status, 1);
        return;
    }
    if (A.seq_len && tid == 0 && blockIdx.x == 0) A.seq_len[b] = pos + n;
    int first = 0;
    while (first < n && s_src[first] < 0) ++first;
    const int wl = (A.g.kv_lora + A.g.rope_dim) >> 4, wi = A.g.index_dim >> 4;   // chunks
    const int l = blockIdx.x * KC_WARPS + warp;
    if (l >= A.n_layers || first >= n) return;
    const CommitLayer L = A.layers[l];
    const int chunks = wl + (L.index_pool ? wi : 0);
    for (int k0 = first; k0 < n; k0 += 32) {                   // the scales
        const int k = k0 + lane;
        const bool moves = k < n;
        const float sc = moves ? L.latent_scale[s_src[k]] : 0.0f, si = moves && L.index_pool ? L.index_scale[s_src[k]] : 0.0f;
        __syncwarp();
        if (moves) {
            L.latent_scale[s_dst[k]] = sc;
            if (L.index_pool) L.index_scale[s_dst[k]] = si;
        }
        __syncwarp();
    }
    int k = first, c = lane;                                   // this lane's next chunk
    while (c >= chunks) { c -= chunks; ++k; }
    for (int done = 0; done < (n - first) * chunks; done += 32 * KC_CHUNKS) {
        uint4 v[KC_CHUNKS];
        uint4* to[KC_CHUNKS];
#pragma unroll
        for (int u = 0; u < KC_CHUNKS; ++u) {
            to[u] = nullptr;
            if (k < n) {
                const size_t src = s_src[k], dst = s_dst[k];
                const bool lat = c < wl;
                uint4* pool = reinterpret_cast<uint4*>(lat ? L.latent_pool : L.index_pool);
                const int w = lat ? wl : wi, at = lat ? c : c - wl;
                v[u] = pool[src * w + at];
                to[u] = pool + dst * w + at;
            }
            c += 32;
            while (c >= chunks) { c -= chunks; ++k; }
        }
        __syncwarp();                   // all of them are in registers
#pragma unroll
        for (int u = 0; u < KC_CHUNKS; ++u)
            if (to[u]) *to[u] = v[u];
        __syncwarp();
    }
}

}  // namespace

RIVOLI_API int rivoli_kv_commit_paged(const DsaGeom* g, const CommitLayer* layers, int n_layers, const int32_t* block_table,
                                      const int32_t* tree_pos, const int32_t* path, int path_stride, const int32_t* n_path, int B,
                                      int32_t* seq_len, int32_t* status, void* stream) {
    if (int e = rv_check_geom(g)) return e;
    if (!layers || n_layers <= 0 || !block_table || !tree_pos || !path || path_stride <= 0 || !n_path || B <= 0) return 1001;
    if (path_stride > KC_MAX_PATH || B > 65535) return 1002;
    if ((uintptr_t)layers & 7) return 1005;
    // blocks of all layers read these while one writes seq_len
    auto shared = [&](const int32_t* p, size_t n) { return (uintptr_t)seq_len < (uintptr_t)(p + n) && (uintptr_t)p < (uintptr_t)(seq_len + B); };
    if (seq_len && (shared(tree_pos, B) || shared(n_path, B) || shared(path, (size_t)B * path_stride) ||
                    shared(block_table, (size_t)B * g->max_pages_per_seq)))
        return 1005;
    CommitArgs a{*g, layers, n_layers, block_table, tree_pos, path, n_path, path_stride, seq_len, status};
    rv_drain_error();
    rv_launch_dependent(kv_commit_kernel, dim3((n_layers + KC_WARPS - 1) / KC_WARPS, B), dim3(KC_WARPS * 32), 0, (cudaStream_t)stream, a);
    return rv_launch_status();
}
