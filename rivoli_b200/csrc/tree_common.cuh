// What both kernels of the tree attention share: the call's arguments and the reading of a sequence's sizes from the device.
#pragma once

#include "common.cuh"

constexpr int TREE_NODES = 64;             // nodes of a sequence: a bit of a 64-bit mask each

struct TreeArgs {
    const uint16_t* q;                     // [n_nodes][H][kv_lora + rope]
    const uint8_t* pool; const float* pscale; const int32_t* block_table;
    const uint32_t* rows; long long row_stride; const int32_t* n_rows;
    const int32_t* tree_pos; const int32_t* node_start; const uint64_t* node_mask;
    int B, n_nodes, H, page_tokens, max_pages, n_pool_pages;
    float softmax_scale;
    uint16_t* out; float* out_lse;
};

// Sizes of sequence b, clamped so that a bad word can never index past an array: node0 and T its nodes, n its prefix rows.
struct TreeSeq { int node0, T, n, pos; bool listed; };
__device__ __forceinline__ TreeSeq tree_seq(const TreeArgs& A, int b) {
    TreeSeq s;
    s.node0 = max(0, A.node_start[b]);
    s.T = max(0, min(min(A.node_start[b + 1], A.n_nodes) - s.node0, TREE_NODES));
    s.pos = A.tree_pos[b];
    // A row list whose first entry is the dense marker stands for "row j = token j" over the first n_rows tokens. The prefix ends where
    // the tree begins: a selection that was made once the root's row was there may name it, and may count it.
    s.listed = A.rows && A.rows[(size_t)b * A.row_stride] != 0xffffffffu;
    const long long cap = s.listed ? A.row_stride : min((long long)s.pos, (long long)A.max_pages * A.page_tokens);
    s.n = (int)max(0LL, min(min((long long)(A.n_rows ? A.n_rows[b] : s.pos), cap), 0x7fffff00LL));
    return s;
}

// Token of entry j of sequence b (j < n: the prefix, from n on the tree) and its pool row; 0xffffffff: none, attended by nobody.
__device__ __forceinline__ uint32_t tree_token(const TreeArgs& A, const TreeSeq& s, int b, int j) {
    if (j < s.n) {
        if (!s.listed) return (uint32_t)j;
        const uint32_t t = A.rows[(size_t)b * A.row_stride + j];
        return (int)t >= 0 && (int)t < s.pos ? t : 0xffffffffu;
    }
    return (uint32_t)s.pos + (uint32_t)(j - s.n);
}
__device__ __forceinline__ uint32_t tree_pool_row(const TreeArgs& A, int b, uint32_t token) {
    const uint32_t lp = token >> rv_log2(A.page_tokens);
    const int pg = lp < (uint32_t)A.max_pages ? A.block_table[(size_t)b * A.max_pages + lp] : -1;
    return pg >= 0 && pg < A.n_pool_pages ? (uint32_t)pg * (uint32_t)A.page_tokens + (token & (uint32_t)(A.page_tokens - 1)) : 0xffffffffu;
}

// Which of the 64 entries from j0 on a node with this mask sees: all of the prefix (below n), of the tree those whose bit is up.
__device__ __forceinline__ uint64_t tree_visible(uint64_t mask, int T, int n, int j0) {
    if (T < 64) mask &= (1ull << T) - 1;
    const int d = j0 - n;
    if (d >= 64) return 0ull;
    if (d >= 0) return mask >> d;
    if (d <= -64) return ~0ull;
    return (mask << -d) | ((1ull << -d) - 1);
}

int rv_tree_mma(const TreeArgs& a, void* scratch, cudaStream_t st);
bool rv_tree_mma_supported(const DsaGeom* g);
size_t rv_tree_mma_scratch_bytes();
