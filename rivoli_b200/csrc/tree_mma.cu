// Attention of drafted trees over the paged latent cache on the 5th-generation tensor cores, all operands fp8.
//
//     out[r] = sum_j softmax_j((q_r . [L_j | R_j]) * scale) * L_j,    r = (node, head) of one sequence, j = its prefix, then its tree
//
// The arithmetic is that of the decode step's attention (attend_mma.cu): cache rows are consumed as the e4m3 codes they are, q and the
// softmax weights are two e4m3 terms each (2^-8 relative), a row's scale rides in its weight (P' = weight * scale * 2^5), references
// lag behind the running maximum by at most 2^3, sums are f32. What differs is the shape of the work. The nodes of a tree share their
// prefix, so that the rows of a sequence are nodes x heads, 128 to a block, and one tile of 64 cache rows serves them all: the kernel is
// bound by the tensor cores and what feeds them.
//   * A block of 128 rows is a PAIR of CTAs, 64 rows each, and its products are tcgen05 cta_group::2, issued by the pair's first CTA. The
//     hi and lo terms of 64 rows are the 128 rows that a CTA has in S = Q . K^T (M = 256, N = 64 tokens: 32 of each CTA); O += P' . V is
//     M = 128 (64 rows of each CTA, both halves of tensor memory's lanes taking half of the columns), N = 256 dims: 128 of each CTA. Each CTA
//     feeds half of the shared operand and keeps softmax, references and O of its own rows to itself. A tile's 26 instructions take
//     1,105 cycles (measured back to back: 32 and 66 cycles each), against 1,400 and more for one CTA on its own, whose O^T += V^T . P'
//     with 64 columns reads shared memory for longer than it multiplies.
//   * The (row block, tile) pairs of all sequences, in order, are cut into equal runs, one per pair of CTAs. A run that begins or ends
//     inside a row block leaves that block's (maximum, sum, O) in scratch and a second, small kernel joins the parts; all others are
//     written directly. No sequence is too long and no batch too ragged for this.
//   * Barriers and their phases run on over the row blocks: the next block's tiles are fetched while this one's output is written.
//   * The rows of a tile come as K (the CTA's 32 tokens, all columns; held until S is there) and V (all 64 tokens, the CTA's 256 columns; held
//     until O is) in rings of their own. Tiles that lie in a dense prefix are tensor copies of page rows, others are gathered.
// Rows of the tree are tested against each node's mask in the tiles that hold them, the last one or two of a sequence. A hidden row's
// weight is 0, but 0 x NaN is NaN: in V, NaN codes of tree rows become 0 (in K they make a score NaN, which the mask takes away from the
// nodes that do not see the row, and from them alone).
//
// Tensor memory: S twice (64 columns each), q (128: its latent columns are the A operand of the QK products), O (256). Warps: 0-7 softmax
// and epilogue in two groups that take the tiles in turn, 8 QK issue, 9 PV issue (in the pair's second CTA these two pass on that its K and
// V are there), 10-12 gather K, 13-15 V. All waits are bounded (tc_common.cuh).
#include <atomic>

#include "codec.cuh"
#include "common.cuh"
#include "quant.cuh"
#include "tc_common.cuh"
#include "tmap.hpp"
#include "tree_common.cuh"

namespace {

constexpr int TM_TILE = 64, TM_ROWS = 64, TM_BLOCK = 2 * TM_ROWS;   // cache rows of a tile; (node, head) rows of a CTA, of a pair
constexpr int TM_KVL = 512, TM_ROPE = 64, TM_W = TM_KVL + TM_ROPE;
constexpr int TM_OWN = TM_TILE / 2;                  // tokens of a tile whose K a CTA holds
constexpr int NK = 5, NV = 6, NG = 2, GW = 3;        // stages of K and of V; softmax groups, each with a P' buffer; warps that gather K, and V
constexpr int TM_SW = 4 * NG, TM_QKW = TM_SW, TM_PVW = TM_SW + 1, TM_KW = TM_SW + 2, TM_VW = TM_KW + GW;
constexpr int TM_THREADS = (TM_VW + GW) * 32, TM_SOFTMAX = TM_SW * 32, TM_GROUP = 128;
constexpr float TM_POFF = 5.0f, TM_MOST = 256.0f;    // P' = 2^(s - ref + 5) <= 2^8: references lag by 2^3 at most, see attend_mma.cu
constexpr int TM_MIN_UNITS = 4;                      // tiles a pair takes at least, while there are few
constexpr int TM_PAIRS = RV_SMS / 2;

// tensor memory columns
constexpr int TMC_S = 0, TMC_Q = 2 * TM_TILE, TMC_O = TMC_Q + TM_KVL / 4;
static_assert(TMC_O + 256 == 512, "tensor memory budget");

// shared memory (bytes)
constexpr int KCHUNK = TM_OWN * 128, KSTAGE = 4 * KCHUNK + TM_OWN * 64;   // four latent chunks [32 tokens][128 B], 128-byte swizzle; rope [32][64 B], 64-byte swizzle
constexpr int VCHUNK = TM_TILE * 128, VSTAGE = 2 * VCHUNK;                // two chunks [64 tokens][128 B]: columns 128 rank and 256 + 128 rank on
constexpr int SM_V = 0;
constexpr int SM_K = SM_V + NV * VSTAGE;
constexpr int SM_QR = SM_K + NK * KSTAGE;                   // rope columns of q: [128 virtual rows][64 B], 64-byte swizzle
constexpr int SM_P = SM_QR + 8192;                          // per group {hi, lo} [64 rows][64 tokens], 64-byte swizzle
constexpr int PTERM = 4096, PBUF = 2 * PTERM;
constexpr int SM_TOK = SM_P + NG * PBUF;                    // f32 [NV][64]: the tokens' scales
constexpr int SM_SEE = SM_TOK + NV * TM_TILE * 4;           // u64 [NV][2]: tokens that are there; tokens whose scale is no number
constexpr int SM_AHI = SM_SEE + NV * 16;                    // f32 [64] query scale * softmax scale * log2(e)
constexpr int SM_WMAX = SM_AHI + 256;                       // f32 [NG][64]
constexpr int SM_FAC = SM_WMAX + NG * 256;                  // f32 [64]
constexpr int SM_MREF = SM_FAC + 256;                       // f32 [64]
constexpr int SM_BARS = SM_MREF + 256;
constexpr int SM_MISC = SM_BARS + 512;
constexpr int SM_TOTAL = SM_MISC + 64;
static_assert(SM_TOTAL <= 232448, "shared memory budget");
static_assert(SM_K % 1024 == 0 && SM_QR % 1024 == 0 && SM_P % 1024 == 0 && KSTAGE % 1024 == 0, "operand tiles are 1024-byte aligned");

// Barriers marked * are the first CTA's alone: both CTAs arrive there.
struct Bars {
    uint64_t k_full[NK], k_peer[NK] /* * */, k_empty[NK], v_full[NV], v_peer[NV] /* * */, v_empty[NV], tok_full[NV], s_full[NG], s_empty[2] /* * */,
        p_full[NG] /* * */, pv_done[NG], dec[NG], q_full /* * */;
};
static_assert(sizeof(Bars) <= 512, "barrier block");
constexpr int FULL = 33;                                    // arrivals that fill a stage: the copies of 32 lanes, and the gathering warp

// scratch: error word (256 bytes) | per pair the block it has the beginning of, for the joining kernel | (reference, sum) of parts | O of parts
constexpr int SLOTS = 2 * TM_PAIRS;                         // a pair leaves at most the end of one block and the beginning of another
struct Head { int32_t row0, valid, parts, pad; };
constexpr size_t SC_HEAD = 256, SC_ML = SC_HEAD + TM_PAIRS * sizeof(Head), SC_O = (SC_ML + (size_t)SLOTS * TM_BLOCK * 8 + 255) / 256 * 256;
constexpr size_t SC_TOTAL = SC_O + (size_t)SLOTS * TM_BLOCK * TM_KVL * 4;

__device__ __forceinline__ uint32_t sw64_chunk(uint32_t row, uint32_t chunk) { return row * 64u + ((chunk ^ ((row >> 1) & 3u)) << 4); }
__device__ __forceinline__ uint64_t smem_desc(uint32_t saddr, uint32_t lbo_bytes, uint32_t sbo_bytes, uint32_t layout) {
    uint64_t d = 0;
    d |= (uint64_t)((saddr & 0x3FFFFu) >> 4);
    d |= (uint64_t)((lbo_bytes >> 4) & 0x3FFFu) << 16;
    d |= (uint64_t)((sbo_bytes >> 4) & 0x3FFFu) << 32;
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)layout << 61;   // 2 = 128-byte swizzle, 4 = 64-byte swizzle
    return d;
}
__device__ __forceinline__ void mbar_arrive_n(uint64_t* bar, uint32_t n) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0], %1;" ::"r"(tc::smem_u32(bar)), "r"(n) : "memory");
}
// One arrival on the first CTA's barrier, from either CTA (`at`: its address there). What it announces is shared and tensor memory of the
// arriving CTA, which the products read there, through the async proxy and behind this thread's fences: release at the CTA's scope is
// what that takes. (With the scopes of arrivals and waits at the cluster, which orders global memory too, every one of these cost a
// thousand cycles and more: 3,700 cycles a tile.)
__device__ __forceinline__ uint32_t in_first(const void* p) {
    uint32_t at;
    asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(at) : "r"(tc::smem_u32(p)));
    return at;
}
__device__ __forceinline__ void arrive_first(uint32_t at) {
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(at) : "memory");
}
// The bounded wait of a warp, in few instructions: the kernel's loops have to stay in the instruction cache. (With every wait unrolled, the
// weights there twice and the query conversion in one piece, 192 KiB of code, each of a tile's steps waited for its instructions, and a
// tile took 3,700 cycles.)
__device__ __forceinline__ bool wait_for(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int code, int max_polls) {
    const uint32_t a = tc::smem_u32(bar);
    uint32_t ok;
    int left = max_polls;
#pragma unroll 1
    do {
        asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                     : "=r"(ok) : "r"(a), "r"(parity) : "memory");
    } while (!ok && --left > 0 && ((left & 63) || !*abort_flag));
    if (__all_sync(0xffffffffu, ok != 0)) return true;
    if (!*abort_flag) *abort_flag = code;
    return false;
}
// Two f32 in a register pair: the packed forms round each as usual.
typedef unsigned long long f2;
__device__ __forceinline__ f2 pack(float lo, float hi) { f2 r; asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi)); return r; }
__device__ __forceinline__ float2 unpack(f2 v) { float2 r; asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v)); return r; }
__device__ __forceinline__ f2 add2(f2 a, f2 b) { f2 r; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }
__device__ __forceinline__ f2 mul2(f2 a, f2 b) { f2 r; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }
// Tensor copies: K's four chunks of 32 rows, V's two of 64 (y: pool row, z: the first chunk's parity).
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const void* map, int y, uint64_t* bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                 ::"r"(dst), "l"(map), "r"(0), "r"(y), "r"(0), "r"(tc::smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const void* map, int y, int z, uint64_t* bar) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
                 ::"r"(dst), "l"(map), "r"(0), "r"(y), "r"(0), "r"(z), "r"(tc::smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// A word of codes with 0 for NaN (bytes whose low seven bits are all up).
__device__ __forceinline__ uint32_t no_nan(uint32_t v) { return v & ~(((((v & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) >> 7) * 0xffu); }

// A walk over a run of (row block, tile) pairs. Units are numbered tile by tile, block by block, sequence by sequence.
struct Walk {
    int b, rb, t0, t1;             // sequence, row block, tiles [t0, t1) of the current segment
    long long left;                // units of the run from t0 on
    int nt, nrb;                   // tiles and row blocks of the sequence
    TreeSeq s;
};
__device__ __forceinline__ void units_of(const TreeArgs& A, const TreeSeq& s, int& nt, int& nrb) {
    nrb = (s.T * A.H + TM_BLOCK - 1) / TM_BLOCK;
    nt = s.T ? (s.n + s.T + TM_TILE - 1) / TM_TILE : 0;
}
__device__ __forceinline__ bool walk_segment(const TreeArgs& A, Walk& w) {
    if (w.left <= 0) return false;
    while (w.nrb == 0) {           // (only behind the first segment: the run begins in a sequence that has units)
        if (++w.b >= A.B) return false;
        w.s = tree_seq(A, w.b);
        units_of(A, w.s, w.nt, w.nrb);
    }
    w.t1 = (int)min((long long)w.nt, w.t0 + w.left);
    return true;
}
__device__ __forceinline__ void walk_on(const TreeArgs& A, Walk& w) {
    w.left -= w.t1 - w.t0;
    w.t0 = 0;
    if (++w.rb == w.nrb) { w.rb = 0; w.nrb = 0; }
}
// First unit of pair g's run.
__device__ __forceinline__ long long run_begin(long long total, int g, int n) { return total * g / n; }

__global__ void __launch_bounds__(TM_THREADS, 1)
tree_mma_kernel(TreeArgs A, const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap r_map, const __grid_constant__ CUtensorMap v_map, int tma, int* err,
                uint8_t* scratch, int max_polls) {
    extern __shared__ __align__(1024) uint8_t smem[];
    Bars& bars = *reinterpret_cast<Bars*>(smem + SM_BARS);
    float* s_tok = reinterpret_cast<float*>(smem + SM_TOK);
    uint4* s_see = reinterpret_cast<uint4*>(smem + SM_SEE);
    float* s_ahi = reinterpret_cast<float*>(smem + SM_AHI);
    float* s_wmax = reinterpret_cast<float*>(smem + SM_WMAX);
    float* s_fac = reinterpret_cast<float*>(smem + SM_FAC);
    float* s_mref = reinterpret_cast<float*>(smem + SM_MREF);
    uint32_t* tmem_base_s = reinterpret_cast<uint32_t*>(smem + SM_MISC);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + SM_MISC + 4);
    int* s_run = reinterpret_cast<int*>(smem + SM_MISC + 8);               // b, rb, t0 of the run's beginning, number of runs
    long long* s_units = reinterpret_cast<long long*>(smem + SM_MISC + 24);   // its units, all units

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int pair = blockIdx.x >> 1, rank = blockIdx.x & 1;               // (clusters of two along x)
    if (tid == 0) {
#pragma unroll
        for (int s = 0; s < NK; ++s) { tc::mbar_init(&bars.k_full[s], FULL); tc::mbar_init(&bars.k_peer[s], 1); tc::mbar_init(&bars.k_empty[s], 1); }
#pragma unroll
        for (int s = 0; s < NV; ++s) {
            tc::mbar_init(&bars.v_full[s], FULL); tc::mbar_init(&bars.v_peer[s], 1); tc::mbar_init(&bars.v_empty[s], 1);
            tc::mbar_init(&bars.tok_full[s], 1);
        }
#pragma unroll
        for (int s = 0; s < 2; ++s) tc::mbar_init(&bars.s_empty[s], 8);
#pragma unroll
        for (int s = 0; s < NG; ++s) { tc::mbar_init(&bars.s_full[s], 1); tc::mbar_init(&bars.p_full[s], 8); tc::mbar_init(&bars.pv_done[s], 1); tc::mbar_init(&bars.dec[s], 4); }
        tc::mbar_init(&bars.q_full, 2 * TM_SW);
        tc::mbar_init_fence();
        *abort_flag = 0;
    }
    if (warp == TM_QKW) tc::tmem_alloc2(tmem_base_s);
    tc::fence_proxy_async();
    tc::tc_fence_before();
    __syncthreads();
    cluster_sync();                                    // barriers and columns of both CTAs are there
    tc::tc_fence_after();
    const uint32_t tmem = *tmem_base_s;
    const uint32_t TM_S0 = tmem + TMC_S, TM_Q = tmem + TMC_Q, TM_O = tmem + TMC_O;
    rv_grid_dep_wait();
    rv_grid_dep_trigger();

    // ------------------------------ the pair's run -----------------------------------------------
    if (warp == 0) {
        auto scan = [&](int b, long long& inc) {   // units of sequence b, and of all of its 32 up to it
            int nt = 0, nrb = 0;
            if (b < A.B) { const TreeSeq s = tree_seq(A, b); units_of(A, s, nt, nrb); }
            const long long mine = (long long)nt * nrb;
            inc = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) { const long long v = __shfl_up_sync(0xffffffffu, inc, o); if (lane >= o) inc += v; }
            return mine;
        };
        long long total = 0, inc = 0, mine = 0;
        for (int b0 = 0; b0 < A.B; b0 += 32) { mine = scan(b0 + lane, inc); total += __shfl_sync(0xffffffffu, inc, 31); }
        const int n = (int)max(1LL, min((long long)(gridDim.x / 2), total / TM_MIN_UNITS)), g = pair;
        const long long u0 = g < n ? run_begin(total, g, n) : total, u1 = g < n ? run_begin(total, g + 1, n) : total;
        if (lane == 0) { s_units[0] = u1 - u0; s_units[1] = total; s_run[0] = A.B; s_run[1] = s_run[2] = 0; s_run[3] = n; }
        __syncwarp();
        long long before = 0;
        for (int b0 = 0; b0 < A.B && u1 > u0; b0 += 32) {
            if (A.B > 32) mine = scan(b0 + lane, inc);     // (a batch of 32 is scanned already)
            if (u0 >= before + inc - mine && u0 < before + inc) {
                int nt, nrb;
                units_of(A, tree_seq(A, b0 + lane), nt, nrb);
                const long long in = u0 - (before + inc - mine);
                s_run[0] = b0 + lane; s_run[1] = (int)(in / nt); s_run[2] = (int)(in % nt);
            }
            before += __shfl_sync(0xffffffffu, inc, 31);
        }
    }
    __syncthreads();
    Walk w;
    w.b = s_run[0]; w.rb = s_run[1]; w.t0 = s_run[2]; w.left = w.b < A.B ? s_units[0] : 0;
    w.nt = w.nrb = 0;
    if (w.left > 0) { w.s = tree_seq(A, w.b); units_of(A, w.s, w.nt, w.nrb); }

    if (warp >= TM_KW) {
        // ------------------------------ gather ---------------------------------------------------
        // Three warps fetch K (this CTA's 32 tokens of a tile) and write the scales of all 64, three fetch V, a tile in turn. None waits
        // for its copies: they signal the stage themselves. Rows past the end and on unmapped pages are written as zeros.
        // A lane resolves two tokens of a tile, 32 apart: entry -> page -> pool row -> scale, each level asked for a tile or more before it
        // is used (the loads come back through queues that the copies have filled).
        const bool is_k = warp < TM_VW;
        const int shift = rv_log2(A.page_tokens), inside = A.page_tokens - 1;
        constexpr uint32_t NONE = 0xffffffffu;
        bool ok = true;
        const int g = warp - (is_k ? TM_KW : TM_VW), depth = is_k ? NK : NV;
        int s = g, use = 0, sv = g, usev = 0;      // stage and use of it; of V's ring, whose depth the token words share
        int turn = g;                              // tiles of the next segment before this warp's first
        for (; ok && walk_segment(A, w); walk_on(A, w)) {
            const int total = w.s.n + w.s.T;
            {   // the queries of the CTA's rows on their way to L2: they are read when the softmax warps come to this segment
                const int r0 = w.rb * TM_BLOCK + rank * TM_ROWS, bytes = min(TM_ROWS, w.s.T * A.H - r0) * TM_W * 2;
                const char* at = reinterpret_cast<const char*>(A.q + ((size_t)w.s.node0 * A.H + r0) * TM_W);
#pragma unroll 1
                for (int o = ((warp - TM_KW) * 32 + lane) * 128; o < bytes; o += 2 * GW * 32 * 128) asm volatile("prefetch.global.L2 [%0];" ::"l"(at + o));
            }
            const int tj = tma && !w.s.listed ? max(w.t0, min(w.t1, w.s.n / TM_TILE)) : w.t0;   // tiles from here on are gathered
            const int32_t* table = A.block_table + (size_t)w.b * A.max_pages;
            int t = w.t0 + turn;
            // A stage of one's own ring (K: and of the token words') is free.
            auto stage_free = [&]() {
                if (usev > 0) ok = wait_for(&bars.v_empty[sv], (usev & 1) ^ 1, abort_flag, 41, max_polls);
                if (ok && is_k && use > 0) ok = wait_for(&bars.k_empty[s], (use & 1) ^ 1, abort_flag, 42, max_polls);
            };
            // scales of the lane's two tokens and which are there, to the softmax warps; the next stage
            auto stage_done = [&](const float* scl, bool mapped0, bool mapped1) {
                if (is_k) {
                    uint32_t there[2], wild[2];
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        const bool odd = !(scl[u] < INFINITY), live = (u ? mapped1 : mapped0) && !(scl[u] <= 0.0f);   // odd: NaN, or infinite
                        s_tok[sv * TM_TILE + u * 32 + lane] = !live ? 0.0f : odd ? 1.0f : scl[u];
                        there[u] = __ballot_sync(0xffffffffu, live);
                        wild[u] = __ballot_sync(0xffffffffu, live && odd);
                    }
                    if (lane == 0) s_see[sv] = make_uint4(there[0], there[1], wild[0], wild[1]);
                    __syncwarp();
                    if (lane == 0) tc::mbar_arrive(&bars.tok_full[sv]);
                }
                if ((s += GW) >= depth) { s -= depth; ++use; }
                if ((sv += GW) >= NV) { sv -= NV; ++usev; }
            };
            if (t < tj) {
                // Pages of 64 tokens and more, a tile inside one: K is two tensor copies, V is one. The page is asked for two of the warp's
                // tiles ahead, the scales one.
                auto page_of = [&](int x) -> int {
                    const int lp = x * TM_TILE >> shift, pg = x < tj && lp < A.max_pages ? table[lp] : -1;
                    return pg < A.n_pool_pages ? pg : -1;
                };
                auto row_of = [&](int x, int pg) -> uint32_t { return pg >= 0 ? (uint32_t)pg * (uint32_t)A.page_tokens + (uint32_t)(x * TM_TILE & inside) : NONE; };
                uint32_t y = row_of(t, page_of(t));
                int pg1 = page_of(t + GW);
                float scl[2] = {0.0f, 0.0f};
                if (is_k && y != NONE) { scl[0] = A.pscale[y + lane]; scl[1] = A.pscale[y + 32 + lane]; }
#pragma unroll 1
                for (; t < tj; t += GW) {
                    const uint32_t y1 = row_of(t + GW, pg1);
                    pg1 = page_of(t + 2 * GW);
                    float scl1[2] = {0.0f, 0.0f};
                    if (is_k && y1 != NONE) { scl1[0] = A.pscale[y1 + lane]; scl1[1] = A.pscale[y1 + 32 + lane]; }
                    stage_free();
                    if (!ok) break;
                    uint64_t* full = (is_k ? bars.k_full : bars.v_full) + s;
                    const uint32_t at = tc::smem_u32(smem) + (is_k ? SM_K + s * KSTAGE : SM_V + s * VSTAGE);
                    if (__builtin_expect(y == NONE, 0)) {          // a page that is not there: zeros
#pragma unroll 1
                        for (int o = lane * 16; o < (is_k ? KSTAGE : VSTAGE); o += 512)
                            asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(at + o), "r"(0) : "memory");
                        tc::fence_proxy_async();
                        __syncwarp();
                        if (lane == 0) mbar_arrive_n(full, FULL);
                    } else if (tc::elect_one()) {
                        tc::mbar_arrive_expect_tx(full, is_k ? KSTAGE : VSTAGE);
                        if (is_k) {
                            tma_load_3d(at, &k_map, (int)y + rank * TM_OWN, full);
                            tc::tma_load_2d(at + 4 * KCHUNK, &r_map, TM_KVL, (int)y + rank * TM_OWN, full);
                        } else {
                            tma_load_4d(at, &v_map, (int)y, rank, full);
                        }
                        mbar_arrive_n(full, FULL - 1);
                    }
                    __syncwarp();
                    stage_done(scl, y != NONE, y != NONE);
                    y = y1; scl[0] = scl1[0]; scl[1] = scl1[1];
                }
            }
            if (ok && t < w.t1) {
                // A lane resolves two tokens of a tile, 32 apart: entry -> page -> pool row -> scale, each level asked for one of the warp's
                // tiles or more before it is used (the loads come back through queues that the copies have filled).
                auto entry = [&](int x, int u) -> uint32_t {
                    const int j = x * TM_TILE + u * 32 + lane;
                    return x < w.t1 && j < total ? tree_token(A, w.s, w.b, j) : NONE;
                };
                auto page = [&](uint32_t tok) -> int { return tok != NONE && (tok >> shift) < (uint32_t)A.max_pages ? table[tok >> shift] : -1; };
                auto pool_row = [&](uint32_t tok, int pg) -> uint32_t {
                    return pg >= 0 && pg < A.n_pool_pages ? (uint32_t)pg * (uint32_t)A.page_tokens + (tok & (uint32_t)inside) : NONE;
                };
                auto scale = [&](uint32_t r) -> float { return is_k && r != NONE ? A.pscale[r] : 0.0f; };
                uint32_t row[2], row1[2], tok2[2];     // pool rows of this warp's tile t and its next; entries of the one after
                float scl[2];
#pragma unroll
                for (int u = 0; u < 2; ++u) { row[u] = entry(t, u); row1[u] = entry(t + GW, u); tok2[u] = entry(t + 2 * GW, u); }
#pragma unroll
                for (int u = 0; u < 2; ++u) { row[u] = pool_row(row[u], page(row[u])); row1[u] = pool_row(row1[u], page(row1[u])); }
#pragma unroll
                for (int u = 0; u < 2; ++u) scl[u] = scale(row[u]);
                const int c = lane & 15;               // V: two rows an instruction, 16 chunks each
                const uint8_t* from = A.pool + (is_k ? lane * 16 : (2 * (c >> 3) + rank) * 128 + (c & 7) * 16);
                const uint32_t to = is_k ? (lane >> 3) * KCHUNK : (c >> 3) * VCHUNK + (lane >> 4) * 128;
#pragma unroll 1
                for (; t < w.t1; t += GW) {
                    float scl1[2];
                    int pg2[2];
                    uint32_t tok3[2];
#pragma unroll
                    for (int u = 0; u < 2; ++u) { scl1[u] = scale(row1[u]); pg2[u] = page(tok2[u]); tok3[u] = entry(t + 3 * GW, u); }
                    stage_free();
                    if (!ok) break;
                    uint64_t* full = (is_k ? bars.k_full : bars.v_full) + s;
                    const uint32_t at = tc::smem_u32(smem) + (is_k ? SM_K + s * KSTAGE : SM_V + s * VSTAGE);
                    const uint32_t first = is_k && rank ? row[1] : row[0];
#pragma unroll 4
                    for (int it = 0; it < 32; ++it) {
                        const int rl = is_k ? it : 2 * it + (lane >> 4);
                        const uint32_t r = __shfl_sync(0xffffffffu, is_k || it < 16 ? first : row[1], rl & 31);
                        tc::cp_async16_zfill(at + to + (is_k ? it * 128 : it * 256) + (((lane ^ rl) & 7) << 4), r != NONE ? from + (size_t)r * TM_W : A.pool, r != NONE ? 16u : 0u);
                    }
                    if (is_k) {
#pragma unroll 1
                        for (int it = 0; it < 4; ++it) {
                            const int rl = it * 8 + (lane >> 2);
                            const uint32_t r = __shfl_sync(0xffffffffu, first, rl);
                            tc::cp_async16_zfill(at + 4 * KCHUNK + sw64_chunk(rl, lane & 3),
                                                 A.pool + (r != NONE ? (size_t)r * TM_W + TM_KVL + (lane & 3) * 16 : 0), r != NONE ? 16u : 0u);
                        }
                    } else if ((t + 1) * TM_TILE > w.s.n) {
                        // rows of the tree: each lane looks through what it copied itself, once it is there
                        tc::cp_async_commit();
                        tc::cp_async_wait<0>();
                        uint8_t* buf = smem + SM_V + s * VSTAGE + (c >> 3) * VCHUNK;
#pragma unroll 2
                        for (int it = 0; it < 32; ++it) {
                            const int rl = 2 * it + (lane >> 4);
                            uint4* v = reinterpret_cast<uint4*>(buf + tc::sw128_chunk(rl, c & 7));
                            if (t * TM_TILE + rl >= w.s.n) { const uint4 x = *v; *v = make_uint4(no_nan(x.x), no_nan(x.y), no_nan(x.z), no_nan(x.w)); }
                        }
                    }
                    tc::cp_async_mbar_arrive_noinc(full);
                    tc::fence_proxy_async();
                    __syncwarp();
                    if (lane == 0) tc::mbar_arrive(full);
                    stage_done(scl, row[0] != NONE, row[1] != NONE);
#pragma unroll
                    for (int u = 0; u < 2; ++u) { row[u] = row1[u]; scl[u] = scl1[u]; row1[u] = pool_row(tok2[u], pg2[u]); tok2[u] = tok3[u]; }
                }
            }
            turn = t - w.t1;
        }
    } else if (warp == TM_QKW || warp == TM_PVW) {
        if (rank == 1) {
            // ------------------------------ the second CTA: its stages are full -------------------
            uint64_t* full = warp == TM_QKW ? bars.k_full : bars.v_full;
            const uint32_t peer = in_first(warp == TM_QKW ? bars.k_peer : bars.v_peer);
            const int stages = warp == TM_QKW ? NK : NV;
            bool ok = true;
            int s = 0, phase = 0;
            for (; ok && walk_segment(A, w); walk_on(A, w))
                for (int t = w.t0; t < w.t1; ++t) {
                    ok = wait_for(&full[s], phase, abort_flag, 57, max_polls);
                    if (!ok) break;
                    tc::fence_proxy_async();
                    if (lane == 0) arrive_first(peer + s * 8);
                    if (++s == stages) { s = 0; phase ^= 1; }
                }
        } else if (warp == TM_QKW) {
            // ------------------------------ QK issuer: S(i) = Q . K(i)^T -------------------------
            const uint32_t id_qk = tc::idesc_e4m3(256, TM_TILE, 0, 0);
            const uint64_t d_qr = smem_desc(tc::smem_u32(smem + SM_QR), 16, 512, 4);
            bool ok = true;
            int i = 0, seg = 0, s = 0, phase = 0, g = 0;
            for (; ok && walk_segment(A, w); walk_on(A, w), ++seg) {
                ok = wait_for(&bars.q_full, seg & 1, abort_flag, 51, max_polls);
#pragma unroll 1
                for (int t = w.t0; t < w.t1 && ok; ++t, ++i) {
                    const int sb = i & 1;
                    ok = wait_for(&bars.k_full[s], phase, abort_flag, 52, max_polls) && wait_for(&bars.k_peer[s], phase, abort_flag, 56, max_polls) &&
                         wait_for(&bars.s_empty[sb], ((i >> 1) & 1) ^ 1, abort_flag, 53, max_polls);
                    if (!ok) break;
                    tc::fence_proxy_async();   // copies that wrote through the generic proxy, the products read through the async one
                    tc::tc_fence_after();
                    const uint64_t d_k = smem_desc(tc::smem_u32(smem + SM_K + s * KSTAGE), 16, 1024, 2);
                    const uint64_t d_rope = smem_desc(tc::smem_u32(smem + SM_K + s * KSTAGE + 4 * KCHUNK), 16, 512, 4);
                    const uint32_t d = TM_S0 + sb * TM_TILE;
                    if (tc::elect_one()) {
#pragma unroll
                        for (int k = 0; k < 2; ++k) tc::mma2_f8(d, d_qr + (uint64_t)(k * 2), d_rope + (uint64_t)(k * 2), id_qk, k != 0);
#pragma unroll
                        for (int c = 0; c < 4; ++c)
#pragma unroll
                            for (int k = 0; k < 4; ++k)
                                tc::mma2_f8_ta(d, TM_Q + (uint32_t)(c * 32 + k * 8), d_k + (uint64_t)((c * KCHUNK + k * 32) >> 4), id_qk, 1);
                        tc::commit2(&bars.k_empty[s]);
                        tc::commit2(&bars.s_full[g]);
                    }
                    __syncwarp();
                    if (++s == NK) { s = 0; phase ^= 1; }
                    if (++g == NG) g = 0;
                }
            }
        } else {
            // ------------------------------ PV issuer: O += P'(i) . V(i) --------------------------
            const uint32_t id_pv = tc::idesc_e4m3(128, 256, 0, 1);
            bool ok = true;
            int s = 0, phase = 0, pb = 0, p_phase = 0;
            for (; ok && walk_segment(A, w); walk_on(A, w)) {
#pragma unroll 1
                for (int t = w.t0; t < w.t1 && ok; ++t) {
                    ok = wait_for(&bars.v_full[s], phase, abort_flag, 58, max_polls) && wait_for(&bars.v_peer[s], phase, abort_flag, 59, max_polls) &&
                         wait_for(&bars.p_full[pb], p_phase, abort_flag, 54, max_polls);
                    if (!ok) break;
                    tc::fence_proxy_async();
                    tc::tc_fence_after();
                    const uint64_t d_v = smem_desc(tc::smem_u32(smem + SM_V + s * VSTAGE), VCHUNK, 1024, 2);
                    const uint64_t d_p = smem_desc(tc::smem_u32(smem + SM_P + pb * PBUF), 16, 512, 4);
                    if (tc::elect_one()) {
#pragma unroll
                        for (int c = 0; c < 2; ++c)
#pragma unroll
                            for (int k = 0; k < 4; ++k)        // p_hi, then p_lo, 32 tokens each time
                                tc::mma2_f8(TM_O + c * 128, d_p + (uint64_t)(((k >> 1) * PTERM >> 4) + (k & 1) * 2), d_v + (uint64_t)((c * VCHUNK + (k & 1) * 4096) >> 4), id_pv,
                                        t > w.t0 || k != 0);
                        tc::commit2(&bars.v_empty[s]);
                        tc::commit2(&bars.pv_done[pb]);
                    }
                    __syncwarp();
                    if (++s == NV) { s = 0; phase ^= 1; }
                    if (++pb == NG) { pb = 0; p_phase ^= 1; }
                }
            }
        }
    } else {
        // ------------------------------ queries, softmax, epilogue -------------------------------
        // S: lanes 0-15 of a warp's quarter hold the hi terms of 16 rows, lanes 16-31 their lo terms. Read 16 lanes at a time in the
        // fragment form (a thread gets two neighbouring columns of rows lane / 4 and lane / 4 + 8 per eight columns), hi and lo come to the
        // same registers of the same thread: the sum takes no exchange. A thread has 16 tokens of two rows.
        // O: lanes 0-63 hold rows 0-63 in columns 0-127 of each 256 dims, lanes 64-127 the same rows in the other 128.
        const int sq = warp & 3, th = warp >> 2, tb = lane >> 4;
        const int hd = 16 * sq + (lane & 15);              // a row of the conversion and of the epilogue's sums
        const int ra = 16 * sq + (lane >> 2), rb = ra + 8, tq = 2 * (lane & 3);   // rows and first token of the scores
        const int orow = (sq * 32 + lane) & 63;            // O: this thread's row
        const uint32_t lane_base = ((uint32_t)(sq * 32)) << 16;
        const uint32_t q_full = in_first(&bars.q_full), s_empty = in_first(bars.s_empty), p_full = in_first(bars.p_full);
        auto give_up = [&]() { (void)tc::barrier_any(6 + th, TM_GROUP, true); (void)tc::barrier_any(9 + th, TM_GROUP, true); };
        // O has taken tile i. A parity tells a phase from the one before it only: a group asks for its own tile first, whose predecessor
        // in the barrier it has seen, and then for another's within the NG behind it.
        auto pv_done = [&](int i) { return wait_for(&bars.pv_done[i % NG], (i / NG) & 1, abort_flag, 63, max_polls); };
        int i0 = 0;                                        // tiles of the pair before this segment
        bool failed = false;
        for (; !failed && walk_segment(A, w); i0 += w.t1 - w.t0, walk_on(A, w)) {
            const int rows_all = w.s.T * A.H, r0 = w.rb * TM_BLOCK + rank * TM_ROWS, valid = max(0, min(TM_ROWS, rows_all - r0));
            const size_t flat = (size_t)w.s.node0 * A.H + r0;      // first row of the CTA in q, out and out_lse
            // ---- q -> two e4m3 terms per row: hi = e4m3(q / s), s = absmax / 448, lo = e4m3(q / s - hi) ----
            // A warp of the first two groups takes sixteen rows and half th of their columns. They arrive as whole 128-byte lines (lanes 8 k .. 8 k + 7 on one row),
            // are split there and go through shared memory, 64 columns at a time, to the lanes whose tensor-memory row they are. (A
            // lane reading its own row, a line per load, waited 10,500 cycles for them.)
            {
                const uint16_t* q0 = A.q + flat * TM_W;
                uint4 v[18];
                const int rq = 16 * sq + (lane >> 3), xq = 16 * sq + (lane >> 2);          // rows of a latent, of a rope load
#pragma unroll
                for (int c = 0; c < 4; ++c)
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const int r = rq + 4 * k;
                        v[4 * c + k] = r < valid && th < 2 ? *reinterpret_cast<const uint4*>(q0 + (size_t)r * TM_W + th * (TM_KVL / 2) + c * 64 + (lane & 7) * 8) : make_uint4(0u, 0u, 0u, 0u);
                    }
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const int r = xq + 8 * k;
                    v[16 + k] = r < valid && th < 2 ? *reinterpret_cast<const uint4*>(q0 + (size_t)r * TM_W + TM_KVL + th * (TM_ROPE / 2) + (lane & 3) * 8) : make_uint4(0u, 0u, 0u, 0u);
                }
                // largest magnitudes: of latent rows 4 k + lane / 8 and rope rows 8 k + lane / 4, then of row lane % 16
                uint32_t ml4[4], mx2[2];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    ml4[k] = rv_max_bf16x2(rv_max_bf16x2(rv_absmax8(v[k]), rv_absmax8(v[4 + k])), rv_max_bf16x2(rv_absmax8(v[8 + k]), rv_absmax8(v[12 + k])));
#pragma unroll
                    for (int o = 1; o < 8; o <<= 1) ml4[k] = rv_max_bf16x2(ml4[k], __shfl_xor_sync(0xffffffffu, ml4[k], o));
                }
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    mx2[k] = rv_absmax8(v[16 + k]);
#pragma unroll
                    for (int o = 1; o < 4; o <<= 1) mx2[k] = rv_max_bf16x2(mx2[k], __shfl_xor_sync(0xffffffffu, mx2[k], o));
                }
                {
                    const int r = lane & 15;
                    uint32_t a = 0u, x = 0u;
#pragma unroll
                    for (int k = 0; k < 4; ++k) { const uint32_t y = __shfl_sync(0xffffffffu, ml4[k], 8 * (r & 3)); if ((r >> 2) == k) a = y; }
#pragma unroll
                    for (int k = 0; k < 2; ++k) { const uint32_t y = __shfl_sync(0xffffffffu, mx2[k], 4 * (r & 7)); if ((r >> 3) == k) x = y; }
                    if (lane < 16 && th < 2) s_wmax[th * 64 + hd] = __uint_as_float(rv_max_bf16x2(a, x) << 16);
                }
                tc::named_barrier(3, TM_SOFTMAX);          // (also: all groups are through with the block before)
                auto scale_of = [&](int r) { const float amax = fmaxf(s_wmax[r], s_wmax[64 + r]); return amax > 0.0f ? amax / 448.0f : 1.0f; };
                if (th == 0 && tb == 0) { s_ahi[hd] = scale_of(hd) * A.softmax_scale * 1.4426950408889634f; s_mref[hd] = -INFINITY; }
                auto codes8 = [&](const uint4 x, float inv, uint2& hi, uint2& lo) {
                    const uint32_t ww[4] = {x.x, x.y, x.z, x.w};
                    uint16_t ch[4], cl[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const float x0 = __uint_as_float(ww[k] << 16) * inv, x1 = __uint_as_float(ww[k] & 0xffff0000u) * inv;
                        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(ch[k]) : "f"(x1), "f"(x0));
                        const float2 xh = rv_e4m3x2_to_f32x2(ch[k]);
                        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(cl[k]) : "f"(x1 - xh.y), "f"(x0 - xh.x));
                    }
                    hi = make_uint2((uint32_t)ch[0] | ((uint32_t)ch[1] << 16), (uint32_t)ch[2] | ((uint32_t)ch[3] << 16));
                    lo = make_uint2((uint32_t)cl[0] | ((uint32_t)cl[1] << 16), (uint32_t)cl[2] | ((uint32_t)cl[3] << 16));
                };
                // 64 codes of 32 virtual rows (hi 0-15, lo 16-31) in this warp's 2 KiB of the idle P' buffers, 16-byte chunks swizzled by row
                uint8_t* buf = smem + SM_P + (warp & 7) * 2048;
                auto spot = [&](int r, int byte) { return buf + r * 64 + ((((byte >> 4) ^ (r >> 1)) & 3) << 4) + (byte & 15); };
                if (th < 2) {
                    const uint32_t dst = TM_Q + lane_base + th * 64;
                    float inv4[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) inv4[k] = 1.0f / scale_of(rq + 4 * k);
#pragma unroll 1
                    for (int c = 0; c < 4; ++c) {              // (a loop: code that runs once is waited for)
                        __syncwarp();
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            uint2 hi, lo;
                            codes8(v[k], inv4[k], hi, lo);
                            const int r = 4 * k + (lane >> 3);
                            *reinterpret_cast<uint2*>(spot(r, (lane & 7) * 8)) = hi;
                            *reinterpret_cast<uint2*>(spot(16 + r, (lane & 7) * 8)) = lo;
                        }
                        __syncwarp();
                        uint32_t a[16];
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const uint4 x = *reinterpret_cast<const uint4*>(spot(lane, 16 * k));
                            a[4 * k] = x.x; a[4 * k + 1] = x.y; a[4 * k + 2] = x.z; a[4 * k + 3] = x.w;
                        }
                        tc::tmem_st8(dst + c * 16, a);
                        tc::tmem_st8(dst + c * 16 + 8, a + 8);
#pragma unroll
                        for (int k = 0; k < 14; ++k) v[k] = v[k + 4];
                    }
#pragma unroll
                    for (int k = 0; k < 2; ++k) {              // rope columns: straight to the operand tile, eight codes at a time
                        const int r = 8 * k + (lane >> 2);
                        uint2 hi, lo;
                        codes8(v[k], 1.0f / scale_of(16 * sq + r), hi, lo);
                        const int col = th * 32 + (lane & 3) * 8;
                        *reinterpret_cast<uint2*>(smem + SM_QR + sw64_chunk(sq * 32 + r, col >> 4) + (col & 15)) = hi;
                        *reinterpret_cast<uint2*>(smem + SM_QR + sw64_chunk(sq * 32 + 16 + r, col >> 4) + (col & 15)) = lo;
                    }
                }
                tc::tmem_st_wait();
                tc::fence_proxy_async();
                tc::tc_fence_before();
                __syncwarp();
                if (lane == 0) arrive_first(q_full);
                tc::named_barrier(3, TM_SOFTMAX);          // the row scales and references are read by other warps than wrote them
            }

            // ---- the tiles ----
            const float a_a = s_ahi[ra], a_b = s_ahi[rb];
            float l_a = 0.0f, l_b = 0.0f, m_a = -INFINITY, m_b = -INFINITY;   // sums, and the references they are at
            const int i1 = i0 + (w.t1 - w.t0);
            bool ok = true;
            int i = i0 + (th + 2 * NG - i0 % NG) % NG;
            int n = i / NG, sv = i % NV, usev = i / NV;    // the group's tiles before; slot and use of the token words
#pragma unroll 1
            for (; i < i1; i += NG, ++n, usev += sv >= NV - NG, sv += sv >= NV - NG ? NG - NV : NG) {
                const int j0 = (w.t0 + i - i0) * TM_TILE, sb = i & 1;
                ok = wait_for(&bars.tok_full[sv], usev & 1, abort_flag, 61, max_polls) && wait_for(&bars.s_full[th], n & 1, abort_flag, 62, max_polls);
                if (!ok) { give_up(); break; }
                tc::tc_fence_after();
                // x: scores in log2 units; [k][row][token tq + e] of each run k of eight tokens
                f2 x[16];
                const f2* sc = reinterpret_cast<const f2*>(s_tok + sv * TM_TILE + tq);   // [4 k]: scales of run k's two tokens
                const uint32_t s_at = TM_S0 + sb * TM_TILE + lane_base;
#pragma unroll
                for (int hf = 0; hf < 2; ++hf) {
                    uint32_t hi[16], lo[16];
                    tc::tmem_ld16x256(s_at + 32 * hf, hi);
                    tc::tmem_ld16x256(s_at + (16u << 16) + 32 * hf, lo);
                    tc::tmem_ld_wait();
                    if (hf == 1) {
                        tc::tc_fence_before();
                        __syncwarp();
                        if (lane == 0) arrive_first(s_empty + sb * 8);
                    }
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        x[8 * hf + j] = add2(pack(__uint_as_float(hi[2 * j]), __uint_as_float(hi[2 * j + 1])), pack(__uint_as_float(lo[2 * j]), __uint_as_float(lo[2 * j + 1])));
                }
                const uint4 see = s_see[sv];
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const f2 c = sc[4 * k];
                    x[2 * k] = mul2(x[2 * k], mul2(pack(a_a, a_a), c));
                    x[2 * k + 1] = mul2(x[2 * k + 1], mul2(pack(a_b, a_b), c));
                }
                if (__builtin_expect(j0 + TM_TILE > w.s.n || (see.x & see.y) != ~0u || (see.z | see.w), 0)) {
                    // rows of the tree, rows that are not there, scales that are no numbers: what a node does not see scores -inf
                    const uint64_t mask_a = ra < valid ? A.node_mask[w.s.node0 + (r0 + ra) / A.H] : 0ull, mask_b = rb < valid ? A.node_mask[w.s.node0 + (r0 + rb) / A.H] : 0ull;
                    const uint64_t there = (uint64_t)see.y << 32 | see.x, wild = ((uint64_t)see.w << 32 | see.z) >> tq;
                    const uint64_t va = (tree_visible(mask_a, w.s.T, w.s.n, j0) & there) >> tq, vb = (tree_visible(mask_b, w.s.T, w.s.n, j0) & there) >> tq;
#pragma unroll
                    for (int k = 0; k < 16; ++k) {
                        const uint64_t v = (k & 1) ? vb : va;
                        float2 y = unpack(x[k]);
                        const int bit = 8 * (k >> 1);
                        y.x = !((v >> bit) & 1) ? -INFINITY : (wild >> bit) & 1 ? NAN : y.x;
                        y.y = !((v >> (bit + 1)) & 1) ? -INFINITY : (wild >> (bit + 1)) & 1 ? NAN : y.y;
                        x[k] = pack(y.x, y.y);
                    }
                }
                // The weights at the references as they were a tile or two ago, before it is known whether those stand: they nearly always
                // do, and what is waited for meanwhile passes. If not, once more.
                uint32_t hi_w[8], lo_w[8];                 // codes of the pairs of run k: row a's in the low half, row b's in the high one
                float lt_a, lt_b;
                bool again = false, left = false;
#pragma unroll 1
                for (;;) {
                    // P' = 2^(x - ref + 5) * scale as two e4m3 terms (through f16); the sums take 2^(x - ref + 5)
                    const float ka = m_a == -INFINITY ? 0.0f : TM_POFF - m_a, kb = m_b == -INFINITY ? 0.0f : TM_POFF - m_b;
                    f2 la = 0ull, lb = 0ull;
                    __half2 top = __float2half2_rn(0.0f);
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        const volatile f2* cv = sc;
                        const f2 c8 = cv[4 * k];
                        uint32_t ch[2], cl[2];
#pragma unroll
                        for (int r = 0; r < 2; ++r) {
                            const float2 t = unpack(add2(x[2 * k + r], r ? pack(kb, kb) : pack(ka, ka)));
                            float w0, w1;
                            asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(w0) : "f"(t.x));
                            asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(w1) : "f"(t.y));
                            const f2 ww = pack(w0, w1);
                            if (r) lb = add2(lb, ww); else la = add2(la, ww);
                            const float2 p = unpack(mul2(ww, c8));
                            const __half2 ph = __floats2half2_rn(p.x, p.y);
                            top = __hmax2(top, ph);
                            const uint32_t phb = *reinterpret_cast<const uint32_t*>(&ph);
                            uint16_t c, d;
                            uint32_t back;
                            asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(c) : "r"(phb));
                            asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(back) : "h"(c));
                            const __half2 rest = __hsub2(ph, *reinterpret_cast<const __half2*>(&back));
                            asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(d) : "r"(*reinterpret_cast<const uint32_t*>(&rest)));
                            ch[r] = c; cl[r] = d;
                        }
                        hi_w[k] = ch[0] | (ch[1] << 16);
                        lo_w[k] = cl[0] | (cl[1] << 16);
                    }
                    const float2 sa = unpack(la), sbb = unpack(lb);
                    lt_a = sa.x + sa.y; lt_b = sbb.x + sbb.y;
                    if (again) break;
                    const float was_a = m_a, was_b = m_b;
                    // the references as the tile before left them (another group's)
                    const int gb = th ? th - 1 : NG - 1;
                    if (i > i0) {
                        ok = wait_for(&bars.dec[gb], (n & 1) ^ (th == 0), abort_flag, 65, max_polls);
                        const float na = s_mref[ra], nb = s_mref[rb];
                        if (na != m_a) { l_a *= exp2f(m_a - na); m_a = na; }
                        if (nb != m_b) { l_b *= exp2f(m_b - nb); m_b = nb; }
                    }
                    // They stand as long as no P' exceeds 2^(5 + 3) by them (one barrier with an OR). One that has moved meanwhile brings the
                    // P' of before down with it; rows that have none yet are looked at.
                    const float2 t2 = __half22float2(top);
                    float most = fmaxf(t2.x, t2.y);
                    if (m_a != was_a || m_b != was_b) most *= fmaxf(exp2f(was_a - m_a), exp2f(was_b - m_b));
                    const bool grown = most > TM_MOST || was_a == -INFINITY || was_b == -INFINITY;
                    if (__builtin_expect(tc::barrier_any(6 + th, TM_GROUP, grown || !ok), 0)) {
                        // the largest x + log2(scale) of a row is what P' goes by
                        float ta = -INFINITY, tb2 = -INFINITY;
#pragma unroll
                        for (int k = 0; k < 8; ++k) {
                            const float2 s2 = unpack(sc[4 * k]), ya = unpack(x[2 * k]), yb = unpack(x[2 * k + 1]);
                            const float g0 = __log2f(s2.x), g1 = __log2f(s2.y);
                            ta = fmaxf(ta, fmaxf(ya.x + g0, ya.y + g1)); tb2 = fmaxf(tb2, fmaxf(yb.x + g0, yb.y + g1));
                        }
#pragma unroll
                        for (int o = 1; o < 4; o <<= 1) { ta = fmaxf(ta, __shfl_xor_sync(0xffffffffu, ta, o)); tb2 = fmaxf(tb2, __shfl_xor_sync(0xffffffffu, tb2, o)); }
                        // all references take all of their growth (taken by those alone that had to, the next tile's row would have to)
                        auto move = [](float& m, float top_now) -> float {
                            float f = 1.0f;
                            if (m == -INFINITY) { if (top_now > -INFINITY) m = top_now; }
                            else if (top_now > m) { f = exp2f(m - top_now); m = top_now; }
                            return f;
                        };
                        const float fa = move(m_a, ta), fb = move(m_b, tb2);
                        if (tq == 0) { s_fac[ra] = fa; s_mref[ra] = m_a; s_fac[rb] = fb; s_mref[rb] = m_b; }
                        left = tc::barrier_any(9 + th, TM_GROUP, !ok);
                        const float f = s_fac[orow];
                        if (!left && i > i0 && __any_sync(0xffffffffu, f != 1.0f)) {       // O to the new references
                            if (i >= i0 + NG) ok = pv_done(i - NG);
                            if (ok) ok = pv_done(i - 1);
                            tc::tc_fence_after();
                            uint32_t r[32];
#pragma unroll 1
                            for (int c = 0; c < 8; ++c) {
                                tc::tmem_ld32(TM_O + lane_base + c * 32, r);
                                tc::tmem_ld_wait();
#pragma unroll
                                for (int h = 0; h < 32; ++h) r[h] = __float_as_uint(__uint_as_float(r[h]) * f);
                                tc::tmem_st32(TM_O + lane_base + c * 32, r);
                            }
                            tc::tmem_st_wait();
                            tc::tc_fence_before();
                        }
                        l_a *= fa; l_b *= fb;
                    }
                    __syncwarp();
                    if (left) break;
                    if (lane == 0) tc::mbar_arrive(&bars.dec[th]);
                    if (!__any_sync(0xffffffffu, m_a != was_a || m_b != was_b)) break;
                    again = true;
                }
                if (left) { ok = false; break; }                   // (the group has agreed on it)
                if (ok && i >= i0 + NG) ok = pv_done(i - NG);      // the buffer was read by the products of this group's tile before
                if (!ok) { if (i + NG < i1) give_up(); break; }
                l_a += lt_a; l_b += lt_b;
                {
                    uint8_t* prow = smem + SM_P + th * PBUF + ra * 64 + tq;
                    const int sx = (ra >> 1) & 3;              // (the same for row b, 512 bytes on)
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        uint8_t* at = prow + ((((k >> 1) ^ sx) << 4) + (k & 1) * 8);
                        *reinterpret_cast<uint16_t*>(at) = (uint16_t)hi_w[k];
                        *reinterpret_cast<uint16_t*>(at + 512) = (uint16_t)(hi_w[k] >> 16);
                        *reinterpret_cast<uint16_t*>(at + PTERM) = (uint16_t)lo_w[k];
                        *reinterpret_cast<uint16_t*>(at + PTERM + 512) = (uint16_t)(lo_w[k] >> 16);
                    }
                }
                tc::fence_proxy_async();
                __syncwarp();
                if (lane == 0) arrive_first(p_full + th * 8);
            }

            // ---- epilogue of the segment ----
            // l per row: its eight threads (four neighbouring lanes in a warp of each group) meet at the last reference
            const int own = i1 - 1 - (i1 - 1 - th + NG) % NG;  // this group's last tile
            if (ok && own >= i0) ok = pv_done(own);
            if (ok) ok = pv_done(i1 - 1);
            failed = tc::barrier_any(1, TM_SOFTMAX, !ok);  // (all leave the loop over segments together)
            const float m_last = s_mref[hd];
            {
                const float na = s_mref[ra], nb = s_mref[rb];
                if (na != m_a) l_a *= exp2f(m_a - na);
                if (nb != m_b) l_b *= exp2f(m_b - nb);
#pragma unroll
                for (int o = 1; o < 4; o <<= 1) { l_a += __shfl_xor_sync(0xffffffffu, l_a, o); l_b += __shfl_xor_sync(0xffffffffu, l_b, o); }
                if (tq == 0) { s_wmax[th * 64 + ra] = l_a; s_wmax[th * 64 + rb] = l_b; }
            }
            tc::named_barrier(1, TM_SOFTMAX);
            tc::tc_fence_after();
            const bool whole = w.t0 == 0 && w.t1 == w.nt;
            const int slot = 2 * pair + (w.t0 == 0 ? 1 : 0);
            if (th == 0 && lane < 16) {
                // (l and O carry 2^5; NaN stays NaN)
                const float l = s_wmax[hd] + s_wmax[64 + hd];
                if (!whole) reinterpret_cast<float2*>(scratch + SC_ML)[slot * TM_BLOCK + rank * TM_ROWS + hd] = make_float2(m_last, l);
                else if (hd < valid && A.out_lse) A.out_lse[flat + hd] = l == 0.0f ? -INFINITY : (m_last - TM_POFF) * 0.6931471805599453f + logf(l);
                s_fac[hd] = l == 0.0f ? 0.0f : 1.0f / l;
            }
            tc::named_barrier(1, TM_SOFTMAX);              // (the sums are read: the next block's maxima take their place)
            {
                // a row's 32 columns at a time: 64 bytes of bf16, or a part's 128 of f32 as they are, for the joining kernel
                const float inv_l = s_fac[orow];
                float* po = reinterpret_cast<float*>(scratch + SC_O) + ((size_t)slot * TM_BLOCK + rank * TM_ROWS + orow) * TM_KVL;
                uint16_t* to = A.out + (flat + orow) * TM_KVL;
#pragma unroll 1
                for (int c = th; c < 8; c += NG) {
                    const int dim = 256 * (c >> 2) + 128 * (sq >> 1) + 32 * (c & 3);
                    uint32_t r[32];
                    tc::tmem_ld32(TM_O + lane_base + c * 32, r);
                    tc::tmem_ld_wait();
                    if (!whole) {
#pragma unroll
                        for (int k = 0; k < 8; ++k) *reinterpret_cast<uint4*>(po + dim + 4 * k) = make_uint4(r[4 * k], r[4 * k + 1], r[4 * k + 2], r[4 * k + 3]);
                    } else if (orow < valid) {
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            uint32_t p[4];
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(p[e]) : "f"(__uint_as_float(r[8 * k + 2 * e + 1]) * inv_l), "f"(__uint_as_float(r[8 * k + 2 * e]) * inv_l));
                            *reinterpret_cast<uint4*>(to + dim + 8 * k) = make_uint4(p[0], p[1], p[2], p[3]);
                        }
                    }
                }
            }
            if (!whole && w.t0 == 0 && tid == 0 && rank == 0) {
                // this pair has the block's beginning: which runs hold the rest
                const long long total = s_units[1], end = run_begin(total, pair + 1, s_run[3]) + (w.nt - w.t1) - 1;   // the block's last unit
                int last = (int)(end * s_run[3] / total);
                while (run_begin(total, last + 1, s_run[3]) <= end) ++last;
                Head h{(int32_t)flat, min(TM_BLOCK, rows_all - r0), last - pair + 1, 0};
                reinterpret_cast<Head*>(scratch + SC_HEAD)[pair] = h;
                w.left = -1;                               // (told; the walk ends here in any case)
            }
            tc::tc_fence_before();
        }
        // no block begins in this run and ends in another: nothing for the joining kernel
        if (tid == 0 && rank == 0 && w.left >= 0) {
            Head h{0, 0, 0, 0};
            reinterpret_cast<Head*>(scratch + SC_HEAD)[pair] = h;
        }
    }

    tc::tc_fence_before();
    __syncthreads();
    if (warp == TM_QKW) tc::settle(*abort_flag);
    __syncthreads();
    cluster_sync();                                    // neither CTA leaves while the other's products may read its shared memory
    if (warp == TM_QKW) {
        tc::settle(*abort_flag);
        tc::tmem_dealloc2(tmem);
    }
    if (tid == 0 && *abort_flag) atomicCAS(err, 0, *abort_flag);
}

// Joins the parts of the row block whose beginning pair blockIdx.x of the kernel before left, eight of its rows per block: a warp per row.
__global__ void __launch_bounds__(256)
tree_join_kernel(const uint8_t* scratch, uint16_t* out, float* out_lse) {
    rv_grid_dep_wait();
    rv_grid_dep_trigger();
    const int g = blockIdx.x, row = blockIdx.y * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    const Head h = reinterpret_cast<const Head*>(scratch + SC_HEAD)[g];
    if (row >= h.valid) return;
    auto slot = [&](int p) { return p == 0 ? 2 * g + 1 : 2 * (g + p); };
    const float2* ml = reinterpret_cast<const float2*>(scratch + SC_ML);
    float m = -INFINITY, l = 0.0f;
    for (int p = 0; p < h.parts; ++p) m = fmaxf(m, ml[slot(p) * TM_BLOCK + row].x);
    float4 acc[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) acc[c] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int p = 0; p < h.parts; ++p) {
        const float2 part = ml[slot(p) * TM_BLOCK + row];
        if (part.x == -INFINITY && part.y == 0.0f) continue;       // the part saw nothing
        const float f = exp2f(part.x - m);
        l += part.y * f;
        const float4* o = reinterpret_cast<const float4*>(scratch + SC_O) + ((size_t)slot(p) * TM_BLOCK + row) * (TM_KVL / 4);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const float4 x = o[c * 32 + lane];
            acc[c].x = fmaf(x.x, f, acc[c].x); acc[c].y = fmaf(x.y, f, acc[c].y);
            acc[c].z = fmaf(x.z, f, acc[c].z); acc[c].w = fmaf(x.w, f, acc[c].w);
        }
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    uint2* to = reinterpret_cast<uint2*>(out + ((size_t)h.row0 + row) * TM_KVL);
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        uint2 v;
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(v.x) : "f"(acc[c].y * inv), "f"(acc[c].x * inv));
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(v.y) : "f"(acc[c].w * inv), "f"(acc[c].z * inv));
        to[c * 32 + lane] = v;
    }
    if (out_lse && lane == 0) out_lse[h.row0 + row] = l == 0.0f ? -INFINITY : (m - TM_POFF) * 0.6931471805599453f + logf(l);
}

}  // namespace

bool rv_tree_mma_supported(const DsaGeom* g) { return g->kv_lora == TM_KVL && g->rope_dim == TM_ROPE; }
size_t rv_tree_mma_scratch_bytes() { return SC_TOTAL; }

// Pairs that are resident at once: their runs are as long as each other, and a pair that had to wait for another's SMs would double the time.
static int tree_pairs() {
    static std::atomic<int> known{0};
    int n = known.load(std::memory_order_relaxed);
    if (n) return n;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(RV_SMS); cfg.blockDim = dim3(TM_THREADS); cfg.dynamicSmemBytes = SM_TOTAL;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = 2; at[0].val.clusterDim.y = 1; at[0].val.clusterDim.z = 1;
    cfg.attrs = at; cfg.numAttrs = 1;
    if (cudaOccupancyMaxActiveClusters(&n, tree_mma_kernel, &cfg) != cudaSuccess || n <= 0) {
        (void)cudaGetLastError();
        return rv_sm_count() / 2 < TM_PAIRS ? rv_sm_count() / 2 : TM_PAIRS;
    }
    n = n < TM_PAIRS ? n : TM_PAIRS;                   // (the scratch holds the parts of so many runs)
    known.store(n, std::memory_order_relaxed);
    return n;
}

int rv_tree_mma(const TreeArgs& a, void* scratch, cudaStream_t st) {
    rv_allow_smem<tree_mma_kernel>(SM_TOTAL);
    const int pairs = tree_pairs();
    rv_drain_error();
    uint8_t* s = reinterpret_cast<uint8_t*>(scratch);
    // a tile inside a page is a few tensor copies; smaller pages are gathered row by row
    const int tma = a.page_tokens >= TM_TILE;
    CUtensorMap k_map{}, r_map{}, v_map{};
    if (tma) {
        const cuuint64_t rows = (cuuint64_t)a.n_pool_pages * a.page_tokens;
        if (int e = rivoli::make_tmap_bytes(&k_map, a.pool, 3, {128, rows, 4}, {TM_W, 128}, {128, TM_OWN, 4}, true)) return e;
        if (int e = rivoli::make_tmap_bytes(&r_map, a.pool, 2, {TM_W, rows}, {TM_W}, {TM_ROPE, TM_OWN}, false)) return e;
        if (int e = rivoli::make_tmap_bytes(&v_map, a.pool, 4, {128, rows, 2, 2}, {TM_W, 256, 128}, {128, TM_TILE, 2, 1}, true)) return e;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(2 * pairs)); cfg.blockDim = dim3(TM_THREADS); cfg.dynamicSmemBytes = (size_t)SM_TOTAL; cfg.stream = st;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = 2; at[1].val.clusterDim.y = 1; at[1].val.clusterDim.z = 1;
    cfg.attrs = at; cfg.numAttrs = 2;
    (void)cudaLaunchKernelEx(&cfg, tree_mma_kernel, a, k_map, r_map, v_map, tma, reinterpret_cast<int*>(s), s, (int)tc::kMaxPolls);
    if (int e = rv_launch_status()) return e;
    rv_launch_dependent(tree_join_kernel, dim3(pairs, TM_BLOCK / 8), dim3(256), 0, st, (const uint8_t*)s, a.out, a.out_lse);
    return rv_launch_status();
}
