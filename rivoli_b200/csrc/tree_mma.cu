// Attention of drafted trees over the paged latent cache on the 5th-generation tensor cores, all operands fp8.
//
//     out[r] = sum_j softmax_j((q_r . [L_j | R_j]) * scale) * L_j,    r = (node, head) of one sequence, j = its prefix, then its tree
//
// The arithmetic is that of the decode step's attention (attend_mma.cu): cache rows are consumed as the e4m3 codes they are, q is two e4m3
// terms (here to a power of two, which loses none of its bits: the scores are those of the bf16 queries), the softmax weights are two
// each (2^-9 relative down to 2^-7 of the reference, 2^-10 * 2^-5 of it below), a row's scale rides in its weight (P' = weight * scale *
// 2^5), references lag behind the running maximum by at most 2^3, sums are f32. What differs, beside references that come down again where
// a long prefix would vanish under them (TM_LOW), is the shape of the work. The nodes of a tree share their
// prefix, so that the rows of a sequence are nodes x heads, 64 to a block, and one tile of 64 cache rows serves them all: 240 products and
// more per byte from a single node on and sixteen times that at sixteen nodes. The kernel is bound by the tensor cores and what feeds
// them, the cache's tiles come from L2, and what has to be even is the number of (row block, tile) pairs per SM:
//   * one persistent CTA per SM; the pairs of all sequences, in order, are cut into runs of equal cost, one per CTA. A run that begins or ends
//     inside a row block leaves that block's (maximum, sum, O) in scratch and a second, small kernel joins the parts; all others are
//     written directly. No sequence is too long and no batch too ragged for this.
//   * barriers and their phases run on over the row blocks of a CTA: the next block's tiles are fetched while this one's output is
//     written.
//   * the loops are kept small: with every wait's loop in its place and the query conversion in one piece the kernel waited for its own
//     instructions.
// A pair of CTAs per block of 128 rows (cta_group::2, 1,105 cycles of products a tile against 1,400 here) was built and measured: 862 us
// against 781 then for 8 trees of up to 64 nodes x 16,384 rows alone, 982 against 900 back to back, where both are held by the power limit.
// Rows of the tree are tested against each node's mask in the tiles that hold them, the last one or two of a sequence. A hidden row's
// weight is 0, but 0 x NaN is NaN: NaN codes of tree rows are fetched as 0, and the row makes scores NaN where it is seen. Rows that
// nobody sees, for want of a page or of a scale above zero, are fetched as zeros altogether.
//
// Shared memory: a ring of five tiles of 64 rows (36 KiB), the rope columns of q, P' twice, 16 KiB of staging. Tensor memory: S twice
// (64 columns each), q (128: its latent columns are the A operand of the QK products), O^T (4 x 64). Warps: 0-7 softmax and epilogue in two
// groups that take the tiles in turn, 8 QK issue, 9 PV issue, 10-13 gather. All waits are bounded (tc_common.cuh).
#include "codec.cuh"
#include "common.cuh"
#include "quant.cuh"
#include "tc_common.cuh"
#include "tmap.hpp"
#include "tree_common.cuh"

namespace {

constexpr int TM_TILE = 64, TM_ROWS = 64;            // cache rows of a tile, (node, head) rows of a block
constexpr int TM_KVL = 512, TM_ROPE = 64, TM_W = TM_KVL + TM_ROPE;
constexpr int NK = 5, NG = 2, GW = 4;                // stages; softmax groups, each with an S and a P' buffer; gathering warps
constexpr int TM_SW = 4 * NG, TM_QKW = TM_SW, TM_PVW = TM_SW + 1, TM_GW0 = TM_SW + 2;
constexpr int TM_THREADS = (TM_GW0 + GW) * 32, TM_SOFTMAX = TM_SW * 32, TM_GROUP = 128;
constexpr float TM_POFF = 5.0f, TM_MOST = 256.0f;    // P' = 2^(s - ref + 5) <= 2^8: references lag by 2^3 at most, see attend_mma.cu
// P' below 2^-10 comes to nothing in both terms, and is off by up to 2^-10 above. Behind a row that has most of the weight the whole of a
// long prefix would lie there, so references come down, too. What the terms leave of a tile's P' is added up, sign in it. Where that is
// more than TM_FEW of a thread's largest P', in a tile that is all prefix, the row's own sum goes to its account, and the row's largest
// against it; above TM_LOST of those the reference of a row whose P' here are below TM_LOW comes down until its largest is 2^(5 - TM_SPARE),
// and the sums go up with it (f32: no further than TM_ROOM above the account, nor from below 2^TM_LOWEST, so that none overflows). So
// rounding takes 2^-7 of a row's weights at most, whatever their levels and the length, beside 2^-15 of a larger one for each of the 63
// that share its tile. With references that only rise, 65,536 equal rows behind one with half of the weight left 0.4 of the output's
// norm missing. Keeping the account costs 5 % of the time (32 trees over 512 to 8,192 rows 256 us, 244 without), where scores deviate by
// two and three nats, so that references often move, 14 and 47 %.
constexpr float TM_FEW = 1.0f / 128, TM_LOST = 1.0f / 2048, TM_LOW = 2.0f, TM_LOW_AT = -6.0f, TM_SPARE = 2.0f, TM_ROOM = 35.0f, TM_LOWEST = -64.0f;
constexpr int TM_MIN_TILES = 4;                      // tiles a CTA takes at least, while there are few: a CTA per block, or as many as that leaves
// What a row block costs beside its tiles, in tiles: its queries, its output and the pipeline's ramp take 26,000 cycles, a tile some 1,900. A
// run pays it for each block that it touches; the first is the same for all runs, so that the blocks that begin inside a run count
// (32 trees over 512 to 8,192 rows, when it was chosen: 383 us with runs of as many tiles, 280 with runs of equal cost; 31 nodes over
// 32,771 rows: 161 and 157).
constexpr int TM_BLOCK_COST = 16;

// tensor memory columns
constexpr int TMC_S = 0, TMC_Q = 2 * TM_TILE, TMC_O = TMC_Q + TM_KVL / 4;
static_assert(TMC_O + 4 * TM_ROWS == 512, "tensor memory budget");

// shared memory (bytes)
constexpr int KCHUNK = 8192, KSTAGE = 4 * KCHUNK + 4096;    // four latent chunks [64 rows][128 B], 128-byte swizzle; rope [64][64 B], 64-byte swizzle
constexpr int SM_K = 0;
constexpr int SM_QR = SM_K + NK * KSTAGE;                   // rope columns of q: [128 virtual rows][64 B], 64-byte swizzle
constexpr int SM_P = SM_QR + 8192;                          // per group {hi, lo} [64 rows][64 tokens], 64-byte swizzle
constexpr int PTERM = 4096, PBUF = 2 * PTERM;
constexpr int SM_OUT = SM_P + NG * PBUF;                    // staging: per group 8 rows x 512 bf16
constexpr int SM_TOK = SM_OUT + NG * 8192;                  // f32 [NK][64]: the tokens' scales
constexpr int SM_SEE = SM_TOK + NK * TM_TILE * 4;           // u16 [NK][2][4]: tokens that are there; tokens that are seen as NaN
constexpr int SM_AHI = SM_SEE + NK * 16;                    // f32 [64] query scale * softmax scale * log2(e)
constexpr int SM_WMAX = SM_AHI + 256;                       // f32 [NG][64]
constexpr int SM_FAC = SM_WMAX + NG * 256;                  // f32 [64]
constexpr int SM_MREF = SM_FAC + 256;                       // f32 [64]
constexpr int SM_ACCT = SM_MREF + 256;                      // float2 [64]: a row's account, see TM_LOW
constexpr int SM_BARS = SM_ACCT + 512;
constexpr int SM_MISC = SM_BARS + 256;
constexpr int SM_TOTAL = SM_MISC + 64;
static_assert(SM_TOTAL <= 232448, "shared memory budget");
static_assert(SM_QR % 1024 == 0 && SM_P % 1024 == 0 && KSTAGE % 1024 == 0 && SM_SEE % 16 == 0, "operand tiles are 1024-byte aligned");

struct Bars {
    uint64_t k_full[NK], k_empty[NK], s_full[NG], s_empty[NG], p_full[NG], pv_done[NG], dec[NG], q_full;
};
static_assert(sizeof(Bars) <= 256, "barrier block");
constexpr int FULL = GW * 33;                               // arrivals that fill a stage: the copies of 128 lanes, and each gathering warp

// scratch: error word (256 bytes) | whose part a CTA has left, for the joining kernel | (reference, sum) of parts | O of parts
constexpr int SLOTS = 2 * RV_SMS;                           // a CTA leaves at most a later part of one block and the beginning of another
struct Head { int32_t row0, valid, parts, part; };          // of a slot: the block's first row, its rows (0: nothing left here), parts, which one
constexpr size_t SC_HEAD = 256, SC_ML = SC_HEAD + SLOTS * sizeof(Head), SC_O = (SC_ML + (size_t)SLOTS * TM_ROWS * 8 + 255) / 256 * 256;
constexpr size_t SC_TOTAL = SC_O + (size_t)SLOTS * TM_ROWS * TM_KVL * 4;

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
// The bounded wait of a warp, in few instructions: the kernel's loops have to stay in the instruction cache.
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
// Tensor copy of a tile's four chunks of 64 rows (y: pool row).
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const void* map, int y, uint64_t* bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                 ::"r"(dst), "l"(map), "r"(0), "r"(y), "r"(0), "r"(tc::smem_u32(bar)) : "memory");
}
// Bytes of a word whose low seven bits are all up (NaN codes), as their top bits.
__device__ __forceinline__ uint32_t nan_bytes(uint32_t v) { return ((v & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }

// A walk over a run of (row block, tile) pairs. Units are numbered block by block, sequence by sequence: the block's own cost, then its tiles.
struct Walk {
    int b, rb, t0, t1;             // sequence, row block, tiles [t0, t1) of the current segment
    int cost;                      // of a block beside its tiles
    long long left;                // units of the run from t0 on
    int nt, nrb;                   // tiles and row blocks of the sequence
    TreeSeq s;
};
__device__ __forceinline__ void units_of(const TreeArgs& A, const TreeSeq& s, int& nt, int& nrb) {
    nrb = (s.T * A.H + TM_ROWS - 1) / TM_ROWS;
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
    w.left -= w.t1 - w.t0 + w.cost;
    w.t0 = 0;
    if (++w.rb == w.nrb) { w.rb = 0; w.nrb = 0; }
}
// First unit of CTA g's run.
__device__ __forceinline__ long long run_begin(long long total, int g, int n) { return total * g / n; }

__global__ void __launch_bounds__(TM_THREADS, 1)
tree_mma_kernel(TreeArgs A, const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap r_map, int tma, int* err, uint8_t* scratch, int max_polls) {
    extern __shared__ __align__(1024) uint8_t smem[];
    Bars& bars = *reinterpret_cast<Bars*>(smem + SM_BARS);
    float* s_tok = reinterpret_cast<float*>(smem + SM_TOK);
    uint16_t* s_see = reinterpret_cast<uint16_t*>(smem + SM_SEE);
    float* s_ahi = reinterpret_cast<float*>(smem + SM_AHI);
    float* s_wmax = reinterpret_cast<float*>(smem + SM_WMAX);
    float* s_fac = reinterpret_cast<float*>(smem + SM_FAC);
    float* s_mref = reinterpret_cast<float*>(smem + SM_MREF);
    float2* s_acct = reinterpret_cast<float2*>(smem + SM_ACCT);
    uint32_t* tmem_base_s = reinterpret_cast<uint32_t*>(smem + SM_MISC);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + SM_MISC + 4);
    int* s_run = reinterpret_cast<int*>(smem + SM_MISC + 8);               // b, rb, t0 of the run's beginning, number of runs, a block's own cost
    long long* s_units = reinterpret_cast<long long*>(smem + SM_MISC + 32);   // its units, all units

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
#pragma unroll
        for (int s = 0; s < NK; ++s) { tc::mbar_init(&bars.k_full[s], FULL); tc::mbar_init(&bars.k_empty[s], 1); }
#pragma unroll
        for (int s = 0; s < NG; ++s) {
            tc::mbar_init(&bars.s_full[s], 2); tc::mbar_init(&bars.s_empty[s], 4); tc::mbar_init(&bars.p_full[s], 4);
            tc::mbar_init(&bars.pv_done[s], 1); tc::mbar_init(&bars.dec[s], 4);
        }
        tc::mbar_init(&bars.q_full, TM_SW);
        tc::mbar_init_fence();
        *abort_flag = 0;
    }
    if (warp == TM_QKW) tc::tmem_alloc<512>(tmem_base_s);
    tc::fence_proxy_async();
    tc::tc_fence_before();
    __syncthreads();
    tc::tc_fence_after();
    const uint32_t tmem = *tmem_base_s;
    const uint32_t TM_S0 = tmem + TMC_S, TM_Q = tmem + TMC_Q, TM_O = tmem + TMC_O;
    rv_grid_dep_wait();
    rv_grid_dep_trigger();

    // ------------------------------ the CTA's run ------------------------------------------------
    if (warp == 0) {
        int nt = 0, nrb = 0;                       // of sequence b0 + lane
        auto sizes = [&](int b) {
            nt = nrb = 0;
            if (b < A.B) units_of(A, tree_seq(A, b), nt, nrb);
        };
        long long tiles = 0, blocks = 0;
        for (int b0 = 0; b0 < A.B; b0 += 32) { sizes(b0 + lane); tiles += (long long)nt * nrb; blocks += nrb; }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) { tiles += __shfl_xor_sync(0xffffffffu, tiles, o); blocks += __shfl_xor_sync(0xffffffffu, blocks, o); }
        const int cost = blocks > 1 ? TM_BLOCK_COST : 0, g = blockIdx.x;
        const long long total = tiles + cost * blocks;
        const int n = (int)max(1LL, min((long long)gridDim.x, max(blocks, tiles / TM_MIN_TILES)));
        const long long u0 = g < n ? run_begin(total, g, n) : total, u1 = g < n ? run_begin(total, g + 1, n) : total;
        if (lane == 0) { s_units[0] = 0; s_units[1] = total; s_run[0] = A.B; s_run[1] = s_run[2] = 0; s_run[3] = n; s_run[4] = cost; }
        __syncwarp();
        long long before = 0;
        for (int b0 = 0; b0 < A.B && u1 > u0; b0 += 32) {
            if (A.B > 32) sizes(b0 + lane);        // (a batch of 32 is read already)
            const long long mine = (long long)(nt + cost) * nrb;
            long long inc = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) { const long long v = __shfl_up_sync(0xffffffffu, inc, o); if (lane >= o) inc += v; }
            const long long from = before + inc - mine;
            if (u0 >= from && u0 < from + mine) {
                // a run that begins in a block's own cost has that block's first tile, if it reaches it
                const int rb = (int)((u0 - from) / (nt + cost)), in = (int)((u0 - from) % (nt + cost));
                s_run[0] = b0 + lane; s_run[1] = rb; s_run[2] = max(0, in - cost);
                s_units[0] = u1 - u0 - max(0, cost - in);
            }
            before += __shfl_sync(0xffffffffu, inc, 31);
        }
    }
    __syncthreads();
    Walk w;
    w.b = s_run[0]; w.rb = s_run[1]; w.t0 = s_run[2]; w.cost = s_run[4]; w.left = w.b < A.B ? s_units[0] : 0;
    w.nt = w.nrb = 0;
    if (w.left > 0) { w.s = tree_seq(A, w.b); units_of(A, w.s, w.nt, w.nrb); }

    if (warp >= TM_GW0) {
        // ------------------------------ gather ---------------------------------------------------
        // Tiles that lie wholly in a dense prefix, in pages of 64 tokens and more, are two tensor copies each, a tile per warp in turn.
        // Tiles of a row list, of smaller pages, and those that hold rows of the tree or end inside are gathered by all four warps
        // together, sixteen rows each: the copies go row by row with 32 lanes on 32 consecutive 16-byte chunks (one warp per tile took
        // 5,200 cycles to issue them, and a stage was held for that long more). No warp waits for its copies: they signal the stage
        // themselves. Rows past the end, on unmapped pages and without a scale above zero are written as zeros, in a tile of a tensor copy
        // by that tile's warp alone.
        const int g = warp - TM_GW0, shift = rv_log2(A.page_tokens), inside = A.page_tokens - 1;
        constexpr uint32_t NONE = 0xffffffffu;
        bool ok = true;
        int c0 = 0;                                // tiles of the CTA before this segment
        for (; ok && walk_segment(A, w); c0 += w.t1 - w.t0, walk_on(A, w)) {
            const int total = w.s.n + w.s.T;
            {   // the block's queries on their way to L2: they are read when the softmax warps come to this segment
                const int r0 = w.rb * TM_ROWS, bytes = min(TM_ROWS, w.s.T * A.H - r0) * TM_W * 2;
                const char* at = reinterpret_cast<const char*>(A.q + ((size_t)w.s.node0 * A.H + r0) * TM_W);
#pragma unroll 1
                for (int o = (g * 32 + lane) * 128; o < bytes; o += GW * 32 * 128) asm volatile("prefetch.global.L2 [%0];" ::"l"(at + o));
            }
            const int tj = tma && !w.s.listed ? max(w.t0, min(w.t1, w.s.n / TM_TILE)) : w.t0;   // tiles from here on are gathered
            const int32_t* table = A.block_table + (size_t)w.b * A.max_pages;
            int t = w.t0 + ((g - c0) & (GW - 1));
            if (t < tj) {
                // The page is asked for two of the warp's tiles ahead, the scales one.
                auto page_of = [&](int x) -> int {
                    const int lp = x * TM_TILE >> shift, pg = x < tj && lp < A.max_pages ? table[lp] : -1;
                    return pg < A.n_pool_pages ? pg : -1;
                };
                auto row_of = [&](int x, int pg) -> uint32_t { return pg >= 0 ? (uint32_t)pg * (uint32_t)A.page_tokens + (uint32_t)(x * TM_TILE & inside) : NONE; };
                uint32_t y = row_of(t, page_of(t));
                int pg1 = page_of(t + GW);
                float scl[2] = {0.0f, 0.0f};
                if (y != NONE) { scl[0] = A.pscale[y + lane]; scl[1] = A.pscale[y + 32 + lane]; }
#pragma unroll 1
                for (; t < tj; t += GW) {
                    const uint32_t y1 = row_of(t + GW, pg1);
                    pg1 = page_of(t + 2 * GW);
                    float scl1[2] = {0.0f, 0.0f};
                    if (y1 != NONE) { scl1[0] = A.pscale[y1 + lane]; scl1[1] = A.pscale[y1 + 32 + lane]; }
                    const int i = c0 + t - w.t0, s = i % NK, use = i / NK;
                    uint32_t there[2], wild[2];
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        const bool odd = !(scl[u] < INFINITY), live = y != NONE && !(scl[u] <= 0.0f);   // odd: NaN, or infinite
                        there[u] = __ballot_sync(0xffffffffu, live);
                        wild[u] = __ballot_sync(0xffffffffu, live && odd);
                        scl[u] = !live ? 0.0f : odd ? 1.0f : scl[u];
                    }
                    if (use > 0) ok = wait_for(&bars.k_empty[s], (use & 1) ^ 1, abort_flag, 41, max_polls);
                    if (!ok) break;
                    uint8_t* kbuf = smem + SM_K + s * KSTAGE;
                    const uint32_t at = tc::smem_u32(kbuf);
                    uint32_t others = FULL - 1;
                    if (__builtin_expect((there[0] & there[1]) != ~0u, 0)) {   // rows that are not there: row by row, those as zeros
                        const uint8_t* row = A.pool + (y != NONE ? (size_t)y * TM_W : 0);
                        auto live = [&](int r) -> bool { return ((r < 32 ? there[0] : there[1]) >> (r & 31)) & 1; };
#pragma unroll 4
                        for (int r = 0; r < TM_TILE; ++r)
                            tc::cp_async16_zfill(at + (lane >> 3) * KCHUNK + tc::sw128_chunk(r, lane & 7), live(r) ? row + r * TM_W + lane * 16 : A.pool, live(r) ? 16u : 0u);
#pragma unroll 2
                        for (int r = lane >> 2; r < TM_TILE; r += 8)
                            tc::cp_async16_zfill(at + 4 * KCHUNK + sw64_chunk(r, lane & 3), live(r) ? row + r * TM_W + TM_KVL + (lane & 3) * 16 : A.pool, live(r) ? 16u : 0u);
                        tc::cp_async_mbar_arrive_noinc(&bars.k_full[s]);
                        others = FULL - 32;
                    } else if (tc::elect_one()) {
                        tc::mbar_arrive_expect_tx(&bars.k_full[s], KSTAGE);
                        tma_load_3d(at, &k_map, (int)y, &bars.k_full[s]);
                        tc::tma_load_2d(at + 4 * KCHUNK, &r_map, TM_KVL, (int)y, &bars.k_full[s]);
                    }
#pragma unroll
                    for (int u = 0; u < 2; ++u) s_tok[s * TM_TILE + u * 32 + lane] = scl[u];
                    if (lane == 0) *reinterpret_cast<uint4*>(s_see + s * 8) = make_uint4(there[0], there[1], wild[0], wild[1]);
                    __syncwarp();
                    if (lane == 0) mbar_arrive_n(&bars.k_full[s], others);
                    y = y1; scl[0] = scl1[0]; scl[1] = scl1[1];
                }
            }
            // Four tiles at a time: a lane resolves one row of each of two of them. The words of the chain entry -> page -> scale are
            // asked for a batch ahead, a level behind each of the batch's first tiles, and used a tile later at the earliest.
            auto entry = [&](int tb, int u) -> uint32_t {
                const int x = tb + 2 * u + (lane >> 4), j = x * TM_TILE + 16 * g + (lane & 15);
                return x < w.t1 && j < total ? tree_token(A, w.s, w.b, j) : NONE;
            };
            auto page = [&](uint32_t tok) -> int { return tok != NONE && (tok >> shift) < (uint32_t)A.max_pages ? table[tok >> shift] : -1; };
            auto pool_row = [&](uint32_t tok, int pg) -> uint32_t {
                return pg >= 0 && pg < A.n_pool_pages ? (uint32_t)pg * (uint32_t)A.page_tokens + (tok & (uint32_t)inside) : NONE;
            };
            uint32_t row[2], tok_n[2] = {NONE, NONE}, row_n[2] = {NONE, NONE};
            int pg_n[2] = {-1, -1};
            float scl[2], scl_n[2] = {0.0f, 0.0f};
            if (ok && tj < w.t1) {
#pragma unroll
                for (int u = 0; u < 2; ++u) tok_n[u] = entry(tj, u);
#pragma unroll
                for (int u = 0; u < 2; ++u) row[u] = pool_row(tok_n[u], page(tok_n[u]));
#pragma unroll
                for (int u = 0; u < 2; ++u) scl[u] = row[u] != NONE ? A.pscale[row[u]] : 0.0f;
            }
#pragma unroll 1
            for (int tb = tj; tb < w.t1 && ok; tb += 4) {
#pragma unroll
                for (int u = 0; u < 2; ++u) tok_n[u] = entry(tb + 4, u);
#pragma unroll 1
                for (int k = 0; k < 4 && tb + k < w.t1; ++k) {
                    const int x = tb + k, i = c0 + x - w.t0, s = i % NK, use = i / NK, l0 = 16 * (k & 1);
                    if (use > 0) ok = wait_for(&bars.k_empty[s], (use & 1) ^ 1, abort_flag, 42, max_polls);
                    if (!ok) break;
                    uint8_t* kbuf = smem + SM_K + s * KSTAGE;
                    uint8_t* rope = kbuf + 4 * KCHUNK;
                    const float sc = k < 2 ? scl[0] : scl[1];
                    const uint32_t mine = sc <= 0.0f ? NONE : k < 2 ? row[0] : row[1];   // (rows without a scale are nobody's)
#pragma unroll 8
                    for (int it = 0; it < 16; ++it) {
                        const uint32_t r = __shfl_sync(0xffffffffu, mine, l0 + it);
                        tc::cp_async16_zfill(tc::smem_u32(kbuf + (lane >> 3) * KCHUNK + tc::sw128_chunk(16 * g + it, lane & 7)),
                                             A.pool + (r != NONE ? (size_t)r * TM_W + lane * 16 : 0), r != NONE ? 16u : 0u);
                    }
#pragma unroll
                    for (int it = 0; it < 2; ++it) {
                        const int rl = it * 8 + (lane >> 2);
                        const uint32_t r = __shfl_sync(0xffffffffu, mine, l0 + rl);
                        tc::cp_async16_zfill(tc::smem_u32(rope + sw64_chunk(16 * g + rl, lane & 3)),
                                             A.pool + (r != NONE ? (size_t)r * TM_W + TM_KVL + (lane & 3) * 16 : 0), r != NONE ? 16u : 0u);
                    }
                    bool bad = false;              // this lane's row holds a NaN code
                    if ((x + 1) * TM_TILE > w.s.n) {
                        // rows of the tree: each lane looks through the chunks that it copied itself, once they are there
                        tc::cp_async_commit();
                        tc::cp_async_wait<0>();
                        auto clear = [&](uint8_t* at) -> bool {
                            uint4 v = *reinterpret_cast<const uint4*>(at);
                            const uint4 m = make_uint4(nan_bytes(v.x), nan_bytes(v.y), nan_bytes(v.z), nan_bytes(v.w));
                            if (!(m.x | m.y | m.z | m.w)) return false;
                            v.x &= ~((m.x >> 7) * 0xffu); v.y &= ~((m.y >> 7) * 0xffu); v.z &= ~((m.z >> 7) * 0xffu); v.w &= ~((m.w >> 7) * 0xffu);
                            *reinterpret_cast<uint4*>(at) = v;
                            return true;
                        };
                        const int first = w.s.n - x * TM_TILE - 16 * g, end = total - x * TM_TILE - 16 * g;
#pragma unroll 2
                        for (int it = max(0, first); it < min(16, end); ++it)
                            if (__any_sync(0xffffffffu, clear(kbuf + (lane >> 3) * KCHUNK + tc::sw128_chunk(16 * g + it, lane & 7))) && (lane & 15) == it) bad = true;
#pragma unroll 1
                        for (int it = 0; it < 2; ++it) {
                            const int rl = it * 8 + (lane >> 2);
                            const uint32_t hit = __ballot_sync(0xffffffffu, rl >= first && rl < end && clear(rope + sw64_chunk(16 * g + rl, lane & 3)));
                            if (((lane & 15) >> 3) == it && ((hit >> (4 * (lane & 7))) & 15u)) bad = true;
                        }
                    }
                    tc::cp_async_mbar_arrive_noinc(&bars.k_full[s]);
                    {
                        const bool here = (lane >> 4) == (k & 1);
                        const bool odd = bad || !(sc < INFINITY), live = mine != NONE;                         // odd: seen as NaN
                        if (here) s_tok[s * TM_TILE + 16 * g + (lane & 15)] = !live ? 0.0f : odd ? 1.0f : sc;
                        const uint32_t there = __ballot_sync(0xffffffffu, live), wild = __ballot_sync(0xffffffffu, live && odd);
                        if (lane == 0) { s_see[s * 8 + g] = (uint16_t)(there >> l0); s_see[s * 8 + 4 + g] = (uint16_t)(wild >> l0); }
                    }
                    tc::fence_proxy_async();
                    __syncwarp();
                    if (lane == 0) tc::mbar_arrive(&bars.k_full[s]);
                    if (k == 0) {
#pragma unroll
                        for (int u = 0; u < 2; ++u) pg_n[u] = page(tok_n[u]);
                    }
                    if (k == 1) {
#pragma unroll
                        for (int u = 0; u < 2; ++u) { row_n[u] = pool_row(tok_n[u], pg_n[u]); scl_n[u] = row_n[u] != NONE ? A.pscale[row_n[u]] : 0.0f; }
                    }
                }
#pragma unroll
                for (int u = 0; u < 2; ++u) { row[u] = row_n[u]; scl[u] = scl_n[u]; }
            }
        }
    } else if (warp == TM_QKW) {
        // ------------------------------ QK issuer: S(i) = Q . K(i)^T -----------------------------
        const uint32_t id_qk = tc::idesc_e4m3(128, TM_TILE, 0, 0);
        const uint64_t d_qr = smem_desc(tc::smem_u32(smem + SM_QR), 16, 512, 4);
        bool ok = true;
        int i = 0, seg = 0, s = 0, phase = 0;
        for (; ok && walk_segment(A, w); walk_on(A, w), ++seg) {
            ok = wait_for(&bars.q_full, seg & 1, abort_flag, 51, max_polls);
#pragma unroll 1
            for (int t = w.t0; t < w.t1 && ok; ++t, ++i) {
                const int sb = i & 1;
                ok = wait_for(&bars.k_full[s], phase, abort_flag, 52, max_polls) && wait_for(&bars.s_empty[sb], ((i >> 1) & 1) ^ 1, abort_flag, 53, max_polls);
                if (!ok) break;
                tc::fence_proxy_async();   // copies that wrote through the generic proxy, the products read through the async one
                tc::tc_fence_after();
                const uint64_t d_k = smem_desc(tc::smem_u32(smem + SM_K + s * KSTAGE), 16, 1024, 2);
                const uint64_t d_rope = smem_desc(tc::smem_u32(smem + SM_K + s * KSTAGE + 4 * KCHUNK), 16, 512, 4);
                const uint32_t d = TM_S0 + sb * TM_TILE;
                if (tc::elect_one()) {
#pragma unroll
                    for (int k = 0; k < 2; ++k) tc::mma_f8(d, d_qr + (uint64_t)(k * 2), d_rope + (uint64_t)(k * 2), id_qk, k != 0);
#pragma unroll
                    for (int c = 0; c < 4; ++c)
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            tc::mma_f8_ta(d, TM_Q + (uint32_t)(c * 32 + k * 8), d_k + (uint64_t)((c * KCHUNK + k * 32) >> 4), id_qk, 1);
                    tc::mma_commit(&bars.s_full[sb]);
                    tc::mbar_arrive(&bars.s_full[sb]);   // hands the token words on: this thread has seen k_full
                }
                __syncwarp();
                if (++s == NK) { s = 0; phase ^= 1; }
            }
        }
    } else if (warp == TM_PVW) {
        // ------------------------------ PV issuer: O^T += V(i)^T . P'(i) --------------------------
        // Beside it, while it waits for a segment's first weights: whose parts this CTA will have left, for the joining kernel.
        const uint32_t id_pv = tc::idesc_e4m3(128, TM_ROWS, 1, 0);
        Head* heads = reinterpret_cast<Head*>(scratch + SC_HEAD) + 2 * blockIdx.x;
        bool ok = true;
        int i = 0, s = 0, told = 0;                        // told: which of the two slots have a part
        for (; ok && walk_segment(A, w); walk_on(A, w)) {
            if (lane == 0 && (w.t0 > 0 || w.t1 < w.nt)) {
                const long long total = s_units[1];
                const int n = s_run[3], r0 = w.rb * TM_ROWS;
                auto run_of = [&](long long unit) -> int {
                    int g = (int)(unit * n / total);
                    while (run_begin(total, g + 1, n) <= unit) ++g;
                    return g;
                };
                // (a segment that goes on in the next run ends with this one; one that does not, and is no beginning, begins with it)
                const bool on = w.t1 < w.nt;
                const long long at = on ? run_begin(total, blockIdx.x + 1, n) - w.t1 : run_begin(total, blockIdx.x, n) - w.t0;   // the unit of tile 0
                const int first = w.t0 == 0 ? (int)blockIdx.x : run_of(at), last = on ? run_of(at + w.nt - 1) : (int)blockIdx.x;
                heads[w.t0 == 0] = Head{w.s.node0 * A.H + r0, min(TM_ROWS, w.s.T * A.H - r0), last - first + 1, (int)blockIdx.x - first};
                told |= 1 << (w.t0 == 0);
            }
            __syncwarp();
#pragma unroll 1
            for (int t = w.t0; t < w.t1 && ok; ++t, ++i) {
                const int pb = i & 1;
                ok = wait_for(&bars.p_full[pb], (i >> 1) & 1, abort_flag, 54, max_polls);
                if (!ok) break;
                tc::fence_proxy_async();
                tc::tc_fence_after();
                const uint64_t d_v = smem_desc(tc::smem_u32(smem + SM_K + s * KSTAGE), KCHUNK, 1024, 2);
                const uint64_t d_phi = smem_desc(tc::smem_u32(smem + SM_P + pb * PBUF), 16, 512, 4);
                const uint64_t d_plo = smem_desc(tc::smem_u32(smem + SM_P + pb * PBUF + PTERM), 16, 512, 4);
                if (tc::elect_one()) {
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
#pragma unroll
                        for (int k = 0; k < 2; ++k)
                            tc::mma_f8(TM_O + c * 64, d_v + (uint64_t)((c * KCHUNK + k * 4096) >> 4), d_phi + (uint64_t)(k * 2), id_pv, t > w.t0 || k != 0);
#pragma unroll
                        for (int k = 0; k < 2; ++k)
                            tc::mma_f8(TM_O + c * 64, d_v + (uint64_t)((c * KCHUNK + k * 4096) >> 4), d_plo + (uint64_t)(k * 2), id_pv, 1);
                    }
                    tc::mma_commit(&bars.k_empty[s]);
                    tc::mma_commit(&bars.pv_done[pb]);
                }
                __syncwarp();
                if (++s == NK) s = 0;
            }
        }
        if (lane == 0)
            for (int u = 0; u < 2; ++u)
                if (!(told >> u & 1)) heads[u] = Head{0, 0, 0, 0};
    } else {
        // ------------------------------ queries, softmax, epilogue -------------------------------
        // S: lanes 0-15 of a warp's quarter hold the hi terms of 16 rows, lanes 16-31 their lo terms. Read 16 lanes at a time in the
        // fragment form (a thread gets two neighbouring columns of rows lane / 4 and lane / 4 + 8 per eight columns), hi and lo come to the
        // same registers of the same thread: the sum takes no exchange. A thread has 16 tokens of two rows.
        // O^T: a thread's lane is one dim of each block of 128, the columns are the rows.
        const int sq = warp & 3, th = warp >> 2, tb = lane >> 4;
        const int hd = 16 * sq + (lane & 15);              // a row of the conversion and of the epilogue's sums
        const int ra = 16 * sq + (lane >> 2), rb = ra + 8, tq = 2 * (lane & 3);   // rows and first token of the scores
        const int odim = sq * 32 + lane;                   // O^T: this thread's dim
        const uint32_t lane_base = ((uint32_t)(sq * 32)) << 16;
        auto give_up = [&]() { (void)tc::barrier_any(6 + th, TM_GROUP, true); (void)tc::barrier_any(9 + th, TM_GROUP, true); };
        // O has taken tile i. A parity tells a phase from the one before it only: a group asks for its own tile first, whose predecessor
        // in the barrier it has seen, and then for another's within the NG behind it.
        auto pv_done = [&](int i) { return wait_for(&bars.pv_done[i % NG], (i / NG) & 1, abort_flag, 63, max_polls); };
        int i0 = 0;                                        // tiles of the CTA before this segment
        bool failed = false;
        for (; !failed && walk_segment(A, w); i0 += w.t1 - w.t0, walk_on(A, w)) {
            const int rows_all = w.s.T * A.H, r0 = w.rb * TM_ROWS, valid = min(TM_ROWS, rows_all - r0);
            const size_t flat = (size_t)w.s.node0 * A.H + r0;      // first row of the block in q, out and out_lse
            // ---- q -> two e4m3 terms per row: hi = e4m3(q / s), s the power of two at or above absmax / 448, lo = e4m3(q / s - hi) ----
            // With a power of two the terms are q itself: a bf16 has eight bits, hi takes four of them, and what is left is at most eight of
            // the last one's units. Only values below 2^-10 of the row's largest lose bits, to the last subnormal of lo: half of 2^-9 s,
            // 2^-18 of the largest at most. (With s = absmax / 448 each value was 2^-8 off and the sums of the softmax 1e-4.)
            // A warp takes sixteen rows and half th of their columns. They arrive as whole 128-byte lines (lanes 8 k .. 8 k + 7 on one row),
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
                        v[4 * c + k] = r < valid ? *reinterpret_cast<const uint4*>(q0 + (size_t)r * TM_W + th * (TM_KVL / 2) + c * 64 + (lane & 7) * 8) : make_uint4(0u, 0u, 0u, 0u);
                    }
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const int r = xq + 8 * k;
                    v[16 + k] = r < valid ? *reinterpret_cast<const uint4*>(q0 + (size_t)r * TM_W + TM_KVL + th * (TM_ROPE / 2) + (lane & 3) * 8) : make_uint4(0u, 0u, 0u, 0u);
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
                    if (lane < 16) s_wmax[th * 64 + hd] = __uint_as_float(rv_max_bf16x2(a, x) << 16);
                }
                tc::named_barrier(3, TM_SOFTMAX);          // (also: all groups are through with the block before)
                auto scale_of = [&](int r) -> float {          // the power of two at or above absmax / 448
                    const float amax = fmaxf(s_wmax[r], s_wmax[64 + r]);
                    return amax > 0.0f ? fmaxf(__uint_as_float((__float_as_uint(amax / 448.0f) + 0x007fffffu) & 0xff800000u), 1.17549435e-38f) : 1.0f;
                };
                if (th == 0 && tb == 0) { s_ahi[hd] = scale_of(hd) * A.softmax_scale * 1.4426950408889634f; s_mref[hd] = -INFINITY; s_acct[hd] = make_float2(0.0f, 0.0f); }
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
                uint8_t* buf = smem + SM_P + warp * 2048;
                auto spot = [&](int r, int byte) { return buf + r * 64 + ((((byte >> 4) ^ (r >> 1)) & 3) << 4) + (byte & 15); };
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
                tc::tmem_st_wait();
                tc::fence_proxy_async();
                tc::tc_fence_before();
                __syncwarp();
                if (lane == 0) tc::mbar_arrive(&bars.q_full);
                tc::named_barrier(3, TM_SOFTMAX);          // the row scales and references are read by other warps than wrote them
            }

            // ---- the tiles ----
            const float a_a = s_ahi[ra], a_b = s_ahi[rb];
            float l_a = 0.0f, l_b = 0.0f, m_a = -INFINITY, m_b = -INFINITY;   // sums, and the references they are at
            const int i1 = i0 + (w.t1 - w.t0);
            bool ok = true;
            int i = i0 + ((th ^ i0) & 1);
            int sv = i % NK;                               // its stage
#pragma unroll 1
            for (; i < i1; i += NG, sv += sv >= NK - NG ? NG - NK : NG) {
                const int j0 = (w.t0 + i - i0) * TM_TILE, phase = (i >> 1) & 1;
                ok = wait_for(&bars.s_full[th], phase, abort_flag, 62, max_polls);
                if (!ok) { give_up(); break; }
                tc::tc_fence_after();
                // x: scores in log2 units; [k][row][token tq + e] of each run k of eight tokens
                f2 x[16];
                const f2* sc = reinterpret_cast<const f2*>(s_tok + sv * TM_TILE + tq);   // [4 k]: scales of run k's two tokens
                const uint32_t s_at = TM_S0 + th * TM_TILE + lane_base;
#pragma unroll
                for (int hf = 0; hf < 2; ++hf) {
                    uint32_t hi[16], lo[16];
                    tc::tmem_ld16x256(s_at + 32 * hf, hi);
                    tc::tmem_ld16x256(s_at + (16u << 16) + 32 * hf, lo);
                    tc::tmem_ld_wait();
                    if (hf == 1) {
                        tc::tc_fence_before();
                        __syncwarp();
                        if (lane == 0) tc::mbar_arrive(&bars.s_empty[th]);
                    }
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        x[8 * hf + j] = add2(pack(__uint_as_float(hi[2 * j]), __uint_as_float(hi[2 * j + 1])), pack(__uint_as_float(lo[2 * j]), __uint_as_float(lo[2 * j + 1])));
                }
                const uint4 see = *reinterpret_cast<const uint4*>(s_see + sv * 8);
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
                    __half2 top[2] = {__float2half2_rn(0.0f), __float2half2_rn(0.0f)}, gone[2] = {top[0], top[1]};   // of rows a and b: the largest P', and what the terms leave of them
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
                            top[r] = __hmax2(top[r], ph);
                            const uint32_t phb = *reinterpret_cast<const uint32_t*>(&ph);
                            uint16_t c, d;
                            uint32_t back;
                            asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(c) : "r"(phb));
                            asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(back) : "h"(c));
                            const __half2 rest = __hsub2(ph, *reinterpret_cast<const __half2*>(&back));
                            asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(d) : "r"(*reinterpret_cast<const uint32_t*>(&rest)));
                            asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(back) : "h"(d));
                            gone[r] = __hadd2(gone[r], __hsub2(rest, *reinterpret_cast<const __half2*>(&back)));
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
                    if (i > i0) {
                        ok = wait_for(&bars.dec[th ^ 1], ((i - 1) >> 1) & 1, abort_flag, 65, max_polls);
                        const float na = s_mref[ra], nb = s_mref[rb];
                        if (na != m_a) { l_a *= exp2f(m_a - na); m_a = na; }
                        if (nb != m_b) { l_b *= exp2f(m_b - nb); m_b = nb; }
                    }
                    // They stand as long as no P' exceeds 2^(5 + 3) by them (one barrier with an OR). One that has moved meanwhile brings the
                    // P' of before along. Rows that have none yet are looked at, too.
                    __half2 t = __hmax2(__lows2half2(top[0], top[1]), __highs2half2(top[0], top[1]));
                    __half2 g = __hadd2(__lows2half2(gone[0], gone[1]), __highs2half2(gone[0], gone[1]));
                    if (m_a != was_a || m_b != was_b) {
                        const float2 t2 = __half22float2(t), g2 = __half22float2(g);
                        const float fa = exp2f(was_a - m_a), fb = exp2f(was_b - m_b);
                        t = __floats2half2_rn(t2.x * fa, t2.y * fb);
                        g = __floats2half2_rn(g2.x * fa, g2.y * fb);
                    }
                    const bool inside = j0 + TM_TILE <= w.s.n;
                    bool down_a = false, down_b = false;
                    if (__builtin_expect(__any_sync(0xffffffffu, inside && !__hble2(__habs2(g), __hmul2(t, __float2half2_rn(TM_FEW))) && i > i0), 0)) {
                        // (where a group's first tile is all small, its reference comes down below)
#pragma unroll
                        for (int o = 1; o < 4; o <<= 1) {
                            t = __hmax2(t, __shfl_xor_sync(0xffffffffu, t, o));
                            g = __hadd2(g, __shfl_xor_sync(0xffffffffu, g, o));
                        }
                        auto look = [&](float most, float took, float was, int row) -> bool {
                            float2 c = s_acct[row];
                            bool down = false;
                            if (most < TM_LOW && was > -INFINITY && fabsf(took) > TM_FEW * most && took - took == 0.0f) {
                                c.y += took;
                                down = fabsf(c.y) > TM_LOST * (c.x + most);
                                if (down) c.y = 0.0f;
                            }
                            c.x += most;
                            __syncwarp();
                            if (tq == 0) s_acct[row] = c;
                            return down;
                        };
                        const float2 most = __half22float2(t), took = __half22float2(g);
                        down_a = look(most.x, took.x, was_a, ra);
                        down_b = look(most.y, took.y, was_b, rb);
                    }
                    const bool grown = !__hble2(t, __float2half2_rn(TM_MOST)) || was_a == -INFINITY || was_b == -INFINITY || down_a || down_b;
                    if (__builtin_expect(tc::barrier_any(6 + th, TM_GROUP, grown || !ok), 0)) {
                        // the largest x + log2(scale) of a row is what P' goes by (scales below 2^-100 as that: their weights would
                        // pass 2^127)
                        float ta = -INFINITY, tb2 = -INFINITY;
#pragma unroll
                        for (int k = 0; k < 8; ++k) {
                            const float2 s2 = unpack(sc[4 * k]), ya = unpack(x[2 * k]), yb = unpack(x[2 * k + 1]);
                            const float g0 = fmaxf(__log2f(s2.x), -100.0f), g1 = fmaxf(__log2f(s2.y), -100.0f);
                            ta = fmaxf(ta, fmaxf(ya.x + g0, ya.y + g1)); tb2 = fmaxf(tb2, fmaxf(yb.x + g0, yb.y + g1));
                        }
#pragma unroll
                        for (int o = 1; o < 4; o <<= 1) { ta = fmaxf(ta, __shfl_xor_sync(0xffffffffu, ta, o)); tb2 = fmaxf(tb2, __shfl_xor_sync(0xffffffffu, tb2, o)); }
                        // all references take all of their growth (taken by those alone that had to, the next tile's row would have to), and
                        // come down where the account says so
                        auto move = [&](float& m, float was, float t_now, bool down, int row) -> float {
                            float2 c = s_acct[row];
                            down |= was == -INFINITY && inside && t_now < m + TM_LOW_AT;
                            float f = 1.0f;
                            if (t_now > -INFINITY) {
                                const float to = fmaxf(t_now + (down ? TM_SPARE : 0.0f), m - (down && m > TM_LOWEST ? fmaxf(TM_ROOM - __log2f(c.x), 0.0f) : 0.0f));
                                if (m > -INFINITY) f = exp2f(m - to);
                                m = to;
                                c.x = c.x * f + exp2f(t_now - m + TM_POFF);
                            }
                            __syncwarp();
                            if (tq == 0) { s_fac[row] = f; s_mref[row] = m; s_acct[row] = make_float2(c.x, c.y * f); }
                            return f;
                        };
                        const float fa = move(m_a, was_a, ta, down_a, ra), fb = move(m_b, was_b, tb2, down_b, rb);
                        left = tc::barrier_any(9 + th, TM_GROUP, !ok);
                        if (!left && i > i0 && __any_sync(0xffffffffu, s_fac[lane] != 1.0f || s_fac[32 + lane] != 1.0f)) {   // O^T to the new references
                            if (i >= i0 + NG) ok = pv_done(i - NG);
                            if (ok) ok = pv_done(i - 1);
                            tc::tc_fence_after();
                            uint32_t r[32];
#pragma unroll 1
                            for (int c = 0; c < 8; ++c) {
                                tc::tmem_ld32(TM_O + lane_base + c * 32, r);
                                tc::tmem_ld_wait();
#pragma unroll
                                for (int h = 0; h < 32; ++h) r[h] = __float_as_uint(__uint_as_float(r[h]) * s_fac[(c & 1) * 32 + h]);
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
                if (lane == 0) tc::mbar_arrive(&bars.p_full[th]);
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
            const int slot = 2 * blockIdx.x + (w.t0 == 0 ? 1 : 0);
            if (th == 0 && lane < 16) {
                // (l and O carry 2^5; NaN stays NaN)
                const float l = s_wmax[hd] + s_wmax[64 + hd];
                if (!whole) reinterpret_cast<float2*>(scratch + SC_ML)[slot * TM_ROWS + hd] = make_float2(m_last, l);
                else if (hd < valid && A.out_lse) A.out_lse[flat + hd] = l == 0.0f ? -INFINITY : (m_last - TM_POFF) * 0.6931471805599453f + logf(l);
                s_fac[hd] = l == 0.0f ? 0.0f : 1.0f / l;
            }
            tc::named_barrier(1, TM_SOFTMAX);              // (the sums are read: the next block's maxima take their place)
            if (whole) {
                // eight rows at a time through the group's staging, and out as one bulk copy
                uint16_t* stage = reinterpret_cast<uint16_t*>(smem + SM_OUT + th * 8192);
#pragma unroll 1
                for (int g = 0; g < 4; ++g) {
                    const int hg = th * 32 + g * 8;
                    uint32_t r[4][8];
#pragma unroll
                    for (int c = 0; c < 4; ++c) tc::tmem_ld8(TM_O + lane_base + c * 64 + hg, r[c]);
                    tc::tmem_ld_wait();
                    if (sq == 0 && lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
                    tc::named_barrier(4 + th, TM_GROUP);   // the staging is free
                    const float4 f0 = *reinterpret_cast<const float4*>(s_fac + hg), f1 = *reinterpret_cast<const float4*>(s_fac + hg + 4);
                    const float inv_l[8] = {f0.x, f0.y, f0.z, f0.w, f1.x, f1.y, f1.z, f1.w};
                    uint16_t* sp = stage + odim;
#pragma unroll
                    for (int c = 0; c < 4; ++c)
#pragma unroll
                        for (int k = 0; k < 8; k += 2) {
                            uint32_t w2;
                            asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w2) : "f"(__uint_as_float(r[c][k + 1]) * inv_l[k + 1]), "f"(__uint_as_float(r[c][k]) * inv_l[k]));
                            sp[k * TM_KVL + c * 128] = (uint16_t)w2;
                            sp[(k + 1) * TM_KVL + c * 128] = (uint16_t)(w2 >> 16);
                        }
                    tc::fence_proxy_async();
                    tc::named_barrier(4 + th, TM_GROUP);
                    const int n = min(8, valid - hg);
                    if (sq == 0 && lane == 0 && n > 0) {
                        asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;"
                                     ::"l"(A.out + (flat + hg) * TM_KVL), "r"(tc::smem_u32(stage)), "r"(n * TM_KVL * 2) : "memory");
                        asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                    }
                }
            } else {
                // a part: O as it is, for the joining kernel
                float* po = reinterpret_cast<float*>(scratch + SC_O) + (size_t)slot * TM_ROWS * TM_KVL + odim;
#pragma unroll 1
                for (int c = 0; c < 4; ++c) {
                    uint32_t r[32];
                    tc::tmem_ld32(TM_O + lane_base + c * 64 + th * 32, r);
                    tc::tmem_ld_wait();
#pragma unroll
                    for (int h = 0; h < 32; ++h) po[(size_t)(th * 32 + h) * TM_KVL + c * 128] = __uint_as_float(r[h]);
                }
            }
            tc::tc_fence_before();
        }
        if (sq == 0 && lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    }

    tc::tc_fence_before();
    __syncthreads();
    if (warp == TM_QKW) {
        tc::settle(*abort_flag);
        tc::tmem_dealloc<512>(tmem);
    }
    if (tid == 0 && *abort_flag) atomicCAS(err, 0, *abort_flag);
}

// Joins the parts of row blocks, eight rows per blockIdx.y. Up to eight parts: by the CTA of the first, a warp per row. More: the CTAs of
// all parts share the rows, part k takes rows k, k + parts, ... of the eight, all its warps on one row at a time, so that a hundred parts
// have their loads on their way at once (one sequence over 131,072 rows, both kernels: 117 us with a warp per row, 59 so; blocks of two
// parts the other way round: 16 trees of 8 over 2,048 rows 72 us when shared, 64 alone).
constexpr int TJ_WARPS = 8, TJ_ALONE = 8;
// dims 4 d .. 4 d + 3 of a row
__device__ __forceinline__ void join_put(uint16_t* out, int d, float4 x, float inv) {
    uint2 v;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(v.x) : "f"(x.y * inv), "f"(x.x * inv));
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(v.y) : "f"(x.w * inv), "f"(x.z * inv));
    reinterpret_cast<uint2*>(out)[d] = v;
}
__device__ __forceinline__ void join_add(float4& acc, float4 x, float f) {
    acc.x = fmaf(x.x, f, acc.x); acc.y = fmaf(x.y, f, acc.y); acc.z = fmaf(x.z, f, acc.z); acc.w = fmaf(x.w, f, acc.w);
}
__device__ __forceinline__ float join_lse(float m, float l) { return l == 0.0f ? -INFINITY : (m - TM_POFF) * 0.6931471805599453f + logf(l); }
__device__ __forceinline__ bool saw_nothing(float2 part) { return part.x == -INFINITY && part.y == 0.0f; }

__global__ void __launch_bounds__(TJ_WARPS * 32, 4)
tree_join_kernel(const uint8_t* scratch, uint16_t* out, float* out_lse) {
    __shared__ float4 s_o[TJ_WARPS][TM_KVL / 4];
    rv_grid_dep_wait();
    rv_grid_dep_trigger();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const float2* ml = reinterpret_cast<const float2*>(scratch + SC_ML);
    const float4* o4 = reinterpret_cast<const float4*>(scratch + SC_O) + lane;
    const Head* heads = reinterpret_cast<const Head*>(scratch + SC_HEAD) + 2 * blockIdx.x;
    const Head first = heads[1], later = heads[0];
    auto at = [](int g, int p, int row) -> size_t { return (size_t)(p == 0 ? 2 * g + 1 : 2 * (g + p)) * TM_ROWS + row; };   // of part p of the block that begins in CTA g
    const int own = blockIdx.y * 8 + warp;
    if (first.parts <= TJ_ALONE && own < first.valid) {
        const int g = blockIdx.x;
        float m = -INFINITY, l = 0.0f;
        for (int p = 0; p < first.parts; ++p) m = fmaxf(m, ml[at(g, p, own)].x);
        float4 acc[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) acc[c] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (int p = 0; p < first.parts; ++p) {
            const float2 part = ml[at(g, p, own)];
            if (saw_nothing(part)) continue;
            const float f = exp2f(part.x - m);
            l += part.y * f;
#pragma unroll
            for (int c = 0; c < 4; ++c) join_add(acc[c], o4[at(g, p, own) * (TM_KVL / 4) + c * 32], f);
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) join_put(out + ((size_t)first.row0 + own) * TM_KVL, c * 32 + lane, acc[c], l == 0.0f ? 0.0f : 1.0f / l);
        if (out_lse && lane == 0) out_lse[first.row0 + own] = join_lse(m, l);
    }
#pragma unroll 1
    for (int u = 0; u < 2; ++u) {
        const Head h = u ? first : later;
        if (h.parts <= TJ_ALONE) continue;                     // (the same for the whole block)
        const int g = blockIdx.x - h.part;
#pragma unroll 1
        for (int row = blockIdx.y * 8 + h.part; row < min(h.valid, (int)blockIdx.y * 8 + 8); row += h.parts) {
            float m = -INFINITY, l = 0.0f;
            for (int p = lane; p < h.parts; p += 32) m = fmaxf(m, ml[at(g, p, row)].x);
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
            for (int p = lane; p < h.parts; p += 32) {
                const float2 part = ml[at(g, p, row)];
                if (!saw_nothing(part)) l += part.y * exp2f(part.x - m);
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
            float4 acc[4];
#pragma unroll
            for (int c = 0; c < 4; ++c) acc[c] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 1
            for (int p0 = warp; p0 < h.parts; p0 += 2 * TJ_WARPS) {            // two parts on their way at once
                float4 x[2][4];
                float2 part[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int p = p0 + e * TJ_WARPS;
                    part[e] = make_float2(-INFINITY, 0.0f);
                    if (p >= h.parts) continue;
                    part[e] = ml[at(g, p, row)];
#pragma unroll
                    for (int c = 0; c < 4; ++c) x[e][c] = o4[at(g, p, row) * (TM_KVL / 4) + c * 32];
                }
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    if (saw_nothing(part[e])) continue;
                    const float f = exp2f(part[e].x - m);
#pragma unroll
                    for (int c = 0; c < 4; ++c) join_add(acc[c], x[e][c], f);
                }
            }
#pragma unroll
            for (int c = 0; c < 4; ++c) s_o[warp][c * 32 + lane] = acc[c];
            __syncthreads();
            if (threadIdx.x < TM_KVL / 4) {
                float4 x = s_o[0][threadIdx.x];
#pragma unroll
                for (int k = 1; k < TJ_WARPS; ++k) join_add(x, s_o[k][threadIdx.x], 1.0f);
                join_put(out + ((size_t)h.row0 + row) * TM_KVL, threadIdx.x, x, l == 0.0f ? 0.0f : 1.0f / l);
            }
            if (out_lse && threadIdx.x == 0) out_lse[h.row0 + row] = join_lse(m, l);
            __syncthreads();
        }
    }
}

}  // namespace

bool rv_tree_mma_supported(const DsaGeom* g) { return g->kv_lora == TM_KVL && g->rope_dim == TM_ROPE; }
size_t rv_tree_mma_scratch_bytes() { return SC_TOTAL; }

int rv_tree_mma(const TreeArgs& a, void* scratch, cudaStream_t st) {
    rv_allow_smem<tree_mma_kernel>(SM_TOTAL);
    const int sms = rv_sm_count(), grid = sms < RV_SMS ? sms : RV_SMS;   // (the scratch holds the parts of RV_SMS runs)
    rv_drain_error();
    uint8_t* s = reinterpret_cast<uint8_t*>(scratch);
    // a tile inside a page is two tensor copies; smaller pages are gathered row by row
    const int tma = a.page_tokens >= TM_TILE;
    CUtensorMap k_map{}, r_map{};
    if (tma) {
        const cuuint64_t rows = (cuuint64_t)a.n_pool_pages * a.page_tokens;
        if (int e = rivoli::make_tmap_bytes(&k_map, a.pool, 3, {128, rows, 4}, {TM_W, 128}, {128, TM_TILE, 4}, true)) return e;
        if (int e = rivoli::make_tmap_bytes(&r_map, a.pool, 2, {TM_W, rows}, {TM_W}, {TM_ROPE, TM_TILE}, false)) return e;
    }
    rv_launch_dependent(tree_mma_kernel, dim3(grid), dim3(TM_THREADS), (size_t)SM_TOTAL, st, a, k_map, r_map, tma, reinterpret_cast<int*>(s), s, (int)tc::kMaxPolls);
    if (int e = rv_launch_status()) return e;
    rv_launch_dependent(tree_join_kernel, dim3(grid, TM_ROWS / 8), dim3(TJ_WARPS * 32), 0, st, (const uint8_t*)s, a.out, a.out_lse);
    return rv_launch_status();
}
