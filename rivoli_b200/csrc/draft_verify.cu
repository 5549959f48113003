// Drafted tokens against the target's probabilities, with given random numbers, and the token that follows them.
//
// Node 0 of a sequence's tree is the token decided last. From there: the children of the current node are tried in the order of
// their indices; with r the target's probabilities behind the current node (negative, infinite and NaN ones count as 0) and q the
// draft's, child x is accepted if u[x] * q(token) < r(token), and the walk goes on from it. If it is not, what is left is
//     r <- max(r - q, 0) / Z,   Z = sum max(r - q, 0)
// (tokens that were chosen and not drawn, draft = NULL: q is 1 at the token and 0 elsewhere), so that the token that comes out is
// distributed as the target says. Where no child is left the next token is the first v with r(0) + .. + r(v) > u_next * sum r, or the
// last with r(v) > 0 if none; where nothing is left of r (Z = 0) the remaining children are refused and the target's own row is drawn
// from; -1 if that is empty too.
//
// Every r in that chain is max(a p - b q, 0) with two numbers a and b: a rejection needs one pass over the rows (for Z), which also
// leaves the sums by chunk that the draw needs, and nothing is written but the answer. Of tokens that were chosen, one pass a node serves all
// rejections: Z goes down by the token's own probability, and before the draw the few chunks that hold such tokens are summed again
// without them (as they are when Z has come below a thousandth of the whole and would lose its last bits). Sums, products and
// comparisons are in 64 bits: a draw next to a border has to come out the same whatever the order of summation.
//
// A cluster of up to eight blocks per sequence, each a contiguous part of the vocabulary, as many blocks as run at once; every block walks
// the tree itself (the few probabilities that decide are gathered at once for all nodes), and only sums are exchanged, through distributed
// shared memory. A warp's chunks of 2 KiB a row come through a ring of its own (with one chunk in registers at a time a pass of five chunks
// waited 15,000 cycles, so 9,000). 128 sequences of 12 chosen tokens over 151,552 bf16: 26 us, the first pass of all sequences at
// 3.9 TB/s (conversions to 64 bits: 16 a clock and SM), then the few that take two more; 48 of 8 drawn over 131,072 f32: 30 us. For
// few sequences bound by the chain launch, node words, probabilities, pass, exchange, chunk, place: 7.5 us for one of 6 over 32,003.
#include "codec.cuh"
#include "common.cuh"
#include "tc_common.cuh"

namespace {

constexpr int DV_THREADS = 256, DV_WARPS = DV_THREADS / 32;
constexpr int DV_NODES = 64, DV_MAX_VOCAB = 1 << 20, DV_MAX_CLUSTER = 8;

struct VerifyArgs {
    const int32_t* node_start; const int32_t* parent; const int32_t* token;
    const void* target; const void* draft;
    long long target_stride, draft_stride;
    int vocab, chunks;                   // chunks: of a block
    const float* u; const float* u_next;
    int32_t* path; int max_path; int32_t* n_path; int32_t* next;
};

__device__ __forceinline__ float clean(float x) { return x > 0.0f && x < INFINITY ? x : 0.0f; }
__device__ __forceinline__ uint32_t cluster_rank() { uint32_t r; asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ uint32_t cluster_size() { uint32_t r; asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(r)); return r; }
// (aligned: a warp has to come with all its lanes, whatever branch a part of them took before)
__device__ __forceinline__ void cluster_arrive() { __syncwarp(); asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { __syncwarp(); asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_sync() { cluster_arrive(); cluster_wait(); }
__device__ __forceinline__ void put_remote(double* mine, uint32_t rank, double v) {
    uint32_t at;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"((uint32_t)__cvta_generic_to_shared(mine)), "r"(rank));
    asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(at), "d"(v) : "memory");
}
__device__ __forceinline__ uint4 load16(uint32_t at) {
    uint4 w;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(w.x), "=r"(w.y), "=r"(w.z), "=r"(w.w) : "r"(at) : "memory");
    return w;
}
__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

template <class T> struct Row;           // 16 bytes of probabilities
template <> struct Row<float> {
    static constexpr int PER = 4;
    __device__ static uint4 some(const float* p, int v, int end) {             // values from v on, zeros from `end` on
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = v + i < end ? __float_as_uint(p[v + i]) : 0u;
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
    __device__ static float one(const float* p, long long i) { return clean(p[i]); }
    __device__ static void unpack(const uint4 w, float* x) {
        const uint32_t v[4] = {w.x, w.y, w.z, w.w};
        uint32_t bad = 0u;               // a sign, or an exponent of ones that reaches the sign with one more
#pragma unroll
        for (int i = 0; i < 4; ++i) { x[i] = __uint_as_float(v[i]); bad |= v[i] | (v[i] + 0x00800000u); }
        if (__builtin_expect((bad & 0x80000000u) != 0u, 0)) {
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = clean(x[i]);
        }
    }
};
template <> struct Row<uint16_t> {
    static constexpr int PER = 8;
    __device__ static uint4 some(const uint16_t* p, int v, int end) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = (v + 2 * i < end ? (uint32_t)p[v + 2 * i] : 0u) | (v + 2 * i + 1 < end ? (uint32_t)p[v + 2 * i + 1] << 16 : 0u);
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
    __device__ static float one(const uint16_t* p, long long i) { return clean(rv_bf16_to_f32(p[i])); }
    __device__ static void unpack(const uint4 w, float* x) {
        const uint32_t v[4] = {w.x, w.y, w.z, w.w};
        uint32_t bad = 0u;               // (a half that carries into its neighbour had the sign itself)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[2 * i] = __uint_as_float(v[i] << 16); x[2 * i + 1] = __uint_as_float(v[i] & 0xffff0000u);
            bad |= v[i] | (v[i] + 0x00800080u);
        }
        if (__builtin_expect((bad & 0x80008000u) != 0u, 0)) {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = clean(x[i]);
        }
    }
};
constexpr int DV_STEPS = 4;              // 16-byte loads of a lane per chunk and row
// with the draft's rows: three blocks an SM and one chunk ahead; without: four and two
__host__ __device__ constexpr int per_sm(bool draft) { return draft ? 3 : 4; }
__host__ __device__ constexpr int ring_of(bool draft) { return draft ? 2 : 3; }
constexpr int ring_bytes(bool draft) { return DV_WARPS * ring_of(draft) * (draft ? 2 : 1) * DV_STEPS * 512; }
__host__ __device__ constexpr int ring_at(int chunks) { return (chunks + 1) & ~1; }   // (behind the sums, 16-byte aligned)
template <class T> __host__ __device__ constexpr int chunk_of() { return 32 * DV_STEPS * Row<T>::PER; }

template <class T, bool DRAFT, bool VEC>
__global__ void __launch_bounds__(DV_THREADS, per_sm(DRAFT))
draft_verify_kernel(VerifyArgs A) {
    constexpr int PER = Row<T>::PER, CHUNK = chunk_of<T>(), RING = ring_of(DRAFT), ROWS = DRAFT ? 2 : 1;
    extern __shared__ __align__(16) double sums[];             // [chunks] of this block's part, from the last pass; the ring
    __shared__ int s_token[DV_NODES];
    __shared__ float s_u[DV_NODES], s_p[DV_NODES], s_q[DV_NODES];
    __shared__ unsigned long long s_kids[DV_NODES];
    __shared__ int s_out[DV_NODES];                            // tokens left out of r (given drafts)
    __shared__ double s_part[2][DV_MAX_CLUSTER];               // the blocks' sums of a pass, by the pass's parity
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, b = blockIdx.y;
    const uint32_t rank = cluster_rank(), n_rank = cluster_size();
    // Another block's shared memory may be written once that block runs: blocks of a cluster are placed together, but do not start
    // together. The nodes' words are read meanwhile.
    cluster_arrive();
    rv_grid_dep_wait();
    rv_grid_dep_trigger();
    const int start = A.node_start[b], T_all = A.node_start[b + 1] - start, T_n = min(T_all, DV_NODES);
    const T* target = reinterpret_cast<const T*>(A.target);
    const T* draft = reinterpret_cast<const T*>(A.draft);
    if (tid < DV_NODES) s_kids[tid] = 0ull;
    __syncthreads();
    if (tid < T_n) {
        const int par = A.parent[start + tid], tok = A.token[start + tid];
        const bool child = tid > 0 && par >= 0 && par < tid, known = tok >= 0 && tok < A.vocab;
        s_token[tid] = known ? tok : -1;
        s_u[tid] = A.u[start + tid];
        s_p[tid] = child && known ? Row<T>::one(target + (long long)(start + par) * A.target_stride, tok) : 0.0f;
        s_q[tid] = DRAFT ? (child && known ? Row<T>::one(draft + (long long)(start + par) * A.draft_stride, tok) : 0.0f) : 1.0f;
        if (child) atomicOr(&s_kids[par], 1ull << tid);
    }
    __syncthreads();
    int32_t* path = A.path + (size_t)b * A.max_path;
    cluster_wait();                                            // all blocks have started
    if (T_n <= 0) {                                            // (the same for all blocks of the cluster)
        if (rank == 0 && tid == 0) { A.n_path[b] = 0; A.next[b] = -1; }
        return;
    }

    const int lo = (int)rank * A.chunks * CHUNK, hi = min(A.vocab, lo + A.chunks * CHUNK);   // (at most 2^20 + 8 chunks)
    const int n_chunks = hi > lo ? (hi - lo + CHUNK - 1) / CHUNK : 0;
    int parity = 0;
    // r at an index of the current node's rows, up to a factor
    auto value = [&](double a, double bq, float p, float q) -> double { return DRAFT ? fmax(a * (double)p - bq * (double)q, 0.0) : (double)p; };
    auto left_out = [&](int v, int n_out) -> bool {
        bool hit = false;
        for (int i = 0; i < n_out; ++i) hit |= s_out[i] == v;
        return hit;
    };
    // a lane's share of the sum of r over a full chunk
    auto share = [&](const uint4 (&wp)[DV_STEPS], const uint4 (&wq)[DV_STEPS], int at, double a, double bq, int n_out) -> double {
        double s = 0.0, s2 = 0.0;
#pragma unroll
        for (int i = 0; i < DV_STEPS; ++i) {
            float xp[PER], xq[PER];
            Row<T>::unpack(wp[i], xp);
            if (DRAFT) Row<T>::unpack(wq[i], xq);
            if (!DRAFT)
                for (int k = 0; k < n_out; ++k) {
                    const int d = s_out[k] - (at + (i * 32 + lane) * PER);
#pragma unroll
                    for (int e = 0; e < PER; ++e) xp[e] = d == e ? 0.0f : xp[e];
                }
#pragma unroll
            for (int e = 0; e < PER; e += 2) {
                s += value(a, bq, xp[e], DRAFT ? xq[e] : 0.0f);
                s2 += value(a, bq, xp[e + 1], DRAFT ? xq[e + 1] : 0.0f);
            }
        }
        return s + s2;
    };
    // sum of r over chunk c of the rows of node `cur`, without the tokens that are left out (all lanes)
    auto chunk_sum = [&](const T* p, const T* q, int c, double a, double bq, int n_out) -> double {
        const int at = lo + c * CHUNK;
        double s = 0.0;
        if (VEC && at + CHUNK <= hi) {
            uint4 wp[DV_STEPS], wq[DV_STEPS];
#pragma unroll
            for (int i = 0; i < DV_STEPS; ++i) wp[i] = __ldg(reinterpret_cast<const uint4*>(p + at) + i * 32 + lane);
            if (DRAFT) {
#pragma unroll
                for (int i = 0; i < DV_STEPS; ++i) wq[i] = q ? __ldg(reinterpret_cast<const uint4*>(q + at) + i * 32 + lane) : make_uint4(0u, 0u, 0u, 0u);
            }
            s = share(wp, wq, at, a, bq, n_out);
        } else {
            for (int v = at + lane; v < min(at + CHUNK, hi); v += 32)
                if (DRAFT || !left_out(v, n_out)) s += value(a, bq, Row<T>::one(p, v), DRAFT && q ? Row<T>::one(q, v) : 0.0f);
        }
        return warp_sum(s);
    };
    // the chunk sums' sum over the vocabulary, the same in every thread of the cluster
    auto all_sums = [&]() -> double {
        __syncthreads();
        if (warp == 0) {
            double s = 0.0;
            for (int c = lane; c < n_chunks; c += 32) s += sums[c];
            s = warp_sum(s);
            if (lane < (int)n_rank) put_remote(&s_part[parity][rank], lane, s);
        }
        cluster_sync();
        double z = 0.0;
        for (uint32_t i = 0; i < n_rank; ++i) z += s_part[parity][i];
        parity ^= 1;                     // (the next sum goes to the other set: a block may still be reading this one)
        return z;
    };
    // one pass over the rows of node `cur`
    auto pass = [&](int cur, double a, double bq) -> double {
        const T* p = target + (long long)(start + cur) * A.target_stride;
        const T* q = DRAFT && bq != 0.0 ? draft + (long long)(start + cur) * A.draft_stride : nullptr;
        const int n_full = VEC && hi > lo ? (hi - lo) / CHUNK : 0;
        // a warp's chunks come through its own ring, each lane reading what it copied itself
        const uint32_t ring = (uint32_t)__cvta_generic_to_shared(sums + ring_at(A.chunks)) + (warp * RING * ROWS * DV_STEPS * 32 + lane) * 16;
        auto fetch = [&](int c, int slot) {
            if (c < n_full) {
                const uint32_t to = ring + slot * (ROWS * DV_STEPS * 512);
                const T* from = p + lo + c * CHUNK + lane * PER;
#pragma unroll
                for (int i = 0; i < DV_STEPS; ++i) tc::cp_async16(to + i * 512, from + i * 32 * PER);
                if (DRAFT && q) {
                    const T* qf = q + lo + c * CHUNK + lane * PER;
#pragma unroll
                    for (int i = 0; i < DV_STEPS; ++i) tc::cp_async16(to + (DV_STEPS + i) * 512, qf + i * 32 * PER);
                }
            }
            tc::cp_async_commit();
        };
        int slot = 0;
#pragma unroll
        for (int i = 0; i < RING - 1; ++i) fetch(warp + i * DV_WARPS, i);
#pragma unroll 1
        for (int c = warp; c < n_full; c += DV_WARPS) {
            const int over = slot == 0 ? RING - 1 : slot - 1;
            fetch(c + (RING - 1) * DV_WARPS, over);
            tc::cp_async_wait<RING - 1>();
            const uint32_t at = ring + slot * (ROWS * DV_STEPS * 512);
            uint4 wp[DV_STEPS], wq[DV_STEPS];
#pragma unroll
            for (int i = 0; i < DV_STEPS; ++i) {
                wp[i] = load16(at + i * 512);
                if (DRAFT) wq[i] = q ? load16(at + (DV_STEPS + i) * 512) : make_uint4(0u, 0u, 0u, 0u);
            }
            const double s = warp_sum(share(wp, wq, 0, a, bq, 0));
            if (lane == 0) sums[c] = s;
            slot = slot == RING - 1 ? 0 : slot + 1;
        }
        for (int c = n_full + warp; c < n_chunks; c += DV_WARPS) {         // (the last one, or all where nothing is aligned)
            const double s = chunk_sum(p, q, c, a, bq, 0);
            if (lane == 0) sums[c] = s;
        }
        return all_sums();
    };
    // the sums of the chunks that hold a token that is left out, again and without it (two tokens of a chunk: twice the same)
    auto without = [&](int cur, int n_out) -> double {
        const T* p = target + (long long)(start + cur) * A.target_stride;
        for (int k = warp; k < n_out; k += DV_WARPS) {
            const int v = s_out[k];
            if (v < lo || v >= hi) continue;
            const int c = (v - lo) / CHUNK;
            const double s = chunk_sum(p, nullptr, c, 1.0, 0.0, n_out);
            if (lane == 0) sums[c] = s;
        }
        return all_sums();
    };

    int cur = 0, n = 1, n_out = 0;
    double a = 1.0, bq = 0.0, total = 0.0;
    double da = 1.0, db = 0.0;           // the two numbers of the last pass: the chunk sums' scale, and the draw's
    double whole = 0.0;                  // (chosen tokens) the sum of the node's row
    bool have = false, dead = false;     // have: the chunk sums are those of the node; dead: nothing is left of r
    bool apart = false;                  // (chosen tokens) the chunk sums are without the tokens left out
    unsigned long long kids = s_kids[0];
    if (rank == 0 && tid == 0) path[0] = 0;
    while (kids && n < A.max_path) {
        const int j = __ffsll((long long)kids) - 1;
        kids &= kids - 1;
        const double p = s_p[j], q = s_q[j];
        const bool out = !DRAFT && left_out(s_token[j], n_out);
        const double r = DRAFT ? fmax(a * p - bq * q, 0.0) : out ? 0.0 : a * p;
        if (!dead && (double)s_u[j] * q < r) {
            if (rank == 0 && tid == 0) path[n] = j;
            cur = j; ++n; kids = s_kids[j];
            a = 1.0; bq = 0.0; n_out = 0; have = dead = apart = false;
            continue;
        }
        if (dead) continue;
        if (DRAFT) {
            bq += 1.0;
            da = a; db = bq;
            total = pass(cur, da, db);
            have = true;
            if (total > 0.0) { a /= total; bq /= total; }      // r / Z (the draw needs no division)
            else { dead = true; have = false; }
            continue;
        }
        if (!have) { whole = total = pass(cur, 1.0, 0.0); have = true; }
        if (!out && s_token[j] >= 0) {
            __syncthreads();             // (everyone has looked at the list)
            if (tid == 0) s_out[n_out] = s_token[j];
            ++n_out;
            __syncthreads();
            total -= p;
            apart = false;
            if (total < whole * 0.0009765625) { total = without(cur, n_out); apart = true; }
        }
        if (total > 0.0) a = 1.0 / total;
        else { dead = true; have = false; }
    }
    if (!have) { da = 1.0; db = 0.0; n_out = 0; total = pass(cur, da, db); }
    else if (!DRAFT && n_out && !apart) total = without(cur, n_out);
    if (rank == 0 && tid == 0) A.n_path[b] = n;

    // The block whose part holds the draw finds the chunk and the place in it, with one warp.
    const double want = (double)A.u_next[b] * total;
    const double* part = s_part[parity ^ 1];
    int owner = -1, last = -1;
    double before = 0.0, run = 0.0;
    for (uint32_t i = 0; i < n_rank; ++i) {
        const double s = part[i];
        if (s > 0.0) last = (int)i;
        if (owner < 0 && run + s > want && s > 0.0) { owner = (int)i; before = run; }
        run += s;
    }
    const bool none = owner < 0;         // the last value that is not zero
    if (none) { owner = last; before = 0.0; }
    if (last < 0) { if (rank == 0 && tid == 0) A.next[b] = -1; }
    else if (owner == (int)rank && warp == 0) {
        // the first lane whose running sum passes `want`, or the last that has any: its index, and what came before it
        auto find = [&](double mine, double from, bool& hit, double& base) -> int {
            double inc = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) { const double t = __shfl_up_sync(0xffffffffu, inc, o); if (lane >= o) inc += t; }
            const double over = __shfl_up_sync(0xffffffffu, inc, 1);
            const double exc = from + (lane ? over : 0.0);
            const uint32_t m = __ballot_sync(0xffffffffu, mine > 0.0 && from + inc > want && !none), pos = __ballot_sync(0xffffffffu, mine > 0.0);
            hit = m != 0;
            const int who = m ? __ffs(m) - 1 : 31 - __clz(pos | 1u);
            base = __shfl_sync(0xffffffffu, exc, who);
            return who;
        };
        // chunk: lanes take runs of chunks in order
        const int each = (n_chunks + 31) >> 5;
        double mine = 0.0;
        for (int i = 0; i < each; ++i) { const int c = lane * each + i; if (c < n_chunks) mine += sums[c]; }
        bool hit;
        double base;
        const int who = find(mine, before, hit, base);
        int chunk = -1;
        double run2 = base;
        for (int i = 0; i < each; ++i) {                       // (uniform: all lanes look at the same chunks)
            const int c = who * each + i;
            if (c >= n_chunks) break;
            const double s = sums[c];
            if (s > 0.0) {
                chunk = c; base = run2;
                if (hit && run2 + s > want) break;
            }
            run2 += s;
        }
        // place: the chunk's runs of 32 x PER values, all asked for at once, then the run's lanes, then a lane's values
        const T* p = target + (long long)(start + cur) * A.target_stride;
        const T* q = DRAFT && db != 0.0 ? draft + (long long)(start + cur) * A.draft_stride : nullptr;
        const int at = lo + chunk * CHUNK, end = min(at + CHUNK, hi);
        uint4 wp[DV_STEPS], wq[DV_STEPS];
#pragma unroll
        for (int i = 0; i < DV_STEPS; ++i) {
            const int v = at + (i * 32 + lane) * PER;
            wp[i] = wq[i] = make_uint4(0u, 0u, 0u, 0u);
            if (VEC && v + PER <= end) {
                wp[i] = __ldg(reinterpret_cast<const uint4*>(p + v));
                if (DRAFT && q) wq[i] = __ldg(reinterpret_cast<const uint4*>(q + v));
            } else {
                wp[i] = Row<T>::some(p, v, end);
                if (DRAFT && q) wq[i] = Row<T>::some(q, v, end);
            }
        }
        double x[PER];
        auto values = [&](const uint4 a4, const uint4 b4, int v) -> double {
            float xp[PER], xq[PER];
            Row<T>::unpack(a4, xp);
            Row<T>::unpack(b4, xq);
            if (!DRAFT)
                for (int k = 0; k < n_out; ++k) {
                    const int d = s_out[k] - v;
#pragma unroll
                    for (int e = 0; e < PER; ++e) xp[e] = d == e ? 0.0f : xp[e];
                }
            double sum = 0.0;
#pragma unroll
            for (int e = 0; e < PER; ++e) { x[e] = value(da, db, xp[e], xq[e]); sum += x[e]; }
            return sum;
        };
        double s4[DV_STEPS];
#pragma unroll
        for (int i = 0; i < DV_STEPS; ++i) s4[i] = values(wp[i], wq[i], at + (i * 32 + lane) * PER);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1)
#pragma unroll
            for (int i = 0; i < DV_STEPS; ++i) s4[i] += __shfl_xor_sync(0xffffffffu, s4[i], o);
        int pick = -1;                   // the run whose sum passes `want`, or the last that has any
        double start_of = base;
#pragma unroll
        for (int i = 0; i < DV_STEPS; ++i) {
            const double s = s4[i];
            const bool passed = pick >= 0 && hit && !none && start_of > want;   // (a run before has it)
            if (s > 0.0 && !passed) { pick = i; base = run2 = start_of; }
            if (!passed) start_of += s;
            if (s > 0.0 && hit && start_of > want) start_of = INFINITY;         // found: nothing behind it is looked at
        }
        if (pick >= 0) {
            uint4 a4 = wp[0], b4 = wq[0];
#pragma unroll
            for (int i = 1; i < DV_STEPS; ++i)
                if (pick == i) { a4 = wp[i]; b4 = wq[i]; }
            const int v = at + (pick * 32 + lane) * PER;
            const double mine2 = values(a4, b4, v);
            const int who2 = find(mine2, base, hit, run2);
            if (lane == who2) {
                int found = -1;
                bool done = false;
#pragma unroll
                for (int e = 0; e < PER; ++e) {
                    if (x[e] > 0.0 && !done) {
                        found = v + e;
                        done = hit && run2 + x[e] > want;
                    }
                    run2 += x[e];
                }
                A.next[b] = found;
            }
        }
    }
    cluster_sync();                      // no block leaves while another may still write into it
}

template <class T, bool DRAFT, bool VEC>
int launch(const VerifyArgs& a, int n, int B, cudaStream_t st) {
    rv_drain_error();
    const size_t smem = (size_t)ring_at(a.chunks) * sizeof(double) + (VEC ? ring_bytes(DRAFT) : 0);
    rv_allow_smem<draft_verify_kernel<T, DRAFT, VEC>>(ring_at(DV_MAX_VOCAB / chunk_of<T>()) * 8 + ring_bytes(DRAFT));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)n, (unsigned)B); cfg.blockDim = dim3(DV_THREADS);
    cfg.dynamicSmemBytes = smem; cfg.stream = st;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = (unsigned)n; at[1].val.clusterDim.y = 1; at[1].val.clusterDim.z = 1;
    cfg.attrs = at; cfg.numAttrs = 2;
    (void)cudaLaunchKernelEx(&cfg, draft_verify_kernel<T, DRAFT, VEC>, a);
    return rv_launch_status();
}
template <class T>
int dispatch(VerifyArgs& a, int B, cudaStream_t st) {
    // blocks a sequence: as many as run at once, while a part has four chunks
    const int sms = rv_sm_count(), all = (a.vocab + chunk_of<T>() - 1) / chunk_of<T>();
    int n = 1;
    while (n < DV_MAX_CLUSTER && (long long)B * 2 * n <= per_sm(a.draft != nullptr) * sms && all / (2 * n) >= 4) n *= 2;
    a.chunks = (all + n - 1) / n;
    const bool vec = (((uintptr_t)a.target | (uintptr_t)a.draft) & 15) == 0 && a.target_stride * (long long)sizeof(T) % 16 == 0 &&
                     (!a.draft || a.draft_stride * (long long)sizeof(T) % 16 == 0);
    if (a.draft) return vec ? launch<T, true, true>(a, n, B, st) : launch<T, true, false>(a, n, B, st);
    return vec ? launch<T, false, true>(a, n, B, st) : launch<T, false, false>(a, n, B, st);
}

}  // namespace

RIVOLI_API int rivoli_draft_verify(const int32_t* node_start, const int32_t* parent, const int32_t* token, const void* target,
                                   long long target_stride, const void* draft, long long draft_stride, int prob_bits, int vocab,
                                   const float* u, const float* u_next, int B, int32_t* path, int max_path, int32_t* n_path,
                                   int32_t* next, void* stream) {
    if (!node_start || !parent || !token || !target || !u || !u_next || !path || !n_path || !next || B <= 0 || vocab <= 0 || max_path <= 0)
        return 1001;
    if (vocab > DV_MAX_VOCAB || max_path > DV_NODES || B > 65535) return 1002;
    if (prob_bits != 32 && prob_bits != 16) return 1004;
    if (target_stride < vocab || (draft && draft_stride < vocab)) return 1005;
    if (((uintptr_t)target | (uintptr_t)draft) & (prob_bits / 8 - 1)) return 1005;
    VerifyArgs a{node_start, parent, token, target, draft, target_stride, draft_stride, vocab, 0, u, u_next, path, max_path, n_path, next};
    return prob_bits == 32 ? dispatch<float>(a, B, (cudaStream_t)stream) : dispatch<uint16_t>(a, B, (cudaStream_t)stream);
}
