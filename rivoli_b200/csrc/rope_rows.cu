// Rotary positions of bf16 rows: y = scale * R(pos * f) x on `seg` values of every vector of a row.
//
//     (y_u, y_v) = scale * (x_a cos t - x_b sin t, x_a sin t + x_b cos t),   t = pos[row] * inv_freq[i],   i < seg / 2
//
// with (a, b) -> (u, v) by layout: adjacent (2i, 2i+1) in place, half (i, i + seg/2) in place, split (2i, 2i+1) -> (i, i + seg/2),
// which is what rivoli_rope_interleave does to one vector (crates/backend/kernels/activation.hip:362-371).
//
// Angles of far positions need more than 32 bits: the product and its remainder by a turn are taken in 64, which leaves an angle of
// at most pi for the 32-bit sine and cosine (error 1e-7 of a turn's radius, against 2^-9 of the bf16 result). They are computed once
// per (row, pair) into shared memory and serve every vector of the row; the rotation is done in 32 bits and rounded once.
// Bound by memory: each value is read and written once. A lane takes eight pairs (two 16-byte loads and stores). 16,381 rows of 64
// vectors, 64 values out of 256 each, and a shared one: 52 us, 5.2 TB/s. Two or four vectors a lane at once, 4 to 32 rows a block and
// loads ahead of the angles come to between 51 and 64 us: what is left is the reads of 128 bytes out of every 512.
#include "codec.cuh"
#include "common.cuh"

namespace {

constexpr int RR_THREADS = 256, RR_WARPS = RR_THREADS / 32;
constexpr int RR_MAX_SEG = 512;
constexpr int RR_MAX_ROWS = 8;          // rows of a block

struct RopeArgs {
    RopeVecs q, k;                      // k.n_vec = 0: none
    int n_rows, rows, seg, layout;      // rows: of a block
    const int32_t* pos; const double* inv_freq;
    float scale;
};

__device__ __forceinline__ float2 angle_of(int pos, double f, float scale) {
    const double t = (double)pos * f;
    const double n = rint(t * 0.15915494309189535);                 // turns
    double r = fma(-n, 6.283185307179586, t);                       // 2 pi in two terms
    r = fma(-n, 2.4492935982947064e-16, r);
    float s, c;
    sincosf((float)r, &s, &c);
    return make_float2(c * scale, s * scale);
}

__device__ __forceinline__ uint32_t pack2(float a, float b) {
    uint32_t w;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(b), "f"(a));
    return w;
}
__device__ __forceinline__ float2 unpack2(uint32_t w) { return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); }

// Vector v of row `row` (q's vectors first): where its segment is read and written.
__device__ __forceinline__ void place(const RopeArgs& A, long long row, int v, const uint16_t*& src, uint16_t*& dst) {
    const bool is_q = v < A.q.n_vec;
    const RopeVecs& w = is_q ? A.q : A.k;
    const int i = is_q ? v : v - A.q.n_vec;
    src = w.src + row * w.src_row + i * w.src_vec;
    dst = w.dst + row * w.dst_row + i * w.dst_vec;
}

// VEC: segments of a multiple of 16 values, everything on 16-byte boundaries: seg / 16 lanes a vector, as many whole vectors a
// warp as fit. Otherwise a warp per vector, a pair per lane and step. Either way a vector is read by one warp before any of it is
// written, so that a call may rotate in place.
template <bool VEC>
__global__ void __launch_bounds__(RR_THREADS)
rope_rows_kernel(RopeArgs A) {
    extern __shared__ float2 turns[];                               // [rows][seg / 2]
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, half = A.seg >> 1;
    const long long row0 = (long long)blockIdx.x * A.rows;
    const int rows = min((long long)A.rows, A.n_rows - row0);
    rv_grid_dep_wait();
    rv_grid_dep_trigger();
    for (int i = tid; i < rows * half; i += RR_THREADS) {
        const int r = i / half;
        turns[i] = angle_of(A.pos[row0 + r], A.inv_freq[i - r * half], A.scale);
    }
    __syncthreads();
    const int n_vec = A.q.n_vec + A.k.n_vec, total = rows * n_vec;
    if (VEC) {
        const int lanes = A.seg >> 4, per_warp = 32 / lanes, sub = lane / lanes, l = lane - sub * lanes;
        const int step = RR_WARPS * per_warp * gridDim.y;
        for (int at = (blockIdx.y * RR_WARPS + warp) * per_warp; at < total; at += step) {
            const int item = at + sub;
            const bool mine = sub < per_warp && item < total;
            uint4 x = make_uint4(0u, 0u, 0u, 0u), y = x;
            uint16_t* dst = nullptr;
            int r = 0;
            const int off = A.layout == RV_ROPE_HALF ? 8 * l : 16 * l, second = A.layout == RV_ROPE_HALF ? half : 8;
            if (mine) {
                r = item / n_vec;
                const uint16_t* src;
                place(A, row0 + r, item - r * n_vec, src, dst);
                x = *reinterpret_cast<const uint4*>(src + off);
                y = *reinterpret_cast<const uint4*>(src + off + second);
            }
            __syncwarp();
            if (!mine) continue;
            const float4* t4 = reinterpret_cast<const float4*>(turns + r * half + 8 * l);
            const uint32_t w[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
            float u[8], v[8];
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                const float4 cs = t4[i >> 1];                       // (cos, sin) of pairs i and i + 1
                float a0, b0, a1, b1;
                if (A.layout == RV_ROPE_HALF) {
                    const float2 a = unpack2(w[i >> 1]), b = unpack2(w[4 + (i >> 1)]);
                    a0 = a.x; a1 = a.y; b0 = b.x; b1 = b.y;
                } else {
                    const float2 p = unpack2(w[i]), s = unpack2(w[i + 1]);
                    a0 = p.x; b0 = p.y; a1 = s.x; b1 = s.y;
                }
                u[i] = a0 * cs.x - b0 * cs.y; v[i] = a0 * cs.y + b0 * cs.x;
                u[i + 1] = a1 * cs.z - b1 * cs.w; v[i + 1] = a1 * cs.w + b1 * cs.z;
            }
            if (A.layout == RV_ROPE_ADJACENT) {
                x = make_uint4(pack2(u[0], v[0]), pack2(u[1], v[1]), pack2(u[2], v[2]), pack2(u[3], v[3]));
                y = make_uint4(pack2(u[4], v[4]), pack2(u[5], v[5]), pack2(u[6], v[6]), pack2(u[7], v[7]));
                *reinterpret_cast<uint4*>(dst + 16 * l) = x;
                *reinterpret_cast<uint4*>(dst + 16 * l + 8) = y;
            } else {
                x = make_uint4(pack2(u[0], u[1]), pack2(u[2], u[3]), pack2(u[4], u[5]), pack2(u[6], u[7]));
                y = make_uint4(pack2(v[0], v[1]), pack2(v[2], v[3]), pack2(v[4], v[5]), pack2(v[6], v[7]));
                *reinterpret_cast<uint4*>(dst + 8 * l) = x;
                *reinterpret_cast<uint4*>(dst + half + 8 * l) = y;
            }
        }
    } else {
        for (int item = blockIdx.y * RR_WARPS + warp; item < total; item += RR_WARPS * gridDim.y) {
            const int r = item / n_vec;
            const uint16_t* src;
            uint16_t* dst;
            place(A, row0 + r, item - r * n_vec, src, dst);
            uint16_t a[RR_MAX_SEG / 64], b[RR_MAX_SEG / 64];
#pragma unroll
            for (int s = 0; s < RR_MAX_SEG / 64; ++s) {
                const int i = lane + 32 * s;
                if (i >= half) break;
                a[s] = src[A.layout == RV_ROPE_HALF ? i : 2 * i];
                b[s] = src[A.layout == RV_ROPE_HALF ? i + half : 2 * i + 1];
            }
            __syncwarp();
#pragma unroll
            for (int s = 0; s < RR_MAX_SEG / 64; ++s) {
                const int i = lane + 32 * s;
                if (i >= half) break;
                const float2 cs = turns[r * half + i];
                const float x = rv_bf16_to_f32(a[s]), y = rv_bf16_to_f32(b[s]);
                dst[A.layout == RV_ROPE_ADJACENT ? 2 * i : i] = rv_f32_to_bf16(x * cs.x - y * cs.y);
                dst[A.layout == RV_ROPE_ADJACENT ? 2 * i + 1 : i + half] = rv_f32_to_bf16(x * cs.y + y * cs.x);
            }
            __syncwarp();
        }
    }
}

// Segments that are written must not lie on one another: vectors of a row, and rows.
bool apart(const RopeVecs& w, int n_rows, int seg) {
    auto near = [&](int64_t stride) { return stride > -seg && stride < seg; };
    return !(w.n_vec > 1 && near(w.dst_vec)) && !(n_rows > 1 && near(w.dst_row));
}
bool aligned16(const RopeVecs& w) {
    return ((((uintptr_t)w.src | (uintptr_t)w.dst) & 15) | ((w.src_row | w.src_vec | w.dst_row | w.dst_vec) & 7)) == 0;
}

}  // namespace

RIVOLI_API int rivoli_rope_rows_bf16(const RopeVecs* q, const RopeVecs* k, int n_rows, const int32_t* pos, const double* inv_freq,
                                     int seg, int layout, float scale, void* stream) {
    if (!q || n_rows <= 0 || !pos || !inv_freq || seg <= 0 || q->n_vec <= 0 || !q->src || !q->dst) return 1001;
    if (k && (k->n_vec <= 0 || !k->src || !k->dst)) return 1001;
    if (seg > RR_MAX_SEG || q->n_vec > 65536 || (k && k->n_vec > 65536)) return 1002;
    if (layout < RV_ROPE_ADJACENT || layout > RV_ROPE_SPLIT) return 1003;
    if (seg % 2) return 1004;
    if (((uintptr_t)q->src | (uintptr_t)q->dst | (k ? (uintptr_t)k->src | (uintptr_t)k->dst : 0)) & 1) return 1005;
    if (!apart(*q, n_rows, seg) || (k && !apart(*k, n_rows, seg))) return 1005;
    RopeArgs a{*q, k ? *k : RopeVecs{}, n_rows, 1, seg, layout, pos, inv_freq, scale};
    const bool vec = seg % 16 == 0 && aligned16(*q) && (!k || aligned16(*k));
    const int n_vec = a.q.n_vec + a.k.n_vec;
    // As many rows a block as leave four blocks to an SM; with fewer rows than that, several blocks share a row's vectors.
    const int sms = rv_sm_count();
    a.rows = n_rows / (4 * sms);
    a.rows = a.rows < 1 ? 1 : (a.rows > RR_MAX_ROWS ? RR_MAX_ROWS : a.rows);
    const int per_pass = vec ? RR_WARPS * (32 / (seg / 16)) : RR_WARPS;
    const int passes = (a.rows * n_vec + per_pass - 1) / per_pass, blocks = (n_rows + a.rows - 1) / a.rows;
    int split = sms / blocks;
    split = split < 1 ? 1 : (split > passes ? passes : split);
    rv_drain_error();
    const size_t smem = (size_t)a.rows * (seg / 2) * sizeof(float2);
    if (vec) rv_launch_dependent(rope_rows_kernel<true>, dim3(blocks, split), dim3(RR_THREADS), smem, (cudaStream_t)stream, a);
    else rv_launch_dependent(rope_rows_kernel<false>, dim3(blocks, split), dim3(RR_THREADS), smem, (cudaStream_t)stream, a);
    return rv_launch_status();
}
