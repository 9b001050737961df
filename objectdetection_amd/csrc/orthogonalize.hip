// Orthogonalisation of matrices by Newton-Schulz products, and the optimizer step built on it.
//
//   X_0 = G / (|G|_F + eps), transposed where G has more rows than columns (X is m x n, m <= n);
//   per step   A = X X^T,   P = a I + b A + c A A,   X <- P X.
// The odd polynomial a s + b s^3 + c s^5 acts on every singular value s of X and leaves the singular vectors: with
// (a, b, c) = (3.4445, -4.7750, 2.0315) five steps take singular values from 0.003 up to between 0.68 and 1.21 -- the values
// never pass 1.21, so every entry of X and A stays under 1.5 and of P under 3.5.
//
// Everything that happens to X is a polynomial in A_0 = X_0 X_0^T, so steps can also run on m x m matrices alone:
//   X_t = Q X_0,   Q = P_t ... P_1,   A_(k+1) = P_k A_k P_k
// with one product by X at the end of a phase of t steps: 1.5 m^2 n + (2 t - 1.5) m^3 multiply-adds for it (symmetric products
// counted half) against t (1.5 m^2 n + 0.5 m^3).  What it costs is accuracy in the directions of small singular values: a
// rounding of A grows by 3.4445^2 per step there, where a rounding of X grows by 3.4445.
//   - At most 64 rows: A and all that follows in 64 bits, phases of ten steps (further down: "at most 64 rows").
//   - More rows, float32 results: phases of two steps, which keep float32's accuracy (error against 64 bits of 256 x 2304 noise
//     with strong directions: 1.6e-6, one step a phase 1.9e-6), where n >= 2 m; one step a phase on squarer ones, which costs no
//     more there.
//   - More rows, bfloat16 results and the optimizer step: phases of five.  1e-6 to 6e-5 on such matrices, under 7e-4
//     (3.4445^8 2^-24 = 1.2e-3) where the singular values fall like 1 / i^2 or vanish; a bfloat16 result is rounded by 2e-3,
//     and the step multiplies by the learning rate.
//
// The products of more rows run on fp16 pairs (gemm.h, PL = 2) scaled by 2^12 (Q, which grows to 3.4445^k, by less): the largest
// entry becomes 14 300, the smallest step 2^-36.  bf16 products would leave a few percent in the result.
// X is kept twice, by rows (X X^T reduces along n) and by columns (Q X reduces along m): both products then read their
// operands along the reduction.  The m x m matrices are symmetric to the bit: what lies on and over the diagonal is computed, the
// rest mirrored, within the tiles on the diagonal too.  Both halves of such a tile as they come differ by a rounding, and that
// difference grows by 3.4445^2 a step where A has no singular value: five steps on a matrix of rank 3 were off by 1.5 to 2 % with
// it, 2e-4 without; it costs 2 to 3 % of the time.  All matrices of a call share every launch.
//
// Eight 256 x 2304 in float32 take 207 us: 22 launches of 5 to 20 us, each a chain of a few latencies.  A step over the 94
// matrices of the detector's largest preset takes 4.7 ms: 4.0 ms of products at 53 % of the matrix rate of a large library
// product (tiles on the diagonal compute both halves; 128 x 128 tiles are bound by LDS reads and matrix instructions alike) and
// 0.7 ms of norm and layout at the rate of a copy.
#include "common.h"
#include "odamd.h"
#include "offsets.h"

#include <math.h>

namespace {

#include "gemm.h"

constexpr double NS_A = 3.4445, NS_B = -4.7750, NS_C = 2.0315;
constexpr float NS_SCALE = 4096.0f;
constexpr int NS_GROUPS = 112;        // groups of one launch: their table travels in the kernel's arguments (4 KiB at most)
constexpr int NS_FEW_STEPS = 10;      // steps of a phase of matrices of at most 64 rows
constexpr int NS_PARTS = 512;         // partial sums of squares per matrix, at most

// stages: sums of squares, laying out, X X^T (whole, or a part of its reduction), P from A, products of square matrices, Q X,
// Q X to the caller; of matrices of few rows: all in one, G G^T, the steps, Q G
enum { ST_NORM, ST_SPLIT, ST_A, ST_AP, ST_P, ST_Q, ST_X, ST_OUT, ST_WHOLE, ST_GRAM, ST_STEPS, ST_QG };
__host__ __device__ constexpr bool ns_symmetric(int stage) { return stage == ST_A || stage == ST_AP || stage == ST_P || stage == ST_Q; }
__host__ __device__ constexpr bool ns_along_n(int stage) { return stage == ST_A || stage == ST_AP; }   // reduces over n, the others over m
// square matrices: A, a product on the way to the next A, and three that P and Q take in turn; X X^T leaves the sums of a cut
// reduction in all but the first
enum { SQ_A, SQ_T, SQ_B, SQ_COUNT = 5 };

// `count` matrices of one shape, one after the other
struct NsGroup {
    long long src;       // first element of the first matrix in the caller's buffers
    unsigned ws;         // start of the first one's workspace, in 256-byte units
    int m, n;            // m <= n
    int count;
    int tile0;           // tiles of the groups before this one
    int tall;            // the caller's matrix is n x m
};
struct NsTable {
    NsGroup g[NS_GROUPS];
    int n, tiles;
    char* ws;
};
// Up to two products of a stage: out = left right, squares by index, `scale` from the sum to the stored pair.  ST_AP: n parts of
// the reduction instead, at most NS_CUTS.
constexpr int NS_CUTS = SQ_COUNT - SQ_T;   // a part's sums lie in the place of a square that is not in use yet
struct NsJobs {
    int n, turn;         // turn: which of the two column copies of X is the current one
    int left[2], right[2], out[2];
    float scale[2];
};
static_assert(sizeof(NsTable) <= 3700, "kernel arguments are limited to 4 KiB");

__host__ __device__ inline long long ns_up(long long v, int to) { return (v + to - 1) / to * to; }
// Columns of an m x n matrix with few rows that a workgroup takes (t: m in 16-row tiles): all of them, or at least what its
// waves have under way at once, and at most 32 parts.  Parts cost two launches more; one workgroup / parts, us: 16 x 1000 12.3 /
// 14, 16 x 2000 20 / 16, 32 x 1000 35 / 32, 48 x 256 35 / 38, 48 x 512 44 / 40, 64 x 256 59 / 61, 64 x 512 75 / 64.
__host__ __device__ inline int ns_few_cols(int t, int n) {
    return n <= (t == 1 ? 1536 : 1024 / t) ? (int)ns_up(n, 16) : (int)ns_up(ns_up(n, 32) / 32, t <= 2 ? 512 : 128);
}
// Workspace of a matrix that is taken in parts: Q and the partial sums of G G^T, in 64 bits
__host__ __device__ inline long long ns_few_bytes(int t, int cols, int n) {
    return ns_up(8LL * (256 * t * t + ((long long)n + cols - 1) / cols * 128 * t * (t + 1)), 256);
}
// Byte offsets within a matrix's workspace; end is its size.
struct NsLayout { long long sums, x, xt0, xt1, sq, sq_size, end; };
__host__ __device__ inline NsLayout ns_layout(int m, int n) {
    NsLayout l;
    const long long mp = ns_up(m, 32), np = ns_up(n, 32);
    l.sums = 0;
    l.x = NS_PARTS * 8;
    l.xt0 = l.x + ns_up(m * np * 4, 256);
    l.xt1 = l.xt0 + ns_up(n * mp * 4, 256);
    l.sq = l.xt1 + ns_up(n * mp * 4, 256);
    l.sq_size = ns_up(m * mp * 4, 256);
    l.end = l.sq + SQ_COUNT * l.sq_size;
    return l;
}
// Elements one workgroup of the norm pass takes: a multiple of eight that keeps the partial sums within NS_PARTS.
__host__ __device__ inline long long ns_share(int m, int n) {
    const long long total = (long long)m * n, least = (total + NS_PARTS - 1) / NS_PARTS;
    return least < 8192 ? 8192 : ns_up(least, 2048);
}
__host__ __device__ inline int ns_parts(int m, int n) { return (int)(((long long)m * n + ns_share(m, n) - 1) / ns_share(m, n)); }
__host__ __device__ inline int ns_tiles(int stage, int tile, int m, int n) {
    if (stage == ST_WHOLE || stage == ST_STEPS) return 1;
    if (stage == ST_NORM) return ns_parts(m, n);
    const int mt = (int)((m + (long long)tile - 1) / tile), nt = (int)((n + (long long)tile - 1) / tile);
    return stage == ST_GRAM || stage == ST_QG ? nt : ns_symmetric(stage) ? mt * (mt + 1) / 2 : mt * nt;
}

// Chunks of a part
__host__ __device__ inline int ns_cut(int chunks, int cuts) { return (chunks + cuts - 1) / cuts; }

// What the optimizer step works on (orthogonalisation alone: in and out)
struct NsIo {
    const void* in;      // caller's matrices (the gradient, for the optimizer step)
    void* out;
    float* param;
    float* momentum;
    float* ema;
    float mu, grad_scale, shrink, lr02, ema_keep, ema_take;  // shrink: lr weight_decay, lr02: 0.2 lr
    int nesterov;
    double eps;
    float* x;            // matrices of few rows: X between phases of steps, one matrix of the table behind the other
    int scaled;          // and whether `in` is X already
};

struct NsPlace { int m, n, tall, tile, group; long long src; char* ws; };

// Which matrix a tile belongs to.  few: workspaces are those of matrices of few rows, `few` 16-row tiles, in parts of tile_size columns
__device__ __forceinline__ NsPlace ns_find(const NsTable& t, int tile, int stage, int tile_size, int few = 0) {
    // all groups at once: one latency, not one for every halving (78 matrices: 15 us launches are 0.5 us shorter)
    int lo = 0;
    if (t.n > 1) {
        const int lane = threadIdx.x & 63;
        lo = -1;
        for (int i = 0; i < t.n; i += 64) lo += __popcll(__ballot(i + lane < t.n && t.g[i + lane].tile0 <= tile));
    }
    const NsGroup& g = t.g[lo];
    const int each = ns_tiles(stage, tile_size, g.m, g.n), at = tile - g.tile0, which = at / each;
    return {g.m, g.n, g.tall, at - which * each, lo, g.src + (long long)which * g.m * g.n,
            t.ws + (long long)g.ws * 256 + which * (few ? ns_few_bytes(few, tile_size, g.n) : ns_layout(g.m, g.n).end)};
}

// The optimizer's direction from the updated momentum
__device__ __forceinline__ float ns_direction(const NsIo& io, float g, float m) {
    return io.nesterov ? g * io.grad_scale + io.mu * m : m;
}

__device__ __forceinline__ double ns_block_sum(double v, double* shared) {
#pragma unroll
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) shared[wave] = v;
    __syncthreads();
    double s = 0.0;
    for (int i = 0; i < (int)(blockDim.x >> 6); ++i) s += shared[i];
    return s;
}

// A parameter after the step: w (1 - lr weight_decay) - step v, with one rounding against w.  1 - lr weight_decay is not a factor of
// its own: a float32 under one has steps of 6e-8, an eighth of 5e-7 and more than 2e-8.
__device__ __forceinline__ float ns_new_param(const NsIo& io, float w, float step, float v) {
    return w - fmaf(io.shrink, w, step * v);
}

// Eight of the caller's values; zeros for those past the first `cnt`
template <int DT>
__device__ __forceinline__ void ns_load8(const void* base, long long at, int cnt, float v[8]) {
    if constexpr (DT == ODAMD_DTYPE_BF16) {
        const uint16_t* s = (const uint16_t*)base + at;
        if (cnt == 8) {
            const u32x4 u = *(const u32x4_any*)s;
#pragma unroll
            for (int e = 0; e < 4; ++e) { v[2 * e] = __uint_as_float(u[e] << 16); v[2 * e + 1] = __uint_as_float(u[e] & 0xffff0000u); }
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = e < cnt ? bf16_to_f32(s[e]) : 0.0f;
        }
    } else {
        const float* s = (const float*)base + at;
        if (cnt == 8) {
            const f32x4_t u = *(const f32x4_any*)s, w = *(const f32x4_any*)(s + 4);
#pragma unroll
            for (int e = 0; e < 4; ++e) { v[e] = u[e]; v[e + 4] = w[e]; }
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = e < cnt ? s[e] : 0.0f;
        }
    }
}

// Sums of squares in double (gradients of 1e-20 and of 1e20 have a norm too), a fixed share of a matrix per workgroup and
// summed in a fixed order: the result does not change from run to run.  The optimizer step's momentum update happens here.
template <bool MUON, int DT>
__global__ void __launch_bounds__(256) ns_norm_kernel(NsTable t, NsIo io) {
    __shared__ double part[4];
    const NsPlace p = ns_find(t, blockIdx.x, ST_NORM, 0);
    const long long total = (long long)p.m * p.n, share = ns_share(p.m, p.n), from = p.tile * share;
    const long long to = from + share < total ? from + share : total;
    double s = 0.0;
    // eight elements a thread
    float* mom = MUON ? io.momentum + p.src : nullptr;
    for (long long i = from + threadIdx.x * 8; i < to; i += 2048) {
        const int cnt = to - i < 8 ? (int)(to - i) : 8;
        float g[8], m[8];
        ns_load8<DT>(io.in, p.src + i, cnt, g);
        if constexpr (MUON) ns_load8<ODAMD_DTYPE_F32>(mom, i, cnt, m);
        if constexpr (MUON) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                m[e] = io.mu * m[e] + g[e] * io.grad_scale;
                g[e] = ns_direction(io, g[e], m[e]);
            }
            if (cnt == 8) {
                *(f32x4_any*)(mom + i) = f32x4_t{m[0], m[1], m[2], m[3]};
                *(f32x4_any*)(mom + i + 4) = f32x4_t{m[4], m[5], m[6], m[7]};
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (e < cnt) mom[i + e] = m[e];
            }
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) s += (double)g[e] * g[e];
    }
    s = ns_block_sum(s, part);
    if (threadIdx.x == 0) ((double*)p.ws)[p.tile] = s;
}

// X by rows and by columns as fp16 pairs, 64 x 64 elements per workgroup
template <bool MUON, int DT>
__global__ void __launch_bounds__(256) ns_split_kernel(NsTable t, NsIo io) {
    __shared__ double part[4];
    __shared__ float tile[64][65];
    const NsPlace p = ns_find(t, blockIdx.x, ST_SPLIT, 64);
    const NsLayout l = ns_layout(p.m, p.n);
    const int parts = ns_parts(p.m, p.n);
    double mine = 0.0;
    for (int i = threadIdx.x; i < parts; i += 256) mine += ((const double*)p.ws)[i];
    const double sum = ns_block_sum(mine, part);
    const double inv = 1.0 / (sqrt(sum) + io.eps);         // in double: a float32 norm may lie at either end of float32's range
    // in the caller's rows and columns: what lies along its rows goes out as it comes, the other copy through LDS
    const int rows = p.tall ? p.n : p.m, cols = p.tall ? p.m : p.n, ct = (cols + 63) / 64;
    const int r0 = p.tile / ct * 64, c0 = p.tile % ct * 64, c = (threadIdx.x & 7) * 8;
    const int rp = (int)ns_up(rows, 32), cp = (int)ns_up(cols, 32);
    char* along = p.ws + (p.tall ? l.xt0 : l.x);
    char* across = p.ws + (p.tall ? l.x : l.xt0);
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        const int r = (threadIdx.x >> 3) + 32 * q, cnt = r0 + r < rows ? max(0, min(8, cols - c0 - c)) : 0;
        const long long at = p.src + (long long)(r0 + r) * cols + c0 + c;
        float v[8], m[8];
        ns_load8<DT>(io.in, at, cnt, v);
        if constexpr (MUON) {
            ns_load8<ODAMD_DTYPE_F32>(io.momentum, at, cnt, m);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = ns_direction(io, v[e], m[e]);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            v[e] = e < cnt ? (float)(v[e] * inv) : 0.0f;
            tile[r][c + e] = v[e];
        }
        if (r0 + r < rows && c0 + c < cp) store_split8(along + (long long)(r0 + r) * cp * 4 + split_at(c0 + c), v, NS_SCALE);
    }
    __syncthreads();
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        const int r = (threadIdx.x >> 3) + 32 * q;
        float v[8];
        if (c0 + r < cols && r0 + c < rp) {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = tile[c + e][r];
            store_split8(across + (long long)(c0 + r) * rp * 4 + split_at(r0 + c), v, NS_SCALE);
        }
    }
}

// ---- at most 64 rows -------------------------------------------------------------------------------------------------
// All steps run on A = X X^T, in 64 bits (v_mfma_f64_16x16x4_f64, half the rate of the float32 instruction): a rounding of A, 2^-53,
// grows to 2^-53 3.4445^18 = 5e-7 in ten steps, so the result has float32's accuracy, and the caller's matrix is read twice only,
// for G G^T (whose trace is the norm) and for Q G.  What it costs is latency: 3 dependent products of m x m per step.  More steps
// start again from X every ten, which is held in float32 in between.
// T: m in 16-row tiles.  Squares lie in LDS, rows LD doubles apart: sixteen rows at two neighbouring k touch all 64 banks.
template <int T_> struct NsFew {
    static constexpr int T = T_, N = 16 * T, LD = N + 2, SQ = N * LD, TRI = T * (T + 1) / 2;
    static constexpr int WAVES = 8, THREADS = 64 * WAVES;
    static constexpr int KEPT = T <= 2 ? WAVES : WAVES / 2;  // waves whose sums lie in LDS side by side
    static constexpr int SUMS = TRI * 256;                   // G G^T: the tiles on and over the diagonal
    static constexpr int LDS = 8 * (3 * SQ > KEPT * SUMS ? 3 * SQ : KEPT * SUMS);
    static constexpr int AT_ONCE = T <= 2 ? 4 : 1;           // groups of sixteen columns a wave has under way
};
typedef double f64x4_t __attribute__((ext_vector_type(4)));
__device__ __forceinline__ f64x4_t ns_mma64(double a, double b, f64x4_t c) {
    return __builtin_amdgcn_mfma_f64_16x16x4f64(a, b, c, 0, 0, 0);
}
// Four values of the caller's, `stride` apart; zeros for those past the first cnt
template <int DT>
__device__ __forceinline__ void ns_load4(const void* base, long long at, long long stride, int cnt, float v[4]) {
    if constexpr (DT == ODAMD_DTYPE_F32) {
        const float* s = (const float*)base + at;
        if (stride == 1 && cnt == 4) {
            const f32x4_t u = *(const f32x4_any*)s;
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = u[e];
            return;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = e < cnt ? s[e * stride] : 0.0f;
    } else {
        const uint16_t* s = (const uint16_t*)base + at;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = e < cnt ? bf16_to_f32(s[e * stride]) : 0.0f;
    }
}
template <int DT>
__device__ __forceinline__ void ns_store4(void* base, long long at, long long stride, int cnt, const float v[4]) {
    if constexpr (DT == ODAMD_DTYPE_F32) {
        float* d = (float*)base + at;
        if (stride == 1 && cnt == 4) {
            *(f32x4_any*)d = f32x4_t{v[0], v[1], v[2], v[3]};
            return;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (e < cnt) d[e * stride] = v[e];
    } else {
        uint16_t* d = (uint16_t*)base + at;
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (e < cnt) d[e * stride] = f32_to_bf16(v[e]);
    }
}

// G G^T over columns [from, to): every wave's sums side by side in `sums`.  A lane loads four neighbouring columns of a row; that
// instruction e takes column 4 h + e of each group of sixteen does not matter to a sum over them.  The optimizer step's momentum
// update happens here.
template <int T, bool MUON, int DT>
__device__ __forceinline__ void ns_few_gram(const NsIo& io, const NsPlace& p, int from, int to, double* sums) {
    using F = NsFew<T>;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, h = lane >> 4;
    const long long sr = p.tall ? 1 : p.n, sc = p.tall ? p.m : 1;
    f64x4_t acc[F::TRI] = {};
    for (int c0 = from + wave * 16 * F::AT_ONCE; c0 < to; c0 += F::WAVES * 16 * F::AT_ONCE) {
        float x[F::AT_ONCE][T][4], m[F::AT_ONCE][T][4];
#pragma unroll
        for (int g = 0; g < F::AT_ONCE; ++g)
#pragma unroll
            for (int t = 0; t < T; ++t) {
                const int row = 16 * t + r, c = c0 + 16 * g + 4 * h, cnt = row < p.m ? max(0, min(4, to - c)) : 0;
                const long long at = p.src + row * sr + c * sc;
                ns_load4<DT>(io.in, at, sc, cnt, x[g][t]);
                if constexpr (MUON) ns_load4<DT>(io.momentum, at, sc, cnt, m[g][t]);
            }
#pragma unroll
        for (int g = 0; g < F::AT_ONCE; ++g) {
            if constexpr (MUON)
#pragma unroll
                for (int t = 0; t < T; ++t) {
                    const int row = 16 * t + r, c = c0 + 16 * g + 4 * h, cnt = row < p.m ? max(0, min(4, to - c)) : 0;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        m[g][t][e] = io.mu * m[g][t][e] + x[g][t][e] * io.grad_scale;
                        x[g][t][e] = e < cnt ? ns_direction(io, x[g][t][e], m[g][t][e]) : 0.0f;
                    }
                    ns_store4<DT>(io.momentum, p.src + row * sr + c * sc, sc, cnt, m[g][t]);
                }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                int k = 0;
#pragma unroll
                for (int j = 0; j < T; ++j)
#pragma unroll
                    for (int i = 0; i <= j; ++i, ++k) acc[k] = ns_mma64((double)x[g][i][e], (double)x[g][j][e], acc[k]);
            }
        }
    }
    const auto at = [&](int w, int k, int e) -> double& { return sums[(w * F::TRI + k) * 256 + e * 64 + lane]; };
    if constexpr (F::KEPT < F::WAVES) {
        // the second half of the waves hands its sums to the first
        if (wave >= F::KEPT)
#pragma unroll
            for (int k = 0; k < F::TRI; ++k)
#pragma unroll
                for (int e = 0; e < 4; ++e) at(wave - F::KEPT, k, e) = acc[k][e];
        __syncthreads();
        if (wave < F::KEPT)
#pragma unroll
            for (int k = 0; k < F::TRI; ++k)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[k][e] += at(wave, k, e);
    }
    if (wave < F::KEPT)
#pragma unroll
        for (int k = 0; k < F::TRI; ++k)
#pragma unroll
            for (int e = 0; e < 4; ++e) at(wave, k, e) = acc[k][e];
    __syncthreads();
}
// Value u of the sums of all waves, added in order
template <int T>
__device__ __forceinline__ double ns_few_sum(const double* sums, int u) {
    double s = sums[u];
#pragma unroll
    for (int w = 1; w < NsFew<T>::KEPT; ++w) s += sums[w * NsFew<T>::SUMS + u];
    return s;
}

// Q / (|G| + eps) from G G^T (Q where G is X already): value u of it is get(u).  Left in the third square of `lds`.
template <int T, typename GET>
__device__ __forceinline__ double* ns_few_steps(double* lds, int steps, const NsIo& io, GET&& get) {
    using F = NsFew<T>;
    constexpr int EACH = (F::SUMS + F::THREADS - 1) / F::THREADS, LD = F::LD;
    double *a = lds, *p = lds + F::SQ, *q = lds + 2 * F::SQ;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, h = lane >> 4;
    if constexpr (T == 1) {
        // One tile: a lane's results, rows 4 e + h of column r, are by symmetry its operands of the next product, columns 4 e + h of
        // row r, so that one wave takes all steps in registers (16 x 27: 8.1 us, through LDS over 10).
        if (wave == 0) {
            const auto times = [](const f64x4_t& x, const f64x4_t& y) {
                f64x4_t even = {}, odd = {};
                even = ns_mma64(x[0], y[0], even);
                odd = ns_mma64(x[1], y[1], odd);
                even = ns_mma64(x[2], y[2], even);
                odd = ns_mma64(x[3], y[3], odd);
                return even + odd;
            };
            f64x4_t am, pm, qm = {};
            double sum = 0.0;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                am[e] = get(e * 64 + lane);
                sum += r == 4 * e + h ? am[e] : 0.0;
            }
#pragma unroll
            for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o);
            const double inv = io.scaled ? 1.0 : 1.0 / (sqrt(sum) + io.eps);
            am = am * inv * inv;
            for (int step = 0; step < steps; ++step) {
                const f64x4_t s = times(am, am);
#pragma unroll
                for (int e = 0; e < 4; ++e) pm[e] = (r == 4 * e + h ? NS_A : 0.0) + NS_B * am[e] + NS_C * s[e];
                qm = step == 0 ? pm : times(qm, pm);
                // P (P A) and its transpose, of the same products in the same order: their mean is symmetric to the bit
                const f64x4_t t = times(pm, am);
                am = (times(pm, t) + times(t, pm)) * 0.5;
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) q[(4 * e + h) * LD + r] = qm[e] * inv;
        }
        __syncthreads();
        return q;
    }
    double v[EACH];
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
        const int u = i * F::THREADS + (int)threadIdx.x;
        v[i] = u < F::SUMS ? get(u) : 0.0;
    }
    __syncthreads();                                          // the sums' place is the squares'
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
        const int u = i * F::THREADS + (int)threadIdx.x;
        if (u < F::SUMS) {
            int ti, tj;
            gemm_triangle_at(u >> 8, ti, tj);
            const int row = ti * 16 + (u >> 6 & 3) * 4 + (u >> 4 & 3), col = tj * 16 + (u & 15);
            a[row * LD + col] = v[i];
            a[col * LD + row] = v[i];
        }
    }
    __syncthreads();
    double sum = lane < F::N ? a[lane * LD + lane] : 0.0;
#pragma unroll
    for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o);
    const double inv = io.scaled ? 1.0 : 1.0 / (sqrt(sum) + io.eps);
    __syncthreads();
    for (int i = threadIdx.x; i < F::SQ; i += F::THREADS) a[i] = i % LD < F::N ? a[i] * inv * inv : 0.0;
    __syncthreads();
    // tile k (on or over the diagonal) of left right, both symmetric
    const auto product = [&](const double* left, const double* right, int k) {
        int ti, tj;
        gemm_triangle_at(k, ti, tj);
        const double *x = left + (ti * 16 + r) * LD + h, *y = right + (tj * 16 + r) * LD + h;
        f64x4_t acc = {};
#pragma unroll
        for (int s = 0; s < F::N; s += 4) acc = ns_mma64(x[s], y[s], acc);
        return acc;
    };
    const auto put = [&](double* to, int k, f64x4_t val, double scale) {
        int ti, tj;
        gemm_triangle_at(k, ti, tj);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int row = ti * 16 + 4 * e + h, col = tj * 16 + r;
            if (row <= col) to[row * LD + col] = to[col * LD + row] = val[e] * scale;      // symmetric to the bit
        }
    };
    constexpr int TURNS = (2 * F::TRI + F::WAVES - 1) / F::WAVES;
    for (int step = 0; step < steps; ++step) {
        const bool last = step + 1 == steps;
        for (int k = wave; k < F::TRI; k += F::WAVES) {
            f64x4_t s = product(a, a, k);
            int ti, tj;
            gemm_triangle_at(k, ti, tj);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int row = ti * 16 + 4 * e + h, col = tj * 16 + r;
                s[e] = (row == col ? NS_A : 0.0) + NS_B * a[row * LD + col] + NS_C * s[e];
            }
            put(p, k, s, 1.0);
            if (step == 0) put(q, k, s, last ? inv : 1.0);
        }
        __syncthreads();
        // Q <- Q P and A <- P A P, by way of registers: the results take their operands' place
        f64x4_t next[TURNS];
#pragma unroll
        for (int i = 0; i < TURNS; ++i) {
            const int k = i * F::WAVES + wave;
            if (k < F::TRI ? step > 0 : k < 2 * F::TRI && !last) next[i] = k < F::TRI ? product(q, p, k) : product(p, a, k - F::TRI);
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < TURNS; ++i) {
            const int k = i * F::WAVES + wave;
            if (k < F::TRI ? step > 0 : k < 2 * F::TRI && !last) put(k < F::TRI ? q : a, k < F::TRI ? k : k - F::TRI, next[i], last ? inv : 1.0);
        }
        __syncthreads();
        if (last) break;
#pragma unroll
        for (int i = 0; i < TURNS; ++i) {
            const int k = i * F::WAVES + wave;
            if (k < F::TRI) next[i] = product(p, a, k);
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < TURNS; ++i) {
            const int k = i * F::WAVES + wave;
            if (k < F::TRI) put(a, k, next[i], 1.0);
        }
        __syncthreads();
    }
    return q;
}

// Columns [from, to) of Q G to the caller.  A lane holds rows 4 h + e of a tile and one column, of G and of the result: the product
// takes Q's rows in the order that puts them there.
template <int T, bool MUON, int DT>
__device__ __forceinline__ void ns_few_out(const NsIo& io, const NsPlace& p, int from, int to, const double* q) {
    using F = NsFew<T>;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, h = lane >> 4, qr = (r & 3) * 4 + (r >> 2);
    const long long sr = p.tall ? 1 : p.n, sc = p.tall ? p.m : 1;
    const float step = MUON ? io.lr02 * sqrtf((float)p.n) : 0.0f;
    for (int c0 = from + wave * 16 * F::AT_ONCE; c0 < to; c0 += F::WAVES * 16 * F::AT_ONCE) {
        float x[F::AT_ONCE][T][4], m[F::AT_ONCE][T][4];
        const auto place = [&](int g, int t, int& cnt) {
            const int row = 16 * t + 4 * h, c = c0 + 16 * g + r;
            cnt = c < to ? max(0, min(4, p.m - row)) : 0;
            return p.src + row * sr + c * sc;
        };
#pragma unroll
        for (int g = 0; g < F::AT_ONCE; ++g)
#pragma unroll
            for (int t = 0; t < T; ++t) {
                int cnt;
                const long long at = place(g, t, cnt);
                ns_load4<DT>(io.in, at, sr, cnt, x[g][t]);
                if constexpr (MUON) ns_load4<DT>(io.momentum, at, sr, cnt, m[g][t]);
            }
#pragma unroll
        for (int g = 0; g < F::AT_ONCE; ++g) {
            f64x4_t acc[T] = {};
            if constexpr (T > 2) asm volatile("" ::: "memory");   // Q comes from LDS anew: registers do not hold it beside the rest
#pragma unroll
            for (int k = 0; k < T; ++k)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const double b = MUON ? ns_direction(io, x[g][k][e], m[g][k][e]) : x[g][k][e];
#pragma unroll
                    for (int i = 0; i < T; ++i) acc[i] = ns_mma64(q[(16 * i + qr) * F::LD + 16 * k + 4 * h + e], b, acc[i]);
                }
#pragma unroll
            for (int t = 0; t < T; ++t) {
                int cnt;
                const long long at = place(g, t, cnt);
                float v[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = (float)acc[t][e];
                if constexpr (MUON) {
                    float w[4], old[4];
                    ns_load4<DT>(io.param, at, sr, cnt, w);
#pragma unroll
                    for (int e = 0; e < 4; ++e) w[e] = ns_new_param(io, w[e], step, v[e]);
                    ns_store4<DT>(io.param, at, sr, cnt, w);
                    if (io.ema) {
                        ns_load4<DT>(io.ema, at, sr, cnt, old);
#pragma unroll
                        for (int e = 0; e < 4; ++e) old[e] = io.ema_keep * old[e] + io.ema_take * w[e];
                        ns_store4<DT>(io.ema, at, sr, cnt, old);
                    }
                } else {
                    ns_store4<DT>(io.out, at, sr, cnt, v);
                }
            }
        }
    }
}

// The three parts in one workgroup, or (`cols` columns a workgroup) as three launches: partial sums of G G^T; Q; Q G
template <int T, int STAGE, bool MUON, int DT>
__global__ void __launch_bounds__(NsFew<T>::THREADS) ns_few_kernel(NsTable t, NsIo io, int steps, int cols) {
    using F = NsFew<T>;
    extern __shared__ __attribute__((aligned(16))) char space[];
    double* lds = (double*)space;
    const NsPlace p = ns_find(t, blockIdx.x, STAGE, cols, T);
    double* q_at = (double*)p.ws;                             // Q, then the partial sums
    double* parts = q_at + F::N * F::N;
    const int from = p.tile * cols, to = from + min(p.n - from, cols);
    if constexpr (STAGE == ST_WHOLE) {
        ns_few_gram<T, MUON, DT>(io, p, 0, p.n, lds);
        const double* q = ns_few_steps<T>(lds, steps, io, [&](int u) { return ns_few_sum<T>(lds, u); });
        ns_few_out<T, MUON, DT>(io, p, 0, p.n, q);
    } else if constexpr (STAGE == ST_GRAM) {
        ns_few_gram<T, MUON, DT>(io, p, from, to, lds);
        for (int u = threadIdx.x; u < F::SUMS; u += F::THREADS) parts[(long long)p.tile * F::SUMS + u] = ns_few_sum<T>(lds, u);
    } else if constexpr (STAGE == ST_STEPS) {
        const int n_parts = ns_tiles(ST_GRAM, cols, p.m, p.n);
        const double* q = ns_few_steps<T>(lds, steps, io, [&](int u) {
            double s = parts[u];
#pragma unroll 8
            for (int k = 1; k < n_parts; ++k) s += parts[(long long)k * F::SUMS + u];
            return s;
        });
        for (int i = threadIdx.x; i < F::N * F::N; i += F::THREADS) q_at[i] = q[i / F::N * F::LD + i % F::N];
    } else {
        for (int i = threadIdx.x; i < F::N * F::N; i += F::THREADS) lds[i / F::N * F::LD + i % F::N] = q_at[i];
        __syncthreads();
        ns_few_out<T, MUON, DT>(io, p, from, to, lds);
    }
}

// X before the first phase of many (what is left of a phase is float32, and the direction of the optimizer's step is made once), and
// BACK: the result of the last one for the caller.
template <bool MUON, int DT, bool BACK>
__global__ void __launch_bounds__(256) ns_few_move_kernel(NsTable t, NsIo io) {
    const NsPlace p = ns_find(t, blockIdx.x, ST_NORM, 0);
    long long at_x = p.src - t.g[p.group].src;
    for (int i = 0; i < p.group; ++i) at_x += (long long)t.g[i].m * t.g[i].n * t.g[i].count;
    const long long total = (long long)p.m * p.n, share = ns_share(p.m, p.n), from = p.tile * share;
    const long long to = from + share < total ? from + share : total;
    const float step = MUON ? io.lr02 * sqrtf((float)p.n) : 0.0f;
    for (long long i = from + threadIdx.x; i < to; i += 256) {
        const long long at = p.src + i;
        if constexpr (!BACK) {
            float v[4], m[4];
            ns_load4<DT>(io.in, at, 1, 1, v);
            if constexpr (MUON) {
                ns_load4<ODAMD_DTYPE_F32>(io.momentum, at, 1, 1, m);
                m[0] = io.mu * m[0] + v[0] * io.grad_scale;
                io.momentum[at] = m[0];
                v[0] = ns_direction(io, v[0], m[0]);
            }
            io.x[at_x + i] = v[0];
        } else if constexpr (MUON) {
            const float w = ns_new_param(io, io.param[at], step, io.x[at_x + i]);
            io.param[at] = w;
            if (io.ema) io.ema[at] = io.ema_keep * io.ema[at] + io.ema_take * w;
        } else {
            const float v[4] = {io.x[at_x + i]};
            ns_store4<DT>(io.out, at, 1, 1, v);
        }
    }
}

// Eight values of param and ema before the step, from element `at` on; the first `cnt` of them exist.
template <bool MUON> struct NsOld {};
template <> struct NsOld<true> { f32x4_t w[2], e[2]; };
template <bool MUON>
__device__ __forceinline__ NsOld<MUON> ns_old8(const NsIo& io, long long at, int cnt) {
    NsOld<MUON> x = {};
    if constexpr (MUON) {
        if (cnt == 8) {
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                x.w[q] = *(const f32x4_any*)(io.param + at + 4 * q);
                if (io.ema) x.e[q] = *(const f32x4_any*)(io.ema + at + 4 * q);
            }
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                x.w[e >> 2][e & 3] = e < cnt ? io.param[at + e] : 0.0f;
                x.e[e >> 2][e & 3] = e < cnt && io.ema ? io.ema[at + e] : 0.0f;
            }
        }
    }
    return x;
}
// Results for the caller
template <bool MUON, int DT>
__device__ __forceinline__ void ns_emit8(const NsIo& io, float step, long long at, int cnt, const float v[8], const NsOld<MUON>& x) {
    if (cnt <= 0) return;
    if constexpr (MUON) {
        f32x4_t w[2], u[2];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            w[e >> 2][e & 3] = ns_new_param(io, x.w[e >> 2][e & 3], step, v[e]);
            u[e >> 2][e & 3] = io.ema_keep * x.e[e >> 2][e & 3] + io.ema_take * w[e >> 2][e & 3];
        }
        if (cnt == 8) {
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                *(f32x4_any*)(io.param + at + 4 * q) = w[q];
                if (io.ema) *(f32x4_any*)(io.ema + at + 4 * q) = u[q];
            }
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (e < cnt) {
                    io.param[at + e] = w[e >> 2][e & 3];
                    if (io.ema) io.ema[at + e] = u[e >> 2][e & 3];
                }
        }
    } else if constexpr (DT == ODAMD_DTYPE_BF16) {
        uint16_t* o = (uint16_t*)io.out + at;
        if (cnt == 8)
            *(u32x4_any*)o = u32x4{f32x2_to_bf16x2(v[0], v[1]), f32x2_to_bf16x2(v[2], v[3]), f32x2_to_bf16x2(v[4], v[5]), f32x2_to_bf16x2(v[6], v[7])};
        else
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (e < cnt) o[e] = f32_to_bf16(v[e]);
    } else {
        float* o = (float*)io.out + at;
        if (cnt == 8) {
            *(f32x4_any*)o = f32x4_t{v[0], v[1], v[2], v[3]};
            *(f32x4_any*)(o + 4) = f32x4_t{v[4], v[5], v[6], v[7]};
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (e < cnt) o[e] = v[e];
        }
    }
}

// One product of the iteration for every matrix of the table
template <typename TILE, int STAGE, bool MUON, int DT>
__global__ void __launch_bounds__(TILE::THREADS) ns_product_kernel(NsTable t, NsIo io, NsJobs jobs) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int block = (int)blockIdx.x, job = STAGE == ST_AP ? block / t.tiles : STAGE == ST_Q && block >= t.tiles ? 1 : 0;
    const int at = block - job * t.tiles;
    const NsPlace p = ns_find(t, t.n == 1 ? gemm_xcd_remap(at, t.tiles) : gemm_xcd_stretch(at, t.tiles), STAGE, TILE::TM);
    const NsLayout l = ns_layout(p.m, p.n);
    const int mp = (int)ns_up(p.m, 32), np = (int)ns_up(p.n, 32);
    const auto square = [&](int i) { return p.ws + l.sq + i * l.sq_size; };
    int ti, tj;
    if (ns_symmetric(STAGE)) gemm_triangle_at(p.tile, ti, tj);
    else gemm_tile_at(p.tile, (p.m + TILE::TM - 1) / TILE::TM, (p.n + TILE::TN - 1) / TILE::TN, ti, tj);
    const int i0 = ti * TILE::TM, j0 = tj * TILE::TN;
    const int left = job ? jobs.left[1] : jobs.left[0], right = job ? jobs.right[1] : jobs.right[0], to = job ? jobs.out[1] : jobs.out[0];
    const float scale = job ? jobs.scale[1] : jobs.scale[0];
    TILE tile;
    if constexpr (STAGE == ST_A) {
        const GemmOperand x = {p.ws + l.x, (long long)np * 4, p.m};
        tile.run(x, x, i0, j0, 0, np / 32, np, lds);
    } else if constexpr (STAGE == ST_AP) {
        const GemmOperand x = {p.ws + l.x, (long long)np * 4, p.m};
        const int per = ns_cut(np / 32, jobs.n), from = job * per;
        if (from >= np / 32) return;                       // a short matrix has fewer parts
        tile.run(x, x, i0, j0, from, min(np / 32, from + per), np, lds);
        float* sums = (float*)square(SQ_T + job);
        const auto none = [](int, int) { return GemmNothing{}; };
        const auto rows = [&](int i, int j, float v[8], const GemmNothing&) {
            i += i0; j += j0;
            if (i >= p.m || j >= mp) return;
            f32x4_t* at = (f32x4_t*)(sums + (long long)i * mp + j);
            at[0] = f32x4_t{v[0], v[1], v[2], v[3]};
            at[1] = f32x4_t{v[4], v[5], v[6], v[7]};
        };
        tile.template hand_out<true, false, 1>(lds, none, rows, none, rows);
        return;
    } else {
        const GemmOperand a = {square(left), (long long)mp * 4, p.m};
        const GemmOperand b = STAGE == ST_P || STAGE == ST_Q ? GemmOperand{square(right), (long long)mp * 4, p.m}
                                                             : GemmOperand{p.ws + (jobs.turn ? l.xt1 : l.xt0), (long long)mp * 4, p.n};
        tile.run(a, b, i0, j0, 0, mp / 32, mp, lds);
    }

    if constexpr (STAGE == ST_AP) {
    } else if constexpr (STAGE == ST_A || STAGE == ST_P || STAGE == ST_Q) {
        char* out = square(to);
        // row i, columns j .. j+7; P needs A's values of that place
        struct Before { f16x8_t hi, lo; };
        const auto get = [&](int i, int j) {
            Before x = {};
            if (STAGE == ST_P && i < p.m && j < mp) {
                const char* at = square(SQ_A) + (long long)i * mp * 4 + split_at(j);
                x.hi = *(const f16x8_t*)at;
                x.lo = *(const f16x8_t*)(at + 64);
            }
            return x;
        };
        const auto put = [&](int i, int j, float v[8], const Before& x) {
            if (i >= p.m || j >= mp) return;
            if constexpr (STAGE == ST_P) {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    v[e] = (float)(NS_C / NS_SCALE) * v[e] + (float)NS_B * ((float)x.hi[e] + (float)x.lo[e]) + (i == j + e ? (float)(NS_A * NS_SCALE) : 0.0f);
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] *= scale;
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = j + e < p.m ? v[e] : 0.0f;
            store_split8(out + (long long)i * mp * 4 + split_at(j), v, 1.0f);
        };
        const auto get_row = [&](int i, int j) { return get(i0 + i, j0 + j); };
        const auto get_col = [&](int i, int j) { return get(j0 + j, i0 + i); };
        const auto rows = [&](int i, int j, float v[8], const Before& x) { put(i0 + i, j0 + j, v, x); };
        const auto cols = [&](int i, int j, float v[8], const Before& x) { put(j0 + j, i0 + i, v, x); };
        // a tile on the diagonal: the runs that reach it by rows, what lies under them by columns
        const auto upper = [&](int i, int j, float v[8], const Before& x) { if (i < j + 8) rows(i, j, v, x); };
        const auto lower = [&](int i, int j, float v[8], const Before& x) { if (i + 8 <= j) cols(i, j, v, x); };
        if (ti == tj) tile.template hand_out<true, true, 4, true>(lds, get_row, upper, get_col, lower);
        else tile.template hand_out<true, true, 4>(lds, get_row, rows, get_col, cols);
    } else if constexpr (STAGE == ST_X) {
        char* xt = p.ws + (jobs.turn ? l.xt0 : l.xt1);
        const auto none = [](int, int) { return GemmNothing{}; };
        tile.template hand_out<true, true, 1>(lds, none,
            [&](int i, int j, float v[8], const GemmNothing&) {
                i += i0; j += j0;
                if (i >= p.m || j >= np) return;
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = j + e < p.n ? v[e] * scale : 0.0f;
                store_split8(p.ws + l.x + (long long)i * np * 4 + split_at(j), v, 1.0f);
            },
            none,
            [&](int i, int j, float v[8], const GemmNothing&) {
                i += i0; j += j0;
                if (j >= p.n || i >= mp) return;
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = i + e < p.m ? v[e] * scale : 0.0f;
                store_split8(xt + (long long)j * mp * 4 + split_at(i), v, 1.0f);
            });
    } else {
        const float step = MUON ? io.lr02 * sqrtf((float)p.n) : 0.0f;
        // X[i][j .. j+7] of a wide matrix, X[i .. i+7][j] of a tall one: eight neighbours in the caller's buffer either way
        const auto at_row = [&](int i, int j) { return p.src + (long long)(i0 + i) * p.n + j0 + j; };
        const auto at_col = [&](int i, int j) { return p.src + (long long)(j0 + j) * p.m + i0 + i; };
        const auto count_row = [&](int i, int j) { return i0 + i < p.m ? min(8, p.n - j0 - j) : 0; };
        const auto count_col = [&](int i, int j) { return j0 + j < p.n ? min(8, p.m - i0 - i) : 0; };
        const auto emit = [&](long long at, int cnt, float v[8], const NsOld<MUON>& x) {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] *= scale;
            ns_emit8<MUON, DT>(io, step, at, cnt, v, x);
        };
        const auto old_row = [&](int i, int j) { return ns_old8<MUON>(io, at_row(i, j), count_row(i, j)); };
        const auto old_col = [&](int i, int j) { return ns_old8<MUON>(io, at_col(i, j), count_col(i, j)); };
        const auto rows = [&](int i, int j, float v[8], const NsOld<MUON>& x) { emit(at_row(i, j), count_row(i, j), v, x); };
        const auto cols = [&](int i, int j, float v[8], const NsOld<MUON>& x) { emit(at_col(i, j), count_col(i, j), v, x); };
        if (p.tall) tile.template hand_out<false, true, 2>(lds, old_row, rows, old_col, cols);
        else tile.template hand_out<true, false, 2>(lds, old_row, rows, old_col, cols);
    }
}

// A from the parts of a cut reduction, summed in their order: 64 x 64 elements per workgroup, mirrored like a product's tile
__global__ void __launch_bounds__(256) ns_join_kernel(NsTable t, int cuts, float scale) {
    __shared__ float tile[64][65];
    const NsPlace p = ns_find(t, blockIdx.x, ST_AP, 64);
    const NsLayout l = ns_layout(p.m, p.n);
    const int mp = (int)ns_up(p.m, 32), chunks = (int)ns_up(p.n, 32) / 32, per = ns_cut(chunks, cuts), parts = (chunks + per - 1) / per;
    int ti, tj;
    gemm_triangle_at(p.tile, ti, tj);
    const int i0 = ti * 64, j0 = tj * 64, c = (threadIdx.x & 7) * 8;
    char* out = p.ws + l.sq + SQ_A * l.sq_size;
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        const int r = (threadIdx.x >> 3) + 32 * q, i = i0 + r, j = j0 + c;
        if (i >= p.m || j >= mp) continue;
        f32x4_t u[NS_CUTS][2];
#pragma unroll
        for (int k = 0; k < NS_CUTS; ++k)
            if (k < parts) {
                const f32x4_t* at = (const f32x4_t*)((const float*)(p.ws + l.sq + (SQ_T + k) * l.sq_size) + (long long)i * mp + j);
                u[k][0] = at[0];
                u[k][1] = at[1];
            }
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            float s = u[0][e >> 2][e & 3];
#pragma unroll
            for (int k = 1; k < NS_CUTS; ++k)
                if (k < parts) s += u[k][e >> 2][e & 3];
            v[e] = j + e < p.m ? s * scale : 0.0f;
            tile[r][c + e] = v[e];
        }
        if (ti != tj) store_split8(out + (long long)i * mp * 4 + split_at(j), v, 1.0f);
    }
    __syncthreads();
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        const int r = (threadIdx.x >> 3) + 32 * q;          // all rows of a tile over the diagonal exist
        float v[8];
        if (j0 + r >= p.m || i0 + c >= mp) continue;
        // on the diagonal the whole tile, its lower half from the upper one
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = ti == tj && c + e >= r ? tile[r][c + e] : tile[c + e][r];
        store_split8(out + (long long)(j0 + r) * mp * 4 + split_at(i0 + c), v, 1.0f);
    }
}

using NsTile256 = GemmTile<2, true, 256, 256, 4, 2, 1, 2>;
using NsTile128 = GemmTile<2, true, 128, 128, 2, 2, 1, 2>;
using NsTile64 = GemmTile<2, true, 64, 64, 2, 2, 1, 2>;
// two wave groups, where a compute unit has one tile or two (78 matrices, 340 tiles: a step of 282 us instead of 295); with 528 tiles
// of one length their third round costs more than it gains (2048 x 8192: 1173 instead of 1023 us)
using NsTile64Few = GemmTile<2, true, 64, 64, 2, 2, 2, 3>;
using NsTile64Two = GemmTile<2, true, 64, 64, 2, 2, 2, 2>;

// Tiles of a stage over the whole table; -1: more than a launch of `threads` for each takes
int ns_count(NsTable& t, int stage, int tile, int threads) {
    long long at = 0;
    for (int i = 0; i < t.n; ++i) {
        t.g[i].tile0 = at > 0x7fffffff ? 0x7fffffff : (int)at;
        at += (long long)ns_tiles(stage, tile, t.g[i].m, t.g[i].n) * t.g[i].count;
    }
    t.tiles = (int)at;
    return gemm_grid_ok(at, threads) ? (int)at : -1;
}

template <typename TILE, int STAGE, bool MUON, int DT>
int ns_launch_tile(NsTable& t, const NsIo& io, const NsJobs& jobs, hipStream_t s) {
    if (ns_count(t, STAGE, TILE::TM, TILE::THREADS * jobs.n) < 0) return ODAMD_E_LIMIT;
    const auto kernel = ns_product_kernel<TILE, STAGE, MUON, DT>;
    const hipError_t e = odamd_ensure_lds((const void*)kernel, TILE::LDS);
    if (e != hipSuccess) return (int)e;
    kernel<<<t.tiles * jobs.n, TILE::THREADS, TILE::LDS, s>>>(t, io, jobs);
    return (int)hipGetLastError();
}

template <int STAGE, bool MUON, int DT>
int ns_launch64(NsTable& t, const NsIo& io, const NsJobs& jobs, hipStream_t s) {
    const int tiles = ns_count(t, STAGE, 64, NsTile64::THREADS * jobs.n);
    if (tiles < 0) return ODAMD_E_LIMIT;
    const long long all = (long long)tiles * jobs.n;
    return all > 512 ? ns_launch_tile<NsTile64, STAGE, MUON, DT>(t, io, jobs, s)
         : all > 256 ? ns_launch_tile<NsTile64Two, STAGE, MUON, DT>(t, io, jobs, s)
                     : ns_launch_tile<NsTile64Few, STAGE, MUON, DT>(t, io, jobs, s);
}

template <int STAGE, bool MUON, int DT>
int ns_product(NsTable& t, const NsIo& io, const NsJobs& jobs, hipStream_t s) {
    constexpr double epilogue = STAGE == ST_OUT ? (MUON ? 16.0 : DT == ODAMD_DTYPE_BF16 ? 2.0 : 4.0) : STAGE == ST_P ? 12.0 : 8.0;
    int best = 64, cuts = 1;
    double least = -1.0;
    for (int tile : {64, 128, 256})
        for (int cut = 1; cut <= (STAGE == ST_A && tile < 256 ? NS_CUTS : 1); ++cut) {
            GemmLoad load;
            double bytes = 0.0;
            for (int i = 0; i < t.n; ++i) {
                const NsGroup& g = t.g[i];
                const int chunks = (int)(ns_up(ns_along_n(STAGE) ? g.n : g.m, 32) / 32), per = ns_cut(chunks, cut);
                gemm_load_add(load, (double)ns_tiles(STAGE, tile, g.m, g.n) * g.count * jobs.n * ((chunks + per - 1) / per), (double)per);
                bytes += 4.0 * g.m * g.m * g.count;
            }
            // a cut reduction costs a second launch (5 us) and half a square per part, once out and once in
            const double us = gemm_time_us(tile, load, true, epilogue) + (cut > 1 ? 5.0 + cut * bytes / 3.0e6 : 0.0);
            if (least < 0.0 || us < least) {
                best = tile;
                cuts = cut;
                least = us;
            }
        }
    if constexpr (STAGE == ST_A)
        if (cuts > 1) {
            NsJobs parts = jobs;
            parts.n = cuts;
            const int rc = best == 128 ? ns_launch_tile<NsTile128, ST_AP, MUON, DT>(t, io, parts, s) : ns_launch64<ST_AP, MUON, DT>(t, io, parts, s);
            if (rc != 0) return rc;
            if (ns_count(t, ST_AP, 64, 256) < 0) return ODAMD_E_LIMIT;
            ns_join_kernel<<<t.tiles, 256, 0, s>>>(t, cuts, jobs.scale[0]);
            return (int)hipGetLastError();
        }
    if (best == 256) return ns_launch_tile<NsTile256, STAGE, MUON, DT>(t, io, jobs, s);
    if (best == 128) return ns_launch_tile<NsTile128, STAGE, MUON, DT>(t, io, jobs, s);
    return ns_launch64<STAGE, MUON, DT>(t, io, jobs, s);
}

// Exponent that keeps a product of k P's (entries up to 3.4445^k) within fp16, an eighth of a bit to spare for rounding
int ns_q_exponent(int k) {
    const int e = (int)floor(log2(65504.0 / (1.1 * pow(NS_A, k))));
    return e < 12 ? e : 12;
}

int ns_few_rows(const NsTable& t) {   // rows of the tallest matrix, in 16-row tiles
    int rows = 0;
    for (int i = 0; i < t.n; ++i) rows = t.g[i].m > rows ? t.g[i].m : rows;
    return (rows + 15) / 16;
}
int ns_longest(const NsTable& t) {
    int n = 0;
    for (int i = 0; i < t.n; ++i) n = t.g[i].n > n ? t.g[i].n : n;
    return n;
}

// All matrices have at most 16 T rows, the longest `n` columns
template <int T, int STAGE, bool MUON, int DT>
int ns_few_launch(NsTable& t, const NsIo& io, int steps, int cols, hipStream_t s) {
    using F = NsFew<T>;
    if (ns_count(t, STAGE, cols, F::THREADS) < 0) return ODAMD_E_LIMIT;
    const auto kernel = ns_few_kernel<T, STAGE, MUON, DT>;
    const hipError_t e = odamd_ensure_lds((const void*)kernel, F::LDS);
    if (e != hipSuccess) return (int)e;
    kernel<<<t.tiles, F::THREADS, F::LDS, s>>>(t, io, steps, cols);
    return (int)hipGetLastError();
}
template <int T, bool MUON, int DT>
int ns_few(NsTable& t, const NsIo& io, int steps, int n, hipStream_t s) {
    const int cols = ns_few_cols(T, n);
    if (cols >= n) return ns_few_launch<T, ST_WHOLE, MUON, DT>(t, io, steps, cols, s);
    int rc = ns_few_launch<T, ST_GRAM, MUON, DT>(t, io, steps, cols, s);
    if (rc == 0) rc = ns_few_launch<T, ST_STEPS, false, ODAMD_DTYPE_F32>(t, io, steps, cols, s);
    return rc == 0 ? ns_few_launch<T, ST_QG, MUON, DT>(t, io, steps, cols, s) : rc;
}

template <bool MUON, int DT>
int ns_few_phase(NsTable& t, const NsIo& io, int steps, hipStream_t s) {
    const int rows = ns_few_rows(t), cols = ns_longest(t);
    return rows == 1 ? ns_few<1, MUON, DT>(t, io, steps, cols, s) : rows == 2 ? ns_few<2, MUON, DT>(t, io, steps, cols, s)
         : rows == 3 ? ns_few<3, MUON, DT>(t, io, steps, cols, s) : ns_few<4, MUON, DT>(t, io, steps, cols, s);
}
template <bool MUON, int DT, bool BACK>
int ns_few_move(NsTable& t, const NsIo& io, hipStream_t s) {
    if (ns_count(t, ST_NORM, 0, 256) < 0) return ODAMD_E_LIMIT;
    ns_few_move_kernel<MUON, DT, BACK><<<t.tiles, 256, 0, s>>>(t, io);
    return (int)hipGetLastError();
}
// More steps than a phase takes.  X lies in the caller's result where that is float32, else in the workspace.
template <bool MUON, int DT>
int ns_few_phases(NsTable& t, const NsIo& io, int steps, hipStream_t s) {
    constexpr bool OWN = MUON || DT != ODAMD_DTYPE_F32;
    NsTable x = t;
    NsIo mid = {};
    mid.eps = io.eps;
    mid.in = io.in;
    mid.out = io.out;
    int rc = 0;
    if constexpr (OWN) {
        long long at = 0;
        for (int i = 0; i < x.n; ++i) {
            x.g[i].src = at;
            at += (long long)x.g[i].m * x.g[i].n * x.g[i].count;
        }
        mid.in = mid.out = io.x;
        rc = ns_few_move<MUON, DT, false>(t, io, s);
    }
    for (int done = 0; done < steps && rc == 0; done += NS_FEW_STEPS) {
        rc = ns_few_phase<false, ODAMD_DTYPE_F32>(x, mid, steps - done < NS_FEW_STEPS ? steps - done : NS_FEW_STEPS, s);
        mid.in = mid.out;
        mid.scaled = 1;
    }
    if constexpr (OWN)
        if (rc == 0) rc = ns_few_move<MUON, DT, true>(t, io, s);
    return rc;
}

template <bool MUON, int DT>
int ns_run(NsTable& t, const NsIo& io, int steps, hipStream_t s) {
    if (ns_few_rows(t) <= 4) return steps <= NS_FEW_STEPS ? ns_few_phase<MUON, DT>(t, io, steps, s) : ns_few_phases<MUON, DT>(t, io, steps, s);
    constexpr bool LOOSE = MUON || DT == ODAMD_DTYPE_BF16;
    int phase = LOOSE ? 5 : 2;
    for (int i = 0; i < t.n; ++i)
        if (!LOOSE && t.g[i].n < 2 * (long long)t.g[i].m) phase = 1;
    if (ns_count(t, ST_NORM, 0, 256) < 0) return ODAMD_E_LIMIT;
    ns_norm_kernel<MUON, DT><<<t.tiles, 256, 0, s>>>(t, io);
    if (ns_count(t, ST_SPLIT, 64, 256) < 0) return ODAMD_E_LIMIT;
    ns_split_kernel<MUON, DT><<<t.tiles, 256, 0, s>>>(t, io);
    int rc = (int)hipGetLastError();
    NsJobs jobs = {};
    const auto clear = [&] { jobs.n = 0; };
    const auto add = [&](int left, int right, int out, int shift) {
        jobs.left[jobs.n] = left;
        jobs.right[jobs.n] = right;
        jobs.out[jobs.n] = out;
        jobs.scale[jobs.n++] = (float)ldexp(1.0, shift);
    };
    for (int done = 0; done < steps && rc == 0;) {
        const int len = steps - done < phase ? steps - done : phase;
        clear();
        add(0, 0, SQ_A, -12);
        rc = ns_product<ST_A, false, ODAMD_DTYPE_F32>(t, io, jobs, s);
        int q = -1, eq = 0;
        for (int k = 1; k <= len && rc == 0; ++k) {
            const int p = q == SQ_B ? SQ_B + 1 : SQ_B, spare = 3 * SQ_B + 3 - p - (q < 0 ? SQ_B + 1 : q);
            clear();
            add(SQ_A, SQ_A, p, 0);
            rc = ns_product<ST_P, false, ODAMD_DTYPE_F32>(t, io, jobs, s);
            clear();
            if (k < len) add(p, SQ_A, SQ_T, -12);
            if (k > 1) {
                const int e = ns_q_exponent(k);
                add(q, p, spare, e - eq - 12);
                q = spare;
                eq = e;
            } else {
                q = p;
                eq = 12;
            }
            if (jobs.n && rc == 0) rc = ns_product<ST_Q, false, ODAMD_DTYPE_F32>(t, io, jobs, s);
            if (k < len && rc == 0) {
                clear();
                add(SQ_T, p, SQ_A, -12);
                rc = ns_product<ST_Q, false, ODAMD_DTYPE_F32>(t, io, jobs, s);
            }
        }
        done += len;
        clear();
        add(q, 0, 0, done < steps ? -eq : -eq - 12);
        if (rc == 0) rc = done < steps ? ns_product<ST_X, false, ODAMD_DTYPE_F32>(t, io, jobs, s) : ns_product<ST_OUT, MUON, DT>(t, io, jobs, s);
        jobs.turn ^= 1;
    }
    return rc;
}

// 2^31 less what a position passes the last column by
bool ns_shape_ok(long long rows, long long cols) { return rows >= 1 && cols >= 1 && rows * cols <= 0x7fff0000LL; }

void ns_orient(NsGroup& g, int rows, int cols) {
    g.tall = rows > cols;
    g.m = g.tall ? cols : rows;
    g.n = g.tall ? rows : cols;
}

// The table of matrices from number `from` on
void ns_fill(NsTable& t, const odamd_matrix* matrices, int from, int count) {
    t.n = 0;
    for (int k = from; k < count && k < from + NS_GROUPS; ++k) {
        NsGroup g = {};
        ns_orient(g, matrices[k].rows, matrices[k].cols);
        g.src = matrices[k].offset;
        g.count = 1;
        // the longest tiles first: short ones fill the end of a launch
        int to = t.n++;
        for (; to > 0 && (t.g[to - 1].m < g.m || (t.g[to - 1].m == g.m && t.g[to - 1].n < g.n)); --to) t.g[to] = t.g[to - 1];
        t.g[to] = g;
    }
}
// Places the workspaces of the table's matrices one behind the other; the bytes of all of them.  A table of few rows: X of all its
// matrices (`x` bytes) lies before them, and only matrices that are taken in parts need more.
size_t ns_place(NsTable& t, size_t& x) {
    const int rows = ns_few_rows(t), n = ns_longest(t), cols = rows <= 4 ? ns_few_cols(rows, n) : 0;
    size_t at = 0;
    long long all = 0;
    for (int i = 0; i < t.n; ++i) {
        const NsGroup& g = t.g[i];
        t.g[i].ws = (unsigned)(at / 256);
        all += (long long)g.m * g.n * g.count;
        at += (size_t)g.count * (rows > 4 ? ns_layout(g.m, g.n).end : cols < n ? ns_few_bytes(rows, cols, g.n) : 0);
    }
    x = rows <= 4 ? (size_t)ns_up(all * 4, 256) : 0;
    return x + at;
}
// One group
void ns_single(NsTable& t, int batch, int rows, int cols) {
    t.n = 1;
    ns_orient(t.g[0], rows, cols);
    t.g[0].src = 0;
    t.g[0].count = batch;
}

}  // namespace

extern "C" {

size_t odamd_orthogonalize_workspace_bytes(int batch, int rows, int cols) {
    if (batch < 1 || !ns_shape_ok(rows, cols)) return 0;
    NsTable t;
    size_t x;
    ns_single(t, batch, rows, cols);
    return ns_place(t, x);
}

int odamd_orthogonalize(const void* x, void* out, int batch, int rows, int cols, int steps, double eps, int dtype, void* workspace,
                        size_t workspace_bytes, void* stream) {
    if (!x || !out || !workspace || batch < 1 || !ns_shape_ok(rows, cols) || steps < 1 || steps > 32 || !(eps >= 0.0)) return ODAMD_E_ARG;
    if (dtype != ODAMD_DTYPE_F32 && dtype != ODAMD_DTYPE_BF16) return ODAMD_E_ARG;
    if (((uintptr_t)x | (uintptr_t)out) & (dtype == ODAMD_DTYPE_F32 ? 3 : 1)) return ODAMD_E_ALIGN;
    if ((uintptr_t)workspace & 255) return ODAMD_E_ALIGN;
    if (workspace_bytes < odamd_orthogonalize_workspace_bytes(batch, rows, cols)) return ODAMD_E_WORKSPACE;
    NsTable t;
    size_t held;
    ns_single(t, batch, rows, cols);
    ns_place(t, held);
    t.ws = (char*)workspace + held;
    NsIo io = {};
    io.in = x;
    io.out = out;
    io.x = (float*)workspace;
    io.eps = eps;
    return dtype == ODAMD_DTYPE_F32 ? ns_run<false, ODAMD_DTYPE_F32>(t, io, steps, (hipStream_t)stream)
                                    : ns_run<false, ODAMD_DTYPE_BF16>(t, io, steps, (hipStream_t)stream);
}

size_t odamd_muon_workspace_bytes(const odamd_matrix* matrices_host, int n_matrices) {
    if (!matrices_host || n_matrices < 1) return 0;
    for (int k = 0; k < n_matrices; ++k)
        if (!ns_shape_ok(matrices_host[k].rows, matrices_host[k].cols)) return 0;
    size_t most = 0;
    for (int i = 0; i < n_matrices; i += NS_GROUPS) {
        NsTable t;
        size_t x;
        ns_fill(t, matrices_host, i, n_matrices);
        const size_t need = ns_place(t, x);
        most = need > most ? need : most;
    }
    return most;
}

int odamd_muon_ema_step(float* param, const float* grad, float* momentum, float* ema, const odamd_matrix* matrices_host,
                        int n_matrices, double lr, double momentum_decay, int nesterov, double weight_decay, int steps, double eps,
                        double ema_decay, double grad_scale, void* workspace, size_t workspace_bytes, void* stream) {
    if (!param || !grad || !momentum || !matrices_host || !workspace || n_matrices < 1 || steps < 1 || steps > 32 || !(eps >= 0.0)) return ODAMD_E_ARG;
    for (int k = 0; k < n_matrices; ++k)
        if (matrices_host[k].offset < 0 || !ns_shape_ok(matrices_host[k].rows, matrices_host[k].cols)) return ODAMD_E_ARG;
    if (((uintptr_t)param | (uintptr_t)grad | (uintptr_t)momentum | (uintptr_t)ema) & 3) return ODAMD_E_ALIGN;
    if ((uintptr_t)workspace & 255) return ODAMD_E_ALIGN;
    const size_t need = odamd_muon_workspace_bytes(matrices_host, n_matrices);
    if (workspace_bytes < need) return ODAMD_E_WORKSPACE;
    if (need / 256 > 0xffffffffULL) return ODAMD_E_LIMIT;
    NsIo io = {};
    io.in = grad;
    io.param = param;
    io.momentum = momentum;
    io.ema = ema;
    io.mu = (float)momentum_decay;
    io.grad_scale = (float)grad_scale;
    io.shrink = (float)(lr * weight_decay);
    io.lr02 = (float)(0.2 * lr);
    io.ema_keep = (float)ema_decay;
    io.ema_take = (float)(1.0 - ema_decay);
    io.nesterov = nesterov != 0;
    io.eps = eps;
    for (int i = 0; i < n_matrices; i += NS_GROUPS) {
        NsTable t;
        size_t held;
        ns_fill(t, matrices_host, i, n_matrices);
        ns_place(t, held);
        t.ws = (char*)workspace + held;
        io.x = (float*)workspace;
        const int rc = ns_run<true, ODAMD_DTYPE_F32>(t, io, steps, (hipStream_t)stream);
        if (rc != 0) return rc;
    }
    return ODAMD_OK;
}

}  // extern "C"
