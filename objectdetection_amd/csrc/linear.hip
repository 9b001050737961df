// Dense layer: y = act(x W^T + b) + r, and its backward pass.
//
//   dz = dy act'(z),  z = x W^T + b;   dx = dz W,   dW = dz^T x,   db = column sums of dz   (dr = dy, the caller's own)
// bfloat16 operands run on bf16 matrix instructions as they are; float32 operands as fp16 pairs (gemm.h) with a power of
// two per row of each operand, so that a row's largest value sits just under 2^15: 22 bits per value down to 2^-17 of the row's
// largest, and the same absolute step below.  Sums are float32; dz is kept in the operands' type, z in float32 or, beside
// bfloat16, in float16.
// dx reduces over the outputs and dW over the rows: in bfloat16 the products read W, x and dz with the reduction along their
// rows, out of the caller's tensors; float32 pairs need a power of two per column there, so that W, x and dz are laid out
// by columns first (one launch for all three).  Few rows, and the backward pass of small layers, go without matrix instructions.
// Times: (25600, 1024, 4096) bf16 with bias, SiLU and residual 285 us, 243 of them the product (a library product of that size
// takes 206 us), the rest the epilogue's 420 MB; forward and backward of (8192, 1024, 4096) bf16 304 us; (4097, 1155, 1001)
// float32 with GELU 66 us; (1, 1024, 1024) bf16 3 us, a call of it 12 on the host.
#include "common.h"
#include "odamd.h"
#include "offsets.h"

#include <math.h>

namespace {

#include "gemm.h"

template <int DT> struct LinType;
template <> struct LinType<ODAMD_DTYPE_F32> {
    using T = float;
    static constexpr int PL = 2;
    static __device__ __forceinline__ float get(T v) { return v; }
    static __device__ __forceinline__ T put(float v) { return v; }
};
template <> struct LinType<ODAMD_DTYPE_BF16> {
    using T = uint16_t;
    static constexpr int PL = 1;
    static __device__ __forceinline__ float get(T v) { return bf16_to_f32(v); }
    static __device__ __forceinline__ T put(float v) { return f32_to_bf16(v); }
};

__host__ __device__ inline long long lin_up(long long v, int to) { return (v + to - 1) / to * to; }

// Normal distribution function F(z) = erfc(-z / sqrt 2) / 2, whose values at negative z keep their digits: 1 + erf loses all of them
// by z = -5, where F is 3e-7.  Fast form, for results that are rounded to bfloat16: erfc(u) = e^(-u u) t (c1 + c2 t + .. + c6 t^5),
// t = 1 / (1 + 0.42 u), coefficients fitted here to e^(u u) erfc(u) for the smallest error of z F(z): 1.1e-7, and 2.8e-5 of F itself up to
// u = 9.
template <bool FAST>
__device__ __forceinline__ float lin_normal(float z) {
    if constexpr (!FAST) return 0.5f * erfcf(z * -0.70710678118654752f);
    const float t = __builtin_amdgcn_rcpf(fmaf(0.42f * 0.70710678118654752f, fabsf(z), 1.0f));
    const float poly = t * fmaf(t, fmaf(t, fmaf(t, fmaf(t, fmaf(t, -0.166439486f, 0.486273358f), -0.0913507648f), 0.314409716f), 0.218850815f), 0.238255336f);
    const float tail = 0.5f * poly * __builtin_amdgcn_exp2f(z * z * -0.72134752044448170f);
    return z < 0.0f ? tail : 1.0f - tail;
}
// FAST: hardware exponential and reciprocal (an error of 2^-22 or so), where the result is rounded to bfloat16.  The float32 forms
// go through expf / erfcf: their results are held to float32.  With the exact forms a value cost some 40 vector instructions
// and the 25600 x 4096 layer with SiLU 220 us on top of its 250 us product.
template <bool FAST, int ACT>
__device__ __forceinline__ float lin_act(float z) {
    if constexpr (ACT == ODAMD_ACT_SILU) return FAST ? z * sigmoid_fast(z) : z / (1.0f + expf(-z));
    if constexpr (ACT == ODAMD_ACT_GELU) return z * lin_normal<FAST>(z);
    if constexpr (ACT == ODAMD_ACT_RELU) return z < 0.0f ? 0.0f : z;
    return z;
}
// dy act'(z)
template <bool FAST, int ACT>
__device__ __forceinline__ float lin_grad(float dy, float z) {
    if constexpr (ACT == ODAMD_ACT_SILU) {
        const float p = FAST ? sigmoid_fast(z) : 1.0f / (1.0f + expf(-z));
        return dy * (p * (1.0f + z * (1.0f - p)));
    }
    if constexpr (ACT == ODAMD_ACT_GELU) {
        const float g = FAST ? __builtin_amdgcn_exp2f(z * z * -0.72134752044448170f) : expf(-0.5f * z * z);
        return dy * (lin_normal<FAST>(z) + z * g * 0.39894228040143268f);
    }
    if constexpr (ACT == ODAMD_ACT_RELU) return z <= 0.0f ? 0.0f : dy;   // also where dy is an infinity
    return dy;
}
// Calls f with the activation as a compile-time constant
template <typename F>
__host__ __device__ __forceinline__ void lin_with_act(int act, F&& f) {
    switch (act) {
        case ODAMD_ACT_SILU: f(std::integral_constant<int, ODAMD_ACT_SILU>{}); break;
        case ODAMD_ACT_GELU: f(std::integral_constant<int, ODAMD_ACT_GELU>{}); break;
        case ODAMD_ACT_RELU: f(std::integral_constant<int, ODAMD_ACT_RELU>{}); break;
        default: f(std::integral_constant<int, ODAMD_ACT_NONE>{}); break;
    }
}

// Power of two that brings a row whose largest finite magnitude has these bits just under 2^15
__device__ __forceinline__ int lin_shift(unsigned max_bits) {
    return max_bits ? 15 - __builtin_amdgcn_frexp_expf(__uint_as_float(max_bits)) : 0;
}
__device__ __forceinline__ unsigned lin_magnitude(float v) {
    const unsigned b = __float_as_uint(v) & 0x7fffffffu;
    return b < 0x7f800000u ? b : 0u;
}

// ---- what is done with a value of x W^T -----------------------------------------------------------------------------
struct LinEnd {
    const void* bias;
    const void* residual;
    void* y;
    void* z;
    long long r_ld, y_ld, z_ld;
    int act;
};

template <int DT>
__device__ __forceinline__ void lin_load8(const void* base, long long at, int cnt, float v[8]) {
    using T = typename LinType<DT>::T;
    const T* s = (const T*)base + at;
    if (cnt == 8) {
        if constexpr (DT == ODAMD_DTYPE_F32) {
            const f32x4_t a = *(const f32x4_any*)s, b = *(const f32x4_any*)(s + 4);
#pragma unroll
            for (int e = 0; e < 4; ++e) { v[e] = a[e]; v[e + 4] = b[e]; }
        } else {
            const u32x4 a = *(const u32x4_any*)s;
#pragma unroll
            for (int e = 0; e < 4; ++e) { v[2 * e] = __uint_as_float(a[e] << 16); v[2 * e + 1] = __uint_as_float(a[e] & 0xffff0000u); }
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = e < cnt ? LinType<DT>::get(s[e]) : 0.0f;
    }
}
template <int DT>
__device__ __forceinline__ void lin_store8(void* base, long long at, int cnt, const float v[8]) {
    using T = typename LinType<DT>::T;
    T* d = (T*)base + at;
    if (cnt == 8) {
        if constexpr (DT == ODAMD_DTYPE_F32) {
            *(f32x4_any*)d = f32x4_t{v[0], v[1], v[2], v[3]};
            *(f32x4_any*)(d + 4) = f32x4_t{v[4], v[5], v[6], v[7]};
        } else {
            *(u32x4_any*)d = u32x4{f32x2_to_bf16x2(v[0], v[1]), f32x2_to_bf16x2(v[2], v[3]), f32x2_to_bf16x2(v[4], v[5]), f32x2_to_bf16x2(v[6], v[7])};
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (e < cnt) d[e] = LinType<DT>::put(v[e]);
    }
}
// Eight values of the caller's type, as loaded
template <int DT> struct LinRaw { f32x4_t a, b; };
template <> struct LinRaw<ODAMD_DTYPE_BF16> { u32x4 a; };
template <int DT>
__device__ __forceinline__ LinRaw<DT> lin_raw8(const void* base, long long at, int cnt) {
    LinRaw<DT> r = {};
    const typename LinType<DT>::T* s = (const typename LinType<DT>::T*)base + at;
    if (cnt == 8) {
        if constexpr (DT == ODAMD_DTYPE_F32) {
            r.a = *(const f32x4_any*)s;
            r.b = *(const f32x4_any*)(s + 4);
        } else {
            r.a = *(const u32x4_any*)s;
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (e < cnt) {
                if constexpr (DT == ODAMD_DTYPE_F32) {
                    if (e < 4) r.a[e & 3] = s[e];
                    else r.b[e & 3] = s[e];
                } else r.a[e >> 1] |= (uint32_t)s[e] << (16 * (e & 1));
            }
    }
    return r;
}
__device__ __forceinline__ void lin_values(const LinRaw<ODAMD_DTYPE_F32>& r, float v[8]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) { v[e] = r.a[e]; v[e + 4] = r.b[e]; }
}
__device__ __forceinline__ void lin_values(const LinRaw<ODAMD_DTYPE_BF16>& r, float v[8]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) { v[2 * e] = __uint_as_float(r.a[e] << 16); v[2 * e + 1] = __uint_as_float(r.a[e] & 0xffff0000u); }
}
// The pre-activation for the backward pass.  Beside bfloat16 it is kept in float16: three bits more for the slope, at the same
// size (with bfloat16 dW of 4197 rows is 1.45 times as far off as the rounding of its result alone, with float16 1.39: what dz's
// rounding leaves); beyond float16's range every activation is straight, so the end of the range stands for an infinity, and a
// positive value under it stays positive where relu asks for the sign.
template <int DT, int ACT>
__device__ __forceinline__ void lin_store_z8(void* base, long long at, int cnt, const float v[8]) {
    if constexpr (DT == ODAMD_DTYPE_F32) {
        lin_store8<DT>(base, at, cnt, v);
    } else {
        _Float16* d = (_Float16*)base + at;
        f16x8_t u;
#pragma unroll
        for (int e = 0; e < 8; ++e) u[e] = (_Float16)(ACT == ODAMD_ACT_RELU && v[e] > 0.0f ? fmaxf(v[e], 0x1p-24f) : v[e]);
        if (cnt == 8) {
            *(u32x4_any*)d = __builtin_bit_cast(u32x4, u);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (e < cnt) d[e] = u[e];
        }
    }
}
template <int DT>
__device__ __forceinline__ void lin_load_z8(const void* base, long long at, int cnt, float v[8]) {
    if constexpr (DT == ODAMD_DTYPE_F32) {
        lin_load8<DT>(base, at, cnt, v);
    } else {
        const _Float16* s = (const _Float16*)base + at;
        f16x8_t u = {};
        if (cnt == 8) {
            u = __builtin_bit_cast(f16x8_t, *(const u32x4_any*)s);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (e < cnt) u[e] = s[e];
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float z = (float)u[e];
            v[e] = fabsf(z) > 65504.0f ? copysignf(65504.0f, z) : z;
        }
    }
}
// Row i, columns j .. j + cnt - 1 (cnt <= 8): bias[8] and the residual's values are there already
template <int DT, int ACT>
__device__ __forceinline__ void lin_finish8(const LinEnd& p, long long i, int j, int cnt, float v[8], const float bias[8], const LinRaw<DT>& residual) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] += bias[e];
    if (p.z) lin_store_z8<DT, ACT>(p.z, i * p.z_ld + j, cnt, v);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = lin_act<DT == ODAMD_DTYPE_BF16, ACT>(v[e]);
    if (p.residual) {
        float r[8];
        lin_values(residual, r);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] += r[e];
    }
    lin_store8<DT>(p.y, i * p.y_ld + j, cnt, v);
}
template <int DT>
__device__ __forceinline__ void lin_bias8(const LinEnd& p, int j, int cnt, float b[8]) {
    if (p.bias && cnt > 0) {
        lin_load8<DT>(p.bias, j, cnt, b);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) b[e] = 0.0f;
    }
}
template <int DT, int ACT>
__device__ __forceinline__ void lin_finish8(const LinEnd& p, long long i, int j, int cnt, float v[8]) {
    float bias[8];
    lin_bias8<DT>(p, j, cnt, bias);
    lin_finish8<DT, ACT>(p, i, j, cnt, v, bias, p.residual ? lin_raw8<DT>(p.residual, i * p.r_ld + j, cnt) : LinRaw<DT>{});
}

// ---- a few rows: W read once from memory, no matrix instructions -----------------------------------------------------
struct LinRow {
    const void* x;
    const void* w;
    long long x_ld, w_ld;
    int m, k, n;
    LinEnd end;
};
// A workgroup takes four output columns of up to eight rows; its four waves hold all of them and share the reduction, so that x is
// loaded once for four columns and as many waves read W as with a wave per column (8 x 4096 x 4096 bf16: 10.1 us, one column
// a wave 15.7; 1 x 30000 x 64 float32 14.0 and 39.3).  Vectors are loaded from any element on: 1 x 1155 x 1001 float32 takes 3.7 us, by
// single elements 7.9.  What bounds it: reading W (1 x 4096 x 4096 bf16 7.3 us, 4.6 TB/s; 8 x 8192 x 8192 26 us, 5.2 TB/s), with many
// rows the x and W that come out of the caches again.
template <int DT, int MR>
__global__ void __launch_bounds__(256) linear_rows_kernel(LinRow p) {
    using T = typename LinType<DT>::T;
    constexpr int V = 16 / (int)sizeof(T), COLS = 4, N = MR * COLS;
    __shared__ float part[4][N];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col0 = blockIdx.x * COLS, row0 = blockIdx.y * MR;
    // rows and columns past the last one are computed like the last one and not stored: all loads of a step go out together
    const T *x[MR], *w[COLS];
#pragma unroll
    for (int i = 0; i < MR; ++i) x[i] = (const T*)p.x + min(row0 + i, p.m - 1) * p.x_ld;
#pragma unroll
    for (int c = 0; c < COLS; ++c) w[c] = (const T*)p.w + min(col0 + c, p.n - 1) * p.w_ld;
    float acc[N];
#pragma unroll
    for (int i = 0; i < N; ++i) acc[i] = 0.0f;
    const auto add = [&](auto width, int k) {
        constexpr int W = width.value;
        T wv[COLS][W], xv[MR][W];
#pragma unroll
        for (int c = 0; c < COLS; ++c) {
            if constexpr (W > 1) *(u32x4*)wv[c] = *(const u32x4_any*)(w[c] + k);
            else wv[c][0] = w[c][k];
        }
#pragma unroll
        for (int i = 0; i < MR; ++i) {
            if constexpr (W > 1) *(u32x4*)xv[i] = *(const u32x4_any*)(x[i] + k);
            else xv[i][0] = x[i][k];
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < MR; ++i)
#pragma unroll
            for (int c = 0; c < COLS; ++c)
#pragma unroll
                for (int e = 0; e < W; ++e) acc[c * MR + i] = fmaf(LinType<DT>::get(xv[i][e]), LinType<DT>::get(wv[c][e]), acc[c * MR + i]);
    };
    for (int k = (wave * 64 + lane) * V; k + V <= p.k; k += 256 * V) add(std::integral_constant<int, V>{}, k);
    if (wave == 0 && lane < p.k % V) add(std::integral_constant<int, 1>{}, p.k - p.k % V + lane);
    // sums over the lanes: while there are several values, a lane hands half of them on and keeps the other half
    int at = 0, o = 32;
#pragma unroll
    for (int half = N / 2; half >= 1; half /= 2, o >>= 1) {
        const bool upper = lane & o;
#pragma unroll
        for (int i = 0; i < half; ++i) {
            const float first = acc[i], second = acc[i + half];
            acc[i] = (upper ? second : first) + __shfl_xor(upper ? first : second, o);
        }
        at = at * 2 + upper;
    }
    for (; o; o >>= 1) acc[0] += __shfl_xor(acc[0], o);
    part[wave][at] = acc[0];                                // lanes of one value hold the same sum
    __syncthreads();
    const int c = threadIdx.x / MR, i = threadIdx.x % MR, col = col0 + c;
    if (c < COLS && row0 + i < p.m && col < p.n) {
        float v[8] = {};
#pragma unroll
        for (int s = 0; s < 4; ++s) v[0] += part[s][c * MR + i];
        lin_with_act(p.end.act, [&](auto act) { lin_finish8<DT, act.value>(p.end, row0 + i, col, 1, v); });
    }
}

// ---- laying operands out ---------------------------------------------------------------------------------------------
// One matrix (m x n) of the caller's, optionally dz = src act'(z): written by rows and / or (float32) by columns with the
// reduction padded with zeros to whole chunks.
struct LinJob {
    const void* src;
    const void* z;
    long long ld, z_ld;
    char* rows;            // [m][n padded]
    char* cols;            // [n][m padded]
    unsigned* row_max;     // float32: bits of each row's / column's largest magnitude
    unsigned* col_max;
    float* sums;           // [ceil(m / 64)][n] column sums
    int m, n, act, tile0;
};
struct LinJobs { LinJob j[3]; int n; };

__device__ __forceinline__ const LinJob& lin_job(const LinJobs& t, int block) {
    int i = 0;
    if (t.n > 1 && block >= t.j[1].tile0) i = 1;
    if (t.n > 2 && block >= t.j[2].tile0) i = 2;
    return t.j[i];
}
// Eight values of row i from column j on; zeros outside
template <int DT>
__device__ __forceinline__ void lin_values8(const LinJob& p, int i, int j, float v[8]) {
    const int cnt = i < p.m ? max(0, min(8, p.n - j)) : 0;
    if (cnt == 0) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = 0.0f;
        return;
    }
    lin_load8<DT>(p.src, i * p.ld + j, cnt, v);
    if (p.z) {
        float z[8];
        lin_load_z8<DT>(p.z, i * p.z_ld + j, cnt, z);
        lin_with_act(p.act, [&](auto act) {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = lin_grad<DT == ODAMD_DTYPE_BF16, act.value>(v[e], z[e]);
        });
    }
}

__global__ void __launch_bounds__(256) linear_clear_kernel(unsigned* p, long long n) {
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long long)gridDim.x * 256) p[i] = 0u;
}

// Largest magnitudes of rows and columns.  The maximum does not depend on the order of its arguments, so the atomics leave
// the same result every time.
__global__ void __launch_bounds__(256) linear_max_kernel(LinJobs t) {
    __shared__ unsigned best[4][64];
    const LinJob& p = lin_job(t, blockIdx.x);
    const int tile = blockIdx.x - p.tile0, nt = (p.n + 63) / 64, i0 = tile / nt * 64, j0 = tile % nt * 64;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = (threadIdx.x & 7) * 8;
    unsigned col[8] = {};
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        const int i = i0 + (threadIdx.x >> 3) + 32 * q;
        float v[8];
        lin_values8<ODAMD_DTYPE_F32>(p, i, j0 + c, v);
        unsigned row = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const unsigned b = lin_magnitude(v[e]);
            row = b > row ? b : row;
            col[e] = b > col[e] ? b : col[e];
        }
        if (p.row_max) {
#pragma unroll
            for (int o = 1; o < 8; o <<= 1) {
                const unsigned u = __shfl_xor(row, o);
                row = u > row ? u : row;
            }
            if (c == 0 && row && i < p.m) atomicMax(p.row_max + i, row);
        }
    }
    if (!p.col_max) return;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
#pragma unroll
        for (int o = 8; o < 64; o <<= 1) {
            const unsigned u = __shfl_xor(col[e], o);
            col[e] = u > col[e] ? u : col[e];
        }
        if (lane < 8) best[wave][c + e] = col[e];
    }
    __syncthreads();
    if (wave == 0 && j0 + lane < p.n) {
        unsigned mine = 0;
#pragma unroll
        for (int q = 0; q < 4; ++q) mine = best[q][lane] > mine ? best[q][lane] : mine;
        if (mine) atomicMax(p.col_max + j0 + lane, mine);
    }
}

// Eight values of row `at` from column k on, shifted by a power of two (float32 form only)
template <int DT>
__device__ __forceinline__ void lin_lay8(char* base, long long at, int padded, int k, const float v[8], int shift) {
    if constexpr (DT == ODAMD_DTYPE_F32) {
        float s[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) s[e] = ldexpf(v[e], shift);
        store_split8(base + at * padded * 4 + split_at(k), s, 1.0f);
    } else {
        *(u32x4*)(base + (at * padded + k) * 2) = u32x4{f32x2_to_bf16x2(v[0], v[1]), f32x2_to_bf16x2(v[2], v[3]), f32x2_to_bf16x2(v[4], v[5]), f32x2_to_bf16x2(v[6], v[7])};
    }
}
template <int DT> __host__ __device__ constexpr int lin_chunk() { return DT == ODAMD_DTYPE_F32 ? 32 : 64; }

template <int DT>
__global__ void __launch_bounds__(256) linear_lay_kernel(LinJobs t) {
    __shared__ float tile[64][65];
    const LinJob& p = lin_job(t, blockIdx.x);
    const int at = blockIdx.x - p.tile0, nt = (p.n + 63) / 64, i0 = at / nt * 64, j0 = at % nt * 64;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int np = (int)lin_up(p.n, lin_chunk<DT>()), c = (threadIdx.x & 7) * 8;
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        const int r = (threadIdx.x >> 3) + 32 * q;
        float v[8];
        lin_values8<DT>(p, i0 + r, j0 + c, v);
        if (p.rows && i0 + r < p.m && j0 + c < np)
            lin_lay8<DT>(p.rows, i0 + r, np, j0 + c, v, DT == ODAMD_DTYPE_F32 ? lin_shift(p.row_max[i0 + r]) : 0);
        if (p.cols || p.sums)
#pragma unroll
            for (int e = 0; e < 8; ++e) tile[r][c + e] = v[e];
    }
    if (!p.cols && !p.sums) return;
    __syncthreads();
    if (p.sums && wave == 0 && j0 + lane < p.n) {
        float s = 0.0f;
#pragma unroll 8
        for (int q = 0; q < 64; ++q) s += tile[q][lane];
        p.sums[(long long)(i0 / 64) * p.n + j0 + lane] = s;
    }
    if constexpr (DT == ODAMD_DTYPE_F32) {
        const int mp = (int)lin_up(p.m, lin_chunk<DT>());
        if (!p.cols) return;
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            const int r = (threadIdx.x >> 3) + 32 * q;
            float v[8];
            if (j0 + r < p.n && i0 + c < mp) {
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = tile[c + e][r];
                lin_lay8<DT>(p.cols, j0 + r, mp, i0 + c, v, lin_shift(p.col_max[j0 + r]));
            }
        }
    }
}

// By rows only, a wave per row: the row's largest magnitude first, then (out of the caches) its pairs.  bfloat16: a plain copy
// to aligned, padded rows.
template <int DT>
__global__ void __launch_bounds__(256) linear_lay_rows_kernel(LinJobs t) {
    const LinJob& p = lin_job(t, blockIdx.x);
    const int row = (blockIdx.x - p.tile0) * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (row >= p.m) return;
    const long long at = (long long)row * p.ld;
    int shift = 0;
    if constexpr (DT == ODAMD_DTYPE_F32) {
        unsigned b = 0;
        for (int k = lane * 8; k < p.n; k += 512) {
            float v[8];
            lin_load8<DT>(p.src, at + k, min(8, p.n - k), v);
#pragma unroll
            for (int e = 0; e < 8; ++e) { const unsigned u = lin_magnitude(v[e]); b = u > b ? u : b; }
        }
#pragma unroll
        for (int o = 32; o; o >>= 1) { const unsigned u = __shfl_xor(b, o); b = u > b ? u : b; }
        if (lane == 0) p.row_max[row] = b;
        shift = lin_shift(b);
    }
    const int np = (int)lin_up(p.n, lin_chunk<DT>());
    for (int k = lane * 8; k < np; k += 512) {
        float v[8];
        lin_load8<DT>(p.src, at + k, max(0, min(8, p.n - k)), v);
        lin_lay8<DT>(p.rows, row, np, k, v, shift);
    }
}

// ---- the backward pass of a small layer in one launch, without matrix instructions ------------------------------------
// Both gradients are sums of rows of V with coefficients out of dz: dx[i] = sum_r dz[i][r] W[r], dw[i] = sum_r dz[r][i] x[r].  A
// workgroup takes eight rows of a result and 64 of its columns (a column a lane: four a lane leave too few workgroups, 64 x 64 x 64
// 5.7 us instead of 4.2); its waves share the sum, 16 terms each at a time, and add up in LDS.  dz stays in float32 and is in nobody's
// memory: every workgroup makes the eight rows or columns of it that it needs.  Bound by latency in the few workgroups of a small
// layer, by the vector unit in more.  Eight waves for float32, sixteen for bfloat16, whose loads bring half as much (78 x 225 of
// 40 rows: 5.7 us, with eight 7.8).
struct LinSmall {
    const void* dy;
    const void* z;
    const void* v[2];        // W, x
    void* out[2];            // dx, dw
    void* db;
    long long dy_ld, z_ld, v_ld[2], out_ld[2];
    int m, k, n;
    int block1;              // blocks of dx
};
template <int DT> __host__ __device__ constexpr int lin_small_threads() { return DT == ODAMD_DTYPE_F32 ? 512 : 1024; }
template <int DT> __host__ __device__ constexpr int lin_small_terms() { return lin_small_threads<DT>() / 4; }

template <int DT, int ACT>
__global__ void __launch_bounds__(lin_small_threads<DT>()) linear_small_backward_kernel(LinSmall p) {
    using T = typename LinType<DT>::T;
    constexpr int THREADS = lin_small_threads<DT>(), TERMS = lin_small_terms<DT>(), WAVES = THREADS / 64, SHARE = TERMS / WAVES;
    __shared__ __attribute__((aligned(16))) float coef[2][TERMS][8];
    __shared__ float joined[4][8][64];
    __shared__ double bias[WAVES][8];
    const int which = (int)blockIdx.x >= p.block1, block = blockIdx.x - (which ? p.block1 : 0);
    const int rows = which ? p.n : p.m, terms = which ? p.m : p.n, across = (p.k + 63) / 64;
    const int i0 = block / across * 8, c0 = block % across * 64;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = c0 + lane;
    const bool some = p.out[which] != nullptr, sum = which && p.db && c0 == 0;
    const T* v = (const T*)p.v[which];
    // two coefficients a thread, along the rows of dz: result row and term of each
    const auto place = [&](int q, int& i, int& r) {
        i = which ? threadIdx.x & 7 : (int)threadIdx.x / TERMS + 4 * q;
        r = which ? (int)threadIdx.x / 8 + TERMS / 2 * q : threadIdx.x % TERMS;
    };
    const auto fetch = [&](int r0, float to[2]) {
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            int i, r;
            place(q, i, r);
            to[q] = 0.0f;
            if (i0 + i < rows && r0 + r < terms) {
                const long long y = which ? r0 + r : i0 + i;     // row and column of dz
                const int x = which ? i0 + i : r0 + r;
                const float dy = LinType<DT>::get(((const T*)p.dy)[y * p.dy_ld + x]);
                float z[8] = {};
                if constexpr (ACT != ODAMD_ACT_NONE) lin_load_z8<DT>(p.z, y * p.z_ld + x, 1, z);
                to[q] = lin_grad<DT == ODAMD_DTYPE_BF16, ACT>(dy, z[0]);
            }
        }
    };
    float acc[8] = {};
    double total = 0.0;
    float next[2];
    fetch(0, next);
    for (int r0 = 0, turn = 0; r0 < terms; r0 += TERMS, turn ^= 1) {
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            int i, r;
            place(q, i, r);
            coef[turn][r][i] = next[q];
        }
        __syncthreads();                                         // one a round: the other buffer is written two rounds on
        if (r0 + TERMS < terms) fetch(r0 + TERMS, next);
        const int from = wave * SHARE;
        if (some && c < p.k) {
            // terms past the last one have zero coefficients, and the last one's row made zeros (it may hold no number)
            float x[SHARE];
#pragma unroll
            for (int s = 0; s < SHARE; ++s) {
                const float u = LinType<DT>::get(v[min(r0 + from + s, terms - 1) * p.v_ld[which] + c]);
                x[s] = r0 + from + s < terms ? u : 0.0f;
            }
#pragma unroll
            for (int s = 0; s < SHARE; ++s) {
                const f32x4_t a = *(const f32x4_t*)coef[turn][from + s], b = *(const f32x4_t*)(coef[turn][from + s] + 4);
#pragma unroll
                for (int i = 0; i < 8; ++i) acc[i] = fmaf(i < 4 ? a[i & 3] : b[i & 3], x[s], acc[i]);
            }
        }
        if (sum) {
#pragma unroll
            for (int s = 0; s < SHARE / 8; ++s) total += coef[turn][from + (lane >> 3) * (SHARE / 8) + s][lane & 7];
        }
    }
    // four waves at a time add their sums to what the ones before left
#pragma unroll
    for (int g = 0; g < WAVES / 4; ++g) {
        if (wave / 4 == g)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                float& at = joined[wave % 4][i][lane];
                at = g == 0 ? acc[i] : at + acc[i];
            }
        __syncthreads();
    }
    if (sum) {
#pragma unroll
        for (int o = 8; o < 64; o <<= 1) total += __shfl_xor(total, o);
        if (lane < 8) bias[wave][lane] = total;
        __syncthreads();
    }
    const int i = threadIdx.x >> 6;
    if (some && i < 8 && i0 + i < rows && c < p.k) {
        float s = joined[0][i][lane];
#pragma unroll
        for (int w = 1; w < 4; ++w) s += joined[w][i][lane];
        ((T*)p.out[which])[(i0 + i) * p.out_ld[which] + c] = LinType<DT>::put(s);
    }
    if (sum && threadIdx.x < 8 && i0 + (int)threadIdx.x < rows) {
        double s = bias[0][threadIdx.x];
        for (int w = 1; w < WAVES; ++w) s += bias[w][threadIdx.x];
        ((T*)p.db)[i0 + threadIdx.x] = LinType<DT>::put((float)s);
    }
}

// ---- the products ----------------------------------------------------------------------------------------------------
struct LinGemm {
    GemmOperand a, b;
    const unsigned* a_max;   // float32: the rows' largest magnitudes
    const unsigned* b_max;
    float* part;             // split reduction: [split][m][n]
    int m, n, k_len, chunks, per, split;   // chunks of K, chunks per split part
    int a_turned;            // backward pass in bfloat16: B lies with the reduction along its rows, A too where this is set
    LinEnd end;
};
// The column sums of 64-row blocks that db is made of
struct LinSums {
    const float* sums;
    void* db;
    int blocks, n;
};
// A launch: up to two products, and behind their tiles the blocks of db
struct LinLaunch {
    LinGemm g[2];
    LinSums sums;
    int block1, block2;      // first block of the second product, of db
};

template <int DT, int THREADS>
__device__ __forceinline__ void lin_bias_grad(const LinSums& p, int block, double* part) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, j = block * 64 + lane;
    constexpr int W = THREADS / 64;
    double s = 0.0;
    if (j < p.n)
        for (int b = wave; b < p.blocks; b += W) s += p.sums[(long long)b * p.n + j];
    part[wave * 64 + lane] = s;
    __syncthreads();
    if (wave == 0 && j < p.n) {
        for (int q = 1; q < W; ++q) s += part[q * 64 + lane];
        ((typename LinType<DT>::T*)p.db)[j] = LinType<DT>::put((float)s);
    }
}

template <typename TILE, int DT, int ACT, bool PART, bool TURNED>
__global__ void __launch_bounds__(TILE::THREADS) linear_product_kernel(LinLaunch t) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    int block = (int)blockIdx.x;
    if (block >= t.block2) {
        lin_bias_grad<DT, TILE::THREADS>(t.sums, block - t.block2, (double*)lds);
        return;
    }
    const bool second = block >= t.block1;
    const LinGemm& p = second ? t.g[1] : t.g[0];
    block -= second ? t.block1 : 0;
    const int mt = (p.m + TILE::TM - 1) / TILE::TM, nt = (p.n + TILE::TN - 1) / TILE::TN;
    const int id = gemm_xcd_remap(block, (second ? t.block2 - t.block1 : t.block1));
    // PART: a product of the launch may be cut
    const int part = PART ? id / (mt * nt) : 0;
    int ti, tj;
    gemm_tile_at(PART ? id - part * mt * nt : id, mt, nt, ti, tj);
    const int i0 = ti * TILE::TM, j0 = tj * TILE::TN;
    TILE tile;
    const int c0 = part * p.per, c1 = min(p.chunks, (part + 1) * p.per);
    if constexpr (TURNED) {
        if (p.a_turned) tile.template run<true, true>(p.a, p.b, i0, j0, c0, c1, p.k_len, lds);
        else tile.template run<false, true>(p.a, p.b, i0, j0, c0, c1, p.k_len, lds);
    } else {
        tile.run(p.a, p.b, i0, j0, c0, c1, p.k_len, lds);
    }
    // a lane hands out the same eight columns in all its rows: bias and exponents are loaded once
    const int col = j0 + tile.row_column(), cnt = max(0, min(8, p.n - col));
    float bias[8];
    int shift[8];
    lin_bias8<DT>(p.end, col, cnt, bias);
#pragma unroll
    for (int e = 0; e < 8; ++e) shift[e] = DT == ODAMD_DTYPE_F32 && e < cnt ? lin_shift(p.b_max[col + e]) : 0;
    struct Before { LinRaw<DT> residual; unsigned max; };
    const auto before = [&](int i, int) {
        Before x = {};
        if (i0 + i < p.m && cnt > 0) {
            if ((!PART || p.split == 1) && p.end.residual) x.residual = lin_raw8<DT>(p.end.residual, (long long)(i0 + i) * p.end.r_ld + col, cnt);
            if (DT == ODAMD_DTYPE_F32) x.max = p.a_max[i0 + i];
        }
        return x;
    };
    const auto rows = [&](int i, int, float v[8], const Before& x) {
        i += i0;
        if (i >= p.m || cnt <= 0) return;
        if constexpr (DT == ODAMD_DTYPE_F32) {
            const int s = lin_shift(x.max);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = ldexpf(v[e], -(s + shift[e]));
        }
        if (PART && p.split > 1) lin_store8<ODAMD_DTYPE_F32>(p.part, ((long long)part * p.m + i) * p.n + col, cnt, v);
        else lin_finish8<DT, ACT>(p.end, i, col, cnt, v, bias, x.residual);
    };
    const auto none = [](int, int) { return GemmNothing{}; };
    const auto never = [](int, int, float*, const GemmNothing&) {};
    tile.template hand_out<true, false, 8>(lds, before, rows, none, never);
}

// Sums the parts of split reductions in their order
struct LinJoin {
    LinGemm g[2];
    long long runs[2];   // runs of eight columns of each
    int n;
};
template <int DT>
__global__ void __launch_bounds__(256) linear_join_kernel(LinJoin t) {
    for (long long q = (long long)blockIdx.x * 256 + threadIdx.x; q < t.runs[0] + t.runs[1]; q += (long long)gridDim.x * 256) {
        const bool second = q >= t.runs[0];
        const LinGemm& p = second ? t.g[1] : t.g[0];
        const int runs = (p.n + 7) / 8;
        const long long at = second ? q - t.runs[0] : q, i = at / runs;
        const int j = (int)(at - i * runs) * 8, cnt = min(8, p.n - j);
        float v[8], u[8];
        lin_load8<ODAMD_DTYPE_F32>(p.part, i * p.n + j, cnt, v);
        for (int s = 1; s < p.split; ++s) {
            lin_load8<ODAMD_DTYPE_F32>(p.part, ((long long)s * p.m + i) * p.n + j, cnt, u);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] += u[e];
        }
        lin_with_act(p.end.act, [&](auto act) { lin_finish8<DT, act.value>(p.end, i, j, cnt, v); });
    }
}

// ---- host ------------------------------------------------------------------------------------------------------------
// Workspace as one walk over its regions: with base 0 it measures, with the caller's base it hands out.
struct LinSpace {
    char* base;
    long long at = 0;
    char* take(long long bytes) {
        char* p = base + at;
        at += lin_up(bytes, 256);
        return p;
    }
};

struct LinPlan { int tile, longest; double us; };   // longest: chunks a workgroup takes at most
// Tile and length of the parts the reductions are cut into, by the estimated time of the launch (`count` products).  A larger
// tile wins per product; but a 256 x 256 tile fills its compute unit, nothing runs beside its epilogue, and all units reach
// theirs together: (25600, 1024, 4096) with bias, SiLU and residual in bf16 takes 285 us in 256, 300 in 128 and 383 us in
// 64.  Where tiles leave units idle, or two products of a launch differ in length, parts of four chunks or more fill them,
// for the price of a second launch that adds them up (4 us, and their bytes once out and once in).
template <int DT>
LinPlan lin_plan(const LinGemm* g, int count) {
    int all = 1;
    for (int q = 0; q < count; ++q) {
        const int chunks = (g[q].k_len + lin_chunk<DT>() - 1) / lin_chunk<DT>();
        all = chunks > all ? chunks : all;
    }
    LinPlan best = {64, all, 0.0};
    if (count == 0) return best;
    double least = -1.0;
    for (int tile : {64, 128, 256})
        for (int cut = 1; cut <= 32 && (cut == 1 || all / cut >= 4); cut *= 2) {
            const int longest = (all + cut - 1) / cut;
            GemmLoad load;
            double extra = 0.0;
            for (int q = 0; q < count; ++q) {
                const int chunks = (g[q].k_len + lin_chunk<DT>() - 1) / lin_chunk<DT>(), parts = (chunks + longest - 1) / longest;
                const double tiles = (double)((g[q].m + (long long)tile - 1) / tile) * ((g[q].n + (long long)tile - 1) / tile);
                gemm_load_add(load, tiles * parts, (chunks + parts - 1) / parts);
                if (parts > 1) extra += 4.0 / count + parts * (double)g[q].m * g[q].n * 8.0 / 3.0e6;
            }
            const double us = gemm_time_us(tile, load, DT == ODAMD_DTYPE_F32, DT == ODAMD_DTYPE_F32 ? 8.0 : 4.0) + extra;
            if (least < 0.0 || us < least) {
                best = {tile, longest, us};
                least = us;
            }
        }
    return best;
}

template <typename TILE, int DT, int ACT, bool PART, bool TURNED>
int lin_launch(LinLaunch& t, int count, hipStream_t s) {
    long long at = 0;
    for (int q = 0; q < 2; ++q) {
        if (q == 1) t.block1 = (int)at;
        if (q < count) at += (((long long)t.g[q].m + TILE::TM - 1) / TILE::TM) * (((long long)t.g[q].n + TILE::TN - 1) / TILE::TN) * t.g[q].split;
        if (at > 0x3fffffffLL) return ODAMD_E_LIMIT;
    }
    t.block2 = (int)at;
    at += t.sums.db ? (t.sums.n + 63) / 64 : 0;
    if (!gemm_grid_ok(at, TILE::THREADS)) return ODAMD_E_LIMIT;
    const auto kernel = linear_product_kernel<TILE, DT, ACT, PART, TURNED>;
    const hipError_t e = odamd_ensure_lds((const void*)kernel, TILE::LDS);
    if (e != hipSuccess) return (int)e;
    kernel<<<(int)at, TILE::THREADS, TILE::LDS, s>>>(t);
    return (int)hipGetLastError();
}
template <int DT, int ACT, bool PART, bool TURNED>
int lin_launch_tile(LinLaunch& t, int count, int tile, hipStream_t s) {
    constexpr int PL = LinType<DT>::PL;
    constexpr bool F16 = DT == ODAMD_DTYPE_F32;
    if (tile == 256) return lin_launch<GemmTile<PL, F16, 256, 256, 4, 2, 1, 2>, DT, ACT, PART, TURNED>(t, count, s);
    if (tile == 128) return lin_launch<GemmTile<PL, F16, 128, 128, 2, PL == 2 ? 2 : 4, 1, 2>, DT, ACT, PART, TURNED>(t, count, s);
    long long tiles = 0;
    for (int q = 0; q < count; ++q) tiles += (((long long)t.g[q].m + 63) / 64) * (((long long)t.g[q].n + 63) / 64) * t.g[q].split;
    // one tile or two for a compute unit: two wave groups each ((512, 4096, 3200) bf16 28.8 us instead of 35.5; with few chunks
    // there is nothing to share: (6000, 600, 256) 8.9 instead of 8.3)
    if (tiles > 512) return lin_launch<GemmTile<PL, F16, 64, 64, 2, 2, 1, 2>, DT, ACT, PART, TURNED>(t, count, s);
    if (tiles > 256) return lin_launch<GemmTile<PL, F16, 64, 64, 2, 2, 2, 2>, DT, ACT, PART, TURNED>(t, count, s);
    return lin_launch<GemmTile<PL, F16, 64, 64, 2, 2, 2, 3>, DT, ACT, PART, TURNED>(t, count, s);
}
// `count` products (0: db alone), measuring their workspace or running them
template <int DT, bool BACKWARD>
int lin_products(LinLaunch& t, int count, LinSpace& ws, bool go, hipStream_t s) {
    const LinPlan plan = lin_plan<DT>(t.g, count);
    LinJoin join = {};
    for (int q = 0; q < count; ++q) {
        LinGemm& g = t.g[q];
        g.chunks = (g.k_len + lin_chunk<DT>() - 1) / lin_chunk<DT>();
        g.split = (g.chunks + plan.longest - 1) / plan.longest;
        g.per = (g.chunks + g.split - 1) / g.split;
        g.split = (g.chunks + g.per - 1) / g.per;
        if (g.split > 1) {
            g.part = (float*)ws.take((long long)g.split * g.m * g.n * 4);
            join.g[join.n] = g;
            join.runs[join.n++] = (long long)g.m * ((g.n + 7) / 8);
        }
    }
    if (!go) return 0;
    constexpr bool TURNED = BACKWARD && DT == ODAMD_DTYPE_BF16;
    int rc = 0;
    if (join.n == 0) {
        if constexpr (BACKWARD) rc = lin_launch_tile<DT, ODAMD_ACT_NONE, false, TURNED>(t, count, plan.tile, s);
        else lin_with_act(t.g[0].end.act, [&](auto act) { rc = lin_launch_tile<DT, act.value, false, false>(t, count, plan.tile, s); });
        return rc;
    }
    rc = lin_launch_tile<DT, ODAMD_ACT_NONE, true, TURNED>(t, count, plan.tile, s);
    if (rc != 0) return rc;
    const long long blocks = (join.runs[0] + join.runs[1] + 255) / 256;
    linear_join_kernel<DT><<<(int)(blocks < 4096 ? blocks : 4096), 256, 0, s>>>(join);
    return (int)hipGetLastError();
}

// Whether products read the caller's rows as they are: no workspace for these.  A query without the pointer counts on nothing.
template <int DT> bool lin_direct(const void* p, long long ld, int k) {
    return DT == ODAMD_DTYPE_BF16 && p && ((uintptr_t)p & 15) == 0 && ld % 8 == 0 && k % 8 == 0;
}
// Blocks of a launch over the jobs: 64 x 64 tiles, or groups of rows; -1: more than a launch takes
int lin_tiles(LinJobs& t, int unit_rows) {
    long long at = 0;
    for (int i = 0; i < t.n; ++i) {
        t.j[i].tile0 = (int)at;
        at += unit_rows ? (t.j[i].m + unit_rows - 1) / unit_rows : (((long long)t.j[i].m + 63) / 64) * ((t.j[i].n + 63) / 64);
    }
    return gemm_grid_ok(at, 256) ? (int)at : -1;
}

// Whether a layer goes without matrix instructions: up to eight rows always (8 x 4096 x 4096 bf16 10.1 us, in products 13.7), more
// where its workgroups are few.  Products cost a launch or two for laying operands out, the rows a step per eight of them;
// rows / products, us: float32 512 x 256 x 256 (4096 workgroups) 9.2 / 10.6, 1024 x 256 x 256 15.7 / 11.3, 128 x 1024 x 1024
// 13.5 / 18.1, 256 x 1024 x 1024 22.5 / 19.9, 32 x 4096 x 4096 46 / 55; bfloat16 read in place 128 x 256 x 256 (1024) 4.2 / 4.5,
// 256 x 256 x 256 6.8 / 4.5, 64 x 1024 x 1024 8.3 / 7.8; bfloat16 laid out 64 x 513 x 1024 (2048) 7.0 / 8.9, 128 x 513 x 1024
// 11.0 / 9.0.  A long reduction in few workgroups is one chain of loads, which products cut: bfloat16 8 x 30000 x 64 17.9 / 18.4,
// 8 x 100000 x 64 58 / 26 (float32, laid out first there, 86 / 252).
template <int DT>
bool lin_by_rows(int m, int k, int n, bool direct) {
    const long long blocks = ((m + 7LL) / 8) * ((n + 3LL) / 4);
    if (DT == ODAMD_DTYPE_BF16 && direct && k > 32768 && blocks < 256) return false;
    return m <= 8 || blocks <= (DT == ODAMD_DTYPE_F32 ? 4096 : direct ? 1024 : 2048);
}

template <int DT>
int lin_forward_rows(const odamd_linear_desc& d, const LinEnd& end, hipStream_t s) {
    const LinRow p = {d.x, d.w, d.x_ld, d.w_ld, d.m, d.k, d.n, end};
    const dim3 blocks((d.n + 3) / 4, (d.m + 7) / 8);
    if (!gemm_grid_ok(blocks.x, 256)) return ODAMD_E_LIMIT;
    if (d.m == 1) linear_rows_kernel<DT, 1><<<blocks, 256, 0, s>>>(p);
    else if (d.m == 2) linear_rows_kernel<DT, 2><<<blocks, 256, 0, s>>>(p);
    else if (d.m <= 4) linear_rows_kernel<DT, 4><<<blocks, 256, 0, s>>>(p);
    else linear_rows_kernel<DT, 8><<<blocks, 256, 0, s>>>(p);
    return (int)hipGetLastError();
}

// go = false: measures the workspace only
template <int DT>
int lin_forward(const odamd_linear_desc& d, LinSpace& ws, bool go, hipStream_t s) {
    const LinEnd end = {d.bias, d.residual, d.y, d.z, d.r_ld, d.y_ld, d.z_ld, d.act};
    const bool direct = lin_direct<DT>(d.x, d.x_ld, d.k) && lin_direct<DT>(d.w, d.w_ld, d.k);
    if (lin_by_rows<DT>(d.m, d.k, d.n, direct)) return go ? lin_forward_rows<DT>(d, end, s) : 0;
    constexpr int SIZE = DT == ODAMD_DTYPE_F32 ? 4 : 2;
    LinLaunch launch = {};
    LinGemm& g = launch.g[0];
    g.end = end;
    g.m = d.m;
    g.n = d.n;
    g.k_len = d.k;
    LinJobs jobs = {};
    const long long kp = lin_up(d.k, lin_chunk<DT>());
    const auto operand = [&](const void* p, long long ld, int rows, GemmOperand& o, const unsigned*& max) {
        if (lin_direct<DT>(p, ld, d.k)) {
            o = {(const char*)p, ld * SIZE, rows};
            return;
        }
        LinJob& j = jobs.j[jobs.n++];
        j.src = p;
        j.ld = ld;
        j.m = rows;
        j.n = d.k;
        j.rows = ws.take(rows * kp * SIZE);
        j.row_max = DT == ODAMD_DTYPE_F32 ? (unsigned*)ws.take(rows * 4LL) : nullptr;
        max = j.row_max;
        o = {j.rows, kp * SIZE, rows};
    };
    operand(d.x, d.x_ld, d.m, g.a, g.a_max);
    operand(d.w, d.w_ld, d.n, g.b, g.b_max);
    // a laid out operand is padded to whole chunks, one read in place is not: the tail is then read as zeros for both
    if (go && jobs.n) {
        const int blocks = lin_tiles(jobs, 4);
        if (blocks < 0) return ODAMD_E_LIMIT;
        linear_lay_rows_kernel<DT><<<blocks, 256, 0, s>>>(jobs);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return (int)e;
    }
    if (DT == ODAMD_DTYPE_BF16) g.k_len = (int)lin_up(d.k, 8);
    return lin_products<DT, false>(launch, 1, ws, go, s);
}

// What both forms of the backward pass share: the job that makes dz, the two products' sizes and results, db
struct LinBackward {
    LinJobs jobs = {};
    LinLaunch launch = {};
    int count = 0;
    LinGemm *gx = nullptr, *gw = nullptr;
    LinJob& dz() { return jobs.j[0]; }

    LinBackward(const odamd_linear_grad_desc& d, LinSpace& ws) {
        jobs.n = 1;
        dz().src = d.dy;
        dz().ld = d.dy_ld;
        dz().z = d.act != ODAMD_ACT_NONE ? d.z : nullptr;
        dz().z_ld = d.z_ld;
        dz().act = d.act;
        dz().m = d.m;
        dz().n = d.n;
        if (d.dx) {
            gx = &launch.g[count++];
            gx->m = d.m;
            gx->n = d.k;
            gx->end.y = d.dx;
            gx->end.y_ld = d.dx_ld;
        }
        if (d.dw) {
            gw = &launch.g[count++];
            gw->m = d.n;
            gw->n = d.k;
            gw->end.y = d.dw;
            gw->end.y_ld = d.dw_ld;
        }
        if (d.db) {
            const int blocks = (d.m + 63) / 64;
            dz().sums = (float*)ws.take((long long)blocks * d.n * 4);
            launch.sums = {dz().sums, d.db, blocks, d.n};
        }
    }
    LinJob& add(const void* src, long long ld, int m, int n) {
        LinJob& j = jobs.j[jobs.n++];
        j.src = src;
        j.ld = ld;
        j.m = m;
        j.n = n;
        return j;
    }
};

int lin_backward_bf16(const odamd_linear_grad_desc& d, LinSpace& ws, bool go, hipStream_t s) {
    constexpr int DT = ODAMD_DTYPE_BF16;
    LinBackward t(d, ws);
    const long long np = lin_up(d.n, 64), kp = lin_up(d.k, 64);
    // dz by rows serves both products; dy itself where there is no activation and its rows can be read as they are
    GemmOperand dz = {};
    const bool direct = d.act == ODAMD_ACT_NONE && lin_direct<DT>(d.dy, d.dy_ld, d.n);
    if (t.count) {
        if (!direct) t.dz().rows = ws.take(d.m * np * 2);
        dz = direct ? GemmOperand{(const char*)d.dy, d.dy_ld * 2, d.m, d.n} : GemmOperand{t.dz().rows, np * 2, d.m, d.n};
    }
    const auto across = [&](const void* p, long long ld, int rows) {
        if (lin_direct<DT>(p, ld, d.k)) return GemmOperand{(const char*)p, ld * 2, rows, d.k};
        LinJob& j = t.add(p, ld, rows, d.k);
        j.rows = ws.take(rows * kp * 2);
        return GemmOperand{j.rows, kp * 2, rows, d.k};
    };
    if (d.dx) {
        t.gx->a = dz;
        t.gx->b = across(d.w, d.w_ld, d.n);
        t.gx->k_len = (int)lin_up(d.n, 8);
    }
    if (d.dw) {
        t.gw->a = dz;
        t.gw->a_turned = 1;
        t.gw->b = across(d.x, d.x_ld, d.m);
        t.gw->k_len = (int)lin_up(d.m, 8);
    }
    if (go && (t.dz().rows || t.dz().sums || t.jobs.n > 1)) {
        const int blocks = lin_tiles(t.jobs, 0);
        if (blocks < 0) return ODAMD_E_LIMIT;
        linear_lay_kernel<DT><<<blocks, 256, 0, s>>>(t.jobs);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return (int)e;
    }
    return lin_products<DT, true>(t.launch, t.count, ws, go, s);
}

int lin_backward_f32(const odamd_linear_grad_desc& d, LinSpace& ws, bool go, hipStream_t s) {
    constexpr int DT = ODAMD_DTYPE_F32;
    LinBackward t(d, ws);
    const long long mp = lin_up(d.m, 32), np = lin_up(d.n, 32);
    // the largest magnitudes of all operands lie side by side: one launch clears them
    const long long n_max = (long long)d.m + d.n + 2LL * d.k;
    unsigned* maxes = (unsigned*)ws.take(n_max * 4);
    unsigned *z_row = maxes, *z_col = maxes + d.m, *w_col = z_col + d.n, *x_col = w_col + d.k;
    if (d.dx) {
        t.dz().rows = ws.take(d.m * np * 4);
        t.dz().row_max = z_row;
        LinJob& w = t.add(d.w, d.w_ld, d.n, d.k);
        w.cols = ws.take(d.k * np * 4);
        w.col_max = w_col;
        t.gx->a = {t.dz().rows, np * 4, d.m};
        t.gx->b = {w.cols, np * 4, d.k};
        t.gx->a_max = z_row;
        t.gx->b_max = w_col;
        t.gx->k_len = d.n;
    }
    if (d.dw) {
        t.dz().cols = ws.take(d.n * mp * 4);
        t.dz().col_max = z_col;
        LinJob& x = t.add(d.x, d.x_ld, d.m, d.k);
        x.cols = ws.take(d.k * mp * 4);
        x.col_max = x_col;
        t.gw->a = {t.dz().cols, mp * 4, d.n};
        t.gw->b = {x.cols, mp * 4, d.k};
        t.gw->a_max = z_col;
        t.gw->b_max = x_col;
        t.gw->k_len = d.m;
    }
    if (go) {
        const int blocks = lin_tiles(t.jobs, 0);
        if (blocks < 0) return ODAMD_E_LIMIT;
        if (t.count) {
            linear_clear_kernel<<<(int)((n_max + 255) / 256 < 1024 ? (n_max + 255) / 256 : 1024), 256, 0, s>>>(maxes, n_max);
            linear_max_kernel<<<blocks, 256, 0, s>>>(t.jobs);
        }
        linear_lay_kernel<DT><<<blocks, 256, 0, s>>>(t.jobs);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return (int)e;
    }
    return lin_products<DT, true>(t.launch, t.count, ws, go, s);
}

// Whether the backward pass goes that way: by its estimated time, measured as 2.4 us, 2 us (bfloat16: 3) for every step of 128
// (256) terms of the longest sum, or 4.5 (9) ns for every step of any workgroup; products with what lies before them take
// launches of 13.5 us in float32 (three more of them), of 6 us in bfloat16.  Small / products, us, rows x inputs x outputs: float32
// 8 x 64 x 64 4.1 / 14.5, 512 x 64 x 64 10.4 / 21, 1024 x 64 x 64 18 / 23, 128 x 996 x 424 13 / 22, 256 x 1024 x 1024 41 / 33;
// bfloat16 40 x 78 x 225 5.7 / 9.0, 256 x 256 x 256 6.4 / 8.7, 512 x 256 x 256 11.4 / 10.3, 8 x 996 x 424 13 / 9.3.
template <int DT>
bool lin_small(const odamd_linear_grad_desc& d) {
    constexpr bool F32 = DT == ODAMD_DTYPE_F32;
    constexpr int TERMS = lin_small_terms<DT>();
    const double across = (d.k + 63) / 64;
    double longest = 0.0, total = 0.0;
    LinGemm g[2] = {};
    int count = 0;
    const auto add = [&](int rows, int terms, bool product) {
        const double steps = (terms + TERMS - 1) / TERMS;
        longest = steps > longest ? steps : longest;
        total += (rows + 7) / 8 * across * steps;
        if (!product) return;
        g[count].m = rows;
        g[count].n = d.k;
        g[count++].k_len = terms;
    };
    if (d.dx) add(d.m, d.n, true);
    if (d.dw || d.db) add(d.n, d.m, d.dw);
    const double chain = (F32 ? 2.0 : 3.0) * longest, all = (F32 ? 2.0 : 3.0) + (F32 ? 4.5e-3 : 9e-3) * total;
    return 2.4 + (chain > all ? chain : all) < lin_plan<DT>(g, count).us + (F32 ? 13.5 : 6.0);
}
template <int DT>
int lin_small_backward(const odamd_linear_grad_desc& d, hipStream_t s) {
    const long long across = (d.k + 63) / 64, block1 = d.dx ? (d.m + 7) / 8 * across : 0;
    const long long blocks = block1 + (d.dw || d.db ? (d.n + 7) / 8 * across : 0);
    if (!gemm_grid_ok(blocks, lin_small_threads<DT>())) return ODAMD_E_LIMIT;
    const LinSmall p = {d.dy, d.z, {d.w, d.x}, {d.dx, d.dw}, d.db, d.dy_ld, d.z_ld, {d.w_ld, d.x_ld}, {d.dx_ld, d.dw_ld}, d.m, d.k, d.n, (int)block1};
    lin_with_act(d.act, [&](auto act) { linear_small_backward_kernel<DT, act.value><<<(int)blocks, lin_small_threads<DT>(), 0, s>>>(p); });
    return (int)hipGetLastError();
}

template <int DT>
int lin_backward(const odamd_linear_grad_desc& d, LinSpace& ws, bool go, hipStream_t s) {
    if (lin_small<DT>(d)) return go ? lin_small_backward<DT>(d, s) : 0;
    if constexpr (DT == ODAMD_DTYPE_F32) return lin_backward_f32(d, ws, go, s);
    else return lin_backward_bf16(d, ws, go, s);
}
int lin_backward_any(const odamd_linear_grad_desc& d, LinSpace& ws, bool go, hipStream_t s) {
    return d.dtype == ODAMD_DTYPE_F32 ? lin_backward<ODAMD_DTYPE_F32>(d, ws, go, s) : lin_backward<ODAMD_DTYPE_BF16>(d, ws, go, s);
}

constexpr long long LIN_MAX = 0x7fff0000LL;   // 2^31 less what an index passes its end by
bool lin_sizes_ok(int m, int k, int n, int act, int dtype) {
    return m >= 1 && k >= 1 && n >= 1 && m <= LIN_MAX && k <= LIN_MAX && n <= LIN_MAX && act >= ODAMD_ACT_NONE && act <= ODAMD_ACT_RELU
           && (dtype == ODAMD_DTYPE_F32 || dtype == ODAMD_DTYPE_BF16);
}
bool lin_aligned(const void* p, int dtype) { return ((uintptr_t)p & (dtype == ODAMD_DTYPE_F32 ? 3 : 1)) == 0; }

}  // namespace

extern "C" {

size_t odamd_linear_workspace_bytes(const odamd_linear_desc* d) {
    if (!d || !lin_sizes_ok(d->m, d->k, d->n, d->act, d->dtype)) return 0;
    LinSpace ws = {nullptr};
    if (d->dtype == ODAMD_DTYPE_F32) lin_forward<ODAMD_DTYPE_F32>(*d, ws, false, nullptr);
    else lin_forward<ODAMD_DTYPE_BF16>(*d, ws, false, nullptr);
    return (size_t)ws.at;
}

int odamd_linear_forward(const odamd_linear_desc* d, void* workspace, size_t workspace_bytes, void* stream) {
    if (!d || !d->x || !d->w || !d->y || !lin_sizes_ok(d->m, d->k, d->n, d->act, d->dtype)) return ODAMD_E_ARG;
    if (d->x_ld < d->k || d->w_ld < d->k || d->y_ld < d->n || (d->residual && d->r_ld < d->n) || (d->z && d->z_ld < d->n)) return ODAMD_E_SHAPE;
    if (!lin_aligned(d->x, d->dtype) || !lin_aligned(d->w, d->dtype) || !lin_aligned(d->y, d->dtype) || !lin_aligned(d->bias, d->dtype)
        || !lin_aligned(d->residual, d->dtype) || !lin_aligned(d->z, d->dtype) || ((uintptr_t)workspace & 255)) return ODAMD_E_ALIGN;
    const size_t need = odamd_linear_workspace_bytes(d);
    if (need && !workspace) return ODAMD_E_ARG;
    if (workspace_bytes < need) return ODAMD_E_WORKSPACE;
    LinSpace ws = {(char*)workspace};
    return d->dtype == ODAMD_DTYPE_F32 ? lin_forward<ODAMD_DTYPE_F32>(*d, ws, true, (hipStream_t)stream)
                                       : lin_forward<ODAMD_DTYPE_BF16>(*d, ws, true, (hipStream_t)stream);
}

size_t odamd_linear_backward_workspace_bytes(const odamd_linear_grad_desc* d) {
    if (!d || !lin_sizes_ok(d->m, d->k, d->n, d->act, d->dtype)) return 0;
    LinSpace ws = {nullptr};
    lin_backward_any(*d, ws, false, nullptr);
    return (size_t)ws.at;
}

int odamd_linear_backward(const odamd_linear_grad_desc* d, void* workspace, size_t workspace_bytes, void* stream) {
    if (!d || !d->dy || !lin_sizes_ok(d->m, d->k, d->n, d->act, d->dtype)) return ODAMD_E_ARG;
    if (!d->dx && !d->dw && !d->db) return ODAMD_E_ARG;
    if ((d->act != ODAMD_ACT_NONE && !d->z) || (d->dx && !d->w) || (d->dw && !d->x)) return ODAMD_E_ARG;
    if (d->dy_ld < d->n || (d->act != ODAMD_ACT_NONE && d->z_ld < d->n) || (d->dx && (d->w_ld < d->k || d->dx_ld < d->k))
        || (d->dw && (d->x_ld < d->k || d->dw_ld < d->k))) return ODAMD_E_SHAPE;
    if (!lin_aligned(d->dy, d->dtype) || !lin_aligned(d->z, d->dtype) || !lin_aligned(d->x, d->dtype) || !lin_aligned(d->w, d->dtype)
        || !lin_aligned(d->dx, d->dtype) || !lin_aligned(d->dw, d->dtype) || !lin_aligned(d->db, d->dtype) || ((uintptr_t)workspace & 255)) return ODAMD_E_ALIGN;
    const size_t need = odamd_linear_backward_workspace_bytes(d);
    if (need && !workspace) return ODAMD_E_ARG;
    if (workspace_bytes < need) return ODAMD_E_WORKSPACE;
    LinSpace ws = {(char*)workspace};
    return lin_backward_any(*d, ws, true, (hipStream_t)stream);
}

}  // extern "C"
