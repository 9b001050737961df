// Matrix product core of the dense layer and of the Newton-Schulz products: C[m][n] = sum_k A[m][k] B[n][k], both operands
// with the reduction contiguous.  Included by linear.hip and orthogonalize.hip inside their anonymous namespaces.
//
// Two operand forms, one data path:
//   PL = 1: bf16 values, one v_mfma_f32_32x32x16_bf16 per 32 x 32 x 16 block;
//   PL = 2: every value as a pair of fp16 numbers, v = (hi + lo) 2^-s; 32 hi and then their 32 lo lie side by side.  hi holds
//           the upper 11 bits of v, lo the next 11, so hi_a hi_b + hi_a lo_b + lo_a hi_b (three v_mfma_f32_32x32x16_f16)
//           carries a product to 2^-22, the dropped lo_a lo_b.  Float32 operands run at a third of the half-precision matrix
//           rate this way, which is five times the rate of the float32 matrix instructions; 2^s is a power of two, so it
//           costs no rounding.  fp16 has no more exponents than its scale gives it: the caller's scale keeps the largest
//           value under 65504, and the smallest step, 2^-24, lies 2^-39 or less under it.
//
// A workgroup holds a TM x TN tile of C in registers (WGM x WGN waves) and walks K in chunks of 128 bytes per row (64
// bf16 values, or 32 pairs).  A chunk of A and B goes global -> LDS without passing registers
// (global_load_lds_dwordx4), NBUF - 1 rounds ahead; one barrier per round.  A round is one chunk, or KG of them, one for each
// of KG groups of WGM x WGN waves whose sums are added at the end: where there are few tiles, a tile's chunks are a chain of
// latencies (barrier, LDS reads, matrix instructions on one accumulator), and more waves on it hide them.  An LDS row is
// eight 16-byte pieces; piece p of row r lies in slot p ^ (r / 2 & 7): sixteen lanes that read the same piece of sixteen
// consecutive rows, two rows to a sweep of the 64 banks, touch every bank once (with p ^ (r & 7) half of the LDS cycles were
// conflicts).  The DMA writes LDS in lane order: the exchange of the slots is in the global
// address each lane reads.
#ifndef ODAMD_GEMM_H
#define ODAMD_GEMM_H

typedef __attribute__((ext_vector_type(8))) _Float16 f16x8_t;
typedef __attribute__((ext_vector_type(8))) __bf16 bf16v8_t;
typedef __attribute__((ext_vector_type(4))) uint32_t u32x4;

// 16 bytes of zeros: the source of pieces past the end of K
__device__ __attribute__((aligned(16))) const unsigned char g_gemm_zero[16] = {};

__device__ __forceinline__ void gemm_dma16(const char* g, char* l) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)g,
                                     (__attribute__((address_space(3))) void*)l, 16, 0, 0);
}

// Accesses to LDS stay on their side of it, in the compiler's order too.
__device__ __forceinline__ void gemm_barrier() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// Blocks that run on one XCD (block index modulo 8) take neighbouring tiles: they share operand rows in that XCD's L2.
__device__ __forceinline__ int gemm_xcd_remap(int bid, int n) {
    const int q = n >> 3, r = n & 7, xcd = bid & 7, slot = bid >> 3;
    return (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + slot;
}

// The same in stretches of 128 tiles, 16 per XCD: where tiles differ in length, every XCD gets its share of the long ones.
__device__ __forceinline__ int gemm_xcd_stretch(int bid, int n) {
    const int from = bid & ~127, len = min(128, n - from);
    return from + gemm_xcd_remap(bid - from, len);
}

// Tile `t` of an mt x nt grid, walked in bands of 8 tile rows: the tiles in flight share 8 row blocks of A and few of B.
__device__ __forceinline__ void gemm_tile_at(int t, int mt, int nt, int& ti, int& tj) {
    const int band = t / (8 * nt), left = t - band * 8 * nt;
    const int rows = min(8, mt - band * 8);
    tj = left / rows;
    ti = band * 8 + left - tj * rows;
}

// Tile `t` of the upper triangle (ti <= tj) of an nt x nt grid, column by column.
__device__ __forceinline__ void gemm_triangle_at(int t, int& ti, int& tj) {
    int j = (int)((sqrtf(8.0f * (float)t + 1.0f) - 1.0f) * 0.5f);
    while ((j + 1) * (j + 2) / 2 <= t) ++j;
    while (j * (j + 1) / 2 > t) --j;
    tj = j;
    ti = t - j * (j + 1) / 2;
}

// 16-byte accesses at addresses that are only aligned to the element (global memory takes them)
typedef f32x4_t f32x4_any __attribute__((aligned(4)));
typedef u32x4 u32x4_any __attribute__((aligned(2)));

struct GemmOperand {
    const char* p;     // row 0 of the operand
    long long ld;      // bytes per row, a multiple of 16
    int rows;          // rows past the last one are read as the last one; their results are not stored
    int cols = 0;      // reduction along the rows: values per row (rows past the last one are read as zeros, columns past
                       // the last as the last eight; a row's memory holds a multiple of eight)
};

// Eight values of K, four rows each, of the column this lane's read returns
typedef short gemm_s16x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ u32x4 gemm_read_tr(const char* first, const char* second) {
    typedef __attribute__((address_space(3))) gemm_s16x4* lds_ptr;
    const gemm_s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)first);
    const gemm_s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)second);
    const uint2 u = __builtin_bit_cast(uint2, a), v = __builtin_bit_cast(uint2, b);
    return u32x4{u.x, u.y, v.x, v.y};
}
// By how many 32-byte units row k of a chunk with rows of `width` values is turned
template <int WIDTH> __device__ __forceinline__ int gemm_turn(int k) { return WIDTH >= 128 ? (k & 3) * 2 : (k >> 1 & 1) * 2; }

template <bool F16>
__device__ __forceinline__ f32x16_t gemm_mma(u32x4 a, u32x4 b, f32x16_t c) {
    if constexpr (F16)
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16v8_t, a), __builtin_bit_cast(bf16v8_t, b), c, 0, 0, 0);
}

template <int PL_, bool F16_, int TM_, int TN_, int WGM_, int WGN_, int KG_, int NBUF_>
struct GemmTile {
    static constexpr int PL = PL_, TM = TM_, TN = TN_, WGM = WGM_, WGN = WGN_, KG = KG_, NBUF = NBUF_;
    static constexpr bool F16 = F16_;
    static constexpr int NW = WGM * WGN, THREADS = 64 * NW * KG;
    static constexpr int WTM = TM / WGM, WTN = TN / WGN, FM = WTM / 32, FN = WTN / 32;
    static constexpr int BK = PL == 1 ? 64 : 32;                    // values of K per chunk
    static constexpr int BUF = (TM + TN) * 128;                     // bytes of one LDS buffer
    static constexpr int SLAB_LD = WTN + 4;                         // floats per row of a wave's epilogue slab
    static constexpr int SLAB = 32 * SLAB_LD * 4;
    static constexpr int RING = NBUF * KG * BUF;                    // buffer of round i, group g: (i % NBUF) * KG + g
    static constexpr int LDS = RING > NW * SLAB ? RING : NW * SLAB;
    // Pairs work long enough on a fragment to hide the next one's read from registers; bf16 products gain nothing from it
    // (25600 x 4096 x 1024 in 256 x 256: 243 us without, 252 with; pairs, 8192 x 1024 x 2304 in 128 x 128: 105 and 91 us), and a
    // 256 x 256 tile has no registers for it (it spills, and the optimizer step's last product takes 1059 instead of 940 us).
    static constexpr bool PIPE = PL == 2 && KG == 1 && NBUF == 2 && FM * FN <= 4;
    static constexpr int NI = (TM + TN) / 8 / NW;                   // DMA instructions per wave and chunk
    static_assert((TM + TN) % (8 * NW) == 0 && TM % 8 == 0, "whole DMA instructions");
    static_assert((KG - 1) * NW * FM * FN * 4096 <= RING, "the other groups' sums pass through the ring");
    static_assert(NBUF >= 2 && NBUF <= 3 && LDS <= 160 * 1024, "LDS of a compute unit");

    f32x16_t acc[FM][FN];

    // Chunks [c0, c1) of K into acc.  k_len: values of K (PL = 1: a multiple of 8, pieces past it are read as zeros; PL = 2:
    // the rows are padded to whole chunks).  TA, TB: A, B lie with the reduction along their rows.
    template <bool TA = false, bool TB = false>
    __device__ __forceinline__ void run(const GemmOperand& a, const GemmOperand& b, int m0, int n0, int c0, int c1, int k_len,
                                        char* lds) {
        static_assert(PL == 1 || (!TA && !TB), "pairs lie along the reduction");
        const int lane = threadIdx.x & 63, any = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), group = any / NW, wave = any % NW;
        const int wm = wave / WGN, wn = wave % WGN, r = lane & 31, h = lane >> 5;
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
            for (int j = 0; j < FN; ++j)
#pragma unroll
                for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.0f;

        // DMA instruction j of this wave brings 1 KiB of A (the first TM / 8 instructions) or of B
        const char* src[NI];
        int row[NI];                                                // reduction along the rows: this lane's row within a chunk
        // row t * 8 + lane / 8 of the chunk; t is even or odd as the wave is
        static_assert(NW % 2 == 0 && TM % 16 == 0, "a wave's instructions are all even or all odd");
        const int piece = (lane & 7) ^ ((wave & 1) * 4 + (lane >> 4));
        const auto along = [&](const GemmOperand& o, int first, int t) {
            return o.p + (long long)min(first + t * 8 + (lane >> 3), o.rows - 1) * o.ld + piece * 16;
        };
        const auto across = [&](auto width, const GemmOperand& o, int first, int t, int& k) {
            constexpr int W = width.value, SLOTS = W / 8;           // 16-byte slots per row
            k = t * (64 / SLOTS) + lane / SLOTS;
            const int slot = lane % SLOTS, col = first + ((((slot >> 1) ^ gemm_turn<W>(k)) << 1) | (slot & 1)) * 8;
            return o.p + (long long)k * o.ld + column_at(col, o.cols);
        };
#pragma unroll
        for (int j = 0; j < NI; ++j) {
            const int t = wave + j * NW;                            // wave uniform
            row[j] = 0;
            if (t * 8 < TM) {
                if constexpr (TA) src[j] = across(std::integral_constant<int, TM>{}, a, m0, t, row[j]);
                else src[j] = along(a, m0, t);
            } else {
                if constexpr (TB) src[j] = across(std::integral_constant<int, TN>{}, b, n0, t - TM / 8, row[j]);
                else src[j] = along(b, n0, t - TM / 8);
            }
        }
        // Round i of this group: chunk c0 + i KG + group; past the last chunk zeros, so that the groups stay in step
        auto issue = [&](int i) {
            const int c = c0 + i * KG + group;
            char* buf = lds + (i % NBUF * KG + group) * BUF;
            const long long at = (long long)c * 128;
            const long long at_a = TA ? c * 64LL * a.ld : at, at_b = TB ? c * 64LL * b.ld : at;
            const int rows_a = TA ? a.rows : 0x7fffffff, rows_b = TB ? b.rows : 0x7fffffff;
            if ((KG == 1 || c < c1) && (PL == 2 || ((c + 1) * BK <= k_len && (c + 1) * BK <= rows_a && (c + 1) * BK <= rows_b))) {
#pragma unroll
                for (int j = 0; j < NI; ++j)
                    gemm_dma16(src[j] + ((wave + j * NW) * 8 < TM ? at_a : at_b), buf + (wave + j * NW) * 1024);
            } else {
#pragma unroll
                for (int j = 0; j < NI; ++j) {
                    const bool is_a = (wave + j * NW) * 8 < TM, turned = is_a ? TA : TB;
                    const bool in = (KG == 1 || c < c1) && (PL == 2 || (turned ? c * BK + row[j] < (is_a ? rows_a : rows_b) : c * BK + piece * 8 < k_len));
                    gemm_dma16(in ? src[j] + (is_a ? at_a : at_b) : (const char*)g_gemm_zero, buf + (wave + j * NW) * 1024);
                }
            }
        };
        const int rounds = (c1 - c0 + KG - 1) / KG;
        const int a_off = (wm * WTM + r) * 128, b_off = TM * 128 + (wn * WTN + r) * 128, sw = r >> 1 & 7;
        // transposing reads: lane i of sixteen addresses four columns of row i / 4; lanes 32 on take the next eight rows of K
        const int tr_row = h * 8 + (lane >> 2 & 3), tr_unit = lane >> 4 & 1, tr_at = (lane & 3) * 8;
        const auto turned = [&](auto width, const char* base, int col, int s) {
            constexpr int W = width.value;
            const int unit = (col / 16 + tr_unit) ^ gemm_turn<W>(tr_row);
            const char* at = base + (s * 16 + tr_row) * (W * 2) + unit * 32 + tr_at;
            return gemm_read_tr(at, at + 4 * W * 2);
        };
        constexpr int STEPS = BK / 16, SUMS = PL == 1 ? 1 : 3;      // steps of a chunk, matrix instructions per product
        u32x4 fa[PIPE ? 2 : 1][PL][FM], fb[PIPE ? 2 : 1][PL][FN];
        const auto read = [&](const char* buf, int s, int to) {     // the fragments of step s
#pragma unroll
            for (int q = 0; q < PL; ++q) {
                const int slot = ((4 * q + 2 * s + h) ^ sw) * 16;
#pragma unroll
                for (int x = 0; x < FM; ++x) {
                    if constexpr (TA) fa[to][q][x] = turned(std::integral_constant<int, TM>{}, buf, wm * WTM + x * 32, s);
                    else fa[to][q][x] = *(const u32x4*)(buf + a_off + x * 4096 + slot);
                }
#pragma unroll
                for (int y = 0; y < FN; ++y) {
                    if constexpr (TB) fb[to][q][y] = turned(std::integral_constant<int, TN>{}, buf + TM * 128, wn * WTN + y * 32, s);
                    else fb[to][q][y] = *(const u32x4*)(buf + b_off + y * 4096 + slot);
                }
            }
        };
        // B is the instruction's row operand: a lane then holds one row m of C and runs of four columns n
        const auto multiply = [&](int f) {
#pragma unroll
            for (int q = 0; q < SUMS; ++q)
#pragma unroll
                for (int x = 0; x < FM; ++x)
#pragma unroll
                    for (int y = 0; y < FN; ++y)
                        acc[x][y] = gemm_mma<F16>(fb[f][q == 1 ? PL - 1 : 0][y], fa[f][q == 2 ? PL - 1 : 0][x], acc[x][y]);
        };
        if constexpr (PIPE) {
            // The fragments of the next step are read while the matrix cores work on this one's, over the end of a chunk too:
            // in a chunk's last step this wave's fragments of it are in registers and its pieces of the next chunk in LDS; behind
            // the barrier that holds for every wave, and the chunk's buffer may take the one after the next.
            issue(0);
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            gemm_barrier();
            if (rounds > 1) issue(1);
            read(lds, 0, 0);
            for (int i = 0; i < rounds; ++i) {
#pragma unroll
                for (int s = 0; s < STEPS; ++s) {
                    if (s + 1 < STEPS) {
                        read(lds + (i & 1) * BUF, s + 1, (s + 1) & 1);
                    } else {
                        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
                        gemm_barrier();
                        read(lds + (~i & 1) * BUF, 0, (s + 1) & 1); // behind the last chunk: of no use, but within LDS
                        if (i + 2 < rounds) issue(i + 2);
                    }
                    multiply(s & 1);
                    constexpr int READS = PL * (FM + FN);
#pragma unroll
                    for (int q = 0; q < READS; ++q) {               // one LDS read, then its share of the matrix instructions
                        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
                        __builtin_amdgcn_sched_group_barrier(0x008, SUMS * FM * FN / READS, 0);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
        } else {
#pragma unroll
            for (int q = 0; q < NBUF - 1; ++q)
                if (q < rounds) issue(q);
            for (int i = 0; i < rounds; ++i) {
                // this wave's pieces of round i have landed (those of up to NBUF - 2 later rounds may still be on their way)
                // and its reads of round i - 1 have returned; behind the barrier that holds for every wave
                const int ahead = min(NBUF - 2, rounds - 1 - i);
                if (NBUF > 2 && ahead == 1) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(NBUF > 2 ? NI : 0) : "memory");
                else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
                gemm_barrier();
                if (i + NBUF - 1 < rounds) issue(i + NBUF - 1);
#pragma unroll
                for (int s = 0; s < STEPS; ++s) {
                    read(lds + (i % NBUF * KG + group) * BUF, s, 0);
                    multiply(0);
                }
            }
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        gemm_barrier();                               // every wave has read its last fragments: the ring is free
        if constexpr (KG > 1) {
            // the other groups leave their sums in LDS, the first adds them in order
            const auto place = [&](int g, int x, int y, int q) {
                return (f32x4_t*)(lds + ((((g - 1) * NW + wave) * FM * FN + x * FN + y) * 4 + q) * 1024 + lane * 16);
            };
            if (group > 0)
#pragma unroll
                for (int x = 0; x < FM; ++x)
#pragma unroll
                    for (int y = 0; y < FN; ++y)
#pragma unroll
                        for (int q = 0; q < 4; ++q)
                            *place(group, x, y, q) = f32x4_t{acc[x][y][4 * q], acc[x][y][4 * q + 1], acc[x][y][4 * q + 2], acc[x][y][4 * q + 3]};
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            gemm_barrier();
            if (group == 0)
#pragma unroll
                for (int g = 1; g < KG; ++g)
#pragma unroll
                    for (int x = 0; x < FM; ++x)
#pragma unroll
                        for (int y = 0; y < FN; ++y)
#pragma unroll
                            for (int q = 0; q < 4; ++q) {
                                const f32x4_t u = *place(g, x, y, q);
                                acc[x][y][4 * q] += u[0]; acc[x][y][4 * q + 1] += u[1]; acc[x][y][4 * q + 2] += u[2]; acc[x][y][4 * q + 3] += u[3];
                            }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            gemm_barrier();                           // read before the slabs take the place
        }
    }

    // First of the eight columns this lane hands out by rows
    __device__ __forceinline__ int row_column() const {
        return (threadIdx.x >> 6) % NW % WGN * WTN + (threadIdx.x & 63) % (WTN / 8) * 8;
    }

    // Hands the tile out in runs of eight, m and n relative to the tile: rows(m, n, v[8], x) for C[m][n .. n+7] and
    // cols(m, n, v[8], x) for C[m .. m+7][n], x = what load(m, n) of that kind gave before.  Every wave passes 32 rows at a time
    // through a slab of LDS of its own; BATCH of its loads are under way together, the first of them while the slab is
    // written (a load that waits for the store before it costs the epilogue a memory latency for every run).
    // SYM: the tile lies on the diagonal of a symmetric result; runs of eight that cross it have their lower part from the upper one.
    template <bool ROWS, bool COLS, int BATCH, bool SYM = false, typename LR, typename FR, typename LC, typename FC>
    __device__ __forceinline__ void hand_out(char* lds, LR&& load_row, FR&& rows, LC&& load_col, FC&& cols) {
        const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        if (KG > 1 && wave >= NW) return;                           // the first group holds the sums
        const int wm = wave / WGN * WTM, wn = wave % WGN * WTN, r = lane & 31, h = lane >> 5;
        float* slab = (float*)(lds + wave * SLAB);
        constexpr int LPR = WTN / 8, RPP = 64 / LPR;                // lanes per row, rows per pass
        constexpr int PASSES = WTN / 16, B = BATCH < PASSES ? BATCH : PASSES;
        static_assert(PASSES % B == 0, "whole batches");
        const auto row_at = [&](int i, int p) { return wm + i * 32 + p * RPP + lane / LPR; };
        const int row_n = wn + lane % LPR * 8;
        const auto col_m = [&](int i, int p) { return wm + i * 32 + (p * 64 + lane) / WTN * 8; };
        const auto col_n = [&](int p) { return wn + (p * 64 + lane) % WTN; };
#pragma unroll
        for (int i = 0; i < FM; ++i) {
            decltype(load_row(0, 0)) xr[B];
            decltype(load_col(0, 0)) xc[B];
            const auto fetch_rows = [&](int p) {
#pragma unroll
                for (int q = 0; q < B; ++q) xr[q] = load_row(row_at(i, p + q), row_n);
            };
            const auto fetch_cols = [&](int p) {
#pragma unroll
                for (int q = 0; q < B; ++q) xc[q] = load_col(col_m(i, p + q), col_n(p + q));
            };
            if constexpr (ROWS) fetch_rows(0);
            else fetch_cols(0);
#pragma unroll
            for (int j = 0; j < FN; ++j)
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    *(f32x4_t*)(slab + r * SLAB_LD + j * 32 + q * 8 + h * 4) =
                        f32x4_t{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            if constexpr (ROWS) {
#pragma unroll
                for (int p = 0; p < PASSES; ++p) {
                    if (p % B == 0 && p > 0) fetch_rows(p);
                    const float* at = slab + (p * RPP + lane / LPR) * SLAB_LD + lane % LPR * 8;
                    const f32x4_t u = *(const f32x4_t*)at, w = *(const f32x4_t*)(at + 4);
                    float v[8] = {u[0], u[1], u[2], u[3], w[0], w[1], w[2], w[3]};
                    if constexpr (SYM) {
                        const int m = row_at(i, p);             // the block of eight rows and columns lies in this slab
                        if (m >> 3 == row_n >> 3)
#pragma unroll
                            for (int e = 0; e < 8; ++e)
                                if (row_n + e < m) v[e] = slab[(row_n + e - wm - i * 32) * SLAB_LD + m - wn];
                    }
                    rows(row_at(i, p), row_n, v, xr[p % B]);
                }
                if constexpr (COLS) fetch_cols(0);
            }
            if constexpr (COLS) {
#pragma unroll
                for (int p = 0; p < PASSES; ++p) {
                    if (p % B == 0 && p > 0) fetch_cols(p);
                    const int n = (p * 64 + lane) % WTN, g = (p * 64 + lane) / WTN;
                    float v[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[e] = slab[(g * 8 + e) * SLAB_LD + n];
                    cols(col_m(i, p), col_n(p), v, xc[p % B]);
                }
            }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        }
    }
};
struct GemmNothing {};

// v (already scaled) as a pair of fp16 numbers.  A value that is no number, or beyond fp16, keeps that in hi alone.
__device__ __forceinline__ void split_f16(float v, _Float16& hi, _Float16& lo) {
    hi = (_Float16)v;
    const float rest = v - (float)hi;
    lo = fabsf(v) < 65504.0f ? (_Float16)rest : (_Float16)0.0f;
}
// Eight of them, from a multiple of eight on.
__device__ __forceinline__ void store_split8(char* hi_at, const float v[8], float scale) {
    f16x8_t hi, lo;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        _Float16 a, b;
        split_f16(v[e] * scale, a, b);
        hi[e] = a;
        lo[e] = b;
    }
    *(f16x8_t*)hi_at = hi;
    *(f16x8_t*)(hi_at + 64) = lo;
}
// ---- host ------------------------------------------------------------------------------------------------------------
// A launch has fewer than 2^32 threads.
inline bool gemm_grid_ok(long long blocks, int threads) { return blocks * threads <= 0xffffffffLL; }

// ---- which tile ------------------------------------------------------------------------------------------------
// Time of a 128-byte chunk of all tiles of a compute unit, in us, by how many tiles a unit has to run (`rounds`; measured
// with pairs at 4096^3, 8192 x 1024 x 2304 and below).  The larger tile wins per product, the smaller one spreads a small
// product over all 256 units: 4096 x 4096 x 4096 takes 353 / 367 / 512 us in 256 / 128 / 64, 2048 x 1024 x 2048
// - / 44 / 34 us.  bf16 chunks take two thirds of the time.
inline double gemm_chunk_us(int tile, double rounds, bool pairs) {
    if (tile == 256) return 2.75 * (rounds > 1.0 ? rounds : 1.0);
    if (tile == 128) {
        if (rounds <= 1.0) return 0.75;
        if (!pairs) return 0.87 * rounds;
        return rounds <= 2.0 ? 0.75 + 0.51 * (rounds - 1.0) : 0.75 * rounds;      // two tiles of a unit run beside each other
    }
    if (rounds <= 1.0) return 0.3;                                               // two wave groups on a tile
    return 0.25 * rounds > 0.49 ? 0.25 * rounds : 0.49;                          // one: 0.49 alone, and up to two in that time
}
struct GemmLoad { double tiles = 0, chunks = 0, longest = 0; int kinds = 0; };   // chunks: summed over all tiles
inline void gemm_load_add(GemmLoad& l, double tiles, double chunks) {
    l.tiles += tiles;
    if (l.kinds == 0 || chunks != l.longest) ++l.kinds;
    l.chunks += tiles * chunks;
    l.longest = chunks > l.longest ? chunks : l.longest;
}
// `bytes`: what the epilogue moves per element of C.  A unit's share of the memory rate is 20 GB/s; some of it runs beside another
// tile's products, a 256 x 256 tile's least.
inline double gemm_time_us(int tile, const GemmLoad& l, bool pairs, double bytes) {
    double rounds = l.chunks / (256.0 * l.longest), rest = 0.0;
    if (l.kinds == 1) {
        // tiles of one length run in whole rounds; where several share a unit, the last round is not quite one (528 tiles of
        // 64 x 64 on 256 units: 2.7 rounds)
        const double whole = (double)(((long long)l.tiles + 255) / 256);
        rounds = tile < 256 && whole > 1.0 && whole - 0.35 > rounds ? whole - 0.35 : whole;
    } else {
        // of several lengths they pack as they come: a quarter of the longest is left over at the end
        rest = 0.25 * l.longest * (tile == 256 ? 2.75 : tile == 128 ? 0.75 : 0.25);
    }
    const double each = l.tiles / 256.0 > 1.0 ? l.kinds == 1 ? rounds : l.tiles / 256.0 : 1.0;
    return (l.longest * gemm_chunk_us(tile, rounds, pairs) + rest) * (pairs ? 1.0 : 2.0 / 3.0)
           + each * tile * tile * bytes / 20.0e3 * (tile == 256 ? 0.9 : 0.8);
}

#endif
