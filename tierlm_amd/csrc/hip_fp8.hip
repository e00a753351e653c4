/* hip_fp8.hip - 8-bit floating point with a scale per block of 128: packing,
 * the activation quantiser and the matrix product (the reference's FP8 weight
 * format, src/lib/tlm_quant.c:761-776, with its activations in 8 bits too). */
#include "tlm_hip_fp8.h"
#include <type_traits>

namespace {

/* ---- packing: a thread per 16-byte piece, then one per scale ---------------- */
__global__ __launch_bounds__(256) void k_fp8_pack(const uint8_t *__restrict__ W, size_t row_bytes, int64_t rows,
                                                  int64_t n, int nb, int64_t pieces, int vec,
                                                  const float *__restrict__ scale, int64_t stride, int64_t scales,
                                                  uint8_t *__restrict__ dst) {
    const int64_t p = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (p >= pieces) {
        const int64_t i = p - pieces;
        if (i < scales) ((float *)(dst + pieces * 16))[i] = scale[i / nb * stride + i % nb];
        return;
    }
    const int64_t unit = p >> 7;
    const int h = (int)(p >> 6) & 1, l = (int)p & 63;
    const int64_t row = unit / nb * TILE_ROWS + (l & 15);
    const int64_t k0 = unit % nb * FP8_BLOCK + 64 * h + 16 * (l >> 4);
    u32x4 v = {0, 0, 0, 0};
    if (row < rows) {
        const uint8_t *src = W + (size_t)row * row_bytes;
        if (vec && k0 + 16 <= n) {
            v = *(const u32x4 *)(src + k0);
        } else {
#pragma unroll
            for (int j = 0; j < 16; j++)
                if (k0 + j < n) v[j >> 2] |= (uint32_t)src[k0 + j] << (8 * (j & 3));
        }
    }
    *(u32x4 *)(dst + p * 16) = v;
}

/* ---- activation quantiser --------------------------------------------------
 * 16 lanes per block of 128 values, 8 values a lane.  scale = 2^e, e the least
 * integer >= -126 with amax <= 448 * 2^e: dividing by it is exact, so the one
 * rounding is the code's, and a floating code loses no relative precision by it. */
template <class T> __device__ __forceinline__ float ld_f32(const T *p);
template <> __device__ __forceinline__ float ld_f32<float>(const float *p) { return *p; }
template <> __device__ __forceinline__ float ld_f32<_Float16>(const _Float16 *p) { return (float)*p; }
template <> __device__ __forceinline__ float ld_f32<__bf16>(const __bf16 *p) {
    return __uint_as_float((uint32_t) * (const uint16_t *)p << 16);
}

/* 8 values from p on, `left` of them in the row; vector loads at any alignment of the
 * elements (this target's memory pipe takes them) */
template <class T> __device__ __forceinline__ void ld8(float (&v)[8], const T *p, int left) {
    typedef T T8 __attribute__((ext_vector_type(8), aligned(sizeof(T))));
    if (left >= 8) {
        const T8 q = *(const T8 *)p;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const T e = q[j];
            v[j] = ld_f32(&e);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = j < left ? ld_f32(p + j) : 0.0f;
    }
}

/* U blocks a lane group, their loads in flight together */
template <class T, int U>
__global__ __launch_bounds__(256) void k_fp8_quant(const T *__restrict__ x, int64_t xstride, int n, int nb,
                                                   int blocks, uint8_t *__restrict__ codes,
                                                   float *__restrict__ scale) {
    const int sub = threadIdx.x & 15, blk0 = blockIdx.x * 16 * U + (threadIdx.x >> 4);
    float v[U][8];
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int blk = blk0 + 16 * u, t = blk / nb, k0 = (blk - t * nb) * FP8_BLOCK + 8 * sub;
        ld8<T>(v[u], x + t * xstride + k0, blk < blocks ? n - k0 : 0);
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int blk = blk0 + 16 * u;
        uint32_t am = 0;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const uint32_t b = __float_as_uint(v[u][j]) & 0x7FFFFFFFu;   /* order of |v|; NaN and infinity on top */
            am = b > am ? b : am;
        }
        am = group_max_u32<16>(am);
        /* amax = m 2^x, 1 <= m < 2: e = x - 8 for m <= 1.75, else x - 7 */
        const int ex = (int)(am >> 23) - 127;
        int e = (am & 0x7FFFFFu) <= 0x600000u ? ex - 8 : ex - 7;
        e = e < -126 ? -126 : e;
        const bool bad = am >= 0x7F800000u;
        const float inv = __uint_as_float((uint32_t)(127 - e) << 23);
        int c0 = 0, c1 = 0;
        c0 = __builtin_amdgcn_cvt_pk_fp8_f32(v[u][0] * inv, v[u][1] * inv, c0, false);
        c0 = __builtin_amdgcn_cvt_pk_fp8_f32(v[u][2] * inv, v[u][3] * inv, c0, true);
        c1 = __builtin_amdgcn_cvt_pk_fp8_f32(v[u][4] * inv, v[u][5] * inv, c1, false);
        c1 = __builtin_amdgcn_cvt_pk_fp8_f32(v[u][6] * inv, v[u][7] * inv, c1, true);
        if (blk < blocks) {
            const u32x2 o = {bad ? 0u : (uint32_t)c0, bad ? 0u : (uint32_t)c1};
            *(u32x2 *)(codes + (size_t)blk * FP8_BLOCK + 8 * sub) = o;
            if (sub == 0)
                scale[blk] = bad ? __uint_as_float(0x7FC00000u) : am ? __uint_as_float((uint32_t)(127 + e) << 23) : 0.0f;
        }
    }
}

template <class T>
void launch_quant(const void *x, int64_t xstride, int64_t n, int nb, int64_t blocks, void *codes, float *scale,
                  hipStream_t s) {
    /* four blocks a lane group once that still leaves every compute unit several groups */
    const int u = blocks >= 65536 ? 4 : 1;
    const dim3 grid((unsigned)((blocks + 16 * u - 1) / (16 * u)));
    if (u == 4)
        hipLaunchKernelGGL((k_fp8_quant<T, 4>), grid, dim3(256), 0, s, (const T *)x, xstride, (int)n, nb, (int)blocks,
                           (uint8_t *)codes, scale);
    else
        hipLaunchKernelGGL((k_fp8_quant<T, 1>), grid, dim3(256), 0, s, (const T *)x, xstride, (int)n, nb, (int)blocks,
                           (uint8_t *)codes, scale);
}

/* ---- product ----------------------------------------------------------------
 * Y[t][r] = sum over blocks b of sa[t][b] sw[r / 128][b] (codes of t . codes of r):
 * products and their sums of 128 in the matrix cores' float accumulators, then
 * one fma per block.  One scale's power of two goes in with its codes (fp8_scale). */
struct MmArgs {
    const uint8_t *W;
    const float *sw;
    const uint8_t *x;
    const float *sa;
    void *y;
    int64_t rows, ystride, T;
    int nb, dt;
};

/* four rows of one token's result, in the type of Y; one store at any alignment of the elements (1323 tokens
 * of 6997 x 1480, float results, one element a store: 53 us, now 39.5) */
typedef f32x4 f32x4any __attribute__((aligned(4)));
typedef u16x4 u16x4any __attribute__((aligned(2)));
__device__ __forceinline__ void store4(const MmArgs &a, int64_t t, int64_t r, f32x4 v) {
    if (a.dt == DT_F32) {
        float *y = (float *)a.y + t * a.ystride + r;
        if (r + 3 < a.rows) *(f32x4any *)y = v;
        else
            for (int q = 0; q < 4; q++)
                if (r + q < a.rows) y[q] = v[q];
        return;
    }
    u16x4 o;
#pragma unroll
    for (int q = 0; q < 4; q++) {
        const _Float16 h = (_Float16)v[q];
        const __bf16 e = (__bf16)v[q];
        o[q] = a.dt == DT_F16 ? __builtin_bit_cast(uint16_t, h) : __builtin_bit_cast(uint16_t, e);
    }
    uint16_t *y = (uint16_t *)a.y + t * a.ystride + r;
    if (r + 3 < a.rows) *(u16x4any *)y = o;
    else
        for (int q = 0; q < 4; q++)
            if (r + q < a.rows) y[q] = o[q];
}

/* ---- product, up to a few hundred tokens -----------------------------------------
 * A group takes RT row tiles and TT token tiles; its KW waves share the blocks of a row, each with
 * the next block's loads under way while it computes one, and add their sums through LDS.
 *   Weights come in the order of the fragments.  Tokens come as rows of whole lines, 8 to an
 * instruction, and pass through LDS of the wave's own (no barrier) to the order of the fragments, pieces
 * at piece ^ row % 8, so that neither side meets a bank twice.  Fetched in that order straight from memory,
 * every quarter of a wave touches 16 lines for 16 bytes each, and those look-ups bound it: 64 tokens
 * of 4096 x 4096 14.6 us, 512 x 16384 46; now 8.2 and 10.
 *   Codes go to the matrix cores as bfloat16 (exact), whose instructions sum in full floats where the 8-bit
 * ones do not; the weights' bytes or the tokens' way through L2 bound either.
 *   One token: 151936 x 2048 in 46-52 us (6.0-6.8 TB/s), 4096 x 4096 4.9, 2048 x 2048 3.5. */
template <int KW, int RT, int TT>
__global__ __launch_bounds__(64 * KW) void k_fp8_rows(MmArgs a) {
    constexpr int XB = TT * FP8_UNIT;   /* a block of the group's tokens */
    constexpr int PW = XB > RT * TT * 1024 ? XB : RT * TT * 1024;
    __shared__ __align__(16) uint8_t s_x[KW * PW];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4,
              c = lane & 15;
    const int tile0 = blockIdx.x * RT, last = (int)fp8_tiles(a.rows) - 1;
    const int64_t t0 = (int64_t)blockIdx.y * TT * 16;
    const int nb = a.nb;
    const GAS uint8_t *w[RT], *x[TT][2];
    const GAS float *sw = (const GAS float *)a.sw + (size_t)(tile0 / 8) * nb, *sa[TT];
#pragma unroll
    for (int i = 0; i < RT; i++)
        w[i] = (const GAS uint8_t *)a.W + (size_t)(tile0 + i < last ? tile0 + i : last) * nb * FP8_UNIT + lane * 16;
#pragma unroll
    for (int j = 0; j < TT; j++) {
        const int64_t t = t0 + 16 * j + c < a.T ? t0 + 16 * j + c : a.T - 1;
        sa[j] = (const GAS float *)a.sa + t * nb;
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int64_t r = t0 + 16 * j + 8 * h + (lane >> 3);
            x[j][h] = (const GAS uint8_t *)a.x + (size_t)(r < a.T ? r : a.T - 1) * nb * FP8_BLOCK + 16 * (lane & 7);
        }
    }
    LAS uint8_t *sx = (LAS uint8_t *)s_x + wave * PW;
    const int at_w = (lane >> 3) * FP8_BLOCK + 16 * ((lane & 7) ^ (lane >> 3));
    const int at_r0 = c * FP8_BLOCK + 16 * (g ^ (c & 7)), at_r1 = c * FP8_BLOCK + 16 * ((4 + g) ^ (c & 7));
    f32x4 acc[RT][TT] = {};
    struct In {
        i32x4 w[RT][2], x[TT][2];
        float ws, xs[TT];
    };
    auto load = [&](In &n, int b) {
#pragma unroll
        for (int j = 0; j < TT; j++) {
            n.xs[j] = sa[j][b];
#pragma unroll
            for (int h = 0; h < 2; h++) n.x[j][h] = *(const GAS i32x4 *)(x[j][h] + b * FP8_BLOCK);
        }
#pragma unroll
        for (int i = 0; i < RT; i++)
#pragma unroll
            for (int h = 0; h < 2; h++) n.w[i][h] = *(const GAS i32x4 *)(w[i] + (size_t)b * FP8_UNIT + 1024 * h);
        n.ws = sw[b];
    };
    auto compute = [&](const In &n) {
#pragma unroll
        for (int j = 0; j < TT; j++)
#pragma unroll
            for (int h = 0; h < 2; h++) *(LAS i32x4 *)(sx + j * FP8_UNIT + h * 1024 + at_w) = n.x[j][h];
        bf16x8 wf[RT][4];
#pragma unroll
        for (int i = 0; i < RT; i++)
#pragma unroll
            for (int k = 0; k < 4; k++) wf[i][k] = fp8_to_bf16(n.w[i][k >> 1][2 * (k & 1)], n.w[i][k >> 1][2 * (k & 1) + 1]);
#pragma unroll
        for (int j = 0; j < TT; j++) {
            const i32x4 q0 = *(const LAS i32x4 *)(sx + j * FP8_UNIT + at_r0), q1 = *(const LAS i32x4 *)(sx + j * FP8_UNIT + at_r1);
            /* the tokens' scale goes in with their codes: the rows' comes by a scalar load, whose wait would be one
             * for the LDS reads too (64 tokens of 512 x 16384: 10.7 us for 9.6) */
            const Fp8Scale xs = fp8_scale(n.xs[j]);
            const bf16x8 xf[4] = {fp8_to_bf16(q0[0], q0[1], xs.pow2), fp8_to_bf16(q0[2], q0[3], xs.pow2),
                                  fp8_to_bf16(q1[0], q1[1], xs.pow2), fp8_to_bf16(q1[2], q1[3], xs.pow2)};
            f32x4 p[RT] = {};
#pragma unroll
            for (int k = 0; k < 4; k++)
#pragma unroll
                for (int i = 0; i < RT; i++) p[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wf[i][k], xf[k], p[i], 0, 0, 0);
            const float sc = n.ws * xs.rest;
#pragma unroll
            for (int i = 0; i < RT; i++)
#pragma unroll
                for (int v = 0; v < 4; v++) acc[i][j][v] = fmaf(p[i][v], sc, acc[i][j][v]);
        }
    };
    In cur;
    int b = wave;
    if (b < nb) {
        load(cur, b);
        for (; b + KW < nb; b += KW) {
            In nxt;
            load(nxt, b + KW);
            compute(cur);
            cur = nxt;
        }
        compute(cur);
    }
#pragma unroll
    for (int i = 0; i < RT; i++)
#pragma unroll
        for (int j = 0; j < TT; j++) *(LAS f32x4 *)(sx + (i * TT + j) * 1024 + lane * 16) = acc[i][j];
    __syncthreads();
    for (int o = threadIdx.x; o < RT * TT * 64; o += 64 * KW) {
        const int m = o >> 6, i = m / TT, j = m % TT, l = o & 63;
        const LAS uint8_t *from = (const LAS uint8_t *)s_x + m * 1024 + l * 16;
        f32x4 s = *(const LAS f32x4 *)from;
#pragma unroll
        for (int q = 1; q < KW; q++) s += *(const LAS f32x4 *)(from + q * PW);
        const int64_t t = t0 + 16 * j + (l & 15), r = (int64_t)(tile0 + i) * 16 + 4 * (l >> 4);
        if (t < a.T && r < a.rows) store4(a, t, r, s);
    }
}

/* ---- product, tiles through LDS -------------------------------------------------
 * A group of WM x WN waves computes WM TM row tiles by WN TN token tiles, a wave TM x TN of
 * them.  A block of 128 values is one stage: direct loads bring its units into LDS, S stages in
 * all.  A stage's sums of 128 products come out of the matrix instructions and are folded into
 * the accumulators with both scales, 4 fmas a lane beside four 16 x 16 x 32 instructions (which
 * take as long as 16 of them, so the fold is free as long as the two overlap).
 *   Weights are in the order of the fragments already.  Tokens come as rows of 128 bytes, whole
 * cache lines, 8 to an instruction; the lanes fetch a row's eight pieces in the order
 * (piece ^ row % 8), so that the 16 lanes that later read one piece of 16 rows meet all
 * banks.
 *   Codes go to the matrix cores as bfloat16 (exact), whose sums are full floats.  The 8-bit
 * instructions run at twice the rate, but align the products of 8 neighbouring values to the
 * largest of them and cut what lies below 2^-13 of its power of two (1.5e-5 of a result on normal data,
 * 5e-5 where values spread over decades): no result's sums may have fewer than a float's bits,
 * a 16-bit result's no more than a float one's.
 *   4096 tokens, 8192 x 4096: 245-258 us, 1.1 PFLOP/s; the 16-bit instructions bound it. */
/* waves a SIMD that the stages' LDS leaves room for, up to two */
constexpr int tile_waves(int s, int waves, int units) { return 2 * s * (units * FP8_UNIT + 256 * waves) <= 160 * 1024 ? 2 : 1; }
template <int S, int WM, int WN, int TM, int TN>
__global__ __launch_bounds__(64 * WM * WN)
    __attribute__((amdgpu_waves_per_eu(tile_waves(S, WM *WN, WM *TM + WN * TN))))
void k_fp8_tile(MmArgs a, int mtiles, int ntiles) {
    constexpr int NWV = WM * WN, MT = WM * TM, NT = WN * TN, UNITS = MT + NT, PER = UNITS / NWV;
    static_assert(MT % NWV == 0 && NT % NWV == 0 && 8 % TM == 0 && (MT % 8 == 0 || 8 % MT == 0), "units are dealt evenly; a wave's rows share a scale");
    /* stages as variables of their own: the compiler then sees that reads of one do not wait
     * for loads into another */
    constexpr int SB = UNITS * FP8_UNIT;
    constexpr int SB4 = S > 2 ? SB : 16;
    __shared__ __align__(16) uint8_t s0[SB], s1[SB], s2[SB4], s3[SB4];
    /* scales: a wave brings those of its share of the tokens, then the row blocks' */
    constexpr int TPW = NT * 16 / NWV;
    constexpr int F = NWV * 64, F4 = S > 2 ? F : 1;
    __shared__ float f0[F], f1[F], f2[F4], f3[F4];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave / WN, wn = wave % WN, g = lane >> 4, c = lane & 15;
    int bm, bn;
    {   /* groups go to the eight XCDs in turn: give each XCD a run of tiles that share rows and tokens */
        const int total = mtiles * ntiles, id = blockIdx.x, xcd = id & 7, at = id >> 3;
        const int q = total >> 3, r = total & 7;
        const int t = xcd * q + (xcd < r ? xcd : r) + at;
        constexpr int BAND = 8;   /* row tiles of a band */
        const int band = t / (BAND * ntiles), in = t % (BAND * ntiles);
        const int width = mtiles - band * BAND < BAND ? mtiles - band * BAND : BAND;
        bm = band * BAND + in % width;
        bn = in / width;
    }
    const int tile0 = bm * MT, last = (int)fp8_tiles(a.rows) - 1;
    const int64_t t0 = (int64_t)bn * NT * 16;
    /* units wave, wave + NWV, ...: a uniform base that moves from block to block, and this lane's offset */
    const GAS uint8_t *base[PER];
    uint32_t off[PER][2];
    const int left = (int)(a.T - 1 - t0 < NT * 16 ? a.T - 1 - t0 : NT * 16);
#pragma unroll
    for (int i = 0; i < PER; i++) {
        const int u = wave + i * NWV;
        if (i * NWV < MT) {
            const int tile = tile0 + u < last ? tile0 + u : last;
            base[i] = (const GAS uint8_t *)a.W + (size_t)tile * a.nb * FP8_UNIT;
            off[i][0] = lane * 16;
            off[i][1] = lane * 16 + 1024;
        } else {
            base[i] = (const GAS uint8_t *)a.x + (size_t)t0 * a.nb * FP8_BLOCK;
            for (int h = 0; h < 2; h++) {
                const int t = (u - MT) * 16 + 8 * h + (lane >> 3);
                off[i][h] = (uint32_t)(t < left ? t : left) * (uint32_t)a.nb * FP8_BLOCK +
                            16 * ((lane & 7) ^ (lane >> 3));
            }
        }
    }
    const int st = wave * TPW + lane, sr = lane - TPW, rlast = last / 8 - tile0 / 8;
    const GAS float *ssrc = lane < TPW ? (const GAS float *)a.sa + (t0 + (st < left ? st : left)) * a.nb
                                       : (const GAS float *)a.sw + (size_t)(tile0 / 8 + (sr < rlast ? sr : rlast)) * a.nb;
    int pos = 0;   /* the block that the next load brings; past the last one it is brought again, unread */
    /* Offsets into a stage, one number each: with the parts of a sum left to the optimiser the compiler
     * loses sight of which variable is read and lets every read wait for every load. */
    int o_unit = wave * FP8_UNIT, o_scale = wave * 64;
    int o_row = wm * TM * FP8_UNIT + lane * 16;
    int o_col0 = (MT + wn * TN) * FP8_UNIT + c * FP8_BLOCK + 16 * (g ^ (c & 7));
    int o_col1 = (MT + wn * TN) * FP8_UNIT + c * FP8_BLOCK + 16 * ((4 + g) ^ (c & 7));
    int o_sa[TN], o_sw = TPW + (tile0 + wm * TM) / 8 - tile0 / 8;
#pragma unroll
    for (int j = 0; j < TN; j++) {
        const int t = (wn * TN + j) * 16;
        o_sa[j] = t / TPW * 64 + t % TPW + c;
        asm("" : "+v"(o_sa[j]));
    }
    asm("" : "+s"(o_unit), "+s"(o_scale), "+v"(o_row), "+v"(o_col0), "+v"(o_col1), "+s"(o_sw));
    auto load = [&](LAS uint8_t *s, LAS float *f) {
        const bool more = ++pos < a.nb;
#pragma unroll
        for (int i = 0; i < PER; i++) {
#pragma unroll
            for (int h = 0; h < 2; h++)
                __builtin_amdgcn_global_load_lds((const GAS void *)(base[i] + off[i][h]),
                                                 (LAS void *)(s + o_unit + i * NWV * FP8_UNIT + h * 1024), 16, 0, 0);
            base[i] += !more ? 0 : i * NWV < MT ? FP8_UNIT : FP8_BLOCK;
        }
        __builtin_amdgcn_global_load_lds((const GAS void *)ssrc, (LAS void *)(f + o_scale), 4, 0, 0);
        ssrc += more ? 1 : 0;
    };
    /* The waves meet once the next stage's loads have landed, those of the S - 2 after it may
     * still be on their way; every wave's reads of the stage before are done by then. */
    constexpr int LOADS = 2 * PER + 1;
    auto meet = [&](auto n) {
        constexpr int N = decltype(n)::value;
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | (7 << 4) | (0 << 8));   /* vmcnt N, lgkmcnt 0 */
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    auto arrive = [&]() { meet(std::integral_constant<int, LOADS * (S - 2)>{}); };
    f32x4 acc[TM][TN] = {};
    auto frag = [&](const LAS uint8_t *s, int i) {
        return fp8_join(*(const LAS i32x4 *)(s + o_row + i * FP8_UNIT), *(const LAS i32x4 *)(s + o_row + i * FP8_UNIT + 1024));
    };
    /* a fragment as the matrix instructions take it: 32 bfloat16 a lane */
    struct Frag {
        bf16x8 k[4];
    };
    auto open = [&](i32x8 q, float pow2 = 1.0f) {
        Frag f;
#pragma unroll
        for (int h = 0; h < 4; h++) f.k[h] = fp8_to_bf16(q[2 * h], q[2 * h + 1], pow2);
        return f;
    };
    auto dot = [&](const Frag &x, const Frag &y) {
        f32x4 p = {0, 0, 0, 0};
#pragma unroll
        for (int h = 0; h < 4; h++) p = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x.k[h], y.k[h], p, 0, 0, 0);
        return p;
    };
    struct Cols {
        i32x8 b[TN];
        float sc[TN], w;
    };
    auto columns = [&](Cols &k, const LAS uint8_t *s, const LAS float *f, int j) {
        k.b[j] = fp8_join(*(const LAS i32x4 *)(s + o_col0 + j * FP8_UNIT), *(const LAS i32x4 *)(s + o_col1 + j * FP8_UNIT));
        k.sc[j] = f[o_sa[j]];
        if (j == 0) k.w = f[o_sw];
    };
    /* One block: the matrix instructions of row tile i run beside the fmas of the ones before
     * (a ring of RING results) and the reads of row tile i + 1.  Once row tile TM - 1 is in
     * registers the stage is free: the waves meet, the next block's loads go out into it, and the
     * next block's columns are read from the other stage under the last instructions. */
    constexpr int RING = TN < 4 ? TN : 4;
    i32x8 av[2];
    auto compute = [&](Cols &k, Cols &kn, LAS uint8_t *s, LAS float *f, const LAS uint8_t *sn, const LAS float *fn) {
        f32x4 p[RING];
        const Fp8Scale ws = fp8_scale(k.w);
        float sc[TN];
        Frag bf[TN];
#pragma unroll
        for (int j = 0; j < TN; j++) bf[j] = open(k.b[j]);
#pragma unroll
        for (int j = 0; j < TN; j++) sc[j] = ws.rest * k.sc[j];
        auto fold = [&](int m) {
            const int i = m / TN, j = m % TN;
#pragma unroll
            for (int v = 0; v < 4; v++) acc[i][j][v] = fmaf(p[m % RING][v], sc[j], acc[i][j][v]);
        };
#pragma unroll
        for (int i = 0; i < TM; i++) {
            const Frag af = open(av[i & 1], ws.pow2);
            if (i + 1 < TM) av[(i + 1) & 1] = frag(s, i + 1);
            if (i + 1 == TM) {
                arrive();
                load(s, f);
            }
#pragma unroll
            for (int j = 0; j < TN; j++) {
                const int m = i * TN + j;
                p[m % RING] = dot(af, bf[j]);
                if (m >= RING - 1) fold(m - RING + 1);
                if (i + 1 == TM) columns(kn, sn, fn, j);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        av[TM & 1] = frag(sn, 0);
#pragma unroll
        for (int m = TM * TN - RING + 1; m < TM * TN; m++) fold(m);
        __builtin_amdgcn_sched_barrier(0);
    };
    static_assert(TM % 2 == 0 && (S == 2 || S == 4), "av[0] holds every block's first row tile");
    LAS uint8_t *const sv[4] = {(LAS uint8_t *)s0, (LAS uint8_t *)s1, (LAS uint8_t *)s2, (LAS uint8_t *)s3};
    LAS float *const ft[4] = {(LAS float *)f0, (LAS float *)f1, (LAS float *)f2, (LAS float *)f3};
    Cols k[2];
#pragma unroll
    for (int i = 0; i < S; i++) load(sv[i], ft[i]);
    meet(std::integral_constant<int, LOADS *(S - 1)>{});
#pragma unroll
    for (int j = 0; j < TN; j++) columns(k[0], sv[0], ft[0], j);
    av[0] = frag(sv[0], 0);
    auto step = [&](auto n) {
        constexpr int I = decltype(n)::value;
        compute(k[I & 1], k[(I + 1) & 1], sv[I], ft[I], sv[(I + 1) % S], ft[(I + 1) % S]);
    };
#define STEP(I) step(std::integral_constant<int, I>{})
    for (int r = a.nb / S; r > 0; r--) {
        STEP(0);
        STEP(1);
        if constexpr (S > 2) {
            STEP(2);
            STEP(3);
        }
    }
    const int rest = a.nb % S;
    if (rest > 0) STEP(0);
    if constexpr (S > 2) {
        if (rest > 1) STEP(1);
        if (rest > 2) STEP(2);
    }
#undef STEP
    meet(std::integral_constant<int, 0>{});   /* no load may land in LDS that another group owns by then */
#pragma unroll
    for (int j = 0; j < TN; j++) {
        const int64_t t = t0 + (wn * TN + j) * 16 + c;
        if (t >= a.T) continue;
#pragma unroll
        for (int i = 0; i < TM; i++) {
            const int64_t r = (int64_t)(tile0 + wm * TM + i) * 16 + 4 * g;
            if (r < a.rows) store4(a, t, r, acc[i][j]);
        }
    }
}

template <int S, int WM, int WN, int TM, int TN> void launch_tile(const MmArgs &a, hipStream_t s) {
    const int64_t mt = (a.rows + WM * TM * 16 - 1) / (WM * TM * 16), nt = (a.T + WN * TN * 16 - 1) / (WN * TN * 16);
    hipLaunchKernelGGL((k_fp8_tile<S, WM, WN, TM, TN>), dim3((unsigned)(mt * nt)), dim3(64 * WM * WN), 0, s, a,
                       (int)mt, (int)nt);
}
template <int KW, int RT, int TT> void launch_rows(const MmArgs &a, hipStream_t s) {
    const dim3 grid((unsigned)((fp8_tiles(a.rows) + RT - 1) / RT), (unsigned)((a.T + 16 * TT - 1) / (16 * TT)));
    hipLaunchKernelGGL((k_fp8_rows<KW, RT, TT>), grid, dim3(64 * KW), 0, s, a);
}

/* Which kernel.  Up to 16 tokens the weights' bytes bound it: row groups of 16 rows, or of 32 that share the
 * tokens' reads, from 9 tokens on with a group for every compute unit, for fewer with four (8192 x 4096: 16
 * tokens 8.6 us in groups of 32, 9.8 in 16; 4 tokens 8.7 and 8.1; 151936 x 2048, 4 tokens 46.6 and 52); 16 waves
 * a group for long rows (512 x 16384, one token 7.6 us against 9.8 with 8; 151936 x 2048, 16 tokens 52 and 57.5).
 *   More tokens: the kernel whose estimate is least.  With `steps` blocks of a row a wave and q groups on the
 * fullest unit,  us = start + max(steps * run, q * (group + steps * block)):  run is a step's latency, block its
 * share of the unit's throughput, group what a group costs besides.  Fitted to sweeps of float results, random
 * sizes and multiples of large powers of two, over 17..4096 tokens, 64..60000 rows and 2..128 blocks, weights from
 * memory: over their 971 sizes the least estimate's kernel took 2.0% longer than the fastest of the eleven, in the
 * geometric mean, and at worst 45%; the largest kernel with a group for every unit took 9%.  4096 x 4096: 32 tokens
 * 6.4 us in 32 x 16 and 8.5 in 32 x 32, 128 tokens 10.1 in 64 x 32 and 12.2 in 32 x 32.  Results of every type take
 * the same kernel: a 16-bit result is the float one's rounding. */
struct Kernel {
    const char *name;   /* rows and tokens of a group; waves, or stages */
    void (*launch)(const MmArgs &, hipStream_t);
    int m, n, waves;    /* rows and tokens of a group; the waves that share a row's blocks */
    float start, group, run, block;
};
constexpr Kernel KERNELS[] = {
    {"rows_16x16_w8", launch_rows<8, 1, 1>, 16, 16, 8, 2.0f, 0.0f, 0.54f, 0.455f},
    {"rows_32x16_w8", launch_rows<8, 2, 1>, 32, 16, 8, 2.0f, 0.0f, 0.66f, 0.69f},
    {"rows_32x32_w4", launch_rows<4, 2, 2>, 32, 32, 4, 2.5f, 0.0f, 0.4f, 0.51f},
    {"rows_32x32_w8", launch_rows<8, 2, 2>, 32, 32, 8, 2.25f, 0.0f, 0.3f, 1.0f},
    {"rows_64x32_w4", launch_rows<4, 4, 2>, 64, 32, 4, 2.85f, 0.0f, 0.9f, 0.81f},
    {"rows_64x32_w8", launch_rows<8, 4, 2>, 64, 32, 8, 1.35f, 0.95f, 1.5f, 1.51f},
    {"rows_64x64_w4", launch_rows<4, 4, 4>, 64, 64, 4, 1.7f, 2.0f, 0.05f, 1.34f},
    {"tile_64x64_s2", launch_tile<2, 2, 2, 2, 2>, 64, 64, 1, 2.85f, 0.05f, 0.46f, 0.329f},
    {"tile_128x64_s2", launch_tile<2, 2, 2, 4, 2>, 128, 64, 1, 3.35f, 0.14f, 0.65f, 0.505f},
    {"tile_128x64_s4", launch_tile<4, 2, 2, 4, 2>, 128, 64, 1, 2.25f, 1.75f, 0.60f, 0.594f},
    {"tile_128x128_s2", launch_tile<2, 2, 2, 4, 4>, 128, 128, 1, 4.25f, 0.0f, 0.95f, 0.829f},
    /* few tokens of long rows alone */
    {"rows_16x16_w16", launch_rows<16, 1, 1>, 16, 16, 16},
    {"rows_32x16_w16", launch_rows<16, 2, 1>, 32, 16, 16}};
enum { ROWS16 = 0, ROWS32 = 1, TILES = 7, FITTED = 11, ROWS16W16 = 11, ROWS32W16 = 12 };
const Kernel &choose(int64_t rows, int nb, int64_t T) {
    constexpr int64_t CUS = 256;
    auto count = [&](int m, int n) { return ((rows + m - 1) / m) * ((T + n - 1) / n); };
    if (T <= 16) {
        if (count(32, 16) >= (T > 8 ? CUS : 4 * CUS)) return KERNELS[nb < 16 ? ROWS32 : ROWS32W16];
        return KERNELS[nb < 64 ? ROWS16 : ROWS16W16];
    }
    int pick = -1;
    float least = 0.0f;
    for (int i = 0; i < FITTED; i++) {
        const Kernel &c = KERNELS[i];
        if (i < TILES && T > 65535 * (int64_t)c.n) continue;   /* their tokens are the grid's second axis */
        const float steps = (float)((nb + c.waves - 1) / c.waves), q = (float)((count(c.m, c.n) + CUS - 1) / CUS);
        const float run = steps * c.run, full = q * (c.group + steps * c.block);
        const float us = c.start + (run > full ? run : full);
        if (pick < 0 || us < least) {
            pick = i;
            least = us;
        }
    }
    return KERNELS[pick];
}

bool aligned(const void *p, size_t a) { return ((uintptr_t)p & (a - 1)) == 0; }
int type_bytes(int dt) { return dt == DT_F32 ? 4 : dt == DT_F16 || dt == DT_BF16 ? 2 : 0; }

}  // namespace

/* Row and length limits keep every launch inside the grid limits; sizes in bytes
 * are 64-bit throughout. */
constexpr int64_t MOST_TOKENS = (int64_t)1 << 20, MOST_RESULTS = (int64_t)1 << 35;   /* 2^31 threads in the smallest tiles */
static int fp8_dims(const char *who, int64_t rows, int64_t n) {
    if (rows < 1 || n < 1 || rows > ((int64_t)1 << 25) || n > ((int64_t)1 << 22))
        return tlmh_seterr(TLM_HIP_EINVAL, "%s: rows=%lld n=%lld outside 1..2^25 and 1..2^22", who, (long long)rows,
                           (long long)n);
    return TLM_HIP_OK;
}

extern "C" {

size_t tlm_hip_fp8_packed_bytes(int64_t rows, int64_t n) {
    if (fp8_dims("fp8_packed_bytes", rows, n)) return 0;
    const size_t sc = (size_t)fp8_blocks(rows) * (size_t)fp8_blocks(n) * 4;
    return fp8_code_bytes(rows, n) + ((sc + 15) & ~(size_t)15);
}

int tlm_hip_fp8_pack(const void *W, size_t row_bytes, const float *scale, int64_t scale_stride, int64_t rows,
                     int64_t n, void *dst, void *stream) {
    if (int rc = fp8_dims("fp8_pack", rows, n)) return rc;
    if (!W || !scale || !dst) return tlmh_seterr(TLM_HIP_EINVAL, "fp8_pack: NULL argument");
    if (row_bytes < (size_t)n || scale_stride < fp8_blocks(n))
        return tlmh_seterr(TLM_HIP_EINVAL, "fp8_pack: row_bytes=%zu scale_stride=%lld are short for n=%lld", row_bytes,
                           (long long)scale_stride, (long long)n);
    if (!aligned(dst, 16) || !aligned(scale, 4))
        return tlmh_seterr(TLM_HIP_EINVAL, "fp8_pack: dst must be 16-byte and scale 4-byte aligned");
    if (int rc = tlmh_refuse_failed(FAILED_FP8, "fp8_pack")) return rc;
    const int nb = (int)fp8_blocks(n);
    const int64_t pieces = (int64_t)(fp8_code_bytes(rows, n) / 16), ns = fp8_blocks(rows) * nb;
    const int64_t groups = (pieces + ns + 255) / 256;
    if (groups > 0x7FFFFFFF / 256)
        return tlmh_seterr(TLM_HIP_ERANGE, "fp8_pack: %lld x %lld is too large for one launch", (long long)rows,
                           (long long)n);
    const int vec = aligned(W, 16) && row_bytes % 16 == 0;
    hipLaunchKernelGGL(k_fp8_pack, dim3((unsigned)groups), dim3(256), 0, (hipStream_t)stream, (const uint8_t *)W,
                       row_bytes, rows, n, nb, pieces, vec, scale, scale_stride, ns, (uint8_t *)dst);
    return tlmh_check(hipGetLastError(), "fp8_pack launch");
}

int tlm_hip_fp8_quantize(int dt, const void *x, int64_t xstride, int64_t n, int64_t ntok, void *codes, float *scale,
                         void *stream) {
    if (int rc = fp8_dims("fp8_quantize", 1, n)) return rc;
    if (!type_bytes(dt)) return tlmh_seterr(TLM_HIP_EUNSUP, "fp8_quantize: dtype %d (F32, F16 and BF16 only)", dt);
    if (ntok < 0) return tlmh_seterr(TLM_HIP_EINVAL, "fp8_quantize: ntok=%lld", (long long)ntok);
    if (ntok == 0) return TLM_HIP_OK;
    if (!x || !codes || !scale) return tlmh_seterr(TLM_HIP_EINVAL, "fp8_quantize: NULL argument");
    if (xstride < n && ntok > 1)
        return tlmh_seterr(TLM_HIP_EINVAL, "fp8_quantize: row stride %lld below n=%lld", (long long)xstride,
                           (long long)n);
    if (!aligned(x, (size_t)type_bytes(dt)) || !aligned(codes, 16) || !aligned(scale, 4))
        return tlmh_seterr(TLM_HIP_EINVAL, "fp8_quantize: x must have its type's alignment, codes 16, scale 4 bytes");
    const int nb = (int)fp8_blocks(n);
    if (ntok > ((int64_t)1 << 26) / nb)
        return tlmh_seterr(TLM_HIP_ERANGE, "fp8_quantize: %lld tokens of %d blocks are too many for one launch",
                           (long long)ntok, nb);
    if (int rc = tlmh_refuse_failed(FAILED_FP8, "fp8_quantize")) return rc;
    const int64_t blocks = ntok * nb;
    hipStream_t s = (hipStream_t)stream;
    if (dt == DT_F32) launch_quant<float>(x, xstride, n, nb, blocks, codes, scale, s);
    else if (dt == DT_F16) launch_quant<_Float16>(x, xstride, n, nb, blocks, codes, scale, s);
    else launch_quant<__bf16>(x, xstride, n, nb, blocks, codes, scale, s);
    return tlmh_check(hipGetLastError(), "fp8_quantize launch");
}

int tlm_hip_fp8_matmul(const void *Wp, int64_t rows, int64_t n, const void *codes, const float *scale, int64_t ntok,
                       int dt, void *Y, int64_t ystride, void *stream) {
    if (int rc = fp8_dims("fp8_matmul", rows, n)) return rc;
    if (!type_bytes(dt)) return tlmh_seterr(TLM_HIP_EUNSUP, "fp8_matmul: dtype %d (F32, F16 and BF16 only)", dt);
    if (ntok < 0) return tlmh_seterr(TLM_HIP_EINVAL, "fp8_matmul: ntok=%lld", (long long)ntok);
    if (ntok == 0) return TLM_HIP_OK;
    if (!Wp || !codes || !scale || !Y) return tlmh_seterr(TLM_HIP_EINVAL, "fp8_matmul: NULL argument");
    if (ystride < rows && ntok > 1)
        return tlmh_seterr(TLM_HIP_EINVAL, "fp8_matmul: row stride %lld below rows=%lld", (long long)ystride,
                           (long long)rows);
    if (!aligned(Wp, 16) || !aligned(codes, 16) || !aligned(scale, 4) || !aligned(Y, (size_t)type_bytes(dt)))
        return tlmh_seterr(TLM_HIP_EINVAL,
                           "fp8_matmul: the matrix and the codes must be 16-byte, scale 4-byte aligned, Y as its type");
    if (ntok > MOST_TOKENS || ntok * rows > MOST_RESULTS)
        return tlmh_seterr(TLM_HIP_ERANGE, "fp8_matmul: %lld tokens of %lld rows are too many for one launch",
                           (long long)ntok, (long long)rows);
    if (int rc = tlmh_refuse_failed(FAILED_FP8, "fp8_matmul")) return rc;
    const MmArgs a = {(const uint8_t *)Wp, (const float *)((const uint8_t *)Wp + fp8_code_bytes(rows, n)),
                      (const uint8_t *)codes, scale, Y, rows, ystride, ntok, (int)fp8_blocks(n), dt};
    choose(rows, a.nb, ntok).launch(a, (hipStream_t)stream);
    return tlmh_check(hipGetLastError(), "fp8_matmul launch");
}

const char *tlm_hip_fp8_matmul_kernel(int64_t rows, int64_t n, int64_t ntok) {
    if (fp8_dims("fp8_matmul_kernel", rows, n)) return nullptr;
    if (ntok < 1 || ntok > MOST_TOKENS || ntok * rows > MOST_RESULTS) {
        tlmh_seterr(TLM_HIP_ERANGE, "fp8_matmul_kernel: no launch for %lld tokens of %lld rows", (long long)ntok,
                    (long long)rows);
        return nullptr;
    }
    return choose(rows, (int)fp8_blocks(n), ntok).name;
}

}  // extern "C"
