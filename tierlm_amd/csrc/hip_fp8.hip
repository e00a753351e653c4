/* hip_fp8.hip - 8-bit floating point with a scale per block of 128: packing,
 * the activation quantiser and the matrix product (the reference's FP8 weight
 * format, src/lib/tlm_quant.c:761-776, with its activations in 8 bits too). */
#include "tlm_hip_fp8.h"

namespace {

/* ---- packing: a thread per 16-byte piece ---------------------------------- */
__global__ __launch_bounds__(256) void k_fp8_pack(const uint8_t *__restrict__ W, size_t row_bytes, int64_t rows,
                                                  int64_t n, int nb, int64_t pieces, int vec,
                                                  uint8_t *__restrict__ dst) {
    const int64_t p = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (p >= pieces) return;
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

__global__ __launch_bounds__(256) void k_fp8_pack_scale(const float *__restrict__ s, int64_t stride, int nb,
                                                        int64_t count, float *__restrict__ dst) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i < count) dst[i] = s[i / nb * stride + i % nb];
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

template <class T>
__global__ __launch_bounds__(256) void k_fp8_quant(const T *__restrict__ x, int64_t xstride, int64_t n, int nb,
                                                   int64_t blocks, uint8_t *__restrict__ codes,
                                                   float *__restrict__ scale) {
    const int64_t blk = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4);
    const int sub = threadIdx.x & 15;
    const bool live = blk < blocks;
    const int64_t t = live ? blk / nb : 0;
    const int64_t k0 = (live ? blk % nb : 0) * FP8_BLOCK + 8 * sub;
    const T *src = x + t * xstride + k0;
    float v[8];
    uint32_t am = 0;
#pragma unroll
    for (int j = 0; j < 8; j++) {
        v[j] = live && k0 + j < n ? ld_f32(src + j) : 0.0f;
        const uint32_t b = __float_as_uint(v[j]) & 0x7FFFFFFFu;   /* order of |v|; NaN and infinity on top */
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
    c0 = __builtin_amdgcn_cvt_pk_fp8_f32(v[0] * inv, v[1] * inv, c0, false);
    c0 = __builtin_amdgcn_cvt_pk_fp8_f32(v[2] * inv, v[3] * inv, c0, true);
    c1 = __builtin_amdgcn_cvt_pk_fp8_f32(v[4] * inv, v[5] * inv, c1, false);
    c1 = __builtin_amdgcn_cvt_pk_fp8_f32(v[6] * inv, v[7] * inv, c1, true);
    if (!live) return;
    u32x2 o = {(uint32_t)c0, (uint32_t)c1};
    if (bad) o = (u32x2){0u, 0u};
    *(u32x2 *)(codes + blk * FP8_BLOCK + 8 * sub) = o;
    if (sub == 0)
        scale[blk] = bad ? __uint_as_float(0x7FC00000u) : am ? __uint_as_float((uint32_t)(127 + e) << 23) : 0.0f;
}

/* ---- product ----------------------------------------------------------------
 * Y[t][r] = sum over blocks b of sa[t][b] sw[r / 128][b] (codes of t . codes of r):
 * products and their sums of 128 in the matrix cores' float accumulators, then
 * one fma per block. */
template <class T> __device__ __forceinline__ T to_out(float v);
template <> __device__ __forceinline__ float to_out<float>(float v) { return v; }
template <> __device__ __forceinline__ _Float16 to_out<_Float16>(float v) { return (_Float16)v; }
template <> __device__ __forceinline__ __bf16 to_out<__bf16>(float v) { return (__bf16)v; }

struct MmArgs {
    const uint8_t *W;
    const float *sw;
    const uint8_t *x;
    const float *sa;
    void *y;
    int64_t rows, ystride, T;
    int nb, wide;   /* wide: every run of four rows of Y may be stored at once */
};

template <class T>
__global__ __launch_bounds__(256) void k_fp8_mm(MmArgs a) {
    const int lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;
    const int64_t tiles = fp8_tiles(a.rows);
    const int64_t tile = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (tile >= tiles) return;
    const int64_t t = (int64_t)blockIdx.y * 16 + c, tc = t < a.T ? t : a.T - 1;
    const uint8_t *w = a.W + (size_t)tile * a.nb * FP8_UNIT + lane * 16;
    const uint8_t *x = a.x + (size_t)tc * a.nb * FP8_BLOCK + g * 16;
    const float *sw = a.sw + tile / 8 * a.nb, *sa = a.sa + tc * a.nb;
    f32x4 acc = {0, 0, 0, 0};
    for (int b = 0; b < a.nb; b++) {
        f32x4 p = {0, 0, 0, 0};
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const i32x4 wc = *(const i32x4 *)(w + (size_t)b * FP8_UNIT + 1024 * h);
            const i32x4 xc = *(const i32x4 *)(x + (size_t)b * FP8_BLOCK + 64 * h);
            p = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fp8_to_bf16(wc[0], wc[1]), fp8_to_bf16(xc[0], xc[1]), p, 0, 0, 0);
            p = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fp8_to_bf16(wc[2], wc[3]), fp8_to_bf16(xc[2], xc[3]), p, 0, 0, 0);
        }
        const float s = sw[b] * sa[b];
#pragma unroll
        for (int v = 0; v < 4; v++) acc[v] = fmaf(p[v], s, acc[v]);
    }
    if (t >= a.T) return;
#pragma unroll
    for (int v = 0; v < 4; v++) {
        const int64_t r = tile * 16 + 4 * g + v;
        if (r < a.rows) ((T *)a.y)[t * a.ystride + r] = to_out<T>(acc[v]);
    }
}

/* ---- product, tiles through LDS ------------------------------------------------ */
template <class T, int WM, int WN, int TM, int TN>
__global__ __launch_bounds__(64 * WM * WN) __attribute__((amdgpu_waves_per_eu(WM * WN / 4, WM * WN / 4)))
void k_fp8_tile(MmArgs a, int mtiles, int ntiles) {
    constexpr int NWV = WM * WN, MT = WM * TM, NT = WN * TN, UNITS = MT + NT, PER = UNITS / NWV;
    static_assert(MT % NWV == 0 && NT % NWV == 0 && 8 % TM == 0 && MT % 8 == 0, "units are dealt evenly; a wave's rows share a scale");
    __shared__ __align__(16) uint8_t s0[UNITS * FP8_UNIT], s1[UNITS * FP8_UNIT];
    /* scales: a wave brings those of its share of the tokens, then the row blocks' */
    constexpr int TPW = NT * 16 / NWV;
    __shared__ float f0[NWV * 64], f1[NWV * 64];
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
    auto load = [&](uint8_t *s, float *f) {
        const bool more = ++pos < a.nb;
#pragma unroll
        for (int i = 0; i < PER; i++) {
            const int u = wave + i * NWV;
#pragma unroll
            for (int h = 0; h < 2; h++)
                __builtin_amdgcn_global_load_lds((const GAS void *)(base[i] + off[i][h]),
                                                 (LAS void *)(s + u * FP8_UNIT + h * 1024), 16, 0, 0);
            base[i] += !more ? 0 : i * NWV < MT ? FP8_UNIT : FP8_BLOCK;
        }
        __builtin_amdgcn_global_load_lds((const GAS void *)ssrc, (LAS void *)(f + wave * 64), 4, 0, 0);
        ssrc += more ? 1 : 0;
    };
    f32x4 acc[TM][TN] = {};
    auto frag = [&](const uint8_t *s, int u) {
        const LAS i32x4 *p = (const LAS i32x4 *)(s + u * FP8_UNIT + lane * 16);
        return fp8_join(p[0], p[64]);
    };
    struct Cols {
        i32x8 b[TN];
        float sc[TN], w;
    };
    auto columns = [&](Cols &k, const uint8_t *s, const float *f, int j) {
        const LAS uint8_t *p = (const LAS uint8_t *)s + (MT + wn * TN + j) * FP8_UNIT + c * FP8_BLOCK;
        k.b[j] = fp8_join(*(const LAS i32x4 *)(p + 16 * (g ^ (c & 7))), *(const LAS i32x4 *)(p + 16 * ((4 + g) ^ (c & 7))));
        const int t = (wn * TN + j) * 16;
        k.sc[j] = ((const LAS float *)f)[t / TPW * 64 + t % TPW + c];
        if (j == 0) k.w = ((const LAS float *)f)[TPW + wm * TM / 8];
    };
    /* One block: the matrix instructions of row tile i run beside the fmas of the ones before
     * (a ring of RING results) and the reads of row tile i + 1.  Once row tile TM - 1 is in
     * registers the stage is free: the waves meet, the next block's loads go out into it, and the
     * next block's columns are read from the other stage under the last instructions. */
    constexpr int RING = 4;
    i32x8 av[2];
    auto compute = [&](Cols &k, Cols &kn, uint8_t *s, float *f, const uint8_t *sn, const float *fn, bool on) {
        f32x4 p[RING];
        float sc[TN];
#pragma unroll
        for (int j = 0; j < TN; j++) sc[j] = k.w * k.sc[j];
        auto fold = [&](int m) {
            const int i = m / TN, j = m % TN;
#pragma unroll
            for (int v = 0; v < 4; v++) acc[i][j][v] = fmaf(p[m % RING][v], sc[j], acc[i][j][v]);
        };
#pragma unroll
        for (int i = 0; i < TM; i++) {
            if (i + 1 < TM) av[(i + 1) & 1] = frag(s, wm * TM + i + 1);
            if (i + 1 == TM && on) {
                __syncthreads();
                load(s, f);
            }
#pragma unroll
            for (int j = 0; j < TN; j++) {
                const int m = i * TN + j;
                p[m % RING] = fp8_mfma(av[i & 1], k.b[j], (f32x4){0, 0, 0, 0});
                if (m >= RING - 1) fold(m - RING + 1);
                if (i + 1 == TM && on) columns(kn, sn, fn, j);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        if (on) av[TM & 1] = frag(sn, wm * TM);
#pragma unroll
        for (int m = TM * TN - RING + 1; m < TM * TN; m++) fold(m);
        __builtin_amdgcn_sched_barrier(0);
    };
    static_assert(TM % 2 == 0, "av[0] holds every block's first row tile");
    Cols k0, k1;
    load(s0, f0);
    __syncthreads();
    load(s1, f1);
#pragma unroll
    for (int j = 0; j < TN; j++) columns(k0, s0, f0, j);
    av[0] = frag(s0, wm * TM);
    for (int n2 = a.nb >> 1; n2 > 0; n2--) {
        compute(k0, k1, s0, f0, s1, f1, true);
        compute(k1, k0, s1, f1, s0, f0, true);
    }
    if (a.nb & 1) compute(k0, k1, s0, f0, s1, f1, false);
    __syncthreads();
#pragma unroll
    for (int j = 0; j < TN; j++) {
        const int64_t t = t0 + (wn * TN + j) * 16 + c;
        if (t >= a.T) continue;
        T *y = (T *)a.y + t * a.ystride;
#pragma unroll
        for (int i = 0; i < TM; i++) {
            const int64_t r = (int64_t)(tile0 + wm * TM + i) * 16 + 4 * g;
            typedef T T4 __attribute__((ext_vector_type(4)));
            T4 o;
#pragma unroll
            for (int v = 0; v < 4; v++) o[v] = to_out<T>(acc[i][j][v]);
            if (a.wide && r + 3 < a.rows) {
                *(T4 *)(y + r) = o;
            } else {
#pragma unroll
                for (int v = 0; v < 4; v++)
                    if (r + v < a.rows) y[r + v] = o[v];
            }
        }
    }
}

bool aligned(const void *p, size_t a) { return ((uintptr_t)p & (a - 1)) == 0; }
int type_bytes(int dt) { return dt == DT_F32 ? 4 : dt == DT_F16 || dt == DT_BF16 ? 2 : 0; }

}  // namespace

/* Row and length limits keep every launch inside the grid limits; sizes in bytes
 * are 64-bit throughout. */
static int fp8_dims(const char *who, int64_t rows, int64_t n) {
    if (rows < 1 || n < 1 || rows > ((int64_t)1 << 28) || n > ((int64_t)1 << 24))
        return tlmh_seterr(TLM_HIP_EINVAL, "%s: rows=%lld n=%lld outside 1..2^28 and 1..2^24", who, (long long)rows,
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
    const int nb = (int)fp8_blocks(n);
    const int64_t pieces = (int64_t)(fp8_code_bytes(rows, n) / 16), ns = fp8_blocks(rows) * nb;
    if ((pieces + 255) / 256 > 0x7FFFFFFF / 256)
        return tlmh_seterr(TLM_HIP_ERANGE, "fp8_pack: %lld x %lld is too large for one launch", (long long)rows,
                           (long long)n);
    const int vec = aligned(W, 16) && row_bytes % 16 == 0;
    hipLaunchKernelGGL(k_fp8_pack, dim3((unsigned)((pieces + 255) / 256)), dim3(256), 0, (hipStream_t)stream,
                       (const uint8_t *)W, row_bytes, rows, n, nb, pieces, vec, (uint8_t *)dst);
    hipLaunchKernelGGL(k_fp8_pack_scale, dim3((unsigned)((ns + 255) / 256)), dim3(256), 0, (hipStream_t)stream, scale,
                       scale_stride, nb, ns, (float *)((uint8_t *)dst + fp8_code_bytes(rows, n)));
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
    const int64_t blocks = ntok * nb;
    const dim3 grid((unsigned)((blocks + 15) / 16));
    hipStream_t s = (hipStream_t)stream;
    if (dt == DT_F32)
        hipLaunchKernelGGL(k_fp8_quant<float>, grid, dim3(256), 0, s, (const float *)x, xstride, n, nb, blocks,
                           (uint8_t *)codes, scale);
    else if (dt == DT_F16)
        hipLaunchKernelGGL(k_fp8_quant<_Float16>, grid, dim3(256), 0, s, (const _Float16 *)x, xstride, n, nb, blocks,
                           (uint8_t *)codes, scale);
    else
        hipLaunchKernelGGL(k_fp8_quant<__bf16>, grid, dim3(256), 0, s, (const __bf16 *)x, xstride, n, nb, blocks,
                           (uint8_t *)codes, scale);
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
    if (ntok > 1000000)
        return tlmh_seterr(TLM_HIP_ERANGE, "fp8_matmul: %lld tokens are too many for one launch", (long long)ntok);
    const MmArgs a = {(const uint8_t *)Wp, (const float *)((const uint8_t *)Wp + fp8_code_bytes(rows, n)),
                      (const uint8_t *)codes, scale, Y, rows, ystride, ntok, (int)fp8_blocks(n),
                      aligned(Y, 4 * (size_t)type_bytes(dt)) && (ystride % 4 == 0 || ntok == 1)};
    const dim3 grid((unsigned)((fp8_tiles(rows) + 3) / 4), (unsigned)((ntok + 15) / 16));
    hipStream_t s = (hipStream_t)stream;
    if (ntok >= 256 && dt == DT_BF16) {
        const int mt = (int)((rows + 255) / 256), nt = (int)((ntok + 255) / 256);
        hipLaunchKernelGGL((k_fp8_tile<__bf16, 2, 4, 8, 4>), dim3((unsigned)(mt * nt)), dim3(512), 0, s, a, mt, nt);
        return tlmh_check(hipGetLastError(), "fp8_matmul launch");
    }
    if (dt == DT_F32) hipLaunchKernelGGL(k_fp8_mm<float>, grid, dim3(256), 0, s, a);
    else if (dt == DT_F16) hipLaunchKernelGGL(k_fp8_mm<_Float16>, grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL(k_fp8_mm<__bf16>, grid, dim3(256), 0, s, a);
    return tlmh_check(hipGetLastError(), "fp8_matmul launch");
}

}  // extern "C"
