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
    int nb;
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
                      (const uint8_t *)codes, scale, Y, rows, ystride, ntok, (int)fp8_blocks(n)};
    const dim3 grid((unsigned)((fp8_tiles(rows) + 3) / 4), (unsigned)((ntok + 15) / 16));
    hipStream_t s = (hipStream_t)stream;
    if (dt == DT_F32) hipLaunchKernelGGL(k_fp8_mm<float>, grid, dim3(256), 0, s, a);
    else if (dt == DT_F16) hipLaunchKernelGGL(k_fp8_mm<_Float16>, grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL(k_fp8_mm<__bf16>, grid, dim3(256), 0, s, a);
    return tlmh_check(hipGetLastError(), "fp8_matmul launch");
}

}  // extern "C"
