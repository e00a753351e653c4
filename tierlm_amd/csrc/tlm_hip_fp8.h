/* tlm_hip_fp8.h - 8-bit floating point (OCP E4M3: sign, 4 exponent bits of bias
 * 7, 3 mantissa bits, largest 448, no infinities, NaN 0x7F / 0xFF) on the device:
 * the packed layout and the fragments that the matrix cores read from it.
 *
 * Packed matrix of rows x n, one scale per 128 x 128 block: n is padded to nb
 * blocks of 128 values and the rows to tiles of 16, codes of the padding 0.  Unit
 * (tile, block) of 2048 bytes sits at (tile * nb + block) * 2048, its 128
 * pieces of 16 bytes in the order half h, lane l: piece (h, l) holds row l % 16,
 * values 64 h + 16 (l / 16) + 0..15 of the block, so both halves of a wave's
 * operand are 1 KB contiguous loads (from memory or LDS) without a bank
 * conflict.  The matrix cores pair equal positions of both operands, so any order of
 * a block's values is right as long as activations use the same one.
 * The scales follow, f32, [rows / 128 rounded up][nb].  Included by .hip files. */
#ifndef TLM_HIP_FP8_H
#define TLM_HIP_FP8_H

#include "tlm_hip_internal.h"

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef uint16_t u16x4 __attribute__((ext_vector_type(4)));
typedef uint16_t u16x8 __attribute__((ext_vector_type(8)));

constexpr int FP8_BLOCK = 128;       /* values, and rows, of one scale */
constexpr int FP8_UNIT = 2048;       /* bytes of 16 rows x 128 values */

__host__ __device__ static inline int64_t fp8_blocks(int64_t n) { return (n + FP8_BLOCK - 1) / FP8_BLOCK; }
__host__ __device__ static inline int64_t fp8_tiles(int64_t rows) { return (rows + TILE_ROWS - 1) / TILE_ROWS; }
__host__ __device__ static inline size_t fp8_code_bytes(int64_t rows, int64_t n) {
    return (size_t)fp8_tiles(rows) * (size_t)fp8_blocks(n) * FP8_UNIT;
}

__device__ __forceinline__ i32x8 fp8_join(i32x4 lo, i32x4 hi) {
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}

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

/* A block of 128 values held by 16 lanes, 8 a lane: this lane's codes and the block's scale.
 * scale = 2^e, e the least integer >= -126 with amax <= 448 * 2^e: dividing by it is exact, so the one
 * rounding is the code's, and a floating code loses no relative precision by it. */
struct Fp8Codes {
    u32x2 codes;
    float scale;
};
__device__ __forceinline__ Fp8Codes fp8_encode(const float (&v)[8]) {
    uint32_t am = 0;
#pragma unroll
    for (int j = 0; j < 8; j++) {
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
    return {{bad ? 0u : (uint32_t)c0, bad ? 0u : (uint32_t)c1},
            bad ? __uint_as_float(0x7FC00000u) : am ? __uint_as_float((uint32_t)(127 + e) << 23) : 0.0f};
}

/* eight codes times a power of two (1 / 2^100 to 2^100) as bfloat16: exact (E4M3 has 4 significant
 * bits, from 2^-9 to 448) */
__device__ __forceinline__ bf16x8 fp8_to_bf16(int lo, int hi, float pow2 = 1.0f) {
    const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, pow2, false);
    const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, pow2, true);
    const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, pow2, false);
    const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, pow2, true);
    bf16x8 r;
    r[0] = a[0]; r[1] = a[1]; r[2] = b[0]; r[3] = b[1];
    r[4] = c[0]; r[5] = c[1]; r[6] = d[0]; r[7] = d[1];
    return r;
}

/* A block's scale as pow2 * rest, pow2 its power of two within 2^-100 .. 2^100 (zeros, infinities and NaN: an
 * end of it).  The codes take pow2 as they are converted, which costs nothing; what is then multiplied with the
 * other operand's scale is 1 to 2 (2^-26 to 2^28 at the ends), and the product a normal float.  Multiplied as they
 * come, 2^-126 (the quantiser's least) and 2e-4 left 13 bits, 2^108 and 2^20 an infinity.  (Each element times one
 * scale, then the other: 5 to 7% of the larger tiles' time.) */
struct Fp8Scale {
    float pow2, rest;
};
__device__ __forceinline__ Fp8Scale fp8_scale(float s) {
    constexpr uint32_t LO = (127 - 100) << 23, HI = (127 + 100) << 23;
    uint32_t e = __float_as_uint(s) & 0x7F800000u;
    e = e < LO ? LO : e > HI ? HI : e;
    return {__uint_as_float(e), s * __uint_as_float((254u << 23) - e)};
}

/* A float as three bfloat16 planes, v = p0 + p1 + p2 exactly: each plane takes
 * the next 8 significant bits (the leading 16 bits of what is left), and a
 * float has 24.  (Exact while the last plane stays normal; below 2^-110 bits of a
 * subnormal third plane may be lost.)  An infinity or NaN sits in the first
 * plane alone. */
__device__ __forceinline__ void split3(float v, uint16_t p[3]) {
    const uint32_t b = __float_as_uint(v);
    const bool special = (b & 0x7F800000u) == 0x7F800000u;
    const float r1 = v - __uint_as_float(b & 0xFFFF0000u);
    const uint32_t b1 = __float_as_uint(r1);
    const float r2 = r1 - __uint_as_float(b1 & 0xFFFF0000u);
    p[0] = (uint16_t)(v != v ? 0x7FC0u : b >> 16);
    p[1] = special ? 0 : (uint16_t)(b1 >> 16);
    p[2] = special ? 0 : (uint16_t)(__float_as_uint(r2) >> 16);
}

#endif
