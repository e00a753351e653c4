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
