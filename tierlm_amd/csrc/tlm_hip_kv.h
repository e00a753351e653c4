/* tlm_hip_kv.h - the paged key-value cache: where a position lies, which work a group takes.
 *
 * A page holds P positions (a power of two >= 16) of every key head, as blocks of 16 positions.  Block
 * (page, head, i) of 16 * head_dim elements is number (page * heads + head) * (P / 16) + i of either array:
 *   keys    [head_dim / 16][16 positions][16 values]
 *   values  [head_dim][16 positions]
 * Both are the order in which the matrix cores take their operands: S^T = K Q^T contracts over values, O^T = V^T P^T over
 * positions, and a lane's operand is 8 consecutive elements of the contracted axis.  So every fragment is 16-byte pieces
 * of one contiguous kilobyte, from memory or LDS, with no transposition and no bank conflict, and the scores' result
 * lanes (one query each) hold the very positions that the second product's operand wants.
 *
 * Plain C++ but for the last part: the CPU tests compile it without HIP.  Included by .hip files. */
#ifndef TLM_HIP_KV_H
#define TLM_HIP_KV_H

#include <stdint.h>

#ifdef __HIPCC__
#include "tlm_hip_internal.h"
#define TLM_HD __host__ __device__ __forceinline__
#else
#define TLM_HD inline
#endif

constexpr int KV_BLOCK = 16;      /* positions of a block */

/* What the kernels know of a cache and its batch.  Lengths, row bounds and tables are the device's: they are held to
 * their limits where they are used, and what lies outside holds nothing. */
struct KvView {
    const int32_t *tables, *lens, *cu;   /* cu: null, a row a sequence */
    int64_t table_stride;
    int64_t rows;
    int32_t B, table_pages, n_pages, heads;
    int32_t sh;                          /* log2 of a page's blocks */
    int32_t hd;
};

/* rows of sequence b (first, count) inside [0, rows) whatever cu holds */
struct KvRows {
    int64_t first, n;
};
TLM_HD KvRows kv_rows(const KvView &c, int b) {
    if (!c.cu) return {b, b < c.rows ? 1 : 0};
    int64_t lo = c.cu[b], hi = c.cu[b + 1];
    lo = lo < 0 ? 0 : lo > c.rows ? c.rows : lo;
    hi = hi < lo ? lo : hi > c.rows ? c.rows : hi;
    return {lo, hi - lo};
}
/* positions of sequence b after this call's rows (negative lengths are zero) */
TLM_HD int64_t kv_len(const KvView &c, int b) { return c.lens[b] < 0 ? 0 : c.lens[b]; }
/* positions that its table can name */
TLM_HD int64_t kv_cap(const KvView &c) { return ((int64_t)c.table_pages << c.sh) * KV_BLOCK; }

/* Element offset of block `blk` (16 positions) of a sequence's head: -1 where the table names no page of the cache. */
TLM_HD int64_t kv_block(const KvView &c, int32_t page, int64_t blk, int head) {
    if ((uint32_t)page >= (uint32_t)c.n_pages) return -1;
    const int64_t at = (((int64_t)page * c.heads + head) << c.sh) + (blk & (((int64_t)1 << c.sh) - 1));
    return at * (KV_BLOCK * c.hd);
}
/* Key value e / value value e of position p (mod 16) inside a block */
TLM_HD int kv_key_at(int p, int e) { return e / 16 * 256 + p * 16 + e % 16; }
TLM_HD int kv_value_at(int p, int e) { return e * 16 + p; }

/* ---- append: an item is a block of 16 positions of a sequence ------------- */
/* First position of a sequence's new rows (negative if it has more rows than positions), and the blocks they touch */
TLM_HD int64_t kv_floor16(int64_t p) { return p >= 0 ? p / 16 : -((15 - p) / 16); }
TLM_HD int64_t kv_append_items(int64_t n, int64_t len) {
    return n > 0 ? kv_floor16(len - 1) - kv_floor16(len - n) + 1 : 0;
}
/* as many items as any lengths of B sequences with `rows` rows give (without cu a sequence is an item) */
TLM_HD int64_t kv_append_most(int64_t rows, int64_t B) {
    const int64_t used = rows < B ? rows : B;   /* sequences that can have a row; n rows touch at most (n + 14) / 16 + 1 */
    return (rows + 14 * used) / 16 + used;
}

/* ---- decode: the batch's positions end to end in units of 128, dealt to W workers in equal shares ------------ */
constexpr int KV_UNIT = 128;
/* units of a sequence (an empty one has one too: its zeros are written) */
TLM_HD int kv_units(int64_t len) { return len <= KV_UNIT ? 1 : (int)((len + KV_UNIT - 1) / KV_UNIT); }
/* U units: the first U mod W workers take U / W + 1 of them, the others U / W */
struct KvShares {
    int q, r;
};
TLM_HD KvShares kv_shares(int U, int W) { return {U / W, U % W}; }
TLM_HD int kv_share(KvShares s, int w) { return w * s.q + (w < s.r ? w : s.r); }     /* worker w's first unit */
TLM_HD int kv_worker(KvShares s, int x) {                                            /* unit x's worker */
    const int big = s.r * (s.q + 1);
    return x < big ? x / (s.q + 1) : s.r + (x - big) / s.q;
}
/* Where worker w leaves its sums of a sequence that it does not have to itself: one that began with an earlier worker, or
 * one that begins here (a worker has at most one of each) */
TLM_HD int kv_slot(int w, bool begins) { return 2 * w + (begins ? 1 : 0); }

/* ---- prompt: an item is a tile of a sequence's (token, head) rows ---------- */
TLM_HD int64_t kv_prompt_items(int64_t n, int64_t group, int64_t tile) { return (n * group + tile - 1) / tile; }
TLM_HD int64_t kv_prompt_most(int64_t rows, int64_t B, int64_t group, int64_t tile) {
    const int64_t used = rows < B ? rows : B;
    return (rows * group - used) / tile + used;   /* sum of ceil(x_b / tile), x_b >= 1 */
}

#ifdef __HIPCC__
/* What all calls ask of a cache and a batch; *v is filled for the kernels (hip_kv.hip) */
int kv_check(const char *who, const tlm_hip_kv_cache *c, const tlm_hip_kv_batch *b, int heads, KvView *v);

/* constant memory: what no launch under way writes; uniform reads go through the scalar cache */
#define CAS __attribute__((address_space(4)))

typedef float f32x16 __attribute__((ext_vector_type(16)));

/* 16-bit types of cache and queries and their matrix instructions */
template <class T> struct KvType;
template <> struct KvType<__bf16> {
    typedef __bf16 x8 __attribute__((ext_vector_type(8)));
    static constexpr uint32_t EXP = 0x7F80u;      /* all ones: an infinity or NaN */
    static constexpr float SHIFT = 0.0f;
    static __device__ __forceinline__ f32x4 mma(x8 a, x8 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    }
    static __device__ __forceinline__ f32x16 mma(x8 a, x8 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
    }
};
template <> struct KvType<_Float16> {
    typedef _Float16 x8 __attribute__((ext_vector_type(8)));
    static constexpr uint32_t EXP = 0x7C00u;
    /* probabilities are held times 2^8: with at most 2^6 over the running maximum they stay finite, and those that a long
     * context leaves near 2^-20 stay out of the subnormals */
    static constexpr float SHIFT = 8.0f;
    static __device__ __forceinline__ f32x4 mma(x8 a, x8 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    }
    static __device__ __forceinline__ f32x16 mma(x8 a, x8 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
    }
};
/* How far (in powers of two) scores may rise over the maximum that the running sums are scaled by before those are
 * scaled anew: the probabilities stay finite in either type and in the float sums, and most tiles scale nothing */
constexpr float KV_SLACK = 6.0f;

/* Running maxima are kept as scores are, before their scale: a difference of two scores is exact where it counts (within a
 * factor of two of each other), so weights are 2^(scale2 (s - m) + SHIFT) whatever the scores' size.  (The scaled maximum
 * rounded and then taken from an unrounded product leaves half a step of it: past 2^25 that is more than an exponent.)
 *
 * Does `top` rise over the maximum m by more than the slack (from -infinity: any score does)? */
__device__ __forceinline__ bool kv_rises(float top, float m, float scale2) { return (top - m) * scale2 > KV_SLACK; }
/* What scales sums kept by the maximum m where the maximum is `to` */
__device__ __forceinline__ float kv_factor(float m, float to, float scale2) {
    return __builtin_amdgcn_exp2f((m - (to == -INFINITY ? 0.0f : to)) * scale2);
}
/* A row that sees positions, all with a score of -infinity, has this maximum at the end of its pass: its weights are 0 / 0 and
 * its result NaN.  One that sees none keeps -infinity, and gets zeros. */
constexpr float KV_LOWEST = -3.4028234663852886e38f;
__device__ __forceinline__ float kv_inverse(float l, float m) {
    return l != 0.0f ? __builtin_amdgcn_rcpf(l) : m == -INFINITY ? 0.0f : __builtin_nanf("");   /* to one unit of 2^-23 */
}
/* Values that are not finite come through whatever their weight, also where it or the factor that scales its sum rounds to 0
 * (0 times infinity is NaN): sums that are not finite at the end have the values that made them so looked up and put in their
 * place, and from then on keep them. */
template <class T> __device__ __forceinline__ uint32_t kv_odd(uint32_t e) {   /* of a value's bits: 0 it is finite, 1 +inf, 2 -inf, 3 NaN */
    constexpr uint32_t E = KvType<T>::EXP;
    return (e & E) != E ? 0u : (e & 0x7FFFu) > E ? 3u : e >> 15 ? 2u : 1u;
}
__device__ __forceinline__ float kv_put_odd(float x, uint32_t odd) {         /* odd: of several values or-ed, both infinities are NaN */
    return odd == 0 ? x : odd == 1 ? INFINITY : odd == 2 ? -INFINITY : __builtin_nanf("");
}
template <class T> __device__ __forceinline__ bool kv_any_odd(u32x4 v) {    /* of 8 values */
    constexpr uint32_t E = KvType<T>::EXP;
    bool odd = false;
#pragma unroll
    for (int w = 0; w < 4; w++) odd |= (v[w] & E) == E || (v[w] & (E << 16)) == E << 16;
    return odd;
}
/* the factor for sums that may be infinite: at least 2^-149, which leaves an infinity and is nothing to a finite sum */
__device__ __forceinline__ float kv_not_zero(float f) { return fmaxf(f, 0x1p-149f); }

/* four values of a result, rounded to its type */
__device__ __forceinline__ void kv_store(void *out, int dt, int64_t i, const float (&v)[4]) {
    typedef _Float16 h4 __attribute__((ext_vector_type(4), aligned(2)));
    typedef __bf16 b4 __attribute__((ext_vector_type(4), aligned(2)));
    typedef f32x4 f4 __attribute__((aligned(4)));
    if (dt == DT_F32) *(f4 *)((float *)out + i) = f4{v[0], v[1], v[2], v[3]};
    else if (dt == DT_F16) *(h4 *)((_Float16 *)out + i) = h4{(_Float16)v[0], (_Float16)v[1], (_Float16)v[2], (_Float16)v[3]};
    else *(b4 *)((__bf16 *)out + i) = b4{(__bf16)v[0], (__bf16)v[1], (__bf16)v[2], (__bf16)v[3]};
}

template <class V> __device__ __forceinline__ V kv_bits(u32x4 v) { return __builtin_bit_cast(V, v); }
/* 8 values, zeros from the left-th on */
__device__ __forceinline__ u32x4 kv_upto(u32x4 v, int left) {
#pragma unroll
    for (int w = 0; w < 4; w++) v[w] &= (2 * w < left ? 0xFFFFu : 0u) | (2 * w + 1 < left ? 0xFFFF0000u : 0u);
    return v;
}

/* 8 consecutive elements at any alignment of the type */
template <class T> __device__ __forceinline__ u32x4 kv_load8(const T *p) {
    typedef u32x4 any __attribute__((aligned(2)));
    return *(const any *)p;
}

__device__ __forceinline__ int kv_uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

/* sum of the lanes up to this one */
__device__ __forceinline__ int kv_scan(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, true);    /* row_shr 1, 2, 4, 8: inside 16 lanes */
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);   /* lanes 15 and 47 to the rows behind them */
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);   /* lane 31 to the upper half */
    return v;
}

/* Which sequence item w belongs to, and its number there, by a scan over the sequences' item counts, 64 a round (each
 * wave by itself).  b < 0: there are fewer items.  before: the items of the sequences before it.  Every field is uniform. */
struct KvItem {
    int b, i, n, before;
};
template <class Count> __device__ __forceinline__ KvItem kv_find(int B, int w, const Count &count) {
    const int lane = wave_lane();
    int before = 0;
    auto scan = [&](int b0, int mine, KvItem &it) {
        const int upto = kv_scan(mine);
        const uint64_t in = __ballot(before + upto > w);
        if (in) {
            const int l = __builtin_ctzll(in);
            const int n = __builtin_amdgcn_readlane(mine, l), u = __builtin_amdgcn_readlane(upto, l);
            const int i = w - (before + u - n);
            /* row bounds that overlap can add up past an int */
            it = {i >= 0 && i < n ? b0 + l : -1, i, n, before + u - n};
            return true;
        }
        before += __builtin_amdgcn_readlane(upto, 63);
        return false;
    };
    KvItem it = {-1, 0, 0, 0};
    if (B <= 64) {
        scan(0, lane < B ? count(lane) : 0, it);
        return it;
    }
    for (int b0 = 0; b0 < B; b0 += 256) {     /* four rounds' reads at once */
        int mine[4];
#pragma unroll
        for (int u = 0; u < 4; u++) mine[u] = b0 + 64 * u + lane < B ? count(b0 + 64 * u + lane) : 0;
#pragma unroll
        for (int u = 0; u < 4; u++)
            if (scan(b0 + 64 * u, mine[u], it)) return it;
    }
    return it;
}
#endif

#endif
