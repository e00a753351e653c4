/* hip_kv_prompt.hip - causal attention of prompts packed end to end, over the paged cache (the reference runs its decode
 * step per prompt token, src/lib/tlm_model.c:1105-1113, attn_heads :683-749).  Layout and work items: tlm_hip_kv.h. */
#include "tlm_hip_kv.h"

namespace {

struct PromptArgs {
    KvView c;
    const void *q, *k, *v;
    void *out;
    int64_t qstride;
    float *part, *ml;        /* parts > 1: [tile and key head][parts][rows][HD] sums, [..][2] maximum and weight */
    float scale2;            /* scale log2(e) */
    int G, out_dt, parts;
};

/* Powers of two of weight from which a maximum is far */
constexpr float KV_FAR = 4096.0f;

/* What a page number outside the cache stands for: its positions are masked, and a finite value times weight 0 is 0 */
__device__ const u32x4 kv_nothing[KV_BLOCK * 256 * 2 / 16] = {};

/* Tile w of `tile` (token, head) rows: its sequence, its first row and what its rows see */
struct PromptTile {
    int b, nrow, row0, present, end;
    KvRows rows;
    int64_t p0;
    __device__ __forceinline__ int limit(int token) const {      /* last position that a token sees (-1: none) */
        const int64_t p = p0 + token;
        return (int)(p < 0 ? -1 : p < present ? p : present - 1);
    }
    __device__ __forceinline__ int last_of(int r, int G) const { return limit((r < nrow ? r : nrow - 1) / G); }
    __device__ __forceinline__ PromptTile(const KvView &c, int G, int w, int tile) {
        const KvItem it = kv_find(c.B, w, [&](int b) { return (int)kv_prompt_items(kv_rows(c, b).n, G, tile); });
        b = it.b;
        if (b < 0) return;
        rows = kv_rows(c, b);
        const int64_t len = kv_len(c, b), cap = kv_cap(c);
        nrow = (int)(rows.n * G);
        row0 = (it.n - 1 - it.i) * tile;      /* the longest first */
        p0 = len - rows.n;
        present = (int)(len < cap ? len : cap);
        end = last_of(row0 + tile - 1, G) + 1;
    }
};
/* stages of each of `parts` parts: a whole number for every wave */
__device__ __forceinline__ int prompt_part(int tiles, int parts, int sg) {
    const int per = (tiles + parts - 1) / parts;
    return per < sg ? sg : (per + sg - 1) / sg * sg;
}

/* A group of four waves takes 32 RG rows of one sequence and key head (RG = 4 / SG), a row being a (token, query head of
 * the group) pair: the heads that share keys lie side by side, so a tile of few tokens wastes little of the causal border.
 * A wave holds 32 rows as the columns of S^T = K Q^T and of O^T = V^T P^T (32 x 32 x 16 products), and takes every SG-th
 * stage of 32 TP positions; the SG waves of the same rows add their sums through LDS at the end.  RG waves share a stage: keys
 * and values come by direct loads into LDS, in units of a kilobyte that are one operand each; the next stage is under way
 * while this one is used.
 *
 * Row i of a key operand is position 8 h + 4 u + e of its block for i = 8 u + 4 h + e: a lane's scores are then 8
 * consecutive positions a block, its operand of the second product.
 *
 * 16384 tokens, 32 heads on 4 of 128: 2.09 to 2.19 ms, 1004 to 1052 TFLOP/s (the library's large product 1337).  Matrix
 * instructions run in 50% of a SIMD's cycles, vector ones issue in 38%, and with two waves a SIMD they hardly overlap; three
 * waves (stages of 32 positions), other orders of the loops and raised priorities for either part changed nothing.
 *
 * A masked place's value may be infinite or NaN, and its weight 0 does not silence it: in stages with a border the values
 * that are not finite leave LDS, and rows that see them get them at the end, value by value (rare).  So do rows with sums that
 * are not finite, which may be an infinity times a weight of 0. */
template <class T, int HD, int SG, int TP, bool PARTS>
__global__ __launch_bounds__(256, (SG == 4 && HD > 64) || (SG == 2 && HD > 128) ? 1 : 2) void k_kv_prompt(PromptArgs a) {
    typedef typename KvType<T>::x8 x8;
    constexpr int RG = 4 / SG, ROWS = 32 * RG;
    constexpr int KS = HD / 16, DT = HD / 32;
    constexpr int POS = 32 * TP, BLOCKS = 2 * TP;      /* positions of a stage */
    constexpr int UNITS = 2 * TP * KS;                 /* of a stage: TP KS of keys, BLOCKS DT of values */
    constexpr int ALL = (1 << BLOCKS) - 1;
    /* two objects: reads of one stage do not wait for the loads into the other */
    __shared__ __attribute__((aligned(1024))) uint8_t s_even[SG * UNITS * 1024], s_odds[SG * UNITS * 1024];
    __shared__ int s_odd;                    /* first stage whose product left values out */
    __shared__ float s_ml[2 * RG][2][32];    /* SG > 1 */
    const KvView &c = a.c;
    const int tid = threadIdx.x, lane = tid & 63, wave = kv_uniform(tid >> 6), col = lane & 31, h = lane >> 5;
    const int rg = wave % RG, sg = wave / RG;
    const int kvh = (int)(blockIdx.x % (uint32_t)c.heads), G = a.G, y = (int)(blockIdx.x / (uint32_t)c.heads);
    const int w = PARTS ? y / a.parts : y, mypart = PARTS ? y % a.parts : 0;
    const PromptTile pt(c, G, w, ROWS);
    if (pt.b < 0) return;
    const KvRows &rows = pt.rows;
    const int nrow = pt.nrow, row0 = pt.row0, present = pt.present;
    const int32_t *table = c.tables + pt.b * c.table_stride;

    /* the lane's row, its last visible position (-1: none) */
    const int row = row0 + 32 * rg + col, token = row / G;
    const bool real = row < nrow;
    const int lim = real ? pt.limit(token) : -1;
    const int end = pt.end;                                   /* positions that the group needs */
    const int gfirst = pt.limit(row0 / G), wfirst = pt.limit((row0 + 32 * rg) / G);
    const int wend = row0 + 32 * rg < nrow ? pt.last_of(row0 + 32 * rg + 31, G) + 1 : 0;
    const int tiles = (end + POS - 1) / POS;
    const int per = PARTS ? prompt_part(tiles, a.parts, SG) : tiles;
    const int t0 = mypart * per, t1 = tiles - t0 < per ? tiles : t0 + per;     /* this group's stages */
    if (PARTS && mypart > 0 && t0 >= tiles) return;

    const int64_t H = (int64_t)G * c.heads;
    x8 qf[KS];
#pragma unroll
    for (int ks = 0; ks < KS; ks++) {
        u32x4 v = {0, 0, 0, 0};
        if (real)
            v = kv_load8((const T *)a.q + (rows.first + token) * a.qstride + (int64_t)(kvh * G + row - token * G) * HD +
                         16 * ks + 8 * h);
        qf[ks] = kv_bits<x8>(v);
    }

    const int i16 = col & 15, krow = 8 * ((i16 >> 2) & 1) + 4 * (i16 >> 3) + (i16 & 3);
    const int koff = kv_key_at(krow, 0) + 8 * h, voff = kv_value_at(0, col) + 8 * h;
    const int lastb = end > 0 ? (end - 1) / KV_BLOCK : 0;
    struct Pages {
        int p[BLOCKS];
    };
    auto pages = [&](int tile) {
        const CAS int32_t *t = (const CAS int32_t *)table;
        Pages n;
#pragma unroll
        for (int s = 0; s < BLOCKS; s++) {
            const int blk = BLOCKS * tile + s;
            n.p[s] = t[(blk < lastb ? blk : lastb) >> c.sh];
        }
        return n;
    };
    /* Puts a stage's loads under way; bit s of the result: block s is a page's.  RG waves share the units in order (keys: half t
     * of the positions, 16 values ks; values: block s, 32 values dt): 4 take a quarter each, 2 the keys or the values. */
    auto load = [&](const Pages &n, int tile, uint8_t *to) {
        auto at = [&](const void *base, int s) {
            const int blk = BLOCKS * tile + s;
            const int64_t at = kv_block(c, n.p[s], blk < lastb ? blk : lastb, kvh);
            return at >= 0 ? (const GAS T *)base + at : (const GAS T *)kv_nothing;
        };
        int here = 0;
#pragma unroll
        for (int s = 0; s < BLOCKS; s++) here |= (uint32_t)n.p[s] < (uint32_t)c.n_pages ? 1 << s : 0;
        auto put = [&](const GAS T *src, int u) {
            __builtin_amdgcn_global_load_lds((const GAS void *)src, (LAS void *)(to + u * 1024), 16, 0, 0);
        };
        auto keys = [&](int t, int ks0, int count) {
            const GAS T *b0 = at(a.k, 2 * t), *b1 = at(a.k, 2 * t + 1), *src = (col & 16 ? b1 : b0) + koff;
#pragma unroll
            for (int j = 0; j < count; j++) put(src + 256 * (ks0 + j), t * KS + ks0 + j);
        };
        auto values = [&](int s) {
            const GAS T *src = at(a.v, s) + voff;
#pragma unroll
            for (int dt = 0; dt < DT; dt++) put(src + 512 * dt, TP * KS + s * DT + dt);
        };
        if (RG == 4 && TP == 2) {
            if (rg == 0) keys(0, 0, KS);
            else if (rg == 1) keys(1, 0, KS);
            else if (rg == 2) values(0), values(1);
            else values(2), values(3);
        } else if (RG == 4) {
            if (rg == 0) keys(0, 0, DT);
            else if (rg == 1) keys(0, DT, DT);
            else if (rg == 2) values(0);
            else values(1);
        } else {
            if (RG == 1 || rg == 0) {
                keys(0, 0, KS);
                if (TP == 2) keys(1, 0, KS);
            }
            if (RG == 1 || rg == 1) {
                values(0), values(1);
                if (TP == 2) values(2), values(3);
            }
        }
        return here;
    };

    f32x16 o[DT];
#pragma unroll
    for (int dt = 0; dt < DT; dt++) o[dt] = f32x16{0};
    float m = -INFINITY, l = 0.0f;
    if (tid == 0) s_odd = tiles;

    int ok = 0;
    Pages next = {};
    if (t0 < t1) {
        ok = load(pages(t0 + sg), t0 + sg, s_even + sg * UNITS * 1024);
        next = pages(t0 + SG + sg);
    }
    auto step = [&](int i, uint8_t *stage, uint8_t *other) {
        __builtin_amdgcn_s_waitcnt(0);      /* this stage's own loads; the barrier brings the other waves' */
        __syncthreads();
        const int tile = t0 + SG * i + sg, base = tile * POS, here = ok;
        uint8_t *buf = stage + sg * UNITS * 1024;
        if (t0 + SG * (i + 1) < t1) ok = load(next, tile + SG, other + sg * UNITS * 1024);
        if ((t0 + SG * i + SG) * POS - 1 > gfirst) {
            /* a border: no value that is masked for some row may disturb its product.  The waves of a stage share its blocks. */
            constexpr int EACH = BLOCKS >= RG ? BLOCKS / RG : 1;
            bool odd = false;
            if (rg * EACH < BLOCKS) {
#pragma unroll
                for (int e = 0; e < EACH; e++) {
                    const int s = rg * EACH + e, left = present - (base + 16 * s + 8 * h);
#pragma unroll
                    for (int dt = 0; dt < DT; dt++) {
                        u32x4 *at = (u32x4 *)(buf + (TP * KS + s * DT + dt) * 1024 + lane * 16);
                        u32x4 v = *at;
#pragma unroll
                        for (int w = 0; w < 4; w++) {
                            constexpr uint32_t E = KvType<T>::EXP;
                            const uint32_t there = (2 * w < left ? 0xFFFFu : 0u) | (2 * w + 1 < left ? 0xFFFF0000u : 0u);
                            const uint32_t x = v[w] & there;
                            const uint32_t finite =
                                ((x & E) == E ? 0u : 0xFFFFu) | ((x & (E << 16)) == E << 16 ? 0u : 0xFFFF0000u);
                            odd |= finite != 0xFFFFFFFFu;
                            v[w] = x & finite;
                        }
                        *at = v;
                    }
                }
            }
            if (__any(odd) && lane == 0) atomicMin(&s_odd, tile);
            __syncthreads();
        }
        if (base >= wend) {
            next = pages(tile + 2 * SG);
            return;
        }
        const uint8_t *kb = buf + lane * 16, *vb = buf + TP * KS * 1024 + lane * 16;
        f32x16 s[TP];
#pragma unroll
        for (int t = 0; t < TP; t++) s[t] = f32x16{0};
#pragma unroll
        for (int ks = 0; ks < KS; ks++)
#pragma unroll
            for (int t = 0; t < TP; t++) s[t] = KvType<T>::mma(*(const x8 *)(kb + (t * KS + ks) * 1024), qf[ks], s[t]);
        __builtin_amdgcn_sched_barrier(0);
        next = pages(tile + 2 * SG);    /* scalar loads: behind the reads of LDS, which one counter waits for too */
        const bool whole = base + POS - 1 <= wfirst && here == ALL;
        if (!whole) {
#pragma unroll
            for (int t = 0; t < TP; t++)
#pragma unroll
                for (int r = 0; r < 16; r++) {
                    const int p = base + 32 * t + 16 * (r >> 3) + 8 * h + (r & 7);
                    const bool see = p <= lim && ((here >> (2 * t + (r >> 3))) & 1);
                    s[t][r] = see ? s[t][r] : -INFINITY;
                }
        }
        float top = s[0][0];
#pragma unroll
        for (int t = 0; t < TP; t++)
#pragma unroll
            for (int r = 0; r < 16; r++) top = fmaxf(top, s[t][r]);
        if (__any(kv_rises(top, m, a.scale2))) {
            top = fmaxf(top, __shfl_xor(top, 32, 64));
            /* each row by its own scores: another's do not show in its bits */
            const float to = kv_rises(top, m, a.scale2) ? top : m, f = to == m ? 1.0f : kv_factor(m, to, a.scale2);
            m = to;
            l *= f;
#pragma unroll
            for (int dt = 0; dt < DT; dt++) o[dt] *= f;
        }
        /* scale2 (s - m) + SHIFT.  Near 0 as one operation, scale2 s - (scale2 m - SHIFT), off by 2^-24 of the score; a row
         * whose maximum is far takes the difference first (by itself: the others' bits stay). */
        const float from = m == -INFINITY ? 0.0f : m, zfrom = from * a.scale2;
        const bool far = fabsf(zfrom) > KV_FAR;
        const float add = far ? KvType<T>::SHIFT : KvType<T>::SHIFT - zfrom;
        if (__any(far)) {
            const float first = far ? from : 0.0f;
#pragma unroll
            for (int t = 0; t < TP; t++)
#pragma unroll
                for (int r = 0; r < 16; r++) s[t][r] -= first;
        }
        x8 p[BLOCKS];
#pragma unroll
        for (int t = 0; t < TP; t++)
#pragma unroll
            for (int r = 0; r < 16; r++) {
                const float e = __builtin_amdgcn_exp2f(fmaf(s[t][r], a.scale2, add));
                l += e;
                /* as many bits as the values it is multiplied with: a bf16 result is off by a third more than by its own
                 * rounding (2.1e-3 for 1.6e-3).  Two numbers a weight, as in decode, take 35% more time at 16384 tokens. */
                p[2 * t + (r >> 3)][r & 7] = (T)e;
            }
#pragma unroll
        for (int ks = 0; ks < BLOCKS; ks++)
#pragma unroll
            for (int dt = 0; dt < DT; dt++)
                o[dt] = KvType<T>::mma(*(const x8 *)(vb + (ks * DT + dt) * 1024), p[ks], o[dt]);
    };
    for (int i = 0; t0 + SG * i < t1; i += 2) {
        step(i, s_even, s_odds);
        if (t0 + SG * (i + 1) < t1) step(i + 1, s_odds, s_even);
    }
    l += __shfl_xor(l, 32, 64);
    __syncthreads();
    /* the splits' sums, half of them at a time, always in the same order */
#pragma unroll
    for (int half = SG / 2; half >= 1; half >>= 1) {
        f32x4 *const at = (f32x4 *)(s_even) + ((sg & (half - 1)) * RG + rg) * DT * 4 * 64 + lane;
        float(*const ml)[32] = s_ml[(sg & (half - 1)) * RG + rg];
        if (sg >= half && sg < 2 * half) {
#pragma unroll
            for (int dt = 0; dt < DT; dt++)
#pragma unroll
                for (int r = 0; r < 4; r++)
                    at[(dt * 4 + r) * 64] = f32x4{o[dt][4 * r], o[dt][4 * r + 1], o[dt][4 * r + 2], o[dt][4 * r + 3]};
            if (h == 0) {
                ml[0][col] = m;
                ml[1][col] = l;
            }
        }
        __syncthreads();
        if (sg < half) {
            const float om = ml[0][col], ol = ml[1][col], to = fmaxf(m, om);
            const float fm = kv_factor(m, to, a.scale2), fo = kv_factor(om, to, a.scale2);
            m = to;
            l = l * fm + ol * fo;
#pragma unroll
            for (int dt = 0; dt < DT; dt++)
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const f32x4 w = at[(dt * 4 + r) * 64];
#pragma unroll
                    for (int e = 0; e < 4; e++) o[dt][4 * r + e] = o[dt][4 * r + e] * fm + w[e] * fo;
                }
        }
        __syncthreads();
    }
    if (sg > 0) return;
    const int odd_from = kv_uniform(s_odd);
    f32x4 z = {0, 0, 0, 0};
#pragma unroll
    for (int dt = 0; dt < DT; dt++)
#pragma unroll
        for (int r = 0; r < 16; r++) z[r & 3] = fmaf(o[dt][r], 0.0f, z[r & 3]);
    const float none = z[0] + z[1] + (z[2] + z[3]);
    const bool all = __any(none != none && l == l);
    if (all || odd_from < tiles) {
        /* The values that are not finite in what the wave's rows see, all of it or from the first stage that left some out, 32
         * of head_dim at a time and four blocks' reads together; blocks that hold some once more, value by value.  Two bits a
         * sum: one for each sign, both for NaN.  16384 tokens with a NaN at the first: 7.0 ms for 2.4. */
        const int first = BLOCKS * (all ? t0 : odd_from);
        const int behind = wend == 0 ? 0 : BLOCKS * t1 <= lastb ? BLOCKS * t1 : lastb + 1;
        uint32_t found[DT];
#pragma unroll
        for (int dt = 0; dt < DT; dt++) {
            uint32_t f = 0;
#pragma unroll 1
            for (int b0 = first; b0 < behind; b0 += 4) {
                u32x4 x[4];
#pragma unroll
                for (int u = 0; u < 4; u++) {
                    const int blk = b0 + u < behind ? b0 + u : behind - 1;
                    const int64_t at = kv_block(c, table[blk >> c.sh], blk, kvh);
                    x[u] = at < 0 ? u32x4{0, 0, 0, 0} : *(const u32x4 *)((const T *)a.v + at + 512 * dt + 8 * lane);
                }
                int odd = 0;
#pragma unroll
                for (int u = 0; u < 4; u++) odd |= __any(b0 + u < behind && kv_any_odd<T>(x[u])) ? 1 << u : 0;
                for (; odd; odd &= odd - 1) {
                    const int blk = b0 + __builtin_ctz(odd);
                    const uint16_t *v = (const uint16_t *)a.v + kv_block(c, table[blk >> c.sh], blk, kvh) + 64 * h;
#pragma unroll 1
                    for (int p = 0; p < KV_BLOCK; p++) {
                        const bool sees = blk * KV_BLOCK + p <= lim;
#pragma unroll
                        for (int r = 0; r < 16; r++) {
                            const uint32_t e = kv_odd<T>(v[kv_value_at(p, 32 * dt + 8 * (r >> 2) + (r & 3))]);
                            f |= sees ? e << 2 * r : 0u;
                        }
                    }
                }
                if (!__any(f != ~0u && lim >= (b0 + 4) * KV_BLOCK)) break;     /* all that is left to find out is NaN */
            }
            found[dt] = f;
        }
#pragma unroll
        for (int dt = 0; dt < DT; dt++)
#pragma unroll
            for (int r = 0; r < 16; r++) o[dt][r] = kv_put_odd(o[dt][r], found[dt] >> 2 * r & 3);
    }
    /* No weight at all, though the row reaches into the group's positions: is one of them a page's?  (rare) */
    const int64_t from = (int64_t)t0 * POS;
    if (__any(l == 0.0f && lim >= from)) {
        const int last = BLOCKS * t1 - 1 < lastb ? BLOCKS * t1 - 1 : lastb;
        int named = last + 1;          /* the first block that is */
        for (int b0 = BLOCKS * t0; b0 <= last; b0 += 64) {
            const int page = b0 + lane <= last ? table[(b0 + lane) >> c.sh] : -1;
            const uint64_t in = __ballot((uint32_t)page < (uint32_t)c.n_pages);
            if (in) {
                named = b0 + __builtin_ctzll(in);
                break;
            }
        }
        if (l == 0.0f && named <= last && named * KV_BLOCK <= lim) m = KV_LOWEST;
    }
    if (!real) return;
    if (PARTS && tiles > per) {
        const int64_t at = (((int64_t)w * c.heads + kvh) * a.parts + mypart) * ROWS + 32 * rg + col;
#pragma unroll
        for (int dt = 0; dt < DT; dt++)
#pragma unroll
            for (int r = 0; r < 4; r++)
                *(f32x4 *)(a.part + at * HD + 32 * dt + 8 * r + 4 * h) =
                    f32x4{o[dt][4 * r], o[dt][4 * r + 1], o[dt][4 * r + 2], o[dt][4 * r + 3]};
        if (h == 0) {
            a.ml[2 * at] = m;
            a.ml[2 * at + 1] = l;
        }
        return;
    }
    const float inv = kv_inverse(l, m);
    const int64_t at = ((rows.first + token) * H + kvh * G + (row - token * G)) * HD;
#pragma unroll
    for (int dt = 0; dt < DT; dt++)
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const float v[4] = {o[dt][4 * r] * inv, o[dt][4 * r + 1] * inv, o[dt][4 * r + 2] * inv, o[dt][4 * r + 3] * inv};
            kv_store(a.out, a.out_dt, at + 32 * dt + 8 * r + 4 * h, v);
        }
}

/* The parts of a tile's rows, in order: a group a tile and key head, HD / 4 threads a row. */
template <int HD, int SG, int TP> __global__ __launch_bounds__(256) void k_kv_prompt_join(PromptArgs a) {
    constexpr int ROWS = 128 / SG, L4 = HD / 4, EACH = 256 / L4;
    const KvView &c = a.c;
    const int kvh = (int)(blockIdx.x % (uint32_t)c.heads), w = (int)(blockIdx.x / (uint32_t)c.heads), G = a.G;
    const PromptTile pt(c, G, w, ROWS);
    if (pt.b < 0) return;
    const int tiles = (pt.end + 32 * TP - 1) / (32 * TP), per = prompt_part(tiles, a.parts, SG), n = (tiles + per - 1) / per;
    if (n <= 1) return;
    const int e = threadIdx.x % L4 * 4, r0 = threadIdx.x / L4;
    if (r0 >= EACH) return;
    const int64_t H = (int64_t)G * c.heads, at0 = ((int64_t)w * c.heads + kvh) * a.parts * ROWS;
    for (int r = r0; r < ROWS && pt.row0 + r < pt.nrow; r += EACH) {
        f32x4 o = {0, 0, 0, 0};
        float m = -INFINITY, l = 0.0f;
#pragma unroll 4
        for (int i = 0; i < n; i++) {
            const int64_t at = at0 + (int64_t)i * ROWS + r;
            const float mi = a.ml[2 * at], li = a.ml[2 * at + 1];
            const f32x4 oi = *(const f32x4 *)(a.part + at * HD + e);
            const float to = fmaxf(m, mi), f = kv_factor(m, to, a.scale2), fi = kv_factor(mi, to, a.scale2);
            o = o * kv_not_zero(f) + oi * kv_not_zero(fi);
            l = l * f + li * fi;
            m = to;
        }
        const int row = pt.row0 + r, token = row / G;
        const float inv = kv_inverse(l, m);
        const float v[4] = {o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv};
        kv_store(a.out, a.out_dt, ((pt.rows.first + token) * H + kvh * G + (row - token * G)) * HD + e, v);
    }
}

/* Rows of a group: 128 where that many groups fill the chip (two fit a compute unit; past 128 wide, where of those with 64
 * rows only one does, from half as many on); else 64, the positions dealt to two waves, or 32 and four, while all groups
 * still run at once: a stage takes a lone wave about a microsecond whatever its rows.  us with 128 / 64 / 32 rows, 32 heads on
 * 4 of 128: 4096 tokens 156 / 178 / 395, 2048 59 / 58 / 129, 1024 30 / 24 / 48, 512 19 / 15 / 21, 256 13.3 / 10.6 / 11.2; 128
 * behind 8000 176 / 117 / 80; 8 heads on 2 of 64, 2048 tokens 39 / 26 / 22; 16 on 2 of 256, 4096 tokens 219 / 259, 2048
 * 104 / 77.
 * Where even those leave units idle and the tables reach far (the lengths are the device's), the positions of each tile go to
 * several groups, at least 512 each, and a second launch joins them.  us split / not: 32 heads on 4 of 128, 20 tokens behind
 * 2000 19 / 27, behind 4000 22 / 44, behind 16000 31 / 152; 100 behind 4000 34 / 47, 300 behind 4000 53 / 68; 16 on 2 of 256,
 * 20 behind 4000 54 / 113.  (1024 each: 24, 26, 32; 256 each: 19, 23, 32.) */
struct PromptPlan {
    int sg, parts;
    int64_t tiles;      /* of all key heads */
};
PromptPlan prompt_plan(const tlm_hip_kv_cache *c, const tlm_hip_kv_batch *b, int heads) {
    const int group = heads / c->kv_heads, hd = c->head_dim;
    const int64_t groups = kv_prompt_most(b->rows, b->B, group, 128) * c->kv_heads;
    int sg = groups > (hd <= 128 ? 512 : 256) ? 1 : groups > (hd <= 64 ? 128 : 64) ? 2 : 4;
    if (sg == 4 && hd > 128) sg = 2;      /* four stages twice are more than the LDS */
    const int64_t tiles = kv_prompt_most(b->rows, b->B, group, 128 / sg) * c->kv_heads, cap = (int64_t)b->table_pages * c->page;
    const int64_t room = (sg == 4 ? (hd <= 64 ? 512 : 256) : hd <= 128 ? 512 : 256) / tiles, reach = cap / 512;
    int64_t parts = sg == 1 || reach < 4 ? 1 : room < reach ? room : reach;
    parts = parts > 16 ? 16 : parts;
    return {sg, parts < 1 ? 1 : (int)parts, tiles};
}
size_t prompt_bytes(const PromptPlan &p, int hd) {
    return p.parts == 1 ? 0 : (size_t)p.tiles * p.parts * (128 / p.sg) * (hd + 2) * 4;
}

template <class T, int HD, int SG, int TP> void launch_sg(const PromptArgs &a, const PromptPlan &p, hipStream_t s) {
    if constexpr (SG > 1) {
        if (p.parts > 1) {
            hipLaunchKernelGGL((k_kv_prompt<T, HD, SG, TP, true>), dim3((unsigned)(p.tiles * p.parts)), dim3(256), 0, s, a);
            hipLaunchKernelGGL((k_kv_prompt_join<HD, SG, TP>), dim3((unsigned)p.tiles), dim3(256), 0, s, a);
            return;
        }
    }
    hipLaunchKernelGGL((k_kv_prompt<T, HD, SG, TP, false>), dim3((unsigned)p.tiles), dim3(256), 0, s, a);
}
template <class T, int HD> void launch(const PromptArgs &a, const PromptPlan &p, hipStream_t s) {
    if (p.sg == 1) return launch_sg<T, HD, 1, HD <= 128 ? 2 : 1>(a, p, s);
    if constexpr (HD <= 128)
        if (p.sg == 4) return launch_sg<T, HD, 4, 1>(a, p, s);
    launch_sg<T, HD, 2, HD <= 64 ? 2 : 1>(a, p, s);
}
template <class T> void prompt(const PromptArgs &a, const PromptPlan &p, hipStream_t s) {
    static void (*const by_width[8])(const PromptArgs &, const PromptPlan &, hipStream_t) = {
        launch<T, 32>, launch<T, 64>, launch<T, 96>, launch<T, 128>,
        launch<T, 160>, launch<T, 192>, launch<T, 224>, launch<T, 256>};
    by_width[a.c.hd / 32 - 1](a, p, s);
}

} // namespace

extern "C" {

size_t tlm_hip_kv_prompt_workspace_bytes(const tlm_hip_kv_cache *c, const tlm_hip_kv_batch *b, int heads) {
    KvView v;
    if (kv_check("kv_prompt_workspace_bytes", c, b, heads, &v) || b->B == 0 || b->rows == 0) return 0;
    return prompt_bytes(prompt_plan(c, b, heads), c->head_dim);
}

int tlm_hip_kv_prompt(const tlm_hip_kv_cache *c, const tlm_hip_kv_batch *b, const void *q, int64_t q_stride, int heads,
                      float scale, int out_dt, void *out, void *workspace, void *stream) {
    PromptArgs a;
    if (int rc = kv_check("kv_prompt", c, b, heads, &a.c)) return rc;
    if (!type_bytes(out_dt)) return tlmh_seterr(TLM_HIP_EUNSUP, "kv_prompt: dtype %d (F32, F16 and BF16 only)", out_dt);
    if (!(scale > 0.0f) || scale > 2.0e38f) return tlmh_seterr(TLM_HIP_EINVAL, "kv_prompt: scale must be finite and positive");
    if (b->B == 0 || b->rows == 0) return TLM_HIP_OK;
    if (!q || !out) return tlmh_seterr(TLM_HIP_EINVAL, "kv_prompt: NULL argument");
    if (q_stride < (int64_t)heads * c->head_dim && b->rows > 1)
        return tlmh_seterr(TLM_HIP_EINVAL, "kv_prompt: row stride %lld below %lld", (long long)q_stride,
                           (long long)heads * c->head_dim);
    if (!aligned(q, 2) || !aligned(out, (size_t)type_bytes(out_dt)))
        return tlmh_seterr(TLM_HIP_EINVAL, "kv_prompt: q and out must have their type's alignment");
    if (kv_prompt_most(b->rows, b->B, heads / c->kv_heads, 128) * c->kv_heads > (1 << 23))
        return tlmh_seterr(TLM_HIP_ERANGE, "kv_prompt: %lld rows of %lld sequences are too many for one launch",
                           (long long)b->rows, (long long)b->B);
    const PromptPlan p = prompt_plan(c, b, heads);
    const size_t need = prompt_bytes(p, c->head_dim);
    if (need && (!workspace || !aligned(workspace, 256)))
        return tlmh_seterr(TLM_HIP_EINVAL, "kv_prompt: needs a workspace of %zu bytes, 256-byte aligned", need);
    if (int rc = tlmh_refuse_failed(FAILED_KV, "kv_prompt")) return rc;
    a.q = q;
    a.k = c->k;
    a.v = c->v;
    a.out = out;
    a.qstride = q_stride;
    a.scale2 = scale * 1.44269504088896341f;
    a.G = heads / c->kv_heads;
    a.out_dt = out_dt;
    a.parts = p.parts;
    a.part = (float *)workspace;
    a.ml = need ? a.part + (size_t)p.tiles * p.parts * (128 / p.sg) * c->head_dim : nullptr;
    if (c->dt == DT_F16) prompt<_Float16>(a, p, (hipStream_t)stream);
    else prompt<__bf16>(a, p, (hipStream_t)stream);
    return tlmh_check(hipGetLastError(), "kv_prompt launch");
}

} // extern "C"
