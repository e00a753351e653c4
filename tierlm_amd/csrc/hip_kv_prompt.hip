/* hip_kv_prompt.hip - causal attention of prompts packed end to end, over the paged cache (the reference runs its decode
 * step per prompt token, src/lib/tlm_model.c:1105-1113, attn_heads :683-749).  Layout and work items: tlm_hip_kv.h. */
#include "tlm_hip_kv.h"

int kv_check(const char *who, const tlm_hip_kv_cache *c, const tlm_hip_kv_batch *b, int heads, KvView *v);

namespace {

struct PromptArgs {
    KvView c;
    const void *q, *k, *v;
    void *out;
    int64_t qstride;
    float scale2;            /* scale log2(e) */
    int G, out_dt;
};

__device__ __forceinline__ void store_out(void *out, int dt, int64_t i, const float (&v)[4]) {
    typedef _Float16 h4 __attribute__((ext_vector_type(4), aligned(2)));
    typedef __bf16 b4 __attribute__((ext_vector_type(4), aligned(2)));
    typedef f32x4 f4 __attribute__((aligned(4)));
    if (dt == DT_F32) *(f4 *)((float *)out + i) = f4{v[0], v[1], v[2], v[3]};
    else if (dt == DT_F16) *(h4 *)((_Float16 *)out + i) = h4{(_Float16)v[0], (_Float16)v[1], (_Float16)v[2], (_Float16)v[3]};
    else *(b4 *)((__bf16 *)out + i) = b4{(__bf16)v[0], (__bf16)v[1], (__bf16)v[2], (__bf16)v[3]};
}

/* What a page number outside the cache stands for: its positions are masked, and a finite value times weight 0 is 0 */
__device__ const u32x4 kv_nothing[KV_BLOCK * 256 * 2 / 16] = {};

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
 * A masked place's value may be infinite or NaN, and its weight 0 does not silence it: in stages with a border the values
 * that are not finite leave LDS, and rows that see them get them at the end, value by value (rare). */
template <class T, int HD, int SG, int TP>
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
    const int kvh = (int)(blockIdx.x % (uint32_t)c.heads), G = a.G;
    const KvItem it = kv_find(c.B, (int)(blockIdx.x / (uint32_t)c.heads), [&](int b) {
        return (int)kv_prompt_items(kv_rows(c, b).n, G, ROWS);
    });
    if (it.b < 0) return;
    const KvRows rows = kv_rows(c, it.b);
    const int64_t len = kv_len(c, it.b), cap = kv_cap(c);
    const int nrow = (int)(rows.n * G), row0 = (it.n - 1 - it.i) * ROWS;    /* the longest first */
    const int64_t p0 = len - rows.n;
    const int present = (int)(len < cap ? len : cap);
    const int32_t *table = c.tables + it.b * c.table_stride;

    /* the lane's row, its last visible position (-1: none) */
    const int row = row0 + 32 * rg + col, token = row / G;
    const bool real = row < nrow;
    auto limit = [&](int token) {
        const int64_t p = p0 + token;
        return (int)(p < 0 ? -1 : p < present ? p : present - 1);
    };
    const int lim = real ? limit(token) : -1;
    auto last_of = [&](int r) { return limit((r < nrow ? r : nrow - 1) / G); };
    const int end = last_of(row0 + ROWS - 1) + 1;             /* positions that the group needs */
    const int gfirst = limit(row0 / G), wfirst = limit((row0 + 32 * rg) / G);
    const int wend = row0 + 32 * rg < nrow ? last_of(row0 + 32 * rg + 31) + 1 : 0;
    const int tiles = (end + POS - 1) / POS;

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
    if (tiles > 0) {
        ok = load(pages(sg), sg, s_even + sg * UNITS * 1024);
        next = pages(SG + sg);
    }
    auto step = [&](int i, uint8_t *stage, uint8_t *other) {
        __builtin_amdgcn_s_waitcnt(0);      /* this stage's own loads; the barrier brings the other waves' */
        __syncthreads();
        const int tile = SG * i + sg, base = tile * POS, here = ok;
        uint8_t *buf = stage + sg * UNITS * 1024;
        if (SG * (i + 1) < tiles) ok = load(next, tile + SG, other + sg * UNITS * 1024);
        if ((SG * i + SG) * POS - 1 > gfirst) {
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
        top *= a.scale2;
        if (__any(top > m + KV_SLACK)) {
            top = fmaxf(top, __shfl_xor(top, 32, 64));
            /* each row by its own scores: another's do not show in its bits */
            const float to = top > m + KV_SLACK ? top : m, f = to == m ? 1.0f : __builtin_amdgcn_exp2f(m - to);
            m = to;
            l *= f;
#pragma unroll
            for (int dt = 0; dt < DT; dt++) o[dt] *= f;
        }
        const float sub = (m == -INFINITY ? 0.0f : m) - KvType<T>::SHIFT;
        x8 p[BLOCKS];
#pragma unroll
        for (int t = 0; t < TP; t++)
#pragma unroll
            for (int r = 0; r < 16; r++) {
                const float e = __builtin_amdgcn_exp2f(fmaf(s[t][r], a.scale2, -sub));
                l += e;
                p[2 * t + (r >> 3)][r & 7] = (T)e;    /* as many bits as the values it is multiplied with */
            }
#pragma unroll
        for (int ks = 0; ks < BLOCKS; ks++)
#pragma unroll
            for (int dt = 0; dt < DT; dt++)
                o[dt] = KvType<T>::mma(*(const x8 *)(vb + (ks * DT + dt) * 1024), p[ks], o[dt]);
    };
    for (int i = 0; SG * i < tiles; i += 2) {
        step(i, s_even, s_odds);
        if (SG * (i + 1) < tiles) step(i + 1, s_odds, s_even);
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
            const float om = ml[0][col], ol = ml[1][col], to = fmaxf(m, om), base = to == -INFINITY ? 0.0f : to;
            const float fm = __builtin_amdgcn_exp2f(m - base), fo = __builtin_amdgcn_exp2f(om - base);
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
    if (odd_from < tiles) {
        /* Rows that see a value that is not finite, from the first stage that left one out; where a later stage had it in its
         * product it is added once more, which changes nothing. */
#pragma unroll 1
        for (int blk = BLOCKS * odd_from; blk <= (wend - 1) / KV_BLOCK; blk++) {
            const int64_t at = kv_block(c, table[blk >> c.sh], blk, kvh);
            if (at < 0) continue;
            const uint16_t *v = (const uint16_t *)a.v + at + 64 * h;
#pragma unroll 1
            for (int p = 0; p < KV_BLOCK; p++) {
                const bool sees = blk * KV_BLOCK + p <= lim;
#pragma unroll
                for (int dt = 0; dt < DT; dt++)
#pragma unroll
                    for (int r = 0; r < 16; r++) {
                        const uint32_t e = v[kv_value_at(p, 32 * dt + 8 * (r >> 2) + (r & 3))], E = KvType<T>::EXP;
                        const float x = (e & 0x7FFFu) > E ? __uint_as_float(0x7FC00000u) : e >> 15 ? -INFINITY : INFINITY;
                        o[dt][r] += sees && (e & E) == E ? x : 0.0f;
                    }
            }
        }
    }
    if (!real) return;
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;    /* a row that sees nothing: zeros */
    const int64_t at = ((rows.first + token) * H + kvh * G + (row - token * G)) * HD;
#pragma unroll
    for (int dt = 0; dt < DT; dt++)
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const float v[4] = {o[dt][4 * r] * inv, o[dt][4 * r + 1] * inv, o[dt][4 * r + 2] * inv, o[dt][4 * r + 3] * inv};
            store_out(a.out, a.out_dt, at + 32 * dt + 8 * r + 4 * h, v);
        }
}

/* Rows of a group: 128 where that many groups fill the chip (two fit a compute unit; past 128 wide, where of those with 64
 * rows only one does, from half as many on); else 64, the positions dealt to two waves, or 32 and four, while all groups
 * still run at once: a stage takes a lone wave about a microsecond whatever its rows.  us with 128 / 64 / 32 rows, 32 heads on
 * 4 of 128: 4096 tokens 156 / 178 / 395, 2048 59 / 58 / 129, 1024 30 / 24 / 48, 512 19 / 15 / 21, 256 13.3 / 10.6 / 11.2; 128
 * behind 8000 176 / 117 / 80; 8 heads on 2 of 64, 2048 tokens 39 / 26 / 22; 16 on 2 of 256, 4096 tokens 219 / 259, 2048
 * 104 / 77. */
int split_of(int64_t rows, int64_t B, int group, int kv_heads, int hd) {
    const int64_t groups = kv_prompt_most(rows, B, group, 128) * kv_heads;
    return groups > (hd <= 128 ? 512 : 256) ? 1 : groups > (hd <= 64 ? 128 : 64) ? 2 : 4;
}

template <class T, int HD, int SG, int TP> void launch_sg(const PromptArgs &a, int64_t B, hipStream_t s) {
    const dim3 grid((unsigned)(kv_prompt_most(a.c.rows, B, a.G, 128 / SG) * a.c.heads));
    hipLaunchKernelGGL((k_kv_prompt<T, HD, SG, TP>), grid, dim3(256), 0, s, a);
}
template <class T, int HD> void launch(const PromptArgs &a, int64_t B, hipStream_t s) {
    const int sg = split_of(a.c.rows, B, a.G, a.c.heads, HD);
    if (sg == 1) return launch_sg<T, HD, 1, HD <= 128 ? 2 : 1>(a, B, s);
    if constexpr (HD <= 128)     /* wider, four stages twice are more than the LDS */
        if (sg == 4) return launch_sg<T, HD, 4, 1>(a, B, s);
    launch_sg<T, HD, 2, HD <= 64 ? 2 : 1>(a, B, s);
}
template <class T> void prompt(const PromptArgs &a, int64_t B, hipStream_t s) {
    static void (*const by_width[8])(const PromptArgs &, int64_t, hipStream_t) = {
        launch<T, 32>, launch<T, 64>, launch<T, 96>, launch<T, 128>, launch<T, 160>, launch<T, 192>, launch<T, 224>, launch<T, 256>};
    by_width[a.c.hd / 32 - 1](a, B, s);
}

bool aligned(const void *p, size_t a) { return ((uintptr_t)p & (a - 1)) == 0; }
int type_bytes(int dt) { return dt == DT_F32 ? 4 : dt == DT_F16 || dt == DT_BF16 ? 2 : 0; }

} // namespace

extern "C" int tlm_hip_kv_prompt(const tlm_hip_kv_cache *c, const tlm_hip_kv_batch *b, const void *q, int64_t q_stride,
                                 int heads, float scale, int out_dt, void *out, void *stream) {
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
    if (int rc = tlmh_refuse_failed(FAILED_KV, "kv_prompt")) return rc;
    a.q = q;
    a.k = c->k;
    a.v = c->v;
    a.out = out;
    a.qstride = q_stride;
    a.scale2 = scale * 1.44269504088896341f;
    a.G = heads / c->kv_heads;
    a.out_dt = out_dt;
    if (c->dt == DT_F16) prompt<_Float16>(a, b->B, (hipStream_t)stream);
    else prompt<__bf16>(a, b->B, (hipStream_t)stream);
    return tlmh_check(hipGetLastError(), "kv_prompt launch");
}
