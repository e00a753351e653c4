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

/* A group takes 32 NW rows of one sequence and key head, a row being a (token, query head of the group) pair: the heads
 * that share keys lie side by side, so a tile of few tokens wastes little of the causal border.  A wave holds 32 rows as the
 * columns of S^T = K Q^T and of O^T = V^T P^T (32 x 32 x 16 products).  Keys and values come 64 positions at a time by direct
 * loads into LDS, in units of a kilobyte that are one operand each, two stages: the next 64 are under way while these are
 * used.
 *
 * Row i of a key operand is position 8 h + 4 u + e of its block for i = 8 u + 4 h + e: a lane's scores are then 8
 * consecutive positions a block, its operand of the second product.
 *
 * A masked place's value may be infinite or NaN, and its weight 0 does not silence it: in tiles with a border the values that
 * are not finite leave LDS, and rows that see them get them at the end, value by value (rare).
 */
template <class T, int HD, int NW>
__global__ __launch_bounds__(NW * 64, HD <= 128 ? 2 : 1) void k_kv_prompt(PromptArgs a) {
    typedef typename KvType<T>::x8 x8;
    constexpr int KS = HD / 16, DT = HD / 32;
    constexpr int UNITS = 4 * KS;            /* of a stage: 2 KS of keys, 4 DT of values */
    static_assert(NW == 4, "how a stage is dealt");
    __shared__ __attribute__((aligned(1024))) uint8_t s_buf[2][UNITS * 1024];
    __shared__ int s_odd;                    /* first tile whose product left values out */
    const KvView &c = a.c;
    const int tid = threadIdx.x, lane = tid & 63, wave = kv_uniform(tid >> 6), col = lane & 31, h = lane >> 5;
    const int kvh = (int)(blockIdx.x % (uint32_t)c.heads), G = a.G;
    const KvItem it = kv_find(c.B, (int)(blockIdx.x / (uint32_t)c.heads), [&](int b) {
        return (int)kv_prompt_items(kv_rows(c, b).n, G, 32 * NW);
    });
    if (it.b < 0) return;
    const KvRows rows = kv_rows(c, it.b);
    const int64_t len = kv_len(c, it.b), cap = kv_cap(c);
    const int nrow = (int)(rows.n * G), row0 = (it.n - 1 - it.i) * 32 * NW;    /* the longest first */
    const int64_t p0 = len - rows.n;
    const int present = (int)(len < cap ? len : cap);
    const int32_t *table = c.tables + it.b * c.table_stride;

    /* the lane's row, its last visible position (-1: none) */
    const int row = row0 + 32 * wave + col, token = row / G;
    const bool real = row < nrow;
    auto limit = [&](int token) {
        const int64_t p = p0 + token;
        return (int)(p < 0 ? -1 : p < present ? p : present - 1);
    };
    const int lim = real ? limit(token) : -1;
    auto last_of = [&](int r) { return limit((r < nrow ? r : nrow - 1) / G); };
    const int end = last_of(row0 + 32 * NW - 1) + 1;             /* positions that the group needs */
    const int gfirst = limit(row0 / G), wfirst = limit((row0 + 32 * wave) / G), wend = row0 + 32 * wave < nrow ? last_of(row0 + 32 * wave + 31) + 1 : 0;
    const int tiles = (end + 63) / 64;

    const int64_t H = (int64_t)G * c.heads;
    const int64_t mine = (rows.first + token) * 1;
    x8 qf[KS];
#pragma unroll
    for (int ks = 0; ks < KS; ks++) {
        u32x4 v = {0, 0, 0, 0};
        if (real) v = kv_load8((const T *)a.q + mine * a.qstride + (int64_t)(kvh * G + row - token * G) * HD + 16 * ks + 8 * h);
        qf[ks] = kv_bits<x8>(v);
    }

    /* A stage's units: wave 0 and 1 load the keys of 32 positions each (KS units of 16 values), wave 2 and 3 the values of
     * two blocks each (DT units of 32 values).  Every wave looks its own two blocks' pages up, and whether all four are there. */
    const int i16 = col & 15, krow = 8 * ((i16 >> 2) & 1) + 4 * (i16 >> 3) + (i16 & 3);
    const bool kwave = wave < 2;
    const int off = kwave ? kv_key_at(krow, 0) + 8 * h : kv_value_at(0, col) + 8 * h, step = kwave ? 256 : 512;
    const GAS T *const src = (const GAS T *)(kwave ? a.k : a.v) + off;
    const int lastb = end > 0 ? (end - 1) / KV_BLOCK : 0;
    struct Pages {
        int p0, p1, p2, p3;
    };
    auto pages = [&](int tile) {
        const CAS int32_t *t = (const CAS int32_t *)table;
        auto one = [&](int s) {
            const int blk = 4 * tile + s;
            return t[(blk < lastb ? blk : lastb) >> c.sh];
        };
        return Pages{one(0), one(1), one(2), one(3)};
    };
    struct Blocks {
        int64_t b0, b1;   /* this wave's */
        int ok;           /* bit s: block s is a page's */
    };
    auto blocks = [&](Pages p, int tile) {
        auto at = [&](int page, int s) {
            const int blk = 4 * tile + s;
            const int64_t at = kv_block(c, page, blk < lastb ? blk : lastb, kvh);
            return at >= 0 ? at : 0;      /* inside the cache; masked */
        };
        const uint32_t n = (uint32_t)c.n_pages;
        const int ok = ((uint32_t)p.p0 < n ? 1 : 0) | ((uint32_t)p.p1 < n ? 2 : 0) | ((uint32_t)p.p2 < n ? 4 : 0) |
                       ((uint32_t)p.p3 < n ? 8 : 0);
        const int w = wave & 1;
        return Blocks{at(w ? p.p2 : p.p0, 2 * w), at(w ? p.p3 : p.p1, 2 * w + 1), ok};
    };
    auto load = [&](Blocks n, uint8_t *to) {
        const GAS T *p0 = src + (kwave && (col & 16) ? n.b1 : n.b0);
        const GAS T *p1 = kwave ? p0 + 256 * DT : src + n.b1;
        to += wave * KS * 1024;
#pragma unroll
        for (int j = 0; j < KS; j++)
            __builtin_amdgcn_global_load_lds((const GAS void *)((j < DT ? p0 : p1) + step * (j < DT ? j : j - DT)),
                                             (LAS void *)(to + j * 1024), 16, 0, 0);
    };

    f32x16 o[DT];
#pragma unroll
    for (int dt = 0; dt < DT; dt++) o[dt] = f32x16{0};
    float m = -INFINITY, l = 0.0f;
    if (tid == 0) s_odd = tiles;

    int ok = 0;
    Pages next = {0, 0, 0, 0};
    if (tiles > 0) {
        const Blocks n = blocks(pages(0), 0);
        load(n, s_buf[0]);
        ok = n.ok;
        next = pages(1);
    }
    for (int tile = 0; tile < tiles; tile++) {
        __builtin_amdgcn_s_waitcnt(0);      /* this stage's own loads; the barrier brings the other waves' */
        __syncthreads();
        uint8_t *buf = s_buf[tile & 1];
        const int here = ok;
        if (tile + 1 < tiles) {
            const Blocks n = blocks(next, tile + 1);
            load(n, s_buf[(tile + 1) & 1]);
            ok = n.ok;
        }
        if (tile * 64 + 63 > gfirst || here != 15) {
            /* a border: no value that is masked for some row may disturb its product.  Wave w cleans block w. */
            const int left = ((here >> wave) & 1) ? present - (tile * 64 + 16 * wave + 8 * h) : 0;
            bool odd = false;
#pragma unroll
            for (int dt = 0; dt < DT; dt++) {
                u32x4 *at = (u32x4 *)(buf + (2 * KS + wave * DT + dt) * 1024 + lane * 16);
                u32x4 v = *at;
#pragma unroll
                for (int w = 0; w < 4; w++) {
                    constexpr uint32_t E = KvType<T>::EXP;
                    const uint32_t there = (2 * w < left ? 0xFFFFu : 0u) | (2 * w + 1 < left ? 0xFFFF0000u : 0u), x = v[w] & there;
                    const uint32_t finite = ((x & E) == E ? 0u : 0xFFFFu) | ((x & (E << 16)) == E << 16 ? 0u : 0xFFFF0000u);
                    odd |= finite != 0xFFFFFFFFu;
                    v[w] = x & finite;
                }
                *at = v;
            }
            if (__any(odd) && lane == 0) atomicMin(&s_odd, tile);
            __syncthreads();
        }
        const int base = tile * 64;
        if (base >= wend) {
            next = pages(tile + 2);
            continue;
        }
        const uint8_t *kb = buf + lane * 16, *vb = buf + 2 * KS * 1024 + lane * 16;
        f32x16 s[2];
#pragma unroll
        for (int t = 0; t < 2; t++) {
            s[t] = f32x16{0};
#pragma unroll
            for (int ks = 0; ks < KS; ks++)
                s[t] = KvType<T>::mma(*(const x8 *)(kb + (t * KS + ks) * 1024), qf[ks], s[t]);
        }
        __builtin_amdgcn_sched_barrier(0);
        next = pages(tile + 2);    /* scalar loads: behind the reads of LDS, which one counter waits for too */
        const bool whole = base + 63 <= wfirst && here == 15;
        if (!whole) {
#pragma unroll
            for (int t = 0; t < 2; t++)
#pragma unroll
                for (int r = 0; r < 16; r++) {
                    const int p = base + 32 * t + 16 * (r >> 3) + 8 * h + (r & 7);
                    const bool see = p <= lim && ((here >> (2 * t + (r >> 3))) & 1);
                    s[t][r] = see ? s[t][r] : -INFINITY;
                }
        }
        float top = s[0][0];
#pragma unroll
        for (int t = 0; t < 2; t++)
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
        x8 p[4];
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
            for (int r = 0; r < 16; r++) {
                const float e = __builtin_amdgcn_exp2f(fmaf(s[t][r], a.scale2, -sub));
                l += e;
                p[2 * t + (r >> 3)][r & 7] = (T)e;    /* as many bits as the values it is multiplied with */
            }
#pragma unroll
        for (int dt = 0; dt < DT; dt++)
#pragma unroll
            for (int ks = 0; ks < 4; ks++)
                o[dt] = KvType<T>::mma(*(const x8 *)(vb + (ks * DT + dt) * 1024), p[ks], o[dt]);
    }
    __syncthreads();
    const int odd_from = kv_uniform(s_odd);
    if (odd_from < tiles) {
        /* Rows that see a value that is not finite, from the first tile that left one out; where a later tile had it in its
         * product it is added once more, which changes nothing. */
#pragma unroll 1
        for (int blk = 4 * odd_from; blk <= (wend - 1) / KV_BLOCK; blk++) {
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
    l += __shfl_xor(l, 32, 64);
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

constexpr int TILE = 128;    /* rows of a group */

template <class T, int HD> void launch(const PromptArgs &a, int64_t B, hipStream_t s) {
    const dim3 grid((unsigned)(kv_prompt_most(a.c.rows, B, a.G, TILE) * a.c.heads));
    hipLaunchKernelGGL((k_kv_prompt<T, HD, TILE / 32>), grid, dim3(TILE * 2), 0, s, a);
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
    if (!(scale > 0.0f) || scale > 3.0e38f) return tlmh_seterr(TLM_HIP_EINVAL, "kv_prompt: scale must be finite and positive");
    if (b->B == 0 || b->rows == 0) return TLM_HIP_OK;
    if (!q || !out) return tlmh_seterr(TLM_HIP_EINVAL, "kv_prompt: NULL argument");
    if (q_stride < (int64_t)heads * c->head_dim && b->rows > 1)
        return tlmh_seterr(TLM_HIP_EINVAL, "kv_prompt: row stride %lld below %lld", (long long)q_stride,
                           (long long)heads * c->head_dim);
    if (!aligned(q, 2) || !aligned(out, (size_t)type_bytes(out_dt)))
        return tlmh_seterr(TLM_HIP_EINVAL, "kv_prompt: q and out must have their type's alignment");
    if (kv_prompt_most(b->rows, b->B, heads / c->kv_heads, TILE) * c->kv_heads > (1 << 23))
        return tlmh_seterr(TLM_HIP_ERANGE, "kv_prompt: %lld rows of %lld sequences are too many for one launch",
                           (long long)b->rows, (long long)b->B);
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
