/* hip_kv.hip - the paged key-value cache: appending a batch's rows, and the attention of one new token a
 * sequence (the reference's attn_heads, src/lib/tlm_model.c:683-749, for many sequences over pages of 16-bit keys and
 * values).  Layout and work items: tlm_hip_kv.h; prompts: hip_kv_prompt.hip. */
#include "tlm_hip_kv.h"

namespace {

/* ---- append ------------------------------------------------------------------
 * A group per block of 16 positions and hpg key heads, one or two: its up to 16 new rows of those heads' queries, keys and
 * values.  16 lanes hold a vector: lane s the pairs j = M s .. M s + M - 1 and their partners at hd / 2 + j (M = hd / 32),
 * so the norm is one 16-lane sum and the rotation stays in the lane.  Vectors go in the order of memory, 16 heads of a row at a time (a
 * row a lane group: 87 us for what takes 75), and values are turned over in registers (8 rows of one value to 16 bytes),
 * so the cache's block is written as whole pieces.
 * 8192 rows of 64 + 8 heads of 128, bf16: 75 us, 4.0 TB/s (64 us from an idle device); 61 rows of a decode step 5 to 6 us, a
 * chain of four reads and a launch. */
struct AppendArgs {
    KvView c;
    const void *x;
    int64_t xstride;
    void *q, *k, *v;
    const float *qw, *kw;
    const double *freq;
    float eps, rope_scale;
    int G, hpg;      /* queries a key head, key heads a group */
};

template <class X> __device__ __forceinline__ float to_f32(X v) { return (float)v; }

/* M consecutive elements at any alignment of the type */
template <int M, class X> __device__ __forceinline__ void load_m(float *v, const X *p) {
    if constexpr (M == 2 || M == 4 || M == 8) {
        typedef X XM __attribute__((ext_vector_type(M), aligned(sizeof(X))));
        const XM x = *(const XM *)p;
#pragma unroll
        for (int m = 0; m < M; m++) v[m] = to_f32((X)x[m]);
    } else {
#pragma unroll
        for (int m = 0; m < M; m++) v[m] = to_f32(p[m]);
    }
}
template <int M, class T> __device__ __forceinline__ void store_m(T *p, const float *v) {
    if constexpr (M == 2 || M == 4 || M == 8) {
        typedef T TM __attribute__((ext_vector_type(M), aligned(sizeof(T))));
        TM x;
#pragma unroll
        for (int m = 0; m < M; m++) x[m] = (T)v[m];
        *(TM *)p = x;
    } else {
#pragma unroll
        for (int m = 0; m < M; m++) p[m] = (T)v[m];
    }
}

template <class X, class T, int M> __global__ __launch_bounds__(256) void k_kv_append(AppendArgs a) {
    constexpr int HD = 32 * M;
    __shared__ float s_cs[KV_BLOCK][HD / 2 + 4], s_sn[KV_BLOCK][HD / 2 + 4];
    const KvView &c = a.c;
    const int tid = threadIdx.x;
    KvItem it = {(int)blockIdx.x, 0, 1, 0};     /* a row a sequence: a block each */
    if (c.cu)
        it = kv_find(c.B, (int)blockIdx.x, [&](int b) {
            const KvRows r = kv_rows(c, b);
            return (int)kv_append_items(r.n, kv_len(c, b));
        });
    if (it.b < 0) return;
    const int kv0 = blockIdx.y * a.hpg, nh = c.heads - kv0 < a.hpg ? c.heads - kv0 : a.hpg;     /* the group's key heads */
    const int H = a.G * c.heads, G = a.G * nh;                                                  /* its queries */
    const KvRows r = kv_rows(c, it.b);
    const int64_t p0 = kv_len(c, it.b) - r.n;                   /* position of the first new row */
    const int64_t blk = kv_floor16(p0) + it.i;
    const int64_t lo = blk * KV_BLOCK > p0 ? blk * KV_BLOCK : p0;
    const int64_t end = blk * KV_BLOCK + KV_BLOCK, hi = end < p0 + r.n ? end : p0 + r.n;
    const int n = (int)(hi - lo);
    const X *x = (const X *)a.x + (r.first + lo - p0) * a.xstride;    /* the block's first row */
    T *q = (T *)a.q + (r.first + lo - p0) * (int64_t)H * HD;
    int64_t at = -1;
    if (blk >= 0 && (blk >> c.sh) < c.table_pages)
        at = kv_block(c, c.tables[it.b * c.table_stride + (blk >> c.sh)], blk, kv0);
    const int64_t head = (int64_t)(KV_BLOCK * HD) << c.sh;      /* from a key head's block to the next one's */

    /* sine and cosine of the block's rows, once.  The angle is a double, less whole turns (2 pi as a sum of two
     * doubles): a far position's fraction of a turn keeps its bits, and the functions take a float in [-pi, pi]. */
    if (a.freq) {
        for (int i = tid; i < n * (HD / 2); i += 256) {
            const int t = i / (HD / 2), j = i % (HD / 2);
            const double ang = (double)(lo + t) * a.freq[j], turns = rint(ang * 0.15915494309189535);
            const double rem = __builtin_fma(-turns, 2.4492935982947064e-16, __builtin_fma(-turns, 6.283185307179586, ang));
            float s, co;
            sincosf((float)rem, &s, &co);
            s_cs[t][j] = co * a.rope_scale;
            s_sn[t][j] = s * a.rope_scale;
        }
        __syncthreads();
    }

    /* norm and rotation of the pairs (u, w) of row t */
    const int sub = tid & 15, grp = tid >> 4;
    auto turn = [&](float (&u)[M], float (&w)[M], const float (&nw)[2 * M], bool norm, int t) {
        if (norm) {
            auto mean = [&](float eps) {
                float ss = 0.0f;
#pragma unroll
                for (int m = 0; m < M; m++) ss = fmaf(u[m], u[m], fmaf(w[m], w[m], ss));
                ss += dpp_f32<DPP_XOR1>(ss);
                ss += dpp_f32<DPP_XOR2>(ss);
                ss += dpp_f32<DPP_HALF_MIRROR>(ss);
                ss += dpp_f32<DPP_MIRROR>(ss);
                return fmaf(ss, 1.0f / HD, eps);
            };
            float s = mean(a.eps);
            const bool odd = !(s > 0x1p-100f && s < 0x1p100f);
            if (__any(odd)) {
                /* squares past a float: that vector times a power of two that brings its largest value near 1 (or to 2^-49: no
                 * further than eps's own square stays finite), which the result does not show (rare) */
                uint32_t top = 0;
#pragma unroll
                for (int m = 0; m < M; m++) {
                    const uint32_t x = __float_as_uint(u[m]) & 0x7FFFFFFFu, y = __float_as_uint(w[m]) & 0x7FFFFFFFu;
                    top = max(top, max(x, y));
                }
                const int e = odd ? max((int)(group_max_u32<16>(top) >> 23) - 127, -100) : 0;
#pragma unroll
                for (int m = 0; m < M; m++) {
                    u[m] = ldexpf(u[m], -e);
                    w[m] = ldexpf(w[m], -e);
                }
                s = mean(ldexpf(a.eps, -2 * e));
            }
            const float f = rsqrtf(s);
#pragma unroll
            for (int m = 0; m < M; m++) {
                u[m] = u[m] * f * nw[m];
                w[m] = w[m] * f * nw[M + m];
            }
        }
        if (a.freq) {
#pragma unroll
            for (int m = 0; m < M; m++) {
                const float c = s_cs[t][M * sub + m], s = s_sn[t][M * sub + m], y = u[m];
                u[m] = fmaf(y, c, -(w[m] * s));
                w[m] = fmaf(w[m], c, y * s);
            }
        }
        if (lo + t < 0) {
#pragma unroll
            for (int m = 0; m < M; m++) u[m] = w[m] = 0.0f;
        }
    };
    auto weights = [&](float (&nw)[2 * M], const float *p) {
        if (!p) return;
        load_m<M>(nw, p + M * sub);
        load_m<M>(nw + M, p + HD / 2 + M * sub);
    };
    /* queries row by row as they lie in memory: 16 lane groups, two vectors of each in flight */
    {
        float nw[2 * M], u0[M], w0[M], u1[M], w1[M];
        weights(nw, a.qw);
        struct At {
            int t, j;
        };
        const int dt = 16 / G, dj = 16 % G;
        auto next = [&](At p) {
            p.t += dt;
            p.j += dj;
            if (p.j >= G) {
                p.j -= G;
                p.t++;
            }
            return p;
        };
        const X *src = x + (int64_t)kv0 * a.G * HD + M * sub;
        T *dst = q + (int64_t)kv0 * a.G * HD + M * sub;
        auto load = [&](float (&u)[M], float (&w)[M], At p) {
            if (p.t >= n) return;
            const X *v = src + p.t * a.xstride + p.j * HD;
            load_m<M>(u, v);
            load_m<M>(w, v + HD / 2);
        };
        auto finish = [&](float (&u)[M], float (&w)[M], At p) {
            if (p.t >= n) return;
            turn(u, w, nw, a.qw != nullptr, p.t);
            T *o = dst + (int64_t)p.t * H * HD + p.j * HD;
            store_m<M>(o, u);
            store_m<M>(o + HD / 2, w);
        };
        At p = {grp / G, grp % G}, p1 = next(p);
        load(u0, w0, p);
        while (p.t < n) {
            load(u1, w1, p1);
            finish(u0, w0, p);
            p = next(p1);
            load(u0, w0, p);
            finish(u1, w1, p1);
            p1 = next(p);
        }
    }
    if (at < 0) return;
    /* keys, a lane group a row and head */
    {
        float nw[2 * M];
        weights(nw, a.kw);
        for (int i = grp; i < n * nh; i += 16) {
            const int t = i / nh, j = i - t * nh;
            float u[M], w[M];
            const X *src = x + t * a.xstride + (int64_t)(H + kv0 + j) * HD + M * sub;
            load_m<M>(u, src);
            load_m<M>(w, src + HD / 2);
            turn(u, w, nw, a.kw != nullptr, t);
            T *o = (T *)a.k + at + j * head;
            const int pos = (int)(lo + t - blk * KV_BLOCK);
            if constexpr (16 % M == 0) {    /* M values of one piece */
                store_m<M>(o + kv_key_at(pos, M * sub), u);
                store_m<M>(o + kv_key_at(pos, HD / 2 + M * sub), w);
            } else {
#pragma unroll
                for (int m = 0; m < M; m++) {
                    o[kv_key_at(pos, M * sub + m)] = (T)u[m];
                    o[kv_key_at(pos, HD / 2 + M * sub + m)] = (T)w[m];
                }
            }
        }
    }
    /* values: a thread per value and half block.  (Read ahead of the angles they take the registers of a wave a SIMD and
     * the queries' loads wait behind them: 8192 rows 75 -> 82 us.) */
    const X *src = x + (int64_t)(H + c.heads + kv0) * HD;
    const int first = (int)(lo - blk * KV_BLOCK), last = first + n;
    for (int i = tid; i < 2 * HD * nh; i += 256) {
        const int j = i / (2 * HD), d = i % HD, half = i / HD % 2 * 8;
        if (half >= last || half + 8 <= first) continue;
        T *o = (T *)a.v + at + j * head;
        float v[8];
#pragma unroll
        for (int p = 0; p < 8; p++)
            v[p] = half + p >= first && half + p < last ? to_f32(src[(half + p - first) * a.xstride + j * HD + d]) : 0.0f;
        if (half >= first && half + 8 <= last) {
            store_m<8>(o + kv_value_at(half, d), v);
        } else {
#pragma unroll
            for (int p = 0; p < 8; p++)
                if (half + p >= first && half + p < last) o[kv_value_at(half + p, d)] = (T)v[p];
        }
    }
}

/* ---- decode --------------------------------------------------------------------
 * out = sum_j p_j v_j / sum_j p_j, p_j = 2^(scale log2(e) (q . k_j - m)), one pass over the cache with the running maximum m.
 * A group takes a part of a sequence's positions for one key head and up to 16 NC of its queries; its NW waves take tiles
 * of 32 positions in turn, straight from memory into the matrix cores' operands (no LDS on the way), the next tile's
 * loads in flight, and merge their sums through LDS at the end.  The bytes of the cache bound it: 64 sequences of up to 8192,
 * 64 heads on 4 of 128, in 102 us (5.4 TB/s, some of it from the memory-side cache; a copy 5.14), one of 131071, 32 on 4, in 50.
 *
 * Shares: the lengths are the device's, so every group works its share out for itself.  All sequences' positions lie end
 * to end in units of 128, and W workers a key head take equal parts of that line, across the sequences' ends: however
 * uneven the lengths are, the groups that fill the chip once end together.  A sequence inside one share is written at
 * once; the parts of the others go to the workspace, and k_kv_join adds a sequence's in order.  Where the tables are short
 * (DECODE_WHOLE) each sequence is a group's and one launch does.  With a fixed number of splits a sequence the 64 ragged ones
 * took 14% longer (129 us for 113, with their join; 106 now). */
struct DecodeArgs {
    KvView c;
    const void *q, *k, *v;
    void *out;
    float *part, *ml;        /* [2 W][heads][HD] sums, [2 W][heads][2] maximum and weight */
    int64_t qstride;
    float scale2;            /* scale log2(e) */
    int G, W, out_dt;
    int hb;                  /* heads of a group of the join */
};

__device__ __forceinline__ int decode_len(const KvView &c, int b) {
    const int64_t len = kv_len(c, b), cap = kv_cap(c);
    return (int)(len < cap ? len : cap);
}
/* The batch's lengths and shares, the same in every group.  Up to 64 sequences are read once, a lane each: what follows
 * waits for one read of memory. */
struct DecodeBatch {
    const KvView &c;
    int mine, upto;       /* B <= 64: lane b's length, and the units up to its sequence's end */
    KvShares sh;
    __device__ __forceinline__ DecodeBatch(const KvView &c_, int W) : c(c_), mine(0), upto(0) {
        const int lane = wave_lane();
        int sum = 0;
        if (few()) {
            if (lane < c.B) {
                mine = decode_len(c, lane);
                sum = kv_units(mine);
            }
        } else {
#pragma unroll 4
            for (int b = lane; b < c.B; b += 64) sum += kv_units(decode_len(c, b));
        }
        upto = kv_scan(sum);
        sh = kv_shares(__builtin_amdgcn_readlane(upto, 63), W);
    }
    __device__ __forceinline__ bool few() const { return c.B <= 64; }
    __device__ __forceinline__ int len(int b) const {
        return few() ? __builtin_amdgcn_readlane(mine, b) : kv_uniform(decode_len(c, b));
    }
    /* the sequence of unit x, and x's number in it; b < 0: there is none */
    __device__ __forceinline__ KvItem find(int x) const {
        if (!few()) return kv_find(c.B, x, [&](int b) { return kv_units(decode_len(c, b)); });
        const uint64_t in = __ballot(wave_lane() < c.B && upto > x);
        if (!in) return {-1, 0, 0, 0};
        const int b = __builtin_ctzll(in), n = kv_units(len(b)), u = __builtin_amdgcn_readlane(upto, b);
        return {b, x - (u - n), n, u - n};
    }
    /* units of the sequences before b */
    __device__ __forceinline__ int before(int b) const {
        if (few()) return __builtin_amdgcn_readlane(upto, b) - kv_units(len(b));
        int sum = 0;
#pragma unroll 4
        for (int i = wave_lane(); i < b; i += 64) sum += kv_units(decode_len(c, i));
        return __builtin_amdgcn_readlane(kv_scan(sum), 63);
    }
};

/* Waves a SIMD that the registers must leave room for: where a sequence is a group's, as many groups a unit as narrow heads
 * allow (three of 32, two of 64 and 160 wide; 96 wide one, and the next when half of its waves are done); shares are a group
 * a unit. */
constexpr int decode_waves(int HD, int NW, bool WHOLE) {
    return NW == 8 ? (HD == 32 ? 6 : HD == 64 ? 4 : HD == 96 ? 3 : 2) : WHOLE && HD == 160 ? 2 : 1;
}
template <class T, int HD, int NC, int NW, bool WHOLE>
__global__ __launch_bounds__(NW * 64, decode_waves(HD, NW, WHOLE)) void k_kv_decode(DecodeArgs a) {
    typedef typename KvType<T>::x8 x8;
    constexpr int KS = HD / 32, DT = HD / 16;    /* steps of the first product, result tiles of the second */
    constexpr int LD = HD + 4;                   /* a merged column in LDS: 16 lanes' float4 on all banks */
    __shared__ float s_o[NW / 2][NC * 16 * LD], s_ml[NW / 2][NC * 16 * 2];
    const KvView &c = a.c;
    const int tid = threadIdx.x, lane = tid & 63, wave = kv_uniform(tid >> 6), col = lane & 15, g = lane >> 4;
    const int worker = blockIdx.x, kvh = blockIdx.y;
    const int col0 = blockIdx.z * NC * 16, ncol = a.G - col0 < NC * 16 ? a.G - col0 : NC * 16;
    auto part = [&](int b, int len, int first, int left) {
        const int32_t *table = c.tables + b * c.table_stride;
        const int units = kv_units(len), take = units - first < left ? units - first : left;
        const int begin = first * KV_UNIT, stop = len - begin < take * KV_UNIT ? len : begin + take * KV_UNIT;
        const int tiles = (stop - begin + 31) / 32;     /* 0: an empty sequence */

        /* queries: column col, values 32 ks + 8 g .. + 7 */
        x8 qf[NC][KS];
#pragma unroll
        for (int n = 0; n < NC; n++)
#pragma unroll
            for (int ks = 0; ks < KS; ks++) {
                const int h = n * 16 + col;
                u32x4 v = {0, 0, 0, 0};
                if (h < ncol)
                    v = kv_load8((const T *)a.q + b * a.qstride + (int64_t)(kvh * a.G + col0 + h) * HD + 32 * ks + 8 * g);
                qf[n][ks] = kv_bits<x8>(v);
            }

        /* A tile's two blocks: row i of key tile t is position 8 (i / 4) + 4 t + i % 4 (block i / 8), so that a lane's scores are
         * the positions 8 g .. 8 g + 7 (block g / 2), which are its operand of the second product. */
        auto key_piece = [](int lane) {          /* + 64 t (four positions) + 512 ks */
            const int col = lane & 15, g = lane >> 4, krow = 8 * (col >> 2) + (col & 3);
            return kv_key_at(krow & 15, 0) + (g >> 1) * 256 + (g & 1) * 8;
        };
        auto value_piece = [](int lane) { return kv_value_at(0, lane & 15) + (lane >> 4 & 1) * 8; };     /* + 256 dt */
        struct Tile {
            u32x4 k[2][KS], v[DT];
            int ok;          /* bit i: block i is a page's */
        };
        /* the wave's page numbers, 32 of its tiles at a time: lane 2 i + j holds block j of its i-th tile */
        int pages = 0;
        auto names = [&](int i0) {
            const int blk = begin / KV_BLOCK + 2 * (wave + NW * (i0 + (lane >> 1))) + (lane & 1);
            const int lastb = (stop - 1) / KV_BLOCK;
            pages = blk <= lastb ? table[blk >> c.sh] : -1;
        };
        auto load = [&](Tile &t, int i) {
            const int b0 = begin / KV_BLOCK + 2 * (wave + NW * i);
            int64_t o0 = kv_block(c, __builtin_amdgcn_readlane(pages, 2 * (i & 31)), b0, kvh);
            int64_t o1 = kv_block(c, __builtin_amdgcn_readlane(pages, 2 * (i & 31) + 1), b0 + 1, kvh);
            t.ok = (o0 >= 0 ? 1 : 0) | (o1 >= 0 ? 2 : 0);
            o0 = o0 < 0 ? 0 : o0;    /* block 0 is inside the cache; what it holds is masked */
            o1 = o1 < 0 ? 0 : o1;
            /* a sequence a group: the lane's places anew for each tile, kept they are the registers that narrow heads lack */
            int own = lane;
            if (WHOLE) asm volatile("" : "+v"(own));
            const GAS T *k = (const GAS T *)a.k + ((own & 8) ? o1 : o0) + key_piece(own);
            const GAS T *v = (const GAS T *)a.v + (own >= 32 ? o1 : o0) + value_piece(own);
#pragma unroll
            for (int ks = 0; ks < KS; ks++) {
                t.k[0][ks] = *(const GAS u32x4 *)(k + 512 * ks);
                t.k[1][ks] = *(const GAS u32x4 *)(k + 512 * ks + 64);
            }
#pragma unroll
            for (int dt = 0; dt < DT; dt++) t.v[dt] = *(const GAS u32x4 *)(v + 256 * dt);
        };

        f32x4 o[NC][DT];
        float m[NC], l[NC];
#pragma unroll
        for (int n = 0; n < NC; n++) {
            m[n] = -INFINITY;
            l[n] = 0.0f;
#pragma unroll
            for (int dt = 0; dt < DT; dt++) o[n][dt] = f32x4{0, 0, 0, 0};
        }
        auto compute = [&](Tile &t, int i) {
            const int p0 = begin + 32 * (wave + NW * i) + 8 * g;     /* the lane's first position */
            const bool whole = p0 - 8 * g + 32 <= stop && t.ok == 3;
            const int left = ((t.ok >> (g >> 1)) & 1) ? stop - p0 : 0;
            if (!whole) {    /* what a masked place holds may be anything, and 0 times it not 0 */
#pragma unroll
                for (int dt = 0; dt < DT; dt++) t.v[dt] = kv_upto(t.v[dt], left);
            }
#pragma unroll
            for (int n = 0; n < NC; n++) {
                f32x4 s[2];
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    s[u] = f32x4{0, 0, 0, 0};
#pragma unroll
                    for (int ks = 0; ks < KS; ks++) s[u] = KvType<T>::mma(kv_bits<x8>(t.k[u][ks]), qf[n][ks], s[u]);
                }
                float z[8];
                float top = -INFINITY;
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    z[j] = s[j >> 2][j & 3];
                    if (!whole && j >= left) z[j] = -INFINITY;
                    top = fmaxf(top, z[j]);
                }
                if (__any(kv_rises(top, m[n], a.scale2))) {
                    top = fmaxf(top, __shfl_xor(top, 16, 64));
                    top = fmaxf(top, __shfl_xor(top, 32, 64));
                    /* each column by its own scores: another's do not show in its bits */
                    const float to = kv_rises(top, m[n], a.scale2) ? top : m[n];
                    const float f = to == m[n] ? 1.0f : kv_factor(m[n], to, a.scale2);
                    m[n] = to;
                    l[n] *= f;
#pragma unroll
                    for (int dt = 0; dt < DT; dt++) o[n][dt] *= f;
                }
                /* before any score is above -infinity the maximum is taken as 0 */
                const float base = m[n] == -INFINITY ? 0.0f : m[n];
                /* A weight as two numbers of the cache's type, 16 (bf16) or 22 bits: as one, a bf16 result is off by a third more
                 * than by its own rounding (2.3e-3 for 1.7e-3).  1 to 3% more time, 6% with 64 queries a key head. */
                x8 p, rest;
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const float e = __builtin_amdgcn_exp2f(fmaf(z[j] - base, a.scale2, KvType<T>::SHIFT));
                    l[n] += e;
                    p[j] = (T)e;
                    rest[j] = (T)(e - (float)p[j]);
                }
                if (WHOLE) __builtin_amdgcn_sched_barrier(0);      /* products among them keep all eight weights' floats in registers */
#pragma unroll
                for (int dt = 0; dt < DT; dt++) o[n][dt] = KvType<T>::mma(kv_bits<x8>(t.v[dt]), p, o[n][dt]);
#pragma unroll
                for (int dt = 0; dt < DT; dt++) o[n][dt] = KvType<T>::mma(kv_bits<x8>(t.v[dt]), rest, o[n][dt]);
            }
        };
        const int mine = (tiles - wave + NW - 1) / NW;      /* this wave's tiles */
        if (mine > 0) {
            Tile ta, tb;
            names(0);
            load(ta, 0);
            for (int i = 0; i < mine; i += 2) {
                if (i + 1 < mine) load(tb, i + 1);
                compute(ta, i);
                if (i + 2 < mine) {
                    if (((i + 2) & 31) == 0) names(i + 2);
                    load(ta, i + 2);
                }
                if (i + 1 < mine) compute(tb, i + 1);
            }
        }
        /* No score above -infinity, or sums that are not finite: is there a position, and which of the wave's values are not
         * finite, each lane those that it holds in the operands, then to the lanes of their sums (rare) */
        bool odd = false;
#pragma unroll
        for (int n = 0; n < NC; n++) {
            f32x4 z = {0, 0, 0, 0};
#pragma unroll
            for (int dt = 0; dt < DT; dt++)
#pragma unroll
                for (int r = 0; r < 4; r++) z[r] = fmaf(o[n][dt][r], 0.0f, z[r]);
            const float none = z[0] + z[1] + (z[2] + z[3]);
            odd |= none != none || m[n] == -INFINITY;
        }
        if (__builtin_expect(mine > 0 && __any(odd), 0)) {
            float found[DT] = {};
            bool seen = false;
#pragma unroll 1
            for (int i = 0; i < mine; i++) {
                const int p0 = begin + 32 * (wave + NW * i) + 8 * g, blk = p0 / KV_BLOCK;
                const int64_t at = p0 < stop ? kv_block(c, table[blk >> c.sh], blk, kvh) : -1;
                if (at < 0) continue;
                seen = true;
#pragma unroll
                for (int dt = 0; dt < DT; dt++) {
                    x8 v = kv_bits<x8>(kv_upto(*(const u32x4 *)((const T *)a.v + at + value_piece(lane) + 256 * dt), stop - p0));
#pragma unroll
                    for (int p = 0; p < 8; p++) {     /* 0 for what is finite */
                        const float x = (float)v[p];
                        found[dt] += x - __builtin_amdgcn_fmed3f(x, -3.4028234663852886e38f, 3.4028234663852886e38f);
                    }
                }
            }
#pragma unroll
            for (int dt = 0; dt < DT; dt++) {
                found[dt] += __shfl_xor(found[dt], 16, 64);
                found[dt] += __shfl_xor(found[dt], 32, 64);
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const float is = __shfl(found[dt], 4 * g + r, 64);
#pragma unroll
                    for (int n = 0; n < NC; n++) o[n][dt][r] = is == 0.0f ? o[n][dt][r] : is;
                }
            }
            if (__any(seen)) {
#pragma unroll
                for (int n = 0; n < NC; n++) m[n] = fmaxf(m[n], KV_LOWEST);
            }
        }
        /* the lanes of a column hold different positions' weights */
#pragma unroll
        for (int n = 0; n < NC; n++) {
            l[n] += __shfl_xor(l[n], 16, 64);
            l[n] += __shfl_xor(l[n], 32, 64);
        }
        /* merge the waves, half of them at a time, always in the same order */
#pragma unroll
        for (int half = NW / 2; half >= 1; half >>= 1) {
            if (wave >= half && wave < 2 * half) {
#pragma unroll
                for (int n = 0; n < NC; n++) {
#pragma unroll
                    for (int dt = 0; dt < DT; dt++)
                        *(f32x4 *)&s_o[wave - half][(n * 16 + col) * LD + 16 * dt + 4 * g] = o[n][dt];
                    if (g == 0) {
                        s_ml[wave - half][(n * 16 + col) * 2] = m[n];
                        s_ml[wave - half][(n * 16 + col) * 2 + 1] = l[n];
                    }
                }
            }
            __syncthreads();
            if (wave < half) {
#pragma unroll
                for (int n = 0; n < NC; n++) {
                    const float om = s_ml[wave][(n * 16 + col) * 2], ol = s_ml[wave][(n * 16 + col) * 2 + 1];
                    const float to = fmaxf(m[n], om);
                    const float fm = kv_factor(m[n], to, a.scale2), fo = kv_factor(om, to, a.scale2);
                    m[n] = to;
                    l[n] = l[n] * fm + ol * fo;
                    const float wm = kv_not_zero(fm), wo = kv_not_zero(fo);
#pragma unroll
                    for (int dt = 0; dt < DT; dt++) {
                        const f32x4 w = *(const f32x4 *)&s_o[wave][(n * 16 + col) * LD + 16 * dt + 4 * g];
                        o[n][dt] = o[n][dt] * wm + w * wo;
                    }
                }
            }
            __syncthreads();
        }
        if (wave == 0) {
#pragma unroll
            for (int n = 0; n < NC; n++) {
                const int h = n * 16 + col;
                if (h >= ncol) continue;
                const int64_t head = kvh * a.G + col0 + h, H = (int64_t)a.G * c.heads;
                if (take == units) {
                    const float inv = kv_inverse(l[n], m[n]);
#pragma unroll
                    for (int dt = 0; dt < DT; dt++) {
                        const float v[4] = {o[n][dt][0] * inv, o[n][dt][1] * inv, o[n][dt][2] * inv, o[n][dt][3] * inv};
                        kv_store(a.out, a.out_dt, (b * H + head) * HD + 16 * dt + 4 * g, v);
                    }
                } else {
                    const int64_t w = kv_slot(worker, first == 0) * H + head;
#pragma unroll
                    for (int dt = 0; dt < DT; dt++) *(f32x4 *)(a.part + w * HD + 16 * dt + 4 * g) = o[n][dt];
                    if (g == 0) {
                        a.ml[2 * w] = m[n];
                        a.ml[2 * w + 1] = l[n];
                    }
                }
            }
        }
        return take;
    };
    if (WHOLE) {
        part(worker, kv_uniform(decode_len(c, worker)), 0, 1 << 30);
    } else {
        const DecodeBatch batch(c, a.W);
        const int at = kv_share(batch.sh, worker);
        int left = kv_share(batch.sh, worker + 1) - at;
        if (left == 0) return;
        const KvItem it = batch.find(at);
        if (it.b < 0) return;
        for (int b = it.b, first = it.i; left > 0 && b < c.B; b++, first = 0) left -= part(b, batch.len(b), first, left);
    }
}

/* The sums of the sequences that several workers share: a group per sequence and hb heads, HD / 4 threads a row, the
 * workers' parts dealt to a head's rows, each with a maximum of its own, the rows added through LDS in a fixed order.  4 to
 * 5 us whatever the sizes: a launch and two reads after each other (1024 threads a group, or a group for 32 values: the same). */
template <int HD> __global__ __launch_bounds__(256) void k_kv_join(DecodeArgs a) {
    constexpr int L4 = HD / 4, ROWS = 256 / L4;
    __shared__ float s_o[ROWS][HD], s_ml[ROWS][2];
    const KvView &c = a.c;
    const int b = blockIdx.x, H = a.G * c.heads, tid = threadIdx.x;
    const DecodeBatch batch(c, a.W);
    const int before = batch.before(b), w0 = kv_worker(batch.sh, before);
    const int n = kv_worker(batch.sh, before + kv_units(batch.len(b)) - 1) - w0 + 1;
    if (n == 1) return;
    const int R = ROWS / a.hb, row = tid / L4, e = tid % L4 * 4, hd = row / R, r = row % R;
    const int head = blockIdx.y * a.hb + hd;
    f32x4 o = {0, 0, 0, 0};
    float m = -INFINITY, l = 0.0f;
    if (hd < a.hb && head < H) {
#pragma unroll 4
        for (int i = r; i < n; i += R) {
            const int64_t w = (int64_t)kv_slot(w0 + i, i == 0) * H + head;
            const float mi = a.ml[2 * w], li = a.ml[2 * w + 1];
            const f32x4 oi = *(const f32x4 *)(a.part + w * HD + e);
            const float to = fmaxf(m, mi), f = kv_factor(m, to, a.scale2), fi = kv_factor(mi, to, a.scale2);
            o = o * kv_not_zero(f) + oi * kv_not_zero(fi);
            l = l * f + li * fi;
            m = to;
        }
    }
    if (row < ROWS) {
        *(f32x4 *)&s_o[row][e] = o;
        if (e == 0) {
            s_ml[row][0] = m;
            s_ml[row][1] = l;
        }
    }
    __syncthreads();
    if (r > 0 || hd >= a.hb || head >= H) return;
    float top = m;
    for (int i = 1; i < R; i++) top = fmaxf(top, s_ml[row + i][0]);
    const float f = kv_factor(m, top, a.scale2);
    o *= kv_not_zero(f);
    l *= f;
    for (int i = 1; i < R; i++) {
        const float fi = kv_factor(s_ml[row + i][0], top, a.scale2);
        o += *(const f32x4 *)&s_o[row + i][e] * kv_not_zero(fi);
        l += s_ml[row + i][1] * fi;
    }
    const float inv = kv_inverse(l, top);
    const float v[4] = {o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv};
    kv_store(a.out, a.out_dt, ((int64_t)b * H + head) * HD + e, v);
}

/* ---- launches -------------------------------------------------------------- */
template <class X, class T, int M> void append_m(const AppendArgs &a, dim3 grid, hipStream_t s) {
    hipLaunchKernelGGL((k_kv_append<X, T, M>), grid, dim3(256), 0, s, a);
}
template <class X, class T> void append_hd(const AppendArgs &a, dim3 grid, hipStream_t s) {
    static void (*const by_width[8])(const AppendArgs &, dim3, hipStream_t) = {
        append_m<X, T, 1>, append_m<X, T, 2>, append_m<X, T, 3>, append_m<X, T, 4>,
        append_m<X, T, 5>, append_m<X, T, 6>, append_m<X, T, 7>, append_m<X, T, 8>};
    by_width[a.c.hd / 32 - 1](a, grid, s);
}
template <class T> void append_x(int xdt, const AppendArgs &a, dim3 grid, hipStream_t s) {
    if (xdt == DT_F32) append_hd<float, T>(a, grid, s);
    else if (xdt == DT_F16) append_hd<_Float16, T>(a, grid, s);
    else append_hd<__bf16, T>(a, grid, s);
}

/* A sequence a group of eight waves and one launch, where the tables are as short as this; twice as long where there are groups
 * for every compute unit.  us whole / in shares, 32 heads on 4 of 128: one sequence of 500 8.5 / 9.1, of 1000 10.9 / 9.1; 64 of
 * 500 16.1 / 17.9, of 1000 24.4 / 26.3, of up to 1000 18.9 / 21.2; 256 of 1000 106 / 103; 300 of 8 on 2 of 64 7.7 / 13.7. */
constexpr int64_t DECODE_WHOLE = 512;

struct DecodePlan {
    int whole, W, nc, z, hb;
};
DecodePlan decode_plan(const tlm_hip_kv_cache *c, const tlm_hip_kv_batch *b, int heads) {
    /* Columns of 16 queries a group.  A key head with more queries has a group for every 16, which read the cache again from
     * the caches nearer by; narrow heads, whose tiles are little to read, take 32.  us with 16 / 32 / 64 a group, one number a
     * weight: 48 sequences of up to 8192 with 64 heads on 1 of 128 36.6 / 36.5 / 44.9 (two numbers: 38.7 with 16), 40 on 2 of
     * 128 55 / 55, 128 on 4 of 64 55 / 46; one of 30000 with 64 on 1 of 128 14.6 / 17.8 / 24.8 (15.0), 64 on 2 of 256 22.5 / 28.4
     * (23.2). */
    const int G = heads / c->kv_heads, nc = G > 16 && c->head_dim <= 64 ? 2 : 1, z = (G + nc * 16 - 1) / (nc * 16);
    const int64_t cap = (int64_t)b->table_pages * c->page;
    if (cap <= DECODE_WHOLE || (cap <= 2 * DECODE_WHOLE && b->B * c->kv_heads * z >= 256)) return {1, (int)b->B, nc, z, 0};
    /* A group a compute unit: four waves with two tiles each on their way keep the memory busy, and fewer shares are fewer
     * parts to join.  256 groups / 512 (1024 up to 64 wide): one sequence of 131071, 32 heads on 4 of 128, 52.7 / 55.1 us; 64
     * of up to 8192, 64 on 4, 113 / 118; 60000, 8 on 2 of 64, 13.8 / 18.3; 240 groups 53.6, 114, 14.2; 256 of eight waves
     * 53.6, 116, 14.1. */
    const int W = 256 / (c->kv_heads * z);
    /* the join: about 1024 groups, a head each if there are fewer */
    const int64_t hb = b->B * heads / 1024;
    const int rows = 256 / (c->head_dim / 4);
    return {0, W < 1 ? 1 : W, nc, z, (int)(hb < 1 ? 1 : hb > rows ? rows : hb)};
}
size_t decode_bytes(const tlm_hip_kv_cache *c, const tlm_hip_kv_batch *b, int heads) {
    const DecodePlan p = decode_plan(c, b, heads);
    return p.whole ? 0 : (size_t)2 * p.W * heads * (c->head_dim + 4) * 4;
}

template <class T, int HD, int NC> void decode_nc(const DecodeArgs &a, const DecodePlan &p, hipStream_t s) {
    const dim3 grid((unsigned)p.W, (unsigned)a.c.heads, (unsigned)p.z);
    if (p.whole) {
        constexpr int NW = NC == 1 && HD <= 128 ? 8 : 4;   /* eight waves leave a wave 256 registers */
        hipLaunchKernelGGL((k_kv_decode<T, HD, NC, NW, true>), grid, dim3(NW * 64), 0, s, a);
    } else {
        hipLaunchKernelGGL((k_kv_decode<T, HD, NC, 4, false>), grid, dim3(256), 0, s, a);
        const dim3 join((unsigned)a.c.B, (unsigned)((a.G * a.c.heads + p.hb - 1) / p.hb));
        hipLaunchKernelGGL((k_kv_join<HD>), join, dim3(256), 0, s, a);
    }
}
template <class T, int HD> void decode_hd(const DecodeArgs &a, const DecodePlan &p, hipStream_t s) {
    if constexpr (HD <= 64)
        if (p.nc == 2) return decode_nc<T, HD, 2>(a, p, s);
    decode_nc<T, HD, 1>(a, p, s);
}
template <class T> void decode(const DecodeArgs &a, const DecodePlan &p, hipStream_t s) {
    static void (*const by_width[8])(const DecodeArgs &, const DecodePlan &, hipStream_t) = {
        decode_hd<T, 32>, decode_hd<T, 64>, decode_hd<T, 96>, decode_hd<T, 128>,
        decode_hd<T, 160>, decode_hd<T, 192>, decode_hd<T, 224>, decode_hd<T, 256>};
    by_width[a.c.hd / 32 - 1](a, p, s);
}

} // namespace

int kv_check(const char *who, const tlm_hip_kv_cache *c, const tlm_hip_kv_batch *b, int heads, KvView *v) {
    if (!c || !b) return tlmh_seterr(TLM_HIP_EINVAL, "%s: NULL argument", who);
    if (c->dt != DT_F16 && c->dt != DT_BF16)
        return tlmh_seterr(TLM_HIP_EUNSUP, "%s: cache of dtype %d (F16 and BF16 only)", who, c->dt);
    if (c->head_dim < 32 || c->head_dim > 256 || c->head_dim % 32)
        return tlmh_seterr(TLM_HIP_EUNSUP, "%s: head_dim %d is not a multiple of 32 up to 256", who, c->head_dim);
    if (c->page < KV_BLOCK || c->page > 4096 || (c->page & (c->page - 1)))
        return tlmh_seterr(TLM_HIP_EINVAL, "%s: page of %d positions (a power of two from 16 to 4096)", who, c->page);
    if (c->kv_heads < 1 || c->kv_heads > 4096 || heads < 1 || heads > 16384 || heads % c->kv_heads)
        return tlmh_seterr(TLM_HIP_EINVAL, "%s: %d heads on %d key heads", who, heads, c->kv_heads);
    if (c->n_pages < 1 || c->n_pages > 0x7FFFFFFF)
        return tlmh_seterr(TLM_HIP_EINVAL, "%s: %lld pages", who, (long long)c->n_pages);
    if (b->B < 0 || b->rows < 0 || (!b->cu && b->rows != b->B))
        return tlmh_seterr(TLM_HIP_EINVAL, "%s: %lld rows of %lld sequences", who, (long long)b->rows, (long long)b->B);
    if (b->B > (1 << 20) || b->rows > ((int64_t)1 << 30) || b->rows * heads > ((int64_t)1 << 30))
        return tlmh_seterr(TLM_HIP_ERANGE, "%s: %lld rows of %lld sequences are too many for one launch", who,
                           (long long)b->rows, (long long)b->B);
    if (b->table_pages < 1 || (int64_t)b->table_pages * c->page > (1 << 30))
        return tlmh_seterr(TLM_HIP_EINVAL, "%s: tables of %d pages (1 to 2^30 positions)", who, b->table_pages);
    if (b->B > 1 && b->table_stride < b->table_pages)
        return tlmh_seterr(TLM_HIP_EINVAL, "%s: table stride %lld below %d", who, (long long)b->table_stride, b->table_pages);
    if (b->B > 0 && b->rows > 0) {
        if (!c->k || !c->v || !b->lens || !b->tables) return tlmh_seterr(TLM_HIP_EINVAL, "%s: NULL argument", who);
        if (!aligned(c->k, 16) || !aligned(c->v, 16) || !aligned(b->lens, 4) || !aligned(b->tables, 4) || !aligned(b->cu, 4))
            return tlmh_seterr(TLM_HIP_EINVAL, "%s: keys and values must be 16-byte, lens, tables and cu 4-byte aligned", who);
    }
    int sh = 0;
    while ((KV_BLOCK << sh) < c->page) sh++;
    *v = {b->tables, b->lens, b->cu, b->table_stride, b->rows, (int32_t)b->B, b->table_pages, (int32_t)c->n_pages,
          c->kv_heads, sh, c->head_dim};
    return TLM_HIP_OK;
}

extern "C" {

int tlm_hip_kv_append(const tlm_hip_kv_cache *c, const tlm_hip_kv_batch *b, int dt, const void *qkv, int64_t qkv_stride,
                      int heads, const float *q_norm, const float *k_norm, float eps, const double *inv_freq,
                      float rope_scale, void *q, void *stream) {
    AppendArgs a;
    if (int rc = kv_check("kv_append", c, b, heads, &a.c)) return rc;
    if (!type_bytes(dt)) return tlmh_seterr(TLM_HIP_EUNSUP, "kv_append: dtype %d (F32, F16 and BF16 only)", dt);
    if (!(eps >= 0.0f) || eps > 3.0e38f) return tlmh_seterr(TLM_HIP_EINVAL, "kv_append: eps must be finite and not negative");
    if (b->B == 0 || b->rows == 0) return TLM_HIP_OK;
    if (!qkv || !q) return tlmh_seterr(TLM_HIP_EINVAL, "kv_append: NULL argument");
    const int64_t width = (int64_t)(heads + 2 * c->kv_heads) * c->head_dim;
    if (qkv_stride < width && b->rows > 1)
        return tlmh_seterr(TLM_HIP_EINVAL, "kv_append: row stride %lld below %lld", (long long)qkv_stride, (long long)width);
    if (!aligned(qkv, (size_t)type_bytes(dt)) || !aligned(q, 16) || !aligned(q_norm, 4) || !aligned(k_norm, 4) ||
        !aligned(inv_freq, 8))
        return tlmh_seterr(TLM_HIP_EINVAL, "kv_append: qkv must have its type's alignment, q 16, the norms 4, inv_freq 8 "
                           "bytes");
    if (int rc = tlmh_refuse_failed(FAILED_KV, "kv_append")) return rc;
    const int64_t items = b->cu ? kv_append_most(b->rows, b->B) : b->B;
    if (items * c->kv_heads > (1 << 23))
        return tlmh_seterr(TLM_HIP_ERANGE, "kv_append: %lld rows of %lld sequences are too many for one launch",
                           (long long)b->rows, (long long)b->B);
    a.x = qkv;
    a.xstride = qkv_stride;
    a.q = q;
    a.k = c->k;
    a.v = c->v;
    a.qw = q_norm;
    a.kw = k_norm;
    a.freq = inv_freq;
    a.eps = eps;
    a.rope_scale = rope_scale;
    a.G = heads / c->kv_heads;
    /* Two key heads a group share the rows' angles, worth it once the card is full without the second group: 8192 rows of
     * 16 heads of 64 on 16 39.4 -> 30.6 us (four: 28.5), 32 of 128 on 32 101 -> 90 (four: 97), 1024 sequences of one row,
     * 32 on 8, 22.6 -> 17.7 (four: 16.0); 64 of 64 on 8 45.3 -> 42.4 (four, 1024 groups: 50.9). */
    a.hpg = items * c->kv_heads >= 2 * 2048 ? 2 : 1;
    const dim3 grid((unsigned)items, (unsigned)((c->kv_heads + a.hpg - 1) / a.hpg));
    if (c->dt == DT_F16) append_x<_Float16>(dt, a, grid, (hipStream_t)stream);
    else append_x<__bf16>(dt, a, grid, (hipStream_t)stream);
    return tlmh_check(hipGetLastError(), "kv_append launch");
}

size_t tlm_hip_kv_decode_workspace_bytes(const tlm_hip_kv_cache *c, const tlm_hip_kv_batch *b, int heads) {
    KvView v;
    if (kv_check("kv_decode_workspace_bytes", c, b, heads, &v)) return 0;
    return decode_bytes(c, b, heads);
}

int tlm_hip_kv_decode(const tlm_hip_kv_cache *c, const tlm_hip_kv_batch *b, const void *q, int64_t q_stride, int heads,
                      float scale, int out_dt, void *out, void *workspace, void *stream) {
    DecodeArgs a;
    if (int rc = kv_check("kv_decode", c, b, heads, &a.c)) return rc;
    if (b->cu) return tlmh_seterr(TLM_HIP_EINVAL, "kv_decode: one row a sequence (cu must be NULL)");
    if (!type_bytes(out_dt)) return tlmh_seterr(TLM_HIP_EUNSUP, "kv_decode: dtype %d (F32, F16 and BF16 only)", out_dt);
    if (!(scale > 0.0f) || scale > 2.0e38f) return tlmh_seterr(TLM_HIP_EINVAL, "kv_decode: scale must be finite and positive");
    if (b->B == 0) return TLM_HIP_OK;
    if (!q || !out) return tlmh_seterr(TLM_HIP_EINVAL, "kv_decode: NULL argument");
    if (q_stride < (int64_t)heads * c->head_dim && b->B > 1)
        return tlmh_seterr(TLM_HIP_EINVAL, "kv_decode: row stride %lld below %lld", (long long)q_stride,
                           (long long)heads * c->head_dim);
    if (!aligned(q, 2) || !aligned(out, (size_t)type_bytes(out_dt)))
        return tlmh_seterr(TLM_HIP_EINVAL, "kv_decode: q and out must have their type's alignment");
    const DecodePlan p = decode_plan(c, b, heads);
    /* the batch's units are counted in an int; groups of a launch */
    if (b->B * (((int64_t)b->table_pages * c->page + KV_UNIT - 1) / KV_UNIT) >= (1 << 30) ||
        (int64_t)p.W * c->kv_heads * p.z > (1 << 22) || b->B * heads > (1 << 23))
        return tlmh_seterr(TLM_HIP_ERANGE, "kv_decode: %lld sequences of %d heads are too many for one launch",
                           (long long)b->B, heads);
    if (!p.whole && (!workspace || !aligned(workspace, 256)))
        return tlmh_seterr(TLM_HIP_EINVAL, "kv_decode: needs a workspace of %zu bytes, 256-byte aligned", decode_bytes(c, b, heads));
    if (int rc = tlmh_refuse_failed(FAILED_KV, "kv_decode")) return rc;
    a.q = q;
    a.k = c->k;
    a.v = c->v;
    a.out = out;
    a.part = (float *)workspace;
    a.ml = p.whole ? nullptr : a.part + (size_t)2 * p.W * heads * c->head_dim;
    a.qstride = q_stride;
    a.scale2 = scale * 1.44269504088896341f;
    a.G = heads / c->kv_heads;
    a.W = p.W;
    a.out_dt = out_dt;
    a.hb = p.hb;
    if (c->dt == DT_F16) decode<_Float16>(a, p, (hipStream_t)stream);
    else decode<__bf16>(a, p, (hipStream_t)stream);
    return tlmh_check(hipGetLastError(), "kv_decode launch");
}

} // extern "C"
