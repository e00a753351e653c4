/* hip_fp8_moe.hip - a routed MoE block for up to 64 tokens with 8-bit
 * floating-point weights (E4M3, a scale per 128 x 128) and f32 activations.
 *
 *   out[t] = h[t] + sum_r w_r D_e (silu(G_e x) * U_e x) (+ gate * shared(x)),
 *   x = rmsnorm(h[t]), e = the expert of rank r
 *
 * So few tokens are bound by the weights' bytes, so the activations keep 32
 * bits: a float is three bfloat16 planes exactly (split3), a code is a bfloat16
 * exactly, their products are exact in the matrix cores' float accumulators.
 * The planes are columns of the matrix product: 16 columns hold five tokens' three
 * planes, whose sums are added at the end, smallest first.
 *
 *   K1 router    x, its planes, the router's scores and the selection keys
 *   K1b route    each token's experts and weights
 *   K2 gate/up   16 rows of one expert's gate and up, for all of its tokens: silu(g) * u as
 *                planes; one token, and few in a small block, route in this launch
 *   K3 down      few tokens: 16 rows of one token's result, all its experts, the sum and the
 *                residual; more: 64 rows of one expert's down for all of its tokens, then
 *                K4 combine  the sum in rank order and the residual
 * No launch hands data between its own groups: on this chip a boundary between launches costs
 * about 1.4 us, a barrier across the groups of one 6 us and more, so three launches for one
 * token beat two.
 *
 * Measured, whole layers: Qwen3-30B-A3B (2048 x 768, 128 experts top-8), one token 19.7 us (38 MB,
 * of it router 5, gate/up 10, down 7: launches and dependent reads more than bytes), 8
 * tokens 60 us (4.0 TB/s of the experts that they reach), 64 tokens 155; Qwen3-235B-A22B (4096 x
 * 1536), 64 tokens 461-478 us, 5.0-5.2 TB/s, what a large copy reaches. */
#include "tlm_hip_fp8.h"

namespace {

constexpr int MAXT = TLM_HIP_FP8_MOE_MAX_TOKENS;   /* 64: a token per lane in the lists */
constexpr int MAXE = 256, MAXK = 32;
constexpr int NW = 4;              /* waves per group of K2 and K3: the blocks of a row are dealt to them */
constexpr int TPT = 5;             /* tokens per 16 columns */
constexpr int NT = 2;              /* column tiles at a time */

__host__ __device__ inline size_t al256(size_t v) { return (v + 255) & ~(size_t)255; }

struct Layout {
    size_t xp, key, score, sgate, ids, w, dptr, hid, shid, eo, seo, total;
    int nbd, nbe, nbs;             /* blocks of D, of the expert width, of the shared width */
};

Layout layout(const tlm_hip_moe_desc &d, int64_t T) {
    Layout L;
    L.nbd = (int)fp8_blocks(d.D);
    L.nbe = (int)fp8_blocks(d.de);
    L.nbs = d.ds > 0 ? (int)fp8_blocks(d.ds) : 0;
    size_t o = 0;
    L.xp = o;    o += al256((size_t)T * 3 * L.nbd * FP8_BLOCK * 2);
    L.key = o;   o += al256((size_t)T * d.E * 4);
    L.score = o; o += al256((size_t)T * d.E * 4);
    L.sgate = o; o += al256((size_t)T * 4);
    L.ids = o;   o += al256((size_t)T * d.k * 4);
    L.w = o;     o += al256((size_t)T * d.k * 4);
    L.dptr = o;  o += al256((size_t)T * d.k * 8);
    L.hid = o;   o += al256((size_t)T * d.k * 3 * L.nbe * FP8_BLOCK * 2);
    L.shid = o;  o += al256((size_t)T * 3 * L.nbs * FP8_BLOCK * 2);
    L.eo = o;    o += al256((size_t)T * d.k * d.D * 4);
    L.seo = o;   o += d.ds > 0 ? al256((size_t)T * d.D * 4) : 0;
    L.total = o;
    return L;
}

struct Args {
    tlm_hip_moe_desc d;
    Layout L;
    const float *h;
    float *out;
    int32_t *ids;
    float *w;
    uint8_t *ws;
    int T, slots, by_expert;
    double inv_D;
    int ce, cs;   /* groups among which an expert's, and the shared expert's, tokens are dealt */
};

/* A vector's planes: a block of 128 values is 384 bfloat16, in the order of the matrix cores' operands: load
 * j of 4, group g of 4 lanes' columns, plane, 8 values (64 (j / 2) + 16 g + 8 (j % 2) on).  The
 * 16 lanes of a quarter wave, five vectors' three planes, then ask for 48 bytes of five lines, not for 16
 * bytes of fifteen. */
constexpr int XBLOCK = 3 * FP8_BLOCK;
__device__ __forceinline__ int plane_at(int i, int plane) {
    const int g = (i >> 4) & 3, j = 2 * ((i >> 6) & 1) + ((i >> 3) & 1);
    return (i >> 7) * XBLOCK + ((j * 4 + g) * 3 + plane) * 8 + (i & 7);
}
/* this lane's part of a block, load j at 96 j from it */
__device__ __forceinline__ int plane_lane() { return (int)((threadIdx.x & 63) >> 4) * 24 + (int)((threadIdx.x & 15) % 3) * 8; }

/* a value that all lanes of a wave share, in a scalar register: branches on it are the
 * wave's, and no matrix instruction ends up under a lane mask */
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

/* order of selection values as unsigned integers; -0 as +0, NaN as -infinity.  0 is
 * left for experts that cannot be chosen. */
__device__ __forceinline__ uint32_t order_key(float f) {
    const uint32_t b = __float_as_uint(f != f ? -INFINITY : f + 0.0f);
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
/* with the exponential's table in the wave's lanes: every lane takes part */
__device__ __forceinline__ float silu(float x, const ExpTabLanes &tab) { return x / (1.0f + expf_ref_with(-x, tab)); }

/* Kernel arguments named here are fetched at once, not in turn where each is first used. */
template <class T> __device__ __forceinline__ void arg_now(T v) { asm volatile("" ::"s"(v)); }
template <class... T> __device__ __forceinline__ void args_now(T... v) { (arg_now(v), ...); }

/* ---- K1 ---------------------------------------------------------------------
 * A group per token and four router rows (the shared expert's gate is one more), x in LDS: the
 * rows' first 2048 values are on their way while the token is normalised.  (Four tokens a group, the
 * rows read once for them: 17.9 us for 64 tokens of 4096, longer than the rows' reads from L2.)  Sums of four
 * products in float, those in double: two experts' scores keep their order down to the
 * last bits of a float. */
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));

/* four values of a row of D at i, zeros behind its end */
__device__ __forceinline__ f32x4 row4(const GAS float *p, int i, int D) {
    f32x4 v = {0, 0, 0, 0};
    if (i + 3 < D) {
        v = *(const GAS f32x4u *)(p + i);
    } else {
#pragma unroll
        for (int q = 0; q < 4; q++)
            if (i + q < D) v[q] = p[i + q];
    }
    return v;
}

__global__ __launch_bounds__(256) void k_fm_router(Args a) {
    extern __shared__ __align__(16) float s_x[];
    __shared__ double s_red[4];
    const tlm_hip_moe_desc &d = a.d;
    args_now(d.D, d.E, d.ds, d.router, d.eps, d.ffn_norm, d.router_w, d.router_bias, d.mask, d.experts, d.shared_gate_inp,
             a.h, a.ws, a.inv_D, a.L.xp, a.L.key, a.L.score, a.L.sgate, a.L.nbd);
    const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6), t = blockIdx.y;
    const int D = (int)d.D, Dq = (D + 3) & ~3, e = blockIdx.x * 4 + wave;
    const bool live = e < d.E || (e == d.E && d.ds > 0 && d.shared_gate_inp);
    const GAS float *w = (const GAS float *)(live && e == d.E ? d.shared_gate_inp : d.router_w + (size_t)(live ? e : 0) * D);
    const GAS float *h = (const GAS float *)a.h + (size_t)t * D, *nw = (const GAS float *)d.ffn_norm;
    /* the token and the norm weights first: they are waited for first */
    constexpr int NC = 4;   /* runs of 1024 values held in registers; a longer row's others are read again */
    f32x4 hv[NC], gv[NC];
#pragma unroll
    for (int c = 0; c < NC; c++)
        if (1024 * c < D) {
            hv[c] = row4(h, 4 * tid + 1024 * c, D);
            gv[c] = row4(nw, 4 * tid + 1024 * c, D);
        }
    constexpr int NV = 8;
    f32x4 wv[NV];
#pragma unroll
    for (int j = 0; j < NV; j++) wv[j] = row4(w, 4 * lane + 256 * j, D);
    ExpTabLanes tab;
    tab.load();
    /* an expert without all of its matrices cannot be chosen: no launch after this one follows a null pointer
     * (a lane each, looked at last: waited for here by all lanes they cost 0.4 us) */
    const void *const mat = ((const void *const GAS *)d.experts)[3 * (size_t)(e < d.E ? e : 0) + (lane < 3 ? lane : 0)];
    double ss = 0.0;
#pragma unroll
    for (int c = 0; c < NC; c++)
        if (1024 * c < D)
#pragma unroll
            for (int q = 0; q < 4; q++) ss += (double)hv[c][q] * (double)hv[c][q];
    for (int i = 4 * tid + 1024 * NC; i < Dq; i += 1024) {
        const f32x4 v = row4(h, i, D);
#pragma unroll
        for (int q = 0; q < 4; q++) ss += (double)v[q] * (double)v[q];
    }
    ss = wave_sum_f64(ss);
    if (lane == 0) s_red[wave] = ss;
    __syncthreads();
    ss = (s_red[0] + s_red[1]) + (s_red[2] + s_red[3]);
    /* The token's factor stays double: rounded, it would be off in the same direction for the whole vector (1e-7 of
     * the result in common, where the elements' own roundings average out), and the mean of large squares is no
     * float.  The instruction gives 23 bits, a Newton step 45. */
    const double v = ss * a.inv_D + (double)d.eps;
    double rn = __builtin_amdgcn_rsq(v);
    rn = fma(0.5 * rn, fma(-v * rn, rn, 1.0), rn);
    auto normed = [&](f32x4 h, f32x4 g) {
        f32x4 x;
#pragma unroll
        for (int q = 0; q < 4; q++) x[q] = (float)((double)h[q] * rn) * g[q];
        return x;
    };
    const int Dp = a.L.nbd * FP8_BLOCK;
    uint16_t *xp = (uint16_t *)(a.ws + a.L.xp) + (size_t)t * 3 * Dp;
    auto put = [&](int i, f32x4 v) {
        if (i < Dq) *(f32x4 *)(s_x + i) = v;
        if ((i >> 8) % gridDim.x != blockIdx.x) return;   /* the groups share the planes' writing */
        u16x4 o[3];
#pragma unroll
        for (int q = 0; q < 4; q++) {
            uint16_t p[3];
            split3(v[q], p);
#pragma unroll
            for (int j = 0; j < 3; j++) o[j][q] = p[j];
        }
#pragma unroll
        for (int j = 0; j < 3; j++) *(u16x4 *)(xp + plane_at(i, j)) = o[j];
    };
#pragma unroll
    for (int c = 0; c < NC; c++) {
        const int i = 4 * tid + 1024 * c;
        if (1024 * c < D && i < Dp) put(i, normed(hv[c], gv[c]));   /* zeros behind D */
    }
    for (int i = 4 * tid + 1024 * NC; i < Dp; i += 1024) put(i, normed(row4(h, i, D), row4(nw, i, D)));
    __syncthreads();
    if (!live) return;
    double acc = 0.0;
    for (int i0 = 0; i0 < Dq; i0 += 256 * NV) {
        if (i0 > 0)
#pragma unroll
            for (int j = 0; j < NV; j++) wv[j] = row4(w, i0 + 4 * lane + 256 * j, D);
#pragma unroll
        for (int j = 0; j < NV; j++) {
            const int i = i0 + 4 * lane + 256 * j;
            if (i >= Dq) continue;
            const f32x4 x = *(const f32x4 *)(s_x + i);
            float p = wv[j][0] * x[0];
#pragma unroll
            for (int q = 1; q < 4; q++) p = fmaf(wv[j][q], x[q], p);
            acc += (double)p;
        }
    }
    const float l = (float)wave_sum_f64(acc);   /* the same in every lane */
    const float sig = 1.0f / (1.0f + expf_ref_with(-l, tab));
    const bool whole = __ballot(mat == nullptr) == 0;
    if (lane != 0) return;
    if (e == d.E) {
        ((float *)(a.ws + a.L.sgate))[t] = sig;
        return;
    }
    const float score = d.router == 2 ? sig : l;
    const float sel = d.router == 2 && d.router_bias ? score + d.router_bias[e] : score;
    ((float *)(a.ws + a.L.score))[t * d.E + e] = score;
    ((uint32_t *)(a.ws + a.L.key))[t * d.E + e] = !whole || (d.mask && d.mask[e]) ? 0u : order_key(sel);
}

/* ---- routing ------------------------------------------------------------------
 * Expert e is among token t's k if fewer than k of t's keys are ahead of its own; the count is
 * its rank.  A key is 64 bits, the order of the selection value and then ~e, so that "larger"
 * is the whole order.  Threads tid, tid + W, ... share the count for expert tid (W = 128 or 256
 * at the least E): counted by one thread an expert, the compares alone took 2 us. */
struct Route {
    unsigned long long key[MAXE];
    uint16_t cnt[4][MAXE];
    int ids[MAXK];
    float w[MAXK];
    const void *down[MAXK];
    float redf[8];
    double red[8];
};
/* What thread e holds of its expert for one token: everything that routing reads, asked for at once. */
struct Choice {
    uint32_t key;
    float score;
    const void *gate, *up, *down;
};
__device__ __forceinline__ Choice choice_of(const Args &a, int t, int tid) {
    const bool in = tid < a.d.E;
    const int e = in ? tid : 0;
    const size_t at = (size_t)t * a.d.E + e;
    Choice c;
    c.key = ((const GAS uint32_t *)(a.ws + a.L.key))[at];
    c.score = ((const GAS float *)(a.ws + a.L.score))[at];
    const void *const GAS *tab = (const void *const GAS *)a.d.experts + 3 * (size_t)e;
    c.gate = tab[0];
    c.up = tab[1];
    c.down = tab[2];
    if (!in) c.key = 0u;
    return c;
}
/* The rank of thread tid's expert (MAXE where it cannot be chosen, and past E).  All WV waves. */
template <int WV> __device__ __forceinline__ int rank_of(const Args &a, const Choice &c, Route *R, int tid) {
    const int W = a.d.E <= 128 ? 128 : 256, parts = WV * 64 / W, e = tid & (W - 1), part = tid / W;
    if (tid < MAXE) R->key[tid] = c.key ? (unsigned long long)c.key << 32 | (0xFFFFFFFFu - (uint32_t)tid) : 0ull;
    if (tid < MAXK) {
        R->ids[tid] = -1;
        R->w[tid] = 0.0f;
        R->down[tid] = nullptr;
    }
    __syncthreads();
    const unsigned long long ke = R->key[e];
    if (ke) {
        int n[4] = {0, 0, 0, 0};
        const LAS u32x4 *kp = (const LAS u32x4 *)R->key + part * (W / parts / 2);
#pragma unroll 8
        for (int f = 0; f < W / parts / 2; f++) {   /* two keys a read; keys past E are 0, never larger */
            const u32x4 k = kp[f];
            n[f & 1] += ((unsigned long long)k[1] << 32 | k[0]) > ke ? 1 : 0;
            n[2 + (f & 1)] += ((unsigned long long)k[3] << 32 | k[2]) > ke ? 1 : 0;
        }
        R->cnt[part][e] = (uint16_t)((n[0] + n[1]) + (n[2] + n[3]));
    }
    __syncthreads();
    if (tid >= W || !ke) return MAXE;
    int rank = 0;
    for (int q = 0; q < parts; q++) rank += R->cnt[q][e];
    return rank;
}
/* A token's experts and weights in rank order into the workspace and the caller's arrays: ranks past the
 * number of experts that can be chosen get id -1 and weight 0.  All threads of a group of WV waves. */
template <int WV>
__device__ void route_token(const Args &a, int t, const Choice &c, Route *R, int rank, const ExpTabLanes &tab) {
    const tlm_hip_moe_desc &d = a.d;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, k = d.k;
    const float l = c.score;
    float p = l;
    if (d.router != 2) {   /* softmax over the experts that can be chosen */
        const bool on = c.key && l == l;
        const float m = wave_max_f32(on ? l : -INFINITY);
        if (lane == 0) R->redf[wave] = m;
        __syncthreads();
        float mx = R->redf[0];
        for (int q = 1; q < WV; q++) mx = R->redf[q] > mx ? R->redf[q] : mx;
        const float ex = expf_ref_with(l - mx, tab);   /* every lane takes part */
        const float x = on && mx > -INFINITY ? ex : 0.0f;
        const double sum = wave_sum_f64((double)x);
        if (lane == 0) R->red[wave] = sum;
        __syncthreads();
        const double st = (R->red[0] + R->red[1]) + (R->red[2] + R->red[3]);   /* no expert is past 256 */
        p = st > 0.0 ? (float)((double)x / st) : 0.0f;
    }
    if (rank < k) {
        R->ids[rank] = tid;
        R->w[rank] = p;
        R->down[rank] = c.down;
    }
    __syncthreads();
    if (wave == 0) {   /* renormalise over the chosen, then scale */
        float wr = lane < k ? R->w[lane] : 0.0f;
        if (d.router != 1) {
            double s = 0.0;
            for (int r = 0; r < k; r++) s += (double)rdlane_f32(wr, r);
            if (d.router == 2) s += 1e-20;
            if (s > 0.0) wr = (float)((double)wr / s);
        }
        wr *= d.routed_scale;
        if (lane < k) {
            const int id = R->ids[lane], at = t * k + lane;
            ((int32_t *)(a.ws + a.L.ids))[at] = id;
            ((float *)(a.ws + a.L.w))[at] = wr;
            ((const void **)(a.ws + a.L.dptr))[at] = R->down[lane];
            if (a.ids) a.ids[at] = id;
            if (a.w) a.w[at] = wr;
        }
    }
}
__global__ __launch_bounds__(256) void k_fm_route(Args a) {
    __shared__ __align__(16) Route R;
    args_now(a.d.E, a.d.k, a.d.router, a.d.routed_scale, a.d.experts, a.ids, a.w, a.ws, a.L.key, a.L.score, a.L.ids, a.L.w,
             a.L.dptr);
    const Choice c = choice_of(a, blockIdx.x, threadIdx.x);
    ExpTabLanes tab;
    tab.load();
    const int rank = rank_of<4>(a, c, &R, threadIdx.x);
    route_token<4>(a, blockIdx.x, c, &R, rank, tab);
}

/* ---- an expert's tokens ------------------------------------------------------ */
struct List {
    int n, e, cnt[2][4];
    uint8_t sel[16];
    uint8_t tok[MAXT], rank[MAXT];
};
/* Which tokens of which slot a group takes: every `parts`th run from `part` on. */
struct Part {
    int slot, part, parts;
};
__device__ __forceinline__ Part part_of(const Args &a, int y) {
    if (y >= a.slots * a.ce) return {a.slots, y - a.slots * a.ce, a.cs};
    return {y / a.ce, y % a.ce, a.ce};
}
/* The pairs (token, rank) of slot `slot` and its expert: every token for the shared expert (E); expert
 * `slot`'s; or, with fewer choices than experts, those of the expert that pair `slot` chose, unless an
 * earlier pair chose it too (-1: nothing to do).  All threads; ends in a barrier. */
__device__ int slot_list(const Args &a, int slot, List *s) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, k = a.d.k, pairs = a.T * k;
    const GAS int32_t *ids = (const GAS int32_t *)(a.ws + a.L.ids);
    if (slot == a.slots) {
        if (tid < a.T) {
            s->tok[tid] = (uint8_t)tid;
            s->rank[tid] = 0;
        }
        if (tid == 0) s->n = a.T;
        __syncthreads();
        return a.d.E;
    }
    /* thread tid looks at pairs tid, tid + 256, ...: the first 512 at once */
    int id[2];
#pragma unroll
    for (int j = 0; j < 2; j++) id[j] = tid + 256 * j < pairs ? ids[tid + 256 * j] : -1;
    const int e = a.by_expert ? slot : uniform(ids[slot]);
    if (e < 0) return -1;
    int n = 0;
    for (int p0 = 0; p0 < pairs; p0 += 512) {
        if (p0 > 0)
#pragma unroll
            for (int j = 0; j < 2; j++) id[j] = p0 + tid + 256 * j < pairs ? ids[p0 + tid + 256 * j] : -1;
#pragma unroll
        for (int j = 0; j < 2; j++) {
            const unsigned long long m = __ballot(id[j] == e);
            if (lane == 0) s->cnt[j][wave] = __builtin_popcountll(m);
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 2; j++) {
            int at = n;
            for (int q = 0; q < 4 * j + wave; q++) at += s->cnt[q >> 2][q & 3];
            const unsigned long long m = __ballot(id[j] == e);
            if (id[j] == e) {
                const int p = p0 + tid + 256 * j;
                at += __builtin_popcountll(m & ((1ull << lane) - 1));
                s->tok[at] = (uint8_t)(p / k);
                s->rank[at] = (uint8_t)(p % k);
                if (at == 0) s->e = p;
            }
        }
        for (int q = 0; q < 8; q++) n += s->cnt[q >> 2][q & 3];
        __syncthreads();
    }
    if (tid == 0) s->n = n;
    __syncthreads();
    if (s->n == 0 || (!a.by_expert && s->e != slot)) return -1;
    return e;
}

/* The same list from the keys, for the launch that routes itself (T <= ROUTES): the tokens' keys are asked for
 * before the slot's expert is known, then each token's is ranked by ballots. */
constexpr int ROUTES = 16;
constexpr unsigned GROUPS = 1536;
__device__ int slot_list_keys(const Args &a, int slot, List *s, Route *R) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, k = a.d.k, E = a.d.E;
    if (slot == a.slots) return slot_list(a, slot, s);
    const GAS uint32_t *key = (const GAS uint32_t *)(a.ws + a.L.key);
    constexpr int TW = ROUTES / NW, KE = MAXE / 64;
    uint32_t kf[TW][KE];
#pragma unroll
    for (int j = 0; j < TW; j++) {
        const int t = wave + NW * j;
#pragma unroll
        for (int q = 0; q < KE; q++)
            kf[j][q] = 64 * q < E && t < a.T && lane + 64 * q < E ? key[(size_t)t * E + lane + 64 * q] : 0u;
    }
    int e = slot;
    if (!a.by_expert) {
        const Choice c = choice_of(a, slot / k, tid);
        if (tid == 0) s->e = -1;
        const int rank = rank_of<NW>(a, c, R, tid);
        if (rank == slot % k) s->e = tid;
        __syncthreads();
        e = uniform(s->e);
        if (e < 0) return -1;
    }
#pragma unroll
    for (int j = 0; j < TW; j++) {
        const int t = wave + NW * j;
        uint32_t ke = 0;
#pragma unroll
        for (int q = 0; q < KE; q++)
            if (e >> 6 == q) ke = (uint32_t)__builtin_amdgcn_readlane((int)kf[j][q], e & 63);
        int rank = 0;
#pragma unroll
        for (int q = 0; q < KE; q++)
            if (64 * q < E)
                rank += __builtin_popcountll(__ballot(kf[j][q] > ke || (kf[j][q] == ke && lane + 64 * q < e)));
        if (lane == 0) s->sel[t] = ke && rank < k ? (uint8_t)(rank + 1) : 0;   /* 0 past T: no keys */
    }
    __syncthreads();
    if (wave == 0) {
        const int sel = lane < a.T ? s->sel[lane < ROUTES ? lane : 0] : 0;
        const unsigned long long m = __ballot(sel != 0);
        if (sel) {
            const int at = __builtin_popcountll(m & ((1ull << lane) - 1));
            s->tok[at] = (uint8_t)lane;
            s->rank[at] = (uint8_t)(sel - 1);
        }
        if (lane == 0) s->n = __builtin_popcountll(m);
    }
    __syncthreads();
    if (s->n == 0 || (!a.by_expert && s->tok[0] != slot / k)) return -1;
    return e;
}

/* ---- 16 rows times up to NT * TPT tokens ------------------------------------- */
struct Mat {
    const GAS uint8_t *w;          /* the row tile's units */
    const GAS float *sw;           /* its 128-row block's scales */
};
__device__ __forceinline__ Mat mat_of(const void *packed, int tile, int64_t rows, int nb) {
    const GAS uint8_t *p = (const GAS uint8_t *)packed;
    return {p + (size_t)tile * nb * FP8_UNIT,
            (const GAS float *)(p + fp8_code_bytes(rows, (int64_t)nb * FP8_BLOCK)) + tile / 8 * nb};
}

/* This wave's share of the blocks for NQ column tiles; x[q]: this lane's part of its vector's planes.  One block
 * in flight a wave: with the next one's loads under way too the registers left room for fewer waves
 * (64 tokens of 2048 x 768, 128 experts 155 us, 167 with two).  No branch stands between a matrix
 * instruction and the reads of its result: the compiler here has left out the wait on such a path. */
template <int M, int NQ>
__device__ __forceinline__ void run_tiles(const Mat (&m)[M], int nb, int wave, const GAS uint16_t *const (&x)[NT],
                                          f32x4 (&acc)[M][NT]) {
    const int lane = threadIdx.x & 63;
    for (int b = wave; b < nb; b += NW) {
        i32x4 w[M][2];
        float sw[M];
        bf16x8 xv[NQ][4];
#pragma unroll
        for (int i = 0; i < M; i++) {
            sw[i] = m[i].sw[b];
#pragma unroll
            for (int h = 0; h < 2; h++) w[i][h] = *(const GAS i32x4 *)(m[i].w + (size_t)b * FP8_UNIT + h * 1024 + lane * 16);
        }
#pragma unroll
        for (int q = 0; q < NQ; q++)
#pragma unroll
            for (int j = 0; j < 4; j++) xv[q][j] = *(const GAS bf16x8 *)(x[q] + b * XBLOCK + 96 * j);
        f32x4 p[M][NQ] = {};
#pragma unroll
        for (int j = 0; j < 4; j++)
#pragma unroll
            for (int i = 0; i < M; i++) {
                const i32x4 c = w[i][j >> 1];
                const bf16x8 wv = (j & 1) ? fp8_to_bf16(c[2], c[3]) : fp8_to_bf16(c[0], c[1]);
#pragma unroll
                for (int q = 0; q < NQ; q++) p[i][q] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wv, xv[q][j], p[i][q], 0, 0, 0);
            }
#pragma unroll
        for (int q = 0; q < NQ; q++)
#pragma unroll
            for (int i = 0; i < M; i++)
#pragma unroll
                for (int v = 0; v < 4; v++) acc[i][q][v] = fmaf(p[i][q][v], sw[i], acc[i][q][v]);
    }
}
template <int M>
__device__ __forceinline__ void run_blocks(const Mat (&m)[M], int nb, int wave, const GAS uint16_t *const (&x)[NT],
                                           int nt, f32x4 (&acc)[M][NT]) {
    if (nt == 1) run_tiles<M, 1>(m, nb, wave, x, acc);
    else run_tiles<M, 2>(m, nb, wave, x, acc);
}

typedef f32x4 Sums[NW][NT][64];
/* the waves' and planes' sums for row r of the tile and token i of the pass */
__device__ __forceinline__ float total(const Sums &s, int r, int i) {
    const int q = i / TPT, l0 = (r >> 2) * 16 + 3 * (i % TPT), v = r & 3;
    float p[3];
#pragma unroll
    for (int j = 0; j < 3; j++) p[j] = (s[0][q][l0 + j][v] + s[1][q][l0 + j][v]) + (s[2][q][l0 + j][v] + s[3][q][l0 + j][v]);
    return p[0] + (p[1] + p[2]);
}

/* this lane's columns for the tokens from i0 on: token i0 + TPT q + column / 3, plane
 * column % 3; columns without a token repeat the last one */
__device__ __forceinline__ int column_index(int i0, int q, int n) {
    const int c = threadIdx.x & 15;
    const int i = i0 + TPT * q + (c < 15 ? c / 3 : 4);
    return i < n ? i : n - 1;
}

/* ---- K2 ----------------------------------------------------------------------- */
/* One token: every group routes it (all of its loads at once, then a count), so that nothing waits for
 * a launch of its own; the last row of groups does it for the later launch and for the caller.
 * 8 waves share the blocks of 16 rows of gate and up. */
__global__ __launch_bounds__(512) void k_fm_gateup_one(Args a) {
    constexpr int W = 8;
    __shared__ __align__(16) Route R;
    __shared__ const void *s_m[2];
    __shared__ f32x4 s_g[W][64], s_u[W][64];
    const tlm_hip_moe_desc &d = a.d;
    const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
    const int tile = blockIdx.x, slot = blockIdx.y;
    args_now(d.E, d.k, d.de, d.ds, d.router, d.routed_scale, d.experts, d.sg, d.su, a.ids, a.w, a.ws, a.slots, a.L.xp, a.L.key,
             a.L.score, a.L.ids, a.L.w, a.L.dptr, a.L.hid, a.L.shid, a.L.nbd, a.L.nbe, a.L.nbs);
    const bool shared = slot == a.slots && d.ds > 0;
    const int64_t rows = shared ? d.ds : d.de;
    const int nbo = shared ? a.L.nbs : a.L.nbe;
    if (tile >= nbo * 8) return;
    ExpTabLanes tab;
    tab.load();
    if (!shared) {
        const bool all = slot >= a.slots;   /* the row of groups that routes for the others; one is enough */
        if (all && tile != 0) return;
        const Choice c = choice_of(a, 0, tid);
        const int rank = rank_of<8>(a, c, &R, tid);
        if (all) {
            route_token<8>(a, 0, c, &R, rank, tab);
            return;
        }
        if (tid == 0) s_m[0] = nullptr;
        __syncthreads();
        if (rank == slot) {
            s_m[0] = c.gate;
            s_m[1] = c.up;
        }
        __syncthreads();
        if (!s_m[0]) return;   /* fewer experts than ranks */
    }
    uint16_t *hid = (uint16_t *)(a.ws + (shared ? a.L.shid : a.L.hid));
    const int wo = nbo * FP8_BLOCK, nb = a.L.nbd;
    const bool pad = tile >= fp8_tiles(rows);
    f32x4 acc[2] = {};
    if (!pad) {
        const Mat m[2] = {mat_of(shared ? d.sg : s_m[0], tile, rows, nb), mat_of(shared ? d.su : s_m[1], tile, rows, nb)};
        const GAS uint16_t *x = (const GAS uint16_t *)(a.ws + a.L.xp) + plane_lane();
        struct In {
            i32x4 w[2][2], x[4];
            float sw[2];
        };
        auto load = [&](In &n, int b) {
#pragma unroll
            for (int i = 0; i < 2; i++) {
                n.sw[i] = m[i].sw[b];
#pragma unroll
                for (int h = 0; h < 2; h++)
                    n.w[i][h] = *(const GAS i32x4 *)(m[i].w + (size_t)b * FP8_UNIT + h * 1024 + lane * 16);
            }
#pragma unroll
            for (int j = 0; j < 4; j++) n.x[j] = *(const GAS i32x4 *)(x + b * XBLOCK + 96 * j);
        };
        auto compute = [&](const In &n) {
            f32x4 p[2] = {};
#pragma unroll
            for (int j = 0; j < 4; j++)
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const i32x4 c = n.w[i][j >> 1];
                    p[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16((j & 1) ? fp8_to_bf16(c[2], c[3]) : fp8_to_bf16(c[0], c[1]),
                                                                   __builtin_bit_cast(bf16x8, n.x[j]), p[i], 0, 0, 0);
                }
#pragma unroll
            for (int i = 0; i < 2; i++)
#pragma unroll
                for (int v = 0; v < 4; v++) acc[i][v] = fmaf(p[i][v], n.sw[i], acc[i][v]);
        };
        if (wave < nb) {   /* the next block's loads are under way while one is computed */
            In cur;
            load(cur, wave);
            for (int b = wave + W; b < nb; b += W) {
                In nxt;
                load(nxt, b);
                compute(cur);
                cur = nxt;
            }
            compute(cur);
        }
    }
    s_g[wave][lane] = acc[0];
    s_u[wave][lane] = acc[1];
    __syncthreads();
    if (wave != 0) return;
    const int r = lane & 15;   /* a row; the other lanes repeat it */
    float g[3], u[3];
#pragma unroll
    for (int j = 0; j < 3; j++) {
        const int l = (r >> 2) * 16 + j;
        g[j] = u[j] = 0.0f;
#pragma unroll
        for (int q = 0; q < W; q++) {
            g[j] += s_g[q][l][r & 3];
            u[j] += s_u[q][l][r & 3];
        }
    }
    uint16_t p[3];
    split3(silu(g[0] + (g[1] + g[2]), tab) * (u[0] + (u[1] + u[2])), p);   /* 0 in the padding */
    const size_t at = (size_t)(shared ? 0 : slot) * 3 * wo;
    if (lane < 16)
#pragma unroll
        for (int j = 0; j < 3; j++) hid[at + plane_at(tile * 16 + r, j)] = p[j];
}

/* More tokens: 16 rows of one expert's gate and up for all of its tokens.  KEYS: the routing is not there
 * yet; the groups find it from the keys, and T groups more do it for the later launches. */
template <bool KEYS>
__global__ __launch_bounds__(256) void k_fm_gateup(Args a) {
    __shared__ List s;
    __shared__ Sums s_g, s_u;
    static_assert(sizeof(Route) <= sizeof(Sums) && MAXT >= ROUTES, "the routing's tables fit where the sums come");
    const tlm_hip_moe_desc &d = a.d;
    const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
    ExpTabLanes tab;
    tab.load();
    if (KEYS && (int)blockIdx.y >= a.slots * a.ce + a.cs) {
        Route *R = (Route *)&s_g;
        if ((int)blockIdx.x >= a.T) return;
        const Choice c = choice_of(a, blockIdx.x, tid);
        const int rank = rank_of<NW>(a, c, R, tid);
        route_token<NW>(a, blockIdx.x, c, R, rank, tab);
        return;
    }
    const Part pt = part_of(a, blockIdx.y);
    const int tile = blockIdx.x, slot = pt.slot;
    const bool shared = slot == a.slots;
    const int64_t rows = shared ? d.ds : d.de;
    const int nbo = shared ? a.L.nbs : a.L.nbe;      /* blocks of the width that this launch makes */
    if (tile >= nbo * 8) return;
    const int e = uniform(KEYS ? slot_list_keys(a, slot, &s, (Route *)&s_g) : slot_list(a, slot, &s));
    if (e < 0) return;
    const int n = uniform(s.n);
    uint16_t *hid = (uint16_t *)(a.ws + (shared ? a.L.shid : a.L.hid));
    const int wo = nbo * FP8_BLOCK;
    const bool pad = tile >= fp8_tiles(rows);        /* the padding of the next product's length: zeros */
    const void *const *mats = d.experts + 3 * (size_t)(shared ? 0 : e);
    Mat m[2];
    if (!pad) {
        m[0] = mat_of(shared ? d.sg : mats[0], tile, rows, a.L.nbd);
        m[1] = mat_of(shared ? d.su : mats[1], tile, rows, a.L.nbd);
    }
    const GAS uint16_t *xp = (const GAS uint16_t *)(a.ws + a.L.xp);
    const int Dp = a.L.nbd * FP8_BLOCK;
    for (int i0 = pt.part * NT * TPT; i0 < n; i0 += pt.parts * NT * TPT) {
        const int left = n - i0 < NT * TPT ? n - i0 : NT * TPT;
        if (!pad) {
            const GAS uint16_t *x[NT];
#pragma unroll
            for (int q = 0; q < NT; q++)
                x[q] = xp + (size_t)s.tok[column_index(i0, q, n)] * 3 * Dp + plane_lane();
            f32x4 acc[2][NT] = {};
            run_blocks<2>(m, a.L.nbd, wave, x, (left + TPT - 1) / TPT, acc);
#pragma unroll
            for (int q = 0; q < NT; q++) {
                s_g[wave][q][lane] = acc[0][q];
                s_u[wave][q][lane] = acc[1][q];
            }
        }
        __syncthreads();
        for (int o0 = 0; o0 < left * 16; o0 += 256) {   /* whole waves: the exponential's table is in their lanes */
            const int o = o0 + tid, r = o & 15, i = (o >> 4) < left ? o >> 4 : left - 1;
            const float v = pad ? 0.0f : silu(total(s_g, r, i), tab) * total(s_u, r, i);
            uint16_t p[3];
            split3(v, p);
            const int t = s.tok[i0 + i];
            const size_t at = (size_t)(shared ? t : t * d.k + s.rank[i0 + i]) * 3 * wo;
            if (o < left * 16)
#pragma unroll
                for (int j = 0; j < 3; j++) hid[at + plane_at(tile * 16 + r, j)] = p[j];
        }
        __syncthreads();
    }
}

/* ---- K3 ----------------------------------------------------------------------- */
/* DM row tiles a group: the planes are read once for all of them. */
constexpr int DM = 4;
__global__ __launch_bounds__(256) void k_fm_down(Args a) {
    __shared__ List s;
    __shared__ Sums s_y;
    const tlm_hip_moe_desc &d = a.d;
    const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
    const Part pt = part_of(a, blockIdx.y);
    const int tile0 = blockIdx.x * DM, slot = pt.slot, tiles = (int)fp8_tiles(d.D);
    const bool shared = slot == a.slots;
    const int e = uniform(slot_list(a, slot, &s));
    if (e < 0) return;
    const int n = uniform(s.n), nb = shared ? a.L.nbs : a.L.nbe, wi = nb * FP8_BLOCK;
    const GAS uint16_t *hid = (const GAS uint16_t *)(a.ws + (shared ? a.L.shid : a.L.hid));
    float *eo = (float *)(a.ws + (shared ? a.L.seo : a.L.eo));
    const void *packed = shared ? d.sd : d.experts[3 * (size_t)e + 2];
    Mat m[DM];
#pragma unroll
    for (int i = 0; i < DM; i++) m[i] = mat_of(packed, tile0 + i < tiles ? tile0 + i : tiles - 1, d.D, nb);
    for (int i0 = pt.part * NT * TPT; i0 < n; i0 += pt.parts * NT * TPT) {
        const int left = n - i0 < NT * TPT ? n - i0 : NT * TPT;
        const GAS uint16_t *x[NT];
#pragma unroll
        for (int q = 0; q < NT; q++) {
            const int i = column_index(i0, q, n), t = s.tok[i];
            x[q] = hid + (size_t)(shared ? t : t * d.k + s.rank[i]) * 3 * wi + plane_lane();
        }
        f32x4 acc[DM][NT] = {};
        run_blocks<DM>(m, nb, wave, x, (left + TPT - 1) / TPT, acc);
#pragma unroll
        for (int j = 0; j < DM; j++) {
#pragma unroll
            for (int q = 0; q < NT; q++) s_y[wave][q][lane] = acc[j][q];
            __syncthreads();
            for (int o = tid; o < left * 16; o += 256) {
                const int r = o & 15, i = o >> 4, t = s.tok[i0 + i];
                const int64_t row = (int64_t)(tile0 + j) * 16 + r;
                if (row < d.D) eo[(size_t)(shared ? t : t * d.k + s.rank[i0 + i]) * d.D + row] = total(s_y, r, i);
            }
            __syncthreads();
        }
    }
}

/* ---- K3 for few tokens: down and the sum ------------------------------------------
 * A group takes 16 rows of one token's result: the blocks of all its experts' down rows, and of
 * the shared expert's, are dealt to the waves, each scaled by its expert's weight as it is added.  A
 * matrix that two tokens share is read by both. */
__global__ __launch_bounds__(512) void k_fm_down_few(Args a) {
    constexpr int DW = 8, U = 2;
    __shared__ f32x4 s_sum[DW][64];
    __shared__ const uint8_t *s_ptr[MAXK + 1];
    __shared__ float s_w[MAXK + 1];
    const tlm_hip_moe_desc &d = a.d;
    args_now(d.D, d.k, d.sd, d.shared_gate_inp, a.h, a.out, a.ws, a.L.ids, a.L.w, a.L.dptr, a.L.sgate, a.L.hid, a.L.shid,
             a.L.nbe, a.L.nbs);
    const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
    const int tile = blockIdx.x, t = blockIdx.y, k = d.k, nbe = a.L.nbe, nbs = a.L.nbs;
    const uint8_t *ptr = nullptr;
    float wt = 0.0f;
    if (tid < k) {
        ptr = ((const uint8_t *const GAS *)(a.ws + a.L.dptr))[t * k + tid];
        wt = ((const GAS float *)(a.ws + a.L.w))[t * k + tid];
    }
    if (tid == k && nbs) {
        ptr = (const uint8_t *)d.sd;
        wt = d.shared_gate_inp ? ((const GAS float *)(a.ws + a.L.sgate))[t] : 1.0f;
    }
    const int units = k * nbe + nbs;
    const size_t code_e = (size_t)fp8_tiles(d.D) * nbe * FP8_UNIT, code_s = (size_t)fp8_tiles(d.D) * nbs * FP8_UNIT;
    const GAS uint16_t *hid = (const GAS uint16_t *)(a.ws + a.L.hid) + (size_t)t * k * nbe * XBLOCK + plane_lane();
    const GAS uint16_t *shid = (const GAS uint16_t *)(a.ws + a.L.shid) + (size_t)t * nbs * XBLOCK + plane_lane();
    f32x4 acc = {0, 0, 0, 0};
    struct In {
        i32x4 w[U][2], x[U][4];
        float sc[U];
        bool on[U];
    };
    auto planes = [&](In &n, int u0) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int v = u0 + u * DW < units ? u0 + u * DW : units - 1;   /* past the end: read again, not added */
            const int r = v < k * nbe ? v / nbe : k, b = v - r * nbe;
            const GAS uint16_t *xx = (r < k ? hid + (size_t)r * nbe * XBLOCK : shid) + b * XBLOCK;
#pragma unroll
            for (int j = 0; j < 4; j++) n.x[u][j] = *(const GAS i32x4 *)(xx + 96 * j);
        }
    };
    auto weights = [&](In &n, int u0) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int v = u0 + u * DW < units ? u0 + u * DW : units - 1;
            const int r = v < k * nbe ? v / nbe : k, nb = r < k ? nbe : nbs, b = v - r * nbe;
            const GAS uint8_t *p = (const GAS uint8_t *)s_ptr[r];
            n.on[u] = u0 + u * DW < units && p != nullptr;   /* a rank without an expert adds nothing: */
            const GAS uint8_t *q = (const GAS uint8_t *)a.ws, *z = q;   /* the workspace (over 2 KB) is read for it */
            if (p) {
                q = p + ((size_t)tile * nb + b) * FP8_UNIT;
                z = p + (r < k ? code_e : code_s) + 4 * (tile / 8 * nb + b);
            }
            n.w[u][0] = *(const GAS i32x4 *)(q + lane * 16);
            n.w[u][1] = *(const GAS i32x4 *)(q + lane * 16 + 1024);
            n.sc[u] = s_w[r] * *(const GAS float *)z;
        }
    };
    auto compute = [&](const In &n) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            f32x4 p = {0, 0, 0, 0};
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const i32x4 c = n.w[u][j >> 1];
                const bf16x8 wv = (j & 1) ? fp8_to_bf16(c[2], c[3]) : fp8_to_bf16(c[0], c[1]);
                p = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wv, __builtin_bit_cast(bf16x8, n.x[u][j]), p, 0, 0, 0);
            }
#pragma unroll
            for (int v = 0; v < 4; v++) {
                const float f = fmaf(p[v], n.sc[u], acc[v]);
                acc[v] = n.on[u] ? f : acc[v];
            }
        }
    };
    In cur;
    planes(cur, wave);   /* they do not wait for the routing */
    if (tid <= k) {
        s_ptr[tid] = ptr;
        s_w[tid] = wt;
    }
    __syncthreads();
    if (wave < units) {   /* the next blocks' loads are under way while some are computed */
        weights(cur, wave);
        for (int u0 = wave + DW * U; u0 < units; u0 += DW * U) {
            In nxt;
            weights(nxt, u0);
            planes(nxt, u0);
            compute(cur);
            cur = nxt;
        }
        compute(cur);
    }
    s_sum[wave][lane] = acc;
    __syncthreads();
    const int64_t i = (int64_t)tile * 16 + tid;
    if (tid >= 16 || i >= d.D) return;
    float p[3];
#pragma unroll
    for (int j = 0; j < 3; j++) {
        float v = 0.0f;
#pragma unroll
        for (int q = 0; q < DW; q++) v += s_sum[q][(tid >> 2) * 16 + j][tid & 3];
        p[j] = v;
    }
    const size_t at = (size_t)t * d.D + i;
    a.out[at] = a.h[at] + (p[0] + (p[1] + p[2]));
}

/* ---- K4 ----------------------------------------------------------------------- */
__global__ __launch_bounds__(256) void k_fm_combine(Args a) {
    const tlm_hip_moe_desc &d = a.d;
    const int t = blockIdx.y;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= d.D) return;
    const GAS float *eo = (const GAS float *)(a.ws + a.L.eo) + (size_t)t * d.k * d.D + i;
    const GAS int32_t *ids = (const GAS int32_t *)(a.ws + a.L.ids) + t * d.k;
    const GAS float *w = (const GAS float *)(a.ws + a.L.w) + t * d.k;
    float acc = 0.0f;
    for (int r = 0; r < d.k; r++) {
        const float v = eo[(size_t)r * d.D];
        acc = ids[r] >= 0 ? acc + w[r] * v : acc;   /* a rank without an expert has no result */
    }
    if (d.ds > 0) {
        const float g = d.shared_gate_inp ? ((const GAS float *)(a.ws + a.L.sgate))[t] : 1.0f;
        acc += g * ((const GAS float *)(a.ws + a.L.seo))[(size_t)t * d.D + i];
    }
    a.out[(size_t)t * d.D + i] = a.h[(size_t)t * d.D + i] + acc;
}

/* The shared expert's tokens go to as many groups as their runs of NT * TPT; an expert's to as many as twice
 * the mean list has (a longer list's runs wrap round). */
void spread(Args &a) {
    constexpr int RUN = NT * TPT;
    const int runs = (a.T + RUN - 1) / RUN, twice = (2 * a.T * a.d.k + a.d.E * RUN - 1) / (a.d.E * RUN);
    a.cs = a.d.ds > 0 ? runs : 0;
    a.ce = !a.by_expert ? 1 : twice < runs ? twice : runs;
}

/* Whether down runs per token (k_fm_down_few) or per expert (k_fm_down, then k_fm_combine).  Per token saves
 * a launch and the results' way through memory, reads a matrix once for each token that chose it and takes 8
 * waves for a token's 16 rows: while the matrices read again come to at most 100 MB, and all of its groups fit
 * the chip at once, or there are no more choices than experts and a block for each wave.  Whole layers, per
 * token against per expert: 2048 x 768, 128 experts top-8: 8 tokens (22 MB) 60.4 against 68.2 us, 16 (94 MB)
 * 97 and 101, 24 (217 MB) 122 and 118; 4096 x 1536, 6 tokens (47 MB) 151 and 152, 12 (207 MB) 256 and 244;
 * 1000 x 300, 8 experts top-4, 4 tokens 14.3 and 18.2; more choices than experts and not one round: 3000 x
 * 500, 16 experts top-4, 8 tokens 32.3 and 30.9; two blocks for 8 waves: 512 x 128, 128 experts top-2, 64
 * tokens 32.4 and 30.5. */
bool by_token(const tlm_hip_moe_desc &d, const Layout &L, int64_t T) {
    if (T == 1) return true;
    const double pairs = (double)T * d.k, again = pairs * (double)(T - 1) * d.k / (2.0 * d.E);
    if (again * (double)d.D * (double)d.de > 100e6) return false;
    return fp8_tiles(d.D) * T * 8 <= 256 * 16 || (pairs <= d.E && d.k * L.nbe + L.nbs >= 8);
}

int check(const tlm_hip_moe_desc *d, int64_t T) {
    if (!d) return tlmh_seterr(TLM_HIP_EINVAL, "fp8_moe: NULL descriptor");
    if (d->E <= 0 || d->E > MAXE || d->k <= 0 || d->k > MAXK || d->k > d->E)
        return tlmh_seterr(TLM_HIP_EINVAL, "fp8_moe: E=%d k=%d outside 1 <= k <= E <= %d, k <= %d", d->E, d->k, MAXE,
                           MAXK);
    if (d->router < 0 || d->router > 2) return tlmh_seterr(TLM_HIP_EINVAL, "fp8_moe: router kind %d", d->router);
    if (d->expert_dt != TLM_HIP_DT_FP8 || (d->ds > 0 && d->shared_dt != TLM_HIP_DT_FP8))
        return tlmh_seterr(TLM_HIP_EUNSUP, "fp8_moe: expert dtype %d / shared dtype %d (FP8 only)", d->expert_dt,
                           d->shared_dt);
    if (d->D < 1 || d->D > 16384 || d->de < 1 || d->de > 65536 || d->ds < 0 || d->ds > 65536)
        return tlmh_seterr(TLM_HIP_EINVAL, "fp8_moe: D=%lld de=%lld ds=%lld outside 1..16384, 1..65536, 0..65536",
                           (long long)d->D, (long long)d->de, (long long)d->ds);
    if (T < 0 || T > MAXT)
        return tlmh_seterr(TLM_HIP_ERANGE, "fp8_moe: %lld tokens outside 0..%d", (long long)T, MAXT);
    return TLM_HIP_OK;
}

}  // namespace

extern "C" {

size_t tlm_hip_fp8_moe_workspace_bytes(const tlm_hip_moe_desc *d, int64_t T) {
    return check(d, T) || T == 0 ? 0 : layout(*d, T).total;
}

int tlm_hip_fp8_moe(const tlm_hip_moe_desc *d, const float *h, float *out, int64_t T, int32_t *ids, float *w,
                    void *workspace, void *stream) {
    if (int rc = check(d, T)) return rc;
    if (T == 0) return TLM_HIP_OK;
    if (!h || !out || !workspace || !d->ffn_norm || !d->router_w || !d->experts ||
        (d->ds > 0 && (!d->sg || !d->su || !d->sd)))
        return tlmh_seterr(TLM_HIP_EINVAL, "fp8_moe: NULL argument or weights");
    if ((uintptr_t)workspace & 255u)
        return tlmh_seterr(TLM_HIP_EINVAL, "fp8_moe: workspace must be 256-byte aligned");
    if (((uintptr_t)h | (uintptr_t)out | (uintptr_t)ids | (uintptr_t)w | (uintptr_t)d->ffn_norm |
         (uintptr_t)d->router_w | (uintptr_t)d->router_bias | (uintptr_t)d->shared_gate_inp) & 3u)
        return tlmh_seterr(TLM_HIP_EINVAL, "fp8_moe: tensors must be 4-byte aligned");
    if (((uintptr_t)d->experts & 7u) || (d->ds > 0 && (((uintptr_t)d->sg | (uintptr_t)d->su | (uintptr_t)d->sd) & 15u)))
        return tlmh_seterr(TLM_HIP_EINVAL, "fp8_moe: the table must be 8-byte, packed matrices 16-byte aligned");
    const uintptr_t gap = (uintptr_t)h < (uintptr_t)out ? (uintptr_t)out - (uintptr_t)h : (uintptr_t)h - (uintptr_t)out;
    if (gap && gap < (size_t)T * (size_t)d->D * 4)   /* a token's group reads h where another's has stored */
        return tlmh_seterr(TLM_HIP_EINVAL, "fp8_moe: out must be h itself or not overlap it");
    if (int rc = tlmh_refuse_failed(FAILED_FP8, "fp8_moe")) return rc;
    Args a{};
    a.d = *d;
    a.L = layout(*d, T);
    a.h = h;
    a.out = out;
    a.ids = ids;
    a.w = w;
    a.ws = (uint8_t *)workspace;
    a.T = (int)T;
    a.inv_D = 1.0 / (double)d->D;
    a.by_expert = T > 1 && T * d->k >= d->E;
    a.slots = a.by_expert ? d->E : (int)(T * d->k);
    spread(a);
    const unsigned ny = (unsigned)(a.slots + (d->ds > 0 ? 1 : 0));
    const int wide = a.L.nbe > a.L.nbs ? a.L.nbe : a.L.nbs;
    hipStream_t s = (hipStream_t)stream;
    const unsigned rows = (unsigned)(d->E + (d->ds > 0 && d->shared_gate_inp ? 1 : 0));
    hipLaunchKernelGGL(k_fm_router, dim3((rows + 3) / 4, (unsigned)T), dim3(256), (size_t)((d->D + 3) & ~(int64_t)3) * 4, s, a);
    if (T == 1) {
        hipLaunchKernelGGL(k_fm_gateup_one, dim3((unsigned)wide * 8, ny + 1), dim3(512), 0, s, a);
    } else {
        const unsigned ys = (unsigned)(a.slots * a.ce + a.cs), xs = (unsigned)wide * 8;
        /* Routing in the gate/up launch saves one, and each group the work of a rank: worth it up to
         * 6 groups a compute unit (2048 x 768, 128 experts: 2 tokens, 768 groups, 26.5 against 28.6 us,
         * 4 tokens, 1536 groups, 40.5 and 40.6, 8 tokens, twice as many, 62.8 and 60.6; 1000 x 300, 32
         * experts, 8 tokens, 768 groups, 18.9 and 21.6). */
        if (T <= ROUTES && xs * ys <= GROUPS) {   /* one more row of groups: one a token routes */
            hipLaunchKernelGGL(k_fm_gateup<true>, dim3(xs > (unsigned)T ? xs : (unsigned)T, ys + 1), dim3(64 * NW), 0, s, a);
        } else {
            hipLaunchKernelGGL(k_fm_route, dim3((unsigned)T), dim3(256), 0, s, a);
            hipLaunchKernelGGL(k_fm_gateup<false>, dim3(xs, ys), dim3(64 * NW), 0, s, a);
        }
    }
    if (by_token(*d, a.L, T)) {
        const dim3 grid((unsigned)fp8_tiles(d->D), (unsigned)T);
        hipLaunchKernelGGL(k_fm_down_few, grid, dim3(512), 0, s, a);
    } else {
        hipLaunchKernelGGL(k_fm_down, dim3((unsigned)((fp8_tiles(d->D) + DM - 1) / DM), (unsigned)(a.slots * a.ce + a.cs)),
                           dim3(64 * NW), 0, s, a);
        hipLaunchKernelGGL(k_fm_combine, dim3((unsigned)((d->D + 255) / 256), (unsigned)T), dim3(256), 0, s, a);
    }
    return tlmh_check(hipGetLastError(), "fp8_moe launch");
}

}  // extern "C"
