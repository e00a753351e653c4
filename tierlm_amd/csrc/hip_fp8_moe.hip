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
 *   K1 router   x, its planes, the router's scores and the selection keys
 *   K2 gate/up  a group per 16 rows of one expert's gate and up, for all of its
 *               tokens: silu(g) * u as planes
 *   K3 down     a group per 16 rows of one expert's down: the unweighted results
 *   K4 combine  per token: routing weights, the sum in rank order, the residual
 * K2 and K3 find an expert's tokens themselves from the keys: expert e is among
 * token t's k if fewer than k of t's keys are larger than e's, a count that takes
 * a wave a few ballots. */
#include "tlm_hip_fp8.h"

namespace {

constexpr int MAXT = TLM_HIP_FP8_MOE_MAX_TOKENS;   /* 64: a token per lane in the lists */
constexpr int MAXE = 256, MAXK = 32;
constexpr int NW = 4;              /* waves per group of K2 and K3: the blocks of a row are dealt to them */
constexpr int TPT = 5;             /* tokens per 16 columns */
constexpr int NT = 4;              /* column tiles at a time */

__host__ __device__ inline size_t al256(size_t v) { return (v + 255) & ~(size_t)255; }

struct Layout {
    size_t xp, key, score, sgate, hid, shid, eo, seo, total;
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
};

/* a value that all lanes of a wave share, in a scalar register: branches on it are the
 * wave's, and no matrix instruction ends up under a lane mask */
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

/* order of selection values as unsigned integers; -0 as +0, NaN as -infinity.  0 is
 * left for experts that cannot be chosen. */
__device__ __forceinline__ uint32_t order_key(float f) {
    const uint32_t b = __float_as_uint(f != f ? -INFINITY : f + 0.0f);
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float silu(float x) { return x / (1.0f + expf_ref(-x)); }

/* ---- K1 --------------------------------------------------------------------- */
constexpr int ROUTER_EXPERTS = 8;   /* experts per group */

__global__ __launch_bounds__(256) void k_fm_router(Args a) {
    extern __shared__ __align__(16) float s_x[];
    __shared__ double s_red[4];
    const tlm_hip_moe_desc &d = a.d;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, t = blockIdx.y;
    const int D = (int)d.D;
    const float *h = a.h + (size_t)t * D;
    double ss = 0.0;
    for (int i = tid; i < D; i += 256) {
        const float v = h[i];
        s_x[i] = v;
        ss += (double)v * (double)v;
    }
    ss = wave_sum_f64(ss);
    if (lane == 0) s_red[wave] = ss;
    __syncthreads();
    ss = (s_red[0] + s_red[1]) + (s_red[2] + s_red[3]);
    const float rn = 1.0f / sqrtf((float)(ss / (double)D) + d.eps);
    const int Dp = a.L.nbd * FP8_BLOCK;
    uint16_t *xp = (uint16_t *)(a.ws + a.L.xp) + (size_t)t * 3 * Dp;
    for (int i = tid; i < Dp; i += 256) {
        const float v = i < D ? s_x[i] * rn * d.ffn_norm[i] : 0.0f;
        if (i < D) s_x[i] = v;
        if ((i >> 8) % gridDim.x == blockIdx.x) {   /* the groups share the planes' writing */
            uint16_t p[3];
            split3(v, p);
            xp[i] = p[0];
            xp[Dp + i] = p[1];
            xp[2 * Dp + i] = p[2];
        }
    }
    __syncthreads();
    const int rows = (int)min((int64_t)ROUTER_EXPERTS, (int64_t)d.E - (int64_t)blockIdx.x * ROUTER_EXPERTS);
    const bool gate = d.ds > 0 && d.shared_gate_inp && blockIdx.x == 0;
    for (int r = wave; r < rows + (gate ? 1 : 0); r += 4) {
        const int e = blockIdx.x * ROUTER_EXPERTS + r;
        const float *w = r < rows ? d.router_w + (size_t)e * D : d.shared_gate_inp;
        /* double: two experts' scores keep their order down to the last bit of a float */
        double acc = 0.0;
        for (int i = lane; i < D; i += 64) acc = __builtin_fma((double)w[i], (double)s_x[i], acc);
        acc = wave_sum_f64(acc);
        if (lane != 0) continue;
        const float l = (float)acc;
        if (r == rows) {
            ((float *)(a.ws + a.L.sgate))[t] = 1.0f / (1.0f + expf_ref(-l));
            continue;
        }
        float score = l, sel = l;
        if (d.router == 2) {
            score = 1.0f / (1.0f + expf_ref(-l));
            sel = d.router_bias ? score + d.router_bias[e] : score;
        }
        ((float *)(a.ws + a.L.score))[t * d.E + e] = score;
        ((uint32_t *)(a.ws + a.L.key))[t * d.E + e] = d.mask && d.mask[e] ? 0u : order_key(sel);
    }
}

/* ---- an expert's tokens ------------------------------------------------------ */
struct List {
    int n;
    uint8_t tok[MAXT], rank[MAXT];
};

__device__ __forceinline__ bool ahead(uint32_t kf, int f, uint32_t ke, int e) {
    return kf > ke || (kf == ke && f < e);
}

/* The tokens that chose expert e, ascending, with its rank among their k.  All
 * threads; ends in a barrier. */
__device__ void find_tokens(const Args &a, int e, List *s, uint8_t *s_sel) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, E = a.d.E;
    const uint32_t *key = (const uint32_t *)(a.ws + a.L.key);
    for (int t = wave; t < a.T; t += NW) {
        const uint32_t ke = key[t * E + e];
        int rank = 0;
        for (int f0 = 0; f0 < E; f0 += 64) {
            const int f = f0 + lane;
            const uint32_t kf = f < E ? key[t * E + f] : 0u;
            rank += __builtin_popcountll(__ballot(f < E && kf && ahead(kf, f, ke, e)));
        }
        if (lane == 0) s_sel[t] = ke && rank < a.d.k ? (uint8_t)(rank + 1) : 0;
    }
    __syncthreads();
    if (wave == 0) {
        const int sel = lane < a.T ? s_sel[lane] : 0;
        const unsigned long long m = __ballot(sel != 0);
        if (sel) {
            const int at = __builtin_popcountll(m & ((1ull << lane) - 1));
            s->tok[at] = (uint8_t)lane;
            s->rank[at] = (uint8_t)(sel - 1);
        }
        if (lane == 0) s->n = __builtin_popcountll(m);
    }
    __syncthreads();
}

/* The list of slot `slot`: the shared expert (every token), expert `slot`, or, with
 * fewer choices than experts, the expert of token slot / k at rank slot % k unless an
 * earlier token chose it too.  Returns the expert, or -1 for nothing to do;
 * E for the shared one. */
__device__ int slot_list(const Args &a, int slot, List *s, uint8_t *s_sel, int *s_e) {
    const int tid = threadIdx.x, E = a.d.E;
    if (slot == a.slots) {
        if (tid < a.T) {
            s->tok[tid] = (uint8_t)tid;
            s->rank[tid] = 0;
        }
        if (tid == 0) s->n = a.T;
        __syncthreads();
        return E;
    }
    int e = slot;
    if (!a.by_expert) {
        const uint32_t *key = (const uint32_t *)(a.ws + a.L.key) + (size_t)(slot / a.d.k) * E;
        if (tid == 0) *s_e = -1;
        __syncthreads();
        const uint32_t ke = tid < E ? key[tid] : 0u;
        int rank = 0;
        for (int f = 0; f < E; f++) {
            const uint32_t kf = key[f];
            rank += kf && ahead(kf, f, ke, tid) ? 1 : 0;
        }
        if (tid < E && ke && rank == slot % a.d.k) *s_e = tid;
        __syncthreads();
        e = *s_e;
        if (e < 0) return -1;
    }
    find_tokens(a, e, s, s_sel);
    if (s->n == 0 || (!a.by_expert && s->tok[0] != slot / a.d.k)) return -1;
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

/* This wave's share of the blocks, for NQ column tiles; x[q]: this lane's column of
 * planes.  No branch stands between a matrix instruction and the reads of its result: the
 * compiler here has left out the wait on such a path. */
template <int M, int NQ>
__device__ __forceinline__ void run_tiles(const Mat (&m)[M], int nb, int wave, const uint16_t *const (&x)[NT],
                                          f32x4 (&acc)[M][NT]) {
    const int lane = threadIdx.x & 63;
    for (int b = wave; b < nb; b += NW) {
        i32x4 w[M][2];
        float sw[M];
#pragma unroll
        for (int i = 0; i < M; i++) {
            sw[i] = m[i].sw[b];
#pragma unroll
            for (int h = 0; h < 2; h++)
                w[i][h] = *(const GAS i32x4 *)(m[i].w + (size_t)b * FP8_UNIT + h * 1024 + lane * 16);
        }
        f32x4 p[M][NQ] = {};
#pragma unroll
        for (int j = 0; j < 4; j++) {
            bf16x8 wv[M];
#pragma unroll
            for (int i = 0; i < M; i++) {
                const i32x4 c = w[i][j >> 1];
                wv[i] = (j & 1) ? fp8_to_bf16(c[2], c[3]) : fp8_to_bf16(c[0], c[1]);
            }
#pragma unroll
            for (int q = 0; q < NQ; q++) {
                const bf16x8 xv = *(const GAS bf16x8 *)(x[q] + b * FP8_BLOCK + 64 * (j >> 1) + 8 * (j & 1));
#pragma unroll
                for (int i = 0; i < M; i++)
                    p[i][q] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wv[i], xv, p[i][q], 0, 0, 0);
            }
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
__device__ __forceinline__ void run_blocks(const Mat (&m)[M], int nb, int wave, const uint16_t *const (&x)[NT], int nt,
                                           f32x4 (&acc)[M][NT]) {
    switch (nt) {
    case 1: run_tiles<M, 1>(m, nb, wave, x, acc); break;
    case 2: run_tiles<M, 2>(m, nb, wave, x, acc); break;
    case 3: run_tiles<M, 3>(m, nb, wave, x, acc); break;
    default: run_tiles<M, 4>(m, nb, wave, x, acc); break;
    }
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
__device__ __forceinline__ int column_plane() { return (threadIdx.x & 15) % 3; }

/* ---- K2 ----------------------------------------------------------------------- */
__global__ __launch_bounds__(256) void k_fm_gateup(Args a) {
    __shared__ List s;
    __shared__ uint8_t s_sel[MAXT];
    __shared__ int s_e;
    __shared__ Sums s_g, s_u;
    const tlm_hip_moe_desc &d = a.d;
    const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
    const int tile = blockIdx.x, slot = blockIdx.y;
    const bool shared = slot == a.slots;
    const int64_t rows = shared ? d.ds : d.de;
    const int nbo = shared ? a.L.nbs : a.L.nbe;      /* blocks of the width that this launch makes */
    if (tile >= nbo * 8) return;
    const int e = uniform(slot_list(a, slot, &s, s_sel, &s_e));
    if (e < 0) return;
    const int n = uniform(s.n);
    uint16_t *hid = (uint16_t *)(a.ws + (shared ? a.L.shid : a.L.hid));
    const int wo = nbo * FP8_BLOCK;
    const bool pad = tile >= fp8_tiles(rows);        /* the padding of the next product's length: zeros */
    const void *const *tab = d.experts + 3 * (size_t)(shared ? 0 : e);
    Mat m[2];
    if (!pad) {
        m[0] = mat_of(shared ? d.sg : tab[0], tile, rows, a.L.nbd);
        m[1] = mat_of(shared ? d.su : tab[1], tile, rows, a.L.nbd);
    }
    const uint16_t *xp = (const uint16_t *)(a.ws + a.L.xp);
    const int Dp = a.L.nbd * FP8_BLOCK;
    for (int i0 = 0; i0 < n; i0 += NT * TPT) {
        const int left = n - i0 < NT * TPT ? n - i0 : NT * TPT;
        if (!pad) {
            const uint16_t *x[NT];
#pragma unroll
            for (int q = 0; q < NT; q++)
                x[q] = xp + ((size_t)s.tok[column_index(i0, q, n)] * 3 + column_plane()) * Dp + 16 * (lane >> 4);
            f32x4 acc[2][NT] = {};
            run_blocks<2>(m, a.L.nbd, wave, x, (left + TPT - 1) / TPT, acc);
#pragma unroll
            for (int q = 0; q < NT; q++) {
                s_g[wave][q][lane] = acc[0][q];
                s_u[wave][q][lane] = acc[1][q];
            }
        }
        __syncthreads();
        for (int o = tid; o < left * 16; o += 256) {
            const int r = o & 15, i = o >> 4;
            float v = 0.0f;
            if (!pad) v = silu(total(s_g, r, i)) * total(s_u, r, i);
            uint16_t p[3];
            split3(v, p);
            const int t = s.tok[i0 + i];
            const size_t at = (size_t)(shared ? t : t * d.k + s.rank[i0 + i]) * 3 * wo + tile * 16 + r;
            hid[at] = p[0];
            hid[at + wo] = p[1];
            hid[at + 2 * wo] = p[2];
        }
        __syncthreads();
    }
}

/* ---- K3 ----------------------------------------------------------------------- */
__global__ __launch_bounds__(256) void k_fm_down(Args a) {
    __shared__ List s;
    __shared__ uint8_t s_sel[MAXT];
    __shared__ int s_e;
    __shared__ Sums s_y;
    const tlm_hip_moe_desc &d = a.d;
    const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
    const int tile = blockIdx.x, slot = blockIdx.y;
    const bool shared = slot == a.slots;
    const int e = uniform(slot_list(a, slot, &s, s_sel, &s_e));
    if (e < 0) return;
    const int n = uniform(s.n), nb = shared ? a.L.nbs : a.L.nbe, wi = nb * FP8_BLOCK;
    const uint16_t *hid = (const uint16_t *)(a.ws + (shared ? a.L.shid : a.L.hid));
    float *eo = (float *)(a.ws + (shared ? a.L.seo : a.L.eo));
    const Mat m[1] = {mat_of(shared ? d.sd : d.experts[3 * (size_t)e + 2], tile, d.D, nb)};
    for (int i0 = 0; i0 < n; i0 += NT * TPT) {
        const int left = n - i0 < NT * TPT ? n - i0 : NT * TPT;
        const uint16_t *x[NT];
#pragma unroll
        for (int q = 0; q < NT; q++) {
            const int i = column_index(i0, q, n), t = s.tok[i];
            x[q] = hid + ((size_t)(shared ? t : t * d.k + s.rank[i]) * 3 + column_plane()) * wi + 16 * (lane >> 4);
        }
        f32x4 acc[1][NT] = {};
        run_blocks<1>(m, nb, wave, x, (left + TPT - 1) / TPT, acc);
#pragma unroll
        for (int q = 0; q < NT; q++) s_y[wave][q][lane] = acc[0][q];
        __syncthreads();
        for (int o = tid; o < left * 16; o += 256) {
            const int r = o & 15, i = o >> 4, t = s.tok[i0 + i];
            if (tile * 16 + r < d.D)
                eo[(size_t)(shared ? t : t * d.k + s.rank[i0 + i]) * d.D + tile * 16 + r] = total(s_y, r, i);
        }
        __syncthreads();
    }
}

/* ---- K4 ----------------------------------------------------------------------- */
/* A token's experts and weights in rank order: ranks past the number of experts that
 * can be chosen get id -1 and weight 0.  All threads; ends in a barrier. */
struct Route {
    int ids[MAXK];
    float w[MAXK];
    float redf[NW];
    double red[NW];
};
__device__ void route_token(const Args &a, int t, Route *R) {
    const tlm_hip_moe_desc &d = a.d;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, E = d.E, k = d.k;
    const uint32_t *key = (const uint32_t *)(a.ws + a.L.key) + (size_t)t * E;
    const bool in = tid < E;
    const uint32_t ke = in ? key[tid] : 0u;
    const float l = in ? ((const float *)(a.ws + a.L.score))[t * E + tid] : 0.0f;
    if (tid < MAXK) {
        R->ids[tid] = -1;
        R->w[tid] = 0.0f;
    }
    float p = l;
    if (d.router != 2) {   /* softmax over the experts that can be chosen */
        const bool on = ke && l == l;
        const float m = wave_max_f32(on ? l : -INFINITY);
        if (lane == 0) R->redf[wave] = m;
        __syncthreads();
        float mx = R->redf[0];
        for (int q = 1; q < NW; q++) mx = R->redf[q] > mx ? R->redf[q] : mx;
        const float x = on && mx > -INFINITY ? expf_ref(l - mx) : 0.0f;
        const double sum = wave_sum_f64((double)x);
        if (lane == 0) R->red[wave] = sum;
        __syncthreads();
        const double st = (R->red[0] + R->red[1]) + (R->red[2] + R->red[3]);
        p = st > 0.0 ? (float)((double)x / st) : 0.0f;
    }
    int rank = 0;
    for (int f = 0; f < E; f++) {
        const uint32_t kf = key[f];
        rank += kf && ahead(kf, f, ke, tid) ? 1 : 0;
    }
    __syncthreads();
    if (ke && rank < k) {
        R->ids[rank] = tid;
        R->w[rank] = p;
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
        if (lane < k) R->w[lane] = wr;
    }
    __syncthreads();
}

__global__ __launch_bounds__(256) void k_fm_combine(Args a) {
    __shared__ Route R;
    const tlm_hip_moe_desc &d = a.d;
    const int t = blockIdx.y;
    route_token(a, t, &R);
    if (blockIdx.x == 0 && (int)threadIdx.x < d.k) {
        if (a.ids) a.ids[t * d.k + threadIdx.x] = R.ids[threadIdx.x];
        if (a.w) a.w[t * d.k + threadIdx.x] = R.w[threadIdx.x];
    }
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= d.D) return;
    const float *eo = (const float *)(a.ws + a.L.eo) + (size_t)t * d.k * d.D + i;
    float acc = 0.0f;
    for (int r = 0; r < d.k; r++)
        if (R.ids[r] >= 0) acc += R.w[r] * eo[(size_t)r * d.D];
    if (d.ds > 0) {
        const float g = d.shared_gate_inp ? ((const float *)(a.ws + a.L.sgate))[t] : 1.0f;
        acc += g * ((const float *)(a.ws + a.L.seo))[(size_t)t * d.D + i];
    }
    a.out[(size_t)t * d.D + i] = a.h[(size_t)t * d.D + i] + acc;
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
         (uintptr_t)d->router_w) & 3u)
        return tlmh_seterr(TLM_HIP_EINVAL, "fp8_moe: tensors must be 4-byte aligned");
    Args a{};
    a.d = *d;
    a.L = layout(*d, T);
    a.h = h;
    a.out = out;
    a.ids = ids;
    a.w = w;
    a.ws = (uint8_t *)workspace;
    a.T = (int)T;
    a.by_expert = T * d->k >= d->E;
    a.slots = a.by_expert ? d->E : (int)(T * d->k);
    const unsigned ny = (unsigned)(a.slots + (d->ds > 0 ? 1 : 0));
    const int wide = a.L.nbe > a.L.nbs ? a.L.nbe : a.L.nbs;
    hipStream_t s = (hipStream_t)stream;
    hipLaunchKernelGGL(k_fm_router, dim3((unsigned)((d->E + ROUTER_EXPERTS - 1) / ROUTER_EXPERTS), (unsigned)T),
                       dim3(256), (size_t)d->D * 4, s, a);
    hipLaunchKernelGGL(k_fm_gateup, dim3((unsigned)wide * 8, ny), dim3(64 * NW), 0, s, a);
    hipLaunchKernelGGL(k_fm_down, dim3((unsigned)fp8_tiles(d->D), ny), dim3(64 * NW), 0, s, a);
    hipLaunchKernelGGL(k_fm_combine, dim3((unsigned)((d->D + 255) / 256), (unsigned)T), dim3(256), 0, s, a);
    return tlmh_check(hipGetLastError(), "fp8_moe launch");
}

}  // extern "C"
