/* hip_selftest.hip - start-up self-test of the HIP kernels
 * (src/lib/tlm_quant.c:950-1056: fixed pseudo-random rows with finite scale
 * fields, 9 rows x 1024 values, two repetitions, bit-exact against the scalar
 * rule).  The host scalar rule below exists only to check the kernels; no
 * entry point ever computes a result with it.
 *
 * Checked: the device activation quantisers (bytes), the plain-layout matvec
 * and the packed-layout matvec (bits of every row) for F32, Q8_0, Q4_K, Q5_K,
 * Q6_K and Q8_K, the exponential against this host's libm expf, the
 * matrix cores' float products against v_mul_f32, and the 8-bit floating-point
 * quantiser (codes and scales) and product (within the roundings of a float sum),
 * at one size, of the row groups; the paged cache in both types at every head width, and a prompt's and a decode step's ways
 * through their launches at one width or two each.
 * Returns the number of failing kernels; bit dt of *mask is set for every dtype
 * whose kernels failed, FAILED_EXP for the exponential, FAILED_PRODUCTS for the
 * products, FAILED_FP8 for 8-bit floating point, FAILED_KV for the paged cache. */
#include "tlm_hip_internal.h"
#include "tlm_hip_outer.h"

#include <math.h>
#include <stdlib.h>
#include <string.h>
#include <vector>

namespace {

float h_f16(uint16_t h) {
    uint32_t s = (uint32_t)(h & 0x8000u) << 16, e = (h >> 10) & 31u, m = h & 1023u, u;
    if (e == 31u) u = s | 0x7F800000u | (m << 13) | (m ? 0x00400000u : 0u);
    else if (e == 0u) {
        float v = (float)m * 0x1p-24f;
        memcpy(&u, &v, 4);
        u |= s;
    } else u = s | ((e + 112u) << 23) | (m << 13);
    float f;
    memcpy(&f, &u, 4);
    return f;
}
uint16_t rd16(const uint8_t *p) { return (uint16_t)(p[0] | (p[1] << 8)); }
float rdf(const uint8_t *p) { float f; memcpy(&f, p, 4); return f; }

int h_rne(float v, int lo, int hi) {
    if (v != v) return 0;
    if (v <= (float)lo) return lo;
    if (v >= (float)hi) return hi;
    volatile float t = v + 12582912.0f;
    return (int)(t - 12582912.0f);
}

/* activation rule, src/lib/tlm_quant.c:458-506 */
void h_act(int kind, const float *x, int64_t n, uint8_t *out) {
    const int qk = kind == DT_Q8_K ? 256 : 32, bb = kind == DT_Q8_K ? 292 : 36;
    for (int64_t b = 0; b * qk < n; b++) {
        int nv = (int)(n - b * qk < qk ? n - b * qk : qk);
        const float *v = x + b * qk;
        float amax = 0.0f, d;
        int nan = 0, inf = 0;
        int8_t q[256];
        memset(q, 0, sizeof q);
        for (int i = 0; i < nv; i++) {
            float a = fabsf(v[i]);
            if (a != a) nan = 1; else if (a == INFINITY) inf = 1; else if (a > amax) amax = a;
        }
        if (nan || inf) d = nan ? NAN : INFINITY;
        else if (!(amax > 0.0f)) d = 0.0f;
        else {
            d = amax / 127.0f;
            if (amax >= 0x1p-100f) {
                float id = 127.0f / amax;
                for (int i = 0; i < nv; i++) q[i] = (int8_t)h_rne(v[i] * id, -127, 127);
            } else {
                double id = 127.0 / (double)amax;
                for (int i = 0; i < nv; i++) q[i] = (int8_t)h_rne((float)((double)v[i] * id), -127, 127);
            }
        }
        uint8_t *o = out + b * bb;
        memcpy(o, &d, 4);
        memcpy(o + 4, q, (size_t)qk);
        if (kind == DT_Q8_K)
            for (int g = 0; g < 16; g++) {
                int s = 0;
                for (int i = 0; i < 16; i++) s += q[16 * g + i];
                int16_t s16 = (int16_t)s;
                memcpy(o + 260 + 2 * g, &s16, 2);
            }
    }
}

/* dot rule, src/lib/tlm_quant.c:721-902 */
float h_dot(int dt, const uint8_t *w, const uint8_t *a, int64_t n) {
    if (dt == DT_F32) {
        float r[32] = {0};
        for (int64_t i = 0; i < n; i++) r[i & 31] = fmaf(rdf(w + 4 * i), rdf(a + 4 * i), r[i & 31]);
        float s16[16], s8[8], s4[4];
        for (int l = 0; l < 16; l++) s16[l] = r[l] + r[l + 16];
        for (int l = 0; l < 8; l++) s8[l] = s16[l] + s16[l + 8];
        for (int l = 0; l < 4; l++) s4[l] = s8[l] + s8[l + 4];
        return (s4[0] + s4[2]) + (s4[1] + s4[3]);
    }
    const int bv = dt_block_values(dt), wb = dt_block_bytes(dt), ab = bv == 32 ? 36 : 292;
    float acc = 0.0f;
    for (int64_t b = 0; b < n / bv; b++) {
        const uint8_t *k = w + b * wb, *x = a + b * ab;
        const int8_t *xq = (const int8_t *)(x + 4);
        const float da = rdf(x);
        int32_t is = 0, ms = 0;
        if (dt == DT_Q8_0) {
            for (int i = 0; i < 32; i++) is += (int8_t)k[2 + i] * xq[i];
            acc = fmaf(h_f16(rd16(k)) * da, (float)is, acc);
        } else if (dt == DT_Q8_K) {
            for (int i = 0; i < 256; i++) is += (int8_t)k[4 + i] * xq[i];
            acc = fmaf(rdf(k) * da, (float)is, acc);
        } else if (dt == DT_Q6_K) {
            for (int g = 0; g < 16; g++) {
                int32_t gs = 0;
                for (int j = 0; j < 16; j++) {
                    int e = 16 * g + j, hh = e >> 7, q = (e >> 5) & 3, l = e & 31;
                    int nib = k[64 * hh + 32 * (q & 1) + l];
                    nib = (q & 2) ? nib >> 4 : nib & 15;
                    gs += (nib | (((k[128 + 32 * hh + l] >> (2 * q)) & 3) << 4)) * xq[e];
                }
                int16_t bs;
                memcpy(&bs, x + 260 + 2 * g, 2);
                is += (int8_t)k[192 + g] * (gs - 32 * bs);
            }
            acc = fmaf(h_f16(rd16(k + 208)) * da, (float)is, acc);
        } else {
            const bool q5 = dt == DT_Q5_K;
            const uint8_t *qs = k + (q5 ? 48 : 16), *s12 = k + 4;
            for (int sb = 0; sb < 8; sb++) {
                int c = sb >> 1, hb = sb & 1, sc, mn;
                if (sb < 4) { sc = s12[sb] & 63; mn = s12[4 + sb] & 63; }
                else { sc = (s12[sb + 4] & 15) | ((s12[sb - 4] >> 6) << 4); mn = (s12[sb + 4] >> 4) | ((s12[sb] >> 6) << 4); }
                int32_t s = 0;
                for (int l = 0; l < 32; l++) {
                    int code = hb ? qs[32 * c + l] >> 4 : qs[32 * c + l] & 15;
                    if (q5) code |= ((k[16 + l] >> (2 * c + hb)) & 1) << 4;
                    s += code * xq[32 * sb + l];
                }
                int16_t b0, b1;
                memcpy(&b0, x + 260 + 4 * sb, 2);
                memcpy(&b1, x + 262 + 4 * sb, 2);
                is += sc * s;
                ms += mn * (b0 + b1);
            }
            float sa = h_f16(rd16(k)) * da, sm = h_f16(rd16(k + 2)) * da;
            acc = fmaf(sa, (float)is, acc);
            acc = fmaf(-sm, (float)ms, acc);
        }
    }
    return acc;
}

uint32_t st_rng(uint32_t *s) { *s = *s * 1664525u + 1013904223u; return *s >> 8; }

/* half-precision scale in [-0.01, 0.01] as in the reference's self-test */
void put_scale(uint8_t *p, uint32_t *s) {
    float v = ((float)(st_rng(s) & 0xFFFF) / 65536.0f - 0.5f) * 0.02f;
    /* RNE f32 -> f16 for a normal-range value */
    uint32_t x;
    memcpy(&x, &v, 4);
    uint32_t sign = (x >> 16) & 0x8000u, ax = x & 0x7FFFFFFFu;
    uint16_t h;
    if (ax < 0x38800000u) {   /* |v| < 2^-14: f16 subnormal or zero */
        uint32_t e = ax >> 23, mant = (ax & 0x7FFFFFu) | 0x800000u;
        if (ax <= 0x33000000u) h = (uint16_t)sign;
        else {
            uint32_t sh = 126u - e, q = mant >> sh, rest = mant & ((1u << sh) - 1u), half = 1u << (sh - 1u);
            q += (rest > half) || (rest == half && (q & 1u));
            h = (uint16_t)(sign | q);
        }
    } else {
        uint32_t r = ax - 0x38000000u, q = r >> 13, rest = r & 0x1FFFu;
        q += (rest > 0x1000u) || (rest == 0x1000u && (q & 1u));
        h = (uint16_t)(sign | q);
    }
    p[0] = (uint8_t)h;
    p[1] = (uint8_t)(h >> 8);
}

void make_row(int dt, uint8_t *w, int64_t n, uint32_t *s) {
    const int bv = dt_block_values(dt), wb = dt_block_bytes(dt);
    const size_t bytes = (size_t)(n / bv) * wb;
    for (size_t i = 0; i < bytes; i++) w[i] = (uint8_t)st_rng(s);
    for (int64_t b = 0; b < n / bv; b++) {
        uint8_t *k = w + b * wb;
        if (dt == DT_F32) { float v = (float)(st_rng(s) & 0xFFFF) / 32768.0f - 1.0f; memcpy(k, &v, 4); }
        else if (dt == DT_Q8_0) put_scale(k, s);
        else if (dt == DT_Q4_K || dt == DT_Q5_K) { put_scale(k, s); put_scale(k + 2, s); }
        else if (dt == DT_Q6_K) put_scale(k + 208, s);
        else if (dt == DT_Q8_K) { float d = (float)(st_rng(s) & 0xFFFF) * 1e-7f; memcpy(k, &d, 4); }
    }
}

bool same(float a, float b) {
    if (a != a || b != b) return (a != a) && (b != b);
    uint32_t x, y;
    memcpy(&x, &a, 4);
    memcpy(&y, &b, 4);
    return x == y;
}

/* bad[64 g + l]: whether one of lane l's products of group g (ROWS values of a,
 * 64 of b) is not v_mul_f32's: the same value or both a NaN (a zero's sign is
 * not compared, tlm_hip_outer.h) */
template <int ROWS>
__global__ __launch_bounds__(64) void k_outer_check(const float *__restrict__ a, const float *__restrict__ b,
                                                    uint32_t *__restrict__ bad) {
    using O = Outer<ROWS>;
    const int lane = threadIdx.x;
    a += ROWS * blockIdx.x;
    b += 64 * blockIdx.x;
    const typename O::T p = O::mul(a[lane % ROWS], b[lane]);
    uint32_t diff = 0;
#pragma unroll
    for (int v = 0; v < ROWS; v++) {
        const float want = a[O::row(v, lane)] * b[O::col(v, lane)], got = p[v];
        if (want != got && !(want != want && got != got)) diff = 1;
    }
    bad[64 * blockIdx.x + lane] = diff;
}

/* every shape over pairs of the values where a product rounds, overflows or
 * vanishes, and over random bit patterns; dev: 64 KB */
bool outer_ok(uint8_t *dev, uint32_t *s) {
    const int G = 64;
    static const uint32_t edge[16] = {0x00000000u, 0x00000001u, 0x00000003u, 0x00400001u, 0x007FFFFFu, 0x00800000u,
                                      0x00800001u, 0x1F800000u, 0x20000001u, 0x3F000000u, 0x3F7FFFFFu, 0x3F800001u,
                                      0x40400000u, 0x7F7FFFFFu, 0x7F800000u, 0x7FC00000u};
    std::vector<uint32_t> a(32 * G), b(64 * G), bad(64 * G);
    for (int i = 0; i < 32 * G; i++)   /* the first half: every edge with both signs */
        a[i] = i < 16 * G ? edge[i & 15] | (uint32_t)(i >> 4 & 1) << 31 : st_rng(s) << 16 ^ st_rng(s);
    for (int i = 0; i < 64 * G; i++)
        b[i] = i < 32 * G ? edge[(i + i / 64) & 15] | (uint32_t)(i >> 5 & 1) << 31 : st_rng(s) << 16 ^ st_rng(s);
    float *da = (float *)dev, *db = (float *)(dev + 16384);
    uint32_t *dbad = (uint32_t *)(dev + 32768);
    if (hipMemcpy(da, a.data(), a.size() * 4, hipMemcpyHostToDevice) != hipSuccess ||
        hipMemcpy(db, b.data(), b.size() * 4, hipMemcpyHostToDevice) != hipSuccess)
        return false;
    bool ok = true;
    for (int rows : {32, 16, 4}) {
        if (rows == 32) hipLaunchKernelGGL(k_outer_check<32>, dim3(G), dim3(64), 0, nullptr, da, db, dbad);
        else if (rows == 16) hipLaunchKernelGGL(k_outer_check<16>, dim3(G), dim3(64), 0, nullptr, da, db, dbad);
        else hipLaunchKernelGGL(k_outer_check<4>, dim3(G), dim3(64), 0, nullptr, da, db, dbad);
        ok = ok && hipGetLastError() == hipSuccess &&
             hipMemcpy(bad.data(), dbad, bad.size() * 4, hipMemcpyDeviceToHost) == hipSuccess;
        for (size_t i = 0; ok && i < bad.size(); i++) ok = bad[i] == 0;
    }
    return ok;
}

/* an E4M3 code's value, and the code nearest to v (|v| <= 448, ties to even) by search */
double e4m3(int c) {
    const int e = (c >> 3) & 15, m = c & 7;
    const double v = e ? ldexp(8.0 + m, e - 10) : ldexp((double)m, -9);
    return c & 128 ? -v : v;
}
int to_e4m3(double v) {
    const double a = fabs(v);
    int best = 0;
    for (int c = 1; c < 127; c++) {
        const double d = fabs(e4m3(c) - a), b = fabs(e4m3(best) - a);
        if (d < b || (d == b && !(c & 1))) best = c;
    }
    return best | (signbit(v) ? 128 : 0);
}

/* the quantiser's codes and scales of T rows of n values, by search */
void h_fp8(const float *x, int T, int n, uint8_t *codes, float *scale) {
    const int nb = (n + 127) / 128, np = nb * 128;
    memset(codes, 0, (size_t)T * np);
    for (int t = 0; t < T; t++)
        for (int b = 0; b < nb; b++) {
            const int m = n - 128 * b < 128 ? n - 128 * b : 128;
            double amax = 0.0;
            for (int i = 0; i < m; i++) amax = fmax(amax, fabs((double)x[t * n + 128 * b + i]));
            int e = -126;
            while (amax > ldexp(448.0, e)) e++;
            scale[t * nb + b] = amax > 0.0 ? ldexpf(1.0f, e) : 0.0f;
            for (int i = 0; i < m; i++) codes[t * np + 128 * b + i] = (uint8_t)to_e4m3(ldexp((double)x[t * n + 128 * b + i], -e));
        }
}

/* 3 tokens and 20 rows of 300 values (part blocks and part tiles); dev: 32 KB */
bool fp8_ok(uint8_t *dev, uint32_t *s) {
    constexpr int T = 3, R = 20, N = 300, NB = 3, NP = NB * 128;
    std::vector<float> x(T * N), sx(T * NB), gs(T * NB), y(T * R);
    std::vector<uint8_t> w(R * N), cx(T * NP, 0), gc(T * NP);
    const float sw[NB] = {0.5f, 0.0371f, 3.0f};
    for (auto &v : x) v = ((float)(st_rng(s) & 0xFFFF) / 32768.0f - 1.0f) * ldexpf(1.0f, (int)(st_rng(s) & 7) - 4);
    for (auto &c : w) {
        c = (uint8_t)st_rng(s);
        if ((c & 127) == 127) c = 0;
    }
    h_fp8(x.data(), T, N, cx.data(), sx.data());
    float *dx = (float *)dev, *ds = (float *)(dev + 4096), *dsw = (float *)(dev + 4352), *dy = (float *)(dev + 4608);
    uint8_t *dc = dev + 8192, *dw = dev + 10240, *dp = dev + 16640;
    if (hipMemcpy(dx, x.data(), x.size() * 4, hipMemcpyHostToDevice) != hipSuccess ||
        hipMemcpy(dw, w.data(), w.size(), hipMemcpyHostToDevice) != hipSuccess ||
        hipMemcpy(dsw, sw, sizeof sw, hipMemcpyHostToDevice) != hipSuccess ||
        tlm_hip_fp8_quantize(DT_F32, dx, N, N, T, dc, ds, nullptr) != TLM_HIP_OK ||
        tlm_hip_fp8_pack(dw, N, dsw, NB, R, N, dp, nullptr) != TLM_HIP_OK ||
        tlm_hip_fp8_matmul(dp, R, N, dc, ds, T, DT_F32, dy, R, nullptr) != TLM_HIP_OK ||
        hipMemcpy(gc.data(), dc, gc.size(), hipMemcpyDeviceToHost) != hipSuccess ||
        hipMemcpy(gs.data(), ds, gs.size() * 4, hipMemcpyDeviceToHost) != hipSuccess ||
        hipMemcpy(y.data(), dy, y.size() * 4, hipMemcpyDeviceToHost) != hipSuccess)
        return false;
    if (memcmp(gc.data(), cx.data(), cx.size()) != 0 || memcmp(gs.data(), sx.data(), sx.size() * 4) != 0) return false;
    for (int t = 0; t < T; t++)
        for (int r = 0; r < R; r++) {
            double sum = 0.0, size = 0.0;
            for (int i = 0; i < N; i++) {
                const double p = e4m3(cx[t * NP + i]) * e4m3(w[r * N + i]) * (double)sx[t * NB + i / 128] * (double)sw[i / 128];
                sum += p;
                size += fabs(p);
            }
            if (!(fabs((double)y[t * R + r] - sum) <= (127 + NB + 2) * 0x1p-24 * size)) return false;
        }
    /* the norm in front of the quantiser: 2 x, x itself added, times some positive weights */
    std::vector<float> h(T * N), v(T * N), nw(N), x2(x), gh(T * N);
    for (int i = 0; i < N; i++) nw[i] = 0.5f + (float)(i % 7) * 0.125f;
    for (auto &e : x2) e *= 2.0f;
    for (int t = 0; t < T; t++) {
        double sum = 0.0;
        for (int i = 0; i < N; i++) {
            h[t * N + i] = x2[t * N + i] + x[t * N + i];
            sum += (double)h[t * N + i] * (double)h[t * N + i];
        }
        const float r = (float)(1.0 / sqrt(sum / N + 0x1p-20));
        for (int i = 0; i < N; i++) v[t * N + i] = (h[t * N + i] * r) * nw[i];
    }
    h_fp8(v.data(), T, N, cx.data(), sx.data());
    float *dh = (float *)(dev + 10240), *dn = (float *)dp;
    if (hipMemcpy(dh, x2.data(), x2.size() * 4, hipMemcpyHostToDevice) != hipSuccess ||
        hipMemcpy(dn, nw.data(), nw.size() * 4, hipMemcpyHostToDevice) != hipSuccess ||
        tlm_hip_fp8_add_rmsnorm(DT_F32, dh, N, DT_F32, dx, N, dn, 0x1p-20f, N, T, dh, N, dc, ds, nullptr) != TLM_HIP_OK ||
        hipMemcpy(gc.data(), dc, gc.size(), hipMemcpyDeviceToHost) != hipSuccess ||
        hipMemcpy(gs.data(), ds, gs.size() * 4, hipMemcpyDeviceToHost) != hipSuccess ||
        hipMemcpy(gh.data(), dh, gh.size() * 4, hipMemcpyDeviceToHost) != hipSuccess)
        return false;
    return memcmp(gh.data(), h.data(), h.size() * 4) == 0 && memcmp(gc.data(), cx.data(), cx.size()) == 0 &&
           memcmp(gs.data(), sx.data(), sx.size() * 4) == 0;
}

/* a value rounded to F16 or BF16 (nothing here is past their range), and one read back */
double to_half(int dt, double v) {
    if (v == 0.0) return 0.0;
    int e;
    frexp(v, &e);
    const int bits = dt == DT_F16 ? 11 : 8, least = dt == DT_F16 ? -24 : -133;
    const int unit = e - bits < least ? least : e - bits;
    return ldexp(nearbyint(ldexp(v, -unit)), unit);
}
double from_half(int dt, uint16_t h) {
    if (dt == DT_F16) return h_f16(h);
    const uint32_t u = (uint32_t)h << 16;
    float f;
    memcpy(&f, &u, 4);
    return f;
}

/* The paged cache: two sequences (19 rows, and 3 behind `past` positions that a first call appended) with norms and rotation;
 * their attention as prompts, and of the last rows alone, each with tables of their length and with far-reaching ones. */
struct KvShape {
    int H, KV, HD, past, each;      /* every each-th head is compared */
};
bool kv_shape_ok(uint32_t *s, const KvShape &shape) {
    constexpr int PAGE = 16, WIDE = 128, B = 2;
    const int H = shape.H, KV = shape.KV, HD = shape.HD, FIRST = shape.past, G = H / KV, ROW = (H + 2 * KV) * HD;
    const int n[B] = {19, 3}, len[B] = {19, FIRST + 3}, T = n[0] + n[1], need = (len[1] + PAGE - 1) / PAGE, PAGES = 2 + need + 1;
    const float scale = 1.0f / sqrtf((float)HD);
    std::vector<float> x((size_t)(FIRST + T) * ROW), norm(2 * HD), gy(T * H * HD), gd(B * H * HD);
    std::vector<double> freq(HD / 2), turn((size_t)len[1] * HD);
    std::vector<int32_t> ints(8 + B * WIDE, -1);
    std::vector<uint16_t> gq(T * H * HD);
    for (auto &e : x) e = (float)(st_rng(s) & 0xFFFF) / 16384.0f - 2.0f;
    for (auto &e : norm) e = 0.5f + (float)(st_rng(s) & 0xFF) / 256.0f;
    for (int j = 0; j < HD / 2; j++) freq[j] = pow(1e4, -2.0 * j / HD);
    for (int p = 0; p < len[1]; p++)
        for (int j = 0; j < HD / 2; j++) {
            turn[p * HD + j] = cos(p * freq[j]);
            turn[p * HD + HD / 2 + j] = sin(p * freq[j]);
        }
    const int32_t head[8] = {0, n[0], T, len[0], len[1], 0, FIRST, FIRST};   /* cu, lens; the first call's cu and length */
    for (int i = 0; i < 8; i++) ints[i] = head[i];
    for (int i = 0; i < 2 + need; i++) ints[8 + (i < 2 ? i : WIDE + i - 2)] = (7 * i + 3) % PAGES;       /* 13 or 5 pages */
    const size_t ALIGN = 255, cache = ((size_t)PAGES * KV * PAGE * HD * 2 + ALIGN) & ~ALIGN;
    const size_t rows = (size_t)(FIRST > T ? FIRST : T) * H * HD;
    const int32_t *any = ints.data();        /* the sizes decide, not what is there */
    const tlm_hip_kv_cache sizes = {DT_F16, KV, HD, PAGE, PAGES, (void *)256, (void *)256};
    const tlm_hip_kv_batch wide_p = {B, T, any, any, any, WIDE, WIDE}, wide_d = {B, B, nullptr, any, any, WIDE, WIDE};
    size_t ws = 256;
    for (const size_t w : {tlm_hip_kv_prompt_workspace_bytes(&sizes, &wide_p, H), tlm_hip_kv_decode_workspace_bytes(&sizes, &wide_d, H)})
        ws = w > ws ? w : ws;
    const size_t o_k = (x.size() * 4 + ALIGN) & ~ALIGN, o_v = o_k + cache, o_q = o_v + cache, o_y = o_q + ((rows * 2 + ALIGN) & ~ALIGN),
                 o_i = o_y + ((gy.size() * 4 + ALIGN) & ~ALIGN), o_w = o_i + 8192;
    uint8_t *dev = nullptr;
    if (hipMalloc((void **)&dev, o_w + ws) != hipSuccess) return false;
    const int32_t *di = (const int32_t *)(dev + o_i);
    double *df = (double *)(dev + o_i + 4096);
    float *dn = (float *)(dev + o_i + 4096 + 2048), *dx = (float *)dev;
    void *q = dev + o_q, *y = dev + o_y;
    bool ok = hipMemcpy(dx, x.data(), x.size() * 4, hipMemcpyHostToDevice) == hipSuccess &&
              hipMemcpy(dev + o_i, ints.data(), ints.size() * 4, hipMemcpyHostToDevice) == hipSuccess &&
              hipMemcpy(df, freq.data(), freq.size() * 8, hipMemcpyHostToDevice) == hipSuccess &&
              hipMemcpy(dn, norm.data(), norm.size() * 4, hipMemcpyHostToDevice) == hipSuccess;
    /* a head's row with its norm, turned to position pos */
    auto turned = [&](const float *src, const float *w, int pos, double *o) {
        double ss = 0.0;
        for (int i = 0; i < HD; i++) ss += (double)src[i] * src[i];
        const double r = 1.0 / sqrt(ss / HD + 1e-6), *c = &turn[(size_t)pos * HD], *sn = c + HD / 2;
        for (int j = 0; j < HD / 2; j++) {
            const double a = src[j] * r * w[j], d = src[HD / 2 + j] * r * w[HD / 2 + j];
            o[j] = a * c[j] - d * sn[j];
            o[HD / 2 + j] = d * c[j] + a * sn[j];
        }
    };
    for (int dt : {DT_F16, DT_BF16}) {
        const double half = dt == DT_F16 ? 0x1p-11 : 0x1p-8;
        const tlm_hip_kv_cache c = {dt, KV, HD, PAGE, PAGES, dev + o_k, dev + o_v};
        const tlm_hip_kv_batch first = {1, FIRST, di + 5, di + 7, di + 8 + WIDE, WIDE, need}, b = {B, T, di, di + 3, di + 8, WIDE, need};
        ok = ok && tlm_hip_kv_append(&c, &first, DT_F32, dx, ROW, H, dn, dn + HD, 1e-6f, df, 1.0f, q, nullptr) == TLM_HIP_OK &&
             tlm_hip_kv_append(&c, &b, DT_F32, dx + (size_t)FIRST * ROW, ROW, H, dn, dn + HD, 1e-6f, df, 1.0f, q, nullptr) == TLM_HIP_OK &&
             hipMemcpy(gq.data(), q, gq.size() * 2, hipMemcpyDeviceToHost) == hipSuccess;
        /* Every row and each last row's results, of the heads compared.  A query is within a half step of its definition, f32
         * roundings beside it.  A key next to the border of two steps may be the other one here: a step (two half ones) of each
         * product of a score, so a weight is off by twice the largest score's steps; and each weight is rounded once. */
        std::vector<double> k((size_t)len[1] * HD), v(k.size()), e(len[1]), qv(HD);
        std::vector<float> got[4];       /* prompts, last rows; tables of the length and wide ones */
        for (int i = 0; ok && i < 4; i++) {
            const int pages = i & 1 ? WIDE : need;
            const tlm_hip_kv_batch all = {B, T, di, di + 3, di + 8, WIDE, pages}, last = {B, B, nullptr, di + 3, di + 8, WIDE, pages};
            got[i].resize((size_t)(i < 2 ? T : B) * H * HD);
            ok = (i < 2 ? tlm_hip_kv_prompt(&c, &all, q, H * HD, H, scale, DT_F32, y, dev + o_w, nullptr)
                        : tlm_hip_kv_decode(&c, &last, (const uint16_t *)q + (n[0] - 1) * H * HD, n[1] * H * HD, H, scale, DT_F32, y,
                                            dev + o_w, nullptr)) == TLM_HIP_OK &&
                 hipMemcpy(got[i].data(), y, got[i].size() * 4, hipMemcpyDeviceToHost) == hipSuccess;
        }
        for (int h = 0; ok && h < H; h += shape.each)
            for (int i = 0, t0 = 0; i < B; t0 += n[i++]) {
                for (int p = 0; p < len[i]; p++) {
                    const float *row = x.data() + (size_t)(i == 0 ? FIRST + p : p < FIRST ? p : FIRST + n[0] + p - FIRST) * ROW;
                    turned(row + (H + h / G) * HD, norm.data() + HD, p, &k[p * HD]);
                    for (int d = 0; d < HD; d++) {
                        k[p * HD + d] = to_half(dt, k[p * HD + d]);
                        v[p * HD + d] = to_half(dt, row[(H + KV + h / G) * HD + d]);
                    }
                }
                for (int r = 0; r < n[i]; r++) {
                    const int t = t0 + r, p = len[i] - n[i] + r;
                    double top = -1e300, sum = 0.0, size = 0.0;
                    turned(x.data() + (size_t)(FIRST + t) * ROW + h * HD, norm.data(), p, qv.data());
                    for (int d = 0; d < HD; d++) {
                        const double g = from_half(dt, gq[(t * H + h) * HD + d]);
                        ok = ok && fabs(g - qv[d]) <= half * fabs(qv[d]) + 1e-5;
                        qv[d] = g;
                    }
                    for (int j = 0; j <= p; j++) {
                        double mag = e[j] = 0.0;
                        for (int d = 0; d < HD; d++) {
                            const double u = qv[d] * k[j * HD + d] * scale;
                            e[j] += u;
                            mag += fabs(u);
                        }
                        top = fmax(top, e[j]);
                        size = fmax(size, mag);
                    }
                    for (int j = 0; j <= p; j++) sum += e[j] = exp(e[j] - top);
                    for (int d = 0; d < HD; d++) {
                        double o = 0.0, mag = 0.0;
                        for (int j = 0; j <= p; j++) {
                            const double u = e[j] / sum * v[j * HD + d];
                            o += u;
                            mag += fabs(u);
                        }
                        const double tol = mag * (half * (1.0 + 4.0 * size) + 1e-5) + 1e-6;
                        for (int a = 0; a < (r == n[i] - 1 ? 4 : 2); a++)
                            ok = ok && fabs(got[a][((size_t)(a < 2 ? t : i) * H + h) * HD + d] - o) <= tol;
                    }
                }
            }
    }
    (void)hipDeviceSynchronize();
    (void)hipFree(dev);
    return ok;
}
/* Every head width, in shares and parts; then enough key heads that a prompt's group takes 64 rows (narrow and wide heads) and
 * 128, and more than 16 queries a key head. */
bool kv_ok(uint32_t *s) {
    static const KvShape shapes[] = {
        {4, 2, 32, 150, 1},  {4, 2, 64, 150, 1},   {6, 3, 96, 150, 1},    {8, 2, 128, 150, 1},   {2, 1, 160, 150, 1},  {2, 2, 192, 150, 1},
        {3, 1, 224, 150, 1}, {4, 2, 256, 150, 1},  {34, 1, 64, 150, 11},  {80, 80, 64, 20, 27},  {40, 40, 128, 20, 13},
        {260, 260, 32, 20, 87}, {130, 130, 160, 20, 43}};
    for (const KvShape &shape : shapes)
        if (!kv_shape_ok(s, shape)) return false;
    return true;
}

}  // namespace

int tlmh_selftest(int *failed_mask) {
    const int64_t N = 1024, NF = 1003;
    const int ROWS = 9;
    static const int dts[] = {DT_F32, DT_Q8_0, DT_Q4_K, DT_Q5_K, DT_Q6_K, DT_Q8_K};
    uint32_t s = 0x2545F491u;
    std::vector<float> xf(N);
    for (int64_t i = 0; i < N; i++) xf[i] = (float)(st_rng(&s) & 0xFFFF) / 32768.0f - 1.0f;
    xf[5] = 7.5f;
    xf[700] = -7.5f;
    std::vector<uint8_t> xk(act_bytes(DT_Q8_K, N)), xa(act_bytes(DT_Q8_0, N));
    h_act(DT_Q8_K, xf.data(), N, xk.data());
    h_act(DT_Q8_0, xf.data(), N, xa.data());

    uint8_t *dev = nullptr;
    const size_t wmax = (size_t)ROWS * N * 4, pmax = (size_t)16 * N * 4;
    size_t o_x = 0, o_xk = 8192, o_xa = 16384, o_w = 32768, o_p = o_w + wmax + 256, o_y = o_p + pmax + 256;
    size_t total = o_y + 4096;
    if (hipMalloc((void **)&dev, total) != hipSuccess) return tlmh_seterr(TLM_HIP_ENOMEM, "self-test: device memory");
    int fails = 0, mask = 0;
    std::vector<uint8_t> got(act_bytes(DT_Q8_K, N));
    std::vector<uint8_t> w(wmax);
    bool io_ok = hipMemcpy(dev + o_x, xf.data(), N * 4, hipMemcpyHostToDevice) == hipSuccess;
    /* activation quantisers */
    for (int kind : {DT_Q8_K, DT_Q8_0}) {
        size_t off = kind == DT_Q8_K ? o_xk : o_xa, nbytes = act_bytes(kind, N);
        bool ok = io_ok && launch_quantize_act(kind, (const float *)(dev + o_x), N, dev + off, nullptr) == TLM_HIP_OK &&
                  hipMemcpy(got.data(), dev + off, nbytes, hipMemcpyDeviceToHost) == hipSuccess &&
                  memcmp(got.data(), kind == DT_Q8_K ? xk.data() : xa.data(), nbytes) == 0;
        if (!ok) {
            fails++;
            mask |= 1 << kind;
        }
    }
    /* the activations the dots use are the host rule's bytes */
    io_ok = io_ok && hipMemcpy(dev + o_xk, xk.data(), xk.size(), hipMemcpyHostToDevice) == hipSuccess &&
            hipMemcpy(dev + o_xa, xa.data(), xa.size(), hipMemcpyHostToDevice) == hipSuccess;
    for (int dt : dts) {
        const int64_t n = dt == DT_F32 ? NF : N;
        const size_t rb = dt == DT_F32 ? (size_t)n * 4 : (size_t)(n / dt_block_values(dt)) * dt_block_bytes(dt);
        const int kind = dt_act_kind(dt);
        const uint8_t *hact = kind == DT_Q8_K ? xk.data() : kind == DT_Q8_0 ? xa.data() : (const uint8_t *)xf.data();
        const uint8_t *dact = dev + (kind == DT_Q8_K ? o_xk : kind == DT_Q8_0 ? o_xa : o_x);
        bool ok = io_ok;
        for (int rep = 0; rep < 2 && ok; rep++) {
            float ref[ROWS], y[ROWS];
            for (int r = 0; r < ROWS; r++) {
                make_row(dt, w.data() + rb * r, n, &s);
                ref[r] = h_dot(dt, w.data() + rb * r, hact, n);
            }
            ok = hipMemcpy(dev + o_w, w.data(), rb * ROWS, hipMemcpyHostToDevice) == hipSuccess;
            /* plain layout, rows [0, 9) then [2, 7) */
            ok = ok && launch_matvec_plain(dt, dev + o_w, rb, dact, (float *)(dev + o_y), n, 0, ROWS, nullptr) == 0 &&
                 hipMemcpy(y, dev + o_y, sizeof y, hipMemcpyDeviceToHost) == hipSuccess;
            for (int r = 0; ok && r < ROWS; r++) ok = same(ref[r], y[r]);
            /* packed layout */
            if (ok && dt != DT_F32) {
                ok = launch_pack(dt, dev + o_w, rb, ROWS, n, dev + o_p, nullptr) == 0 &&
                     launch_matvec_packed(dt, dev + o_p, ROWS, n, dact, (float *)(dev + o_y), nullptr) == 0 &&
                     hipMemcpy(y, dev + o_y, sizeof y, hipMemcpyDeviceToHost) == hipSuccess;
                for (int r = 0; ok && r < ROWS; r++) ok = same(ref[r], y[r]);
            }
        }
        if (!ok) {
            fails++;
            mask |= 1 << dt;
        }
    }
    /* the exponential against this host's libm expf (what the reference
     * calls): float bit patterns strided over the whole range, the overflow and
     * underflow edges and two inputs whose result needs the fused shift */
    {
        const int NE = 4096;
        std::vector<float> ex(NE), ey(NE), eg(NE);
        for (int i = 0; i < NE - 6; i++) {
            const uint32_t u = (uint32_t)i * 1048573u;
            memcpy(&ex[i], &u, 4);
        }
        const float edge[6] = {0x1.62e42ep6f, 0x1.62e430p6f, -0x1.9fe368p6f, -0x1.9fe366p6f, 0x1.04845ep+5f,
                               -0x1.f8cbb2p+5f};
        for (int i = 0; i < 6; i++) ex[NE - 6 + i] = edge[i];
        for (int i = 0; i < NE; i++) ey[i] = expf(ex[i]);
        float *dx = (float *)(dev + o_w), *dy = (float *)(dev + o_p);
        bool ok = hipMemcpy(dx, ex.data(), NE * 4, hipMemcpyHostToDevice) == hipSuccess &&
                  launch_expf(dx, dy, NE, nullptr) == TLM_HIP_OK &&
                  hipMemcpy(eg.data(), dy, NE * 4, hipMemcpyDeviceToHost) == hipSuccess;
        for (int i = 0; ok && i < NE; i++) ok = same(ey[i], eg[i]) || (ey[i] != ey[i] && eg[i] != eg[i]);
        if (!ok) {
            fails++;
            mask |= 1 << FAILED_EXP;
        }
    }
    if (!outer_ok(dev + o_p, &s)) {
        fails++;
        mask |= 1 << FAILED_PRODUCTS;
    }
    if (!fp8_ok(dev + o_p, &s)) {
        fails++;
        mask |= 1 << FAILED_FP8;
    }
    if (!kv_ok(&s)) {
        fails++;
        mask |= 1 << FAILED_KV;
    }
    (void)hipDeviceSynchronize();
    (void)hipFree(dev);
    *failed_mask = mask;
    return fails;
}
