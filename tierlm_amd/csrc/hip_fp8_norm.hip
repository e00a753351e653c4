/* hip_fp8_norm.hip - what a sublayer hands on to the next product: the residual's addition, the RMS norm
 * and the E4M3 codes of its result, in one pass. */
#include "tlm_hip_fp8.h"

namespace {

struct NormArgs {
    const void *x, *h;      /* x: null, nothing is added */
    void *out;              /* null: the sum is not stored */
    int64_t xstride, hstride, ostride;
    const float *w;
    uint8_t *codes;
    float *scale;
    double eps;
    int n, nb;
};

template <class T> __device__ __forceinline__ T to_type(float v) { return (T)v; }

/* 8 values rounded to T (to nearest, ties to even), and as they were rounded in v; `left` of them stored */
template <class T> __device__ __forceinline__ void st8(float (&v)[8], T *p, int left) {
    typedef T T8 __attribute__((ext_vector_type(8), aligned(sizeof(T))));
    T8 q;
#pragma unroll
    for (int j = 0; j < 8; j++) {
        q[j] = to_type<T>(v[j]);
        v[j] = (float)q[j];
    }
    if (!p) return;
    if (left >= 8) {
        *(T8 *)p = q;
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++)
            if (j < left) p[j] = q[j];
    }
}

/* A group of NT threads per row, which it holds in registers: 8 consecutive values a thread in each of V rounds (so 16
 * lanes hold a block of 128).
 *   s = h + x rounded to H's type;  r = 1 / sqrt(mean(s^2) + eps);  y = (s r) w;  codes of y
 * The squares are summed in double: with 16384 of them a float sum is off by parts in 10^6, which moves values across the
 * border of two codes; in double the order of the sum does not show in r.  MORE: rows longer than V rounds hold; their
 * rest is read a second time.  8192 x 4096, f32 with bf16 added: 68 us, 5.4 TB/s (a copy 5.14): HBM. */
template <class X, class H, int NT, int V, bool MORE>
__global__ __launch_bounds__(NT) void k_fp8_norm(NormArgs a) {
    constexpr int STEP = NT * 8;
    __shared__ double s_sum[NT / 64];
    const int tid = threadIdx.x;
    const int64_t row = blockIdx.x;
    const H *h = (const H *)a.h + row * a.hstride;
    const X *x = a.x ? (const X *)a.x + row * a.xstride : nullptr;
    H *o = a.out ? (H *)a.out + row * a.ostride : nullptr;
    float v[V][8], u[V][8];
#pragma unroll
    for (int i = 0; i < V; i++) {
        const int k = tid * 8 + i * STEP;
        ld8<H>(v[i], h + k, a.n - k);
        if (x) ld8<X>(u[i], x + k, a.n - k);
    }
    double sum = 0.0;
    auto add = [&](float (&v)[8], const float (&u)[8], int k) {
        if (x) {
#pragma unroll
            for (int j = 0; j < 8; j++) v[j] += u[j];
        }
        st8<H>(v, o ? o + k : nullptr, a.n - k);
#pragma unroll
        for (int j = 0; j < 8; j++) sum = __builtin_fma((double)v[j], (double)v[j], sum);
    };
#pragma unroll
    for (int i = 0; i < V; i++) add(v[i], u[i], tid * 8 + i * STEP);
    if (MORE)
        for (int k = tid * 8 + V * STEP; k < a.n; k += STEP) {
            float p[8], q[8];
            ld8<H>(p, h + k, a.n - k);
            if (x) ld8<X>(q, x + k, a.n - k);
            add(p, q, k);
        }
    sum = wave_sum_f64(sum);
    if (NT > 64) {
        if ((tid & 63) == 0) s_sum[tid >> 6] = sum;
        __syncthreads();
        sum = s_sum[0];
#pragma unroll
        for (int i = 1; i < NT / 64; i++) sum += s_sum[i];
    }
    const float r = (float)(1.0 / sqrt(sum / (double)a.n + a.eps));
    auto finish = [&](const float (&v)[8], int k) {
        float w[8], y[8];
        ld8<float>(w, a.w + k, a.n - k);
#pragma unroll
        for (int j = 0; j < 8; j++) y[j] = j < a.n - k ? (v[j] * r) * w[j] : 0.0f;
        const Fp8Codes c = fp8_encode(y);
        if (k < a.nb * FP8_BLOCK) {
            const int64_t b = row * a.nb;
            *(u32x2 *)(a.codes + b * FP8_BLOCK + k) = c.codes;
            if ((tid & 15) == 0) a.scale[b + k / FP8_BLOCK] = c.scale;
        }
    };
#pragma unroll
    for (int i = 0; i < V; i++) finish(v[i], tid * 8 + i * STEP);
    if (MORE)
        for (int k0 = V * STEP; k0 < a.nb * FP8_BLOCK; k0 += STEP) {   /* whole blocks of 16 lanes leave together */
            const int k = k0 + tid * 8;
            float p[8], q[8];
            /* in place the sum is there already, and adding x again would be wrong */
            const H *src = o ? o : h;
            ld8<H>(p, src + k, a.n - k);
            if (x && !o) {
                ld8<X>(q, x + k, a.n - k);
#pragma unroll
                for (int j = 0; j < 8; j++) p[j] += q[j];
                st8<H>(p, (H *)nullptr, 0);
            }
            finish(p, k);
        }
}

template <class X, class H, int NT, int V, bool MORE> void launch_nt(const NormArgs &a, int64_t T, hipStream_t s) {
    hipLaunchKernelGGL((k_fp8_norm<X, H, NT, V, MORE>), dim3((unsigned)T), dim3(NT), 0, s, a);
}
/* As many threads as hold the row in one round, or two: the row's sum is a wait for all of them, and more rounds are more
 * loads behind it.  us, f32 rows with bf16 added, threads x rounds: 8192 x 512 64 x 1 13.1, 128 14.1, 256 17.3; 8192 x 2048
 * 256 x 1 37.4, 128 x 2 40.8; 8192 x 4096 512 x 1 68.4, 256 x 2 72.6, 128 x 4 80.2; 6710 x 5000 512 x 2 74.7, 1024 x 1 78.4,
 * 256 x 4 86.3; 4096 x 8192 1024 x 1 69.3, 512 x 2 72.1, 256 x 4 78.4; 2048 x 16384 1024 x 2 77.8, 512 x 4 88.2.  One row
 * of 4096 3.6 / 4.2 / 5.5, of 8192 4.2 / 4.9 / 5.7. */
template <class X, class H> void launch(const NormArgs &a, int64_t T, hipStream_t s) {
    if (a.n <= 512) launch_nt<X, H, 64, 1, false>(a, T, s);
    else if (a.n <= 1024) launch_nt<X, H, 128, 1, false>(a, T, s);
    else if (a.n <= 2048) launch_nt<X, H, 256, 1, false>(a, T, s);
    else if (a.n <= 4096) launch_nt<X, H, 512, 1, false>(a, T, s);
    else if (a.n <= 6144) launch_nt<X, H, 512, 2, false>(a, T, s);
    else if (a.n <= 8192) launch_nt<X, H, 1024, 1, false>(a, T, s);
    else launch_nt<X, H, 1024, 2, true>(a, T, s);
}
template <class X> void launch_h(int hdt, const NormArgs &a, int64_t T, hipStream_t s) {
    if (hdt == DT_F32) launch<X, float>(a, T, s);
    else if (hdt == DT_F16) launch<X, _Float16>(a, T, s);
    else launch<X, __bf16>(a, T, s);
}

} // namespace

extern "C" int tlm_hip_fp8_add_rmsnorm(int hdt, const void *h, int64_t hstride, int xdt, const void *x,
                                       int64_t xstride, const float *w, float eps, int64_t n, int64_t ntok, void *out,
                                       int64_t ostride, void *codes, float *scale, void *stream) {
    if (n < 1 || n > ((int64_t)1 << 22))
        return tlmh_seterr(TLM_HIP_EINVAL, "fp8_add_rmsnorm: n=%lld outside 1..2^22", (long long)n);
    if (!type_bytes(hdt) || (x && !type_bytes(xdt)))
        return tlmh_seterr(TLM_HIP_EUNSUP, "fp8_add_rmsnorm: dtypes %d, %d (F32, F16 and BF16 only)", hdt, xdt);
    if (ntok < 0) return tlmh_seterr(TLM_HIP_EINVAL, "fp8_add_rmsnorm: ntok=%lld", (long long)ntok);
    if (!(eps >= 0.0f) || eps > 3.0e38f)
        return tlmh_seterr(TLM_HIP_EINVAL, "fp8_add_rmsnorm: eps must be finite and not negative");
    if (ntok == 0) return TLM_HIP_OK;
    if (!h || !w || !codes || !scale) return tlmh_seterr(TLM_HIP_EINVAL, "fp8_add_rmsnorm: NULL argument");
    if (ntok > 1 && (hstride < n || (x && xstride < n) || (out && ostride < n)))
        return tlmh_seterr(TLM_HIP_EINVAL, "fp8_add_rmsnorm: a row stride is below n=%lld", (long long)n);
    const size_t hb = (size_t)type_bytes(hdt);
    if (!aligned(h, hb) || !aligned(out, hb) || (x && !aligned(x, (size_t)type_bytes(xdt))) || !aligned(w, 4) ||
        !aligned(codes, 16) || !aligned(scale, 4))
        return tlmh_seterr(TLM_HIP_EINVAL, "fp8_add_rmsnorm: rows must have their type's alignment, w and scale 4, "
                           "codes 16 bytes");
    const int64_t nb = fp8_blocks(n);
    if (ntok > ((int64_t)1 << 22) || ntok > ((int64_t)1 << 26) / nb)
        return tlmh_seterr(TLM_HIP_ERANGE, "fp8_add_rmsnorm: %lld tokens of %lld values are too many for one launch",
                           (long long)ntok, (long long)n);
    if (int rc = tlmh_refuse_failed(FAILED_FP8, "fp8_add_rmsnorm")) return rc;
    const NormArgs a = {x, h, out, xstride, hstride, ostride, w, (uint8_t *)codes, scale, (double)eps, (int)n, (int)nb};
    hipStream_t s = (hipStream_t)stream;
    if (!x || xdt == DT_F32) launch_h<float>(hdt, a, ntok, s);
    else if (xdt == DT_F16) launch_h<_Float16>(hdt, a, ntok, s);
    else launch_h<__bf16>(hdt, a, ntok, s);
    return tlmh_check(hipGetLastError(), "fp8_add_rmsnorm launch");
}
