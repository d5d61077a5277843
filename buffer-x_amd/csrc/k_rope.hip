// k_rope.hip -- norm of every query and key head with the rotation by position in the same pass (bx_qk_norm_rope).
//   y = x * w / sqrt(mean(x^2) + eps)   (rms)     or   x * w / max(|x|, eps)   (l2)     or   x * w   (none)
//   (a, b) of rotation pair p of axis s -> (a cos t - b sin t, b cos t + a sin t),  t = pos[token][s] * freqs[p]
// Bound by memory: q and k are read once and written once.
#include "bx_ops.h"

namespace {

struct RopeK {
    const void *q, *k, *pos, *qw, *kw;
    void *qo, *ko;
    const double* freqs;
    const int32_t* m_dev;
    long long qs_t, qs_h, ks_t, ks_h, qos_t, qos_h, kos_t, kos_h, pos_t;
    int T, Hq, Hk, D, pairs, axes, sec[4], norm, half, pos_int;
    float eps;
};

// sin and cos of x to binary64 precision for |x| < 2^50: x - n pi/2 in two fused steps, then the series on [-pi/4, pi/4].  Positions
// times frequencies reach 1e5 rad and more, where a product in f32 has lost the angle.
__device__ __forceinline__ void sincos64(double x, float& s, float& c)
{
    const double n = rint(x * 0.63661977236758134308);
    double r = fma(-n, 1.57079632679489655800e+00, x);
    r = fma(-n, 6.12323399573676603587e-17, r);
    const double z = r * r;
    double a = fma(z, 1.0 / 6227020800.0, -1.0 / 39916800.0);
    a = fma(z, a, 1.0 / 362880.0);
    a = fma(z, a, -1.0 / 5040.0);
    a = fma(z, a, 1.0 / 120.0);
    a = fma(z, a, -1.0 / 6.0);
    const double sn = fma(r * z, a, r);
    double b = fma(z, -1.0 / 87178291200.0, 1.0 / 479001600.0);
    b = fma(z, b, -1.0 / 3628800.0);
    b = fma(z, b, 1.0 / 40320.0);
    b = fma(z, b, -1.0 / 720.0);
    b = fma(z, b, 1.0 / 24.0);
    b = fma(z, b, -0.5);
    const double cs = fma(z, b, 1.0);
    const int m = (int)((long long)n & 3);
    const double so = (m & 1) ? cs : sn, co = (m & 1) ? sn : cs;
    s = (float)((m & 2) ? -so : so);
    c = (float)(((m + 1) & 2) ? -co : co);
}

constexpr int ROPE_PAIRS = 128;      // rotation pairs of a head (D <= 256)

// One workgroup = one token: its angles once for all heads into LDS, then a wave per head.
template <class T>
__global__ __launch_bounds__(256) void rope_kernel(RopeK p)
{
    __shared__ float sc[ROPE_PAIRS], ss[ROPE_PAIRS];
    const int t = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    if (p.m_dev && t >= *p.m_dev) return;
    for (int i = tid; i < p.pairs; i += 256) {
        int ax = 0, e = p.sec[0];
        while (i >= e && ax + 1 < p.axes) e += p.sec[++ax];
        const double at = p.pos_int ? (double)((const int32_t*)p.pos)[(long long)t * p.pos_t + ax] : (double)((const float*)p.pos)[(long long)t * p.pos_t + ax];
        sincos64(at * p.freqs[i], ss[i], sc[i]);
    }
    __syncthreads();
    for (int hh = wave; hh < p.Hq + p.Hk; hh += 4) {
        const bool isq = hh < p.Hq;
        const int hd = isq ? hh : hh - p.Hq;
        const T* x = isq ? (const T*)p.q + (long long)t * p.qs_t + (long long)hd * p.qs_h : (const T*)p.k + (long long)t * p.ks_t + (long long)hd * p.ks_h;
        T* y = isq ? (T*)p.qo + (long long)t * p.qos_t + (long long)hd * p.qos_h : (T*)p.ko + (long long)t * p.kos_t + (long long)hd * p.kos_h;
        const T* w = (const T*)(isq ? p.qw : p.kw);
        // lane holds pairs lane and lane + 64, and the unrotated elements behind the pairs the same way
        float a[2], b[2], u[4];
        int ia[2], ib[2];
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int pr = lane + 64 * i;
            ia[i] = p.half ? pr : 2 * pr;
            ib[i] = p.half ? pr + p.pairs : 2 * pr + 1;
            a[i] = b[i] = 0.0f;
            if (pr < p.pairs) { a[i] = (float)x[ia[i]]; b[i] = (float)x[ib[i]]; }
            sum = fmaf(a[i], a[i], fmaf(b[i], b[i], sum));
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int d = 2 * p.pairs + lane + 64 * i;
            u[i] = d < p.D ? (float)x[d] : 0.0f;
            sum = fmaf(u[i], u[i], sum);
        }
        float f = 1.0f;
        if (p.norm != BX_NORM_NONE) {
            sum = bx_wave_sum(sum);
            f = p.norm == BX_NORM_RMS ? 1.0f / sqrtf(sum / (float)p.D + p.eps) : 1.0f / (sqrtf(sum) < p.eps ? p.eps : sqrtf(sum));
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int pr = lane + 64 * i;
            if (pr >= p.pairs) continue;
            const float av = a[i] * f * (w ? (float)w[ia[i]] : 1.0f), bv = b[i] * f * (w ? (float)w[ib[i]] : 1.0f);
            const float c = sc[pr], s = ss[pr];
            y[ia[i]] = (T)(av * c - bv * s);
            y[ib[i]] = (T)(bv * c + av * s);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int d = 2 * p.pairs + lane + 64 * i;
            if (d < p.D) y[d] = (T)(u[i] * f * (w ? (float)w[d] : 1.0f));
        }
    }
}

}  // namespace

int bxk_qk_norm_rope(hipStream_t s, int n_cu, const bx_qk_norm_rope_args& a)
{
    (void)n_cu;
    RopeK k = {a.q, a.k, a.pos, a.q_weight, a.k_weight, a.q_out, a.k_out, a.freqs, a.m_dev,
               a.q_stride_t, a.q_stride_h, a.k_stride_t, a.k_stride_h, a.q_out_stride_t, a.q_out_stride_h, a.k_out_stride_t, a.k_out_stride_h,
               a.pos_stride_t, (int)a.T, a.q ? a.Hq : 0, a.k ? a.Hk : 0, a.D, 0, a.axes, {0, 0, 0, 0}, a.norm, a.pairs == BX_PAIRS_HALF,
               a.pos_dtype == BX_POS_I32, a.eps};
    for (int i = 0; i < a.axes; ++i) { k.sec[i] = a.sections[i]; k.pairs += a.sections[i]; }
    if (k.T == 0 || k.Hq + k.Hk == 0) return BX_OK;
    if (a.dtype == BX_TYPE_F32) rope_kernel<float><<<k.T, 256, 0, s>>>(k);
    else if (a.dtype == BX_TYPE_F16) rope_kernel<bx_f16><<<k.T, 256, 0, s>>>(k);
    else rope_kernel<bx_bf16><<<k.T, 256, 0, s>>>(k);
    BX_LAUNCH_CHECK();
    return BX_OK;
}
