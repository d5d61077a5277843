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

// 1 / (2 pi), 1152 bits behind the point: as many turns as the largest binary64 number of radians leaves a fraction of
__device__ const unsigned long long TURN[18] = {
    0x28be60db9391054aULL, 0x7f09d5f47d4d3770ULL, 0x36d8a5664f10e410ULL,
    0x7f9458eaf7aef158ULL, 0x6dc91b8e909374b8ULL, 0x01924bba82746487ULL,
    0x3f877ac72c4a69cfULL, 0xba208d7d4baed121ULL, 0x3a671c09ad17df90ULL,
    0x4e64758e60d4ce7dULL, 0x272117e2ef7e4a0eULL, 0xc7fe25fff7816603ULL,
    0xfbcbc462d6829b47ULL, 0xdb4d9fb3c9f2c26dULL, 0xd3d18fd9a797fa8bULL,
    0x5d49eeb1faf97c5eULL, 0xcf41ce7de294a4baULL, 0x9afed7ec47e35742ULL};

// |x| >= 2^52 radians: x = m 2^e with whole m < 2^53, e >= 0.  Of the digits of 1 / (2 pi) those above 2^-e make whole turns; m times the next 128 is,
// modulo 2^128, the fraction of a turn, off by 2^-75 of one.  q = the nearest quarter, r = what is left of it in radians.
__device__ __forceinline__ double far_angle(double x, int& q)
{
    const unsigned long long bits = __builtin_bit_cast(unsigned long long, x) & ~(1ULL << 63);
    const int e = min((int)(bits >> 52) - 1075, 971), at = e >> 6, sh = e & 63;
    const unsigned long long m = (bits & ((1ULL << 52) - 1)) | 1ULL << 52;
    unsigned long long u1 = TURN[at], u0 = TURN[at + 1];
    if (sh > 0) { u1 = u1 << sh | u0 >> (64 - sh); u0 = u0 << sh | TURN[at + 2] >> (64 - sh); }
    const unsigned long long f = m * u1 + __umul64hi(m, u0);
    const unsigned long long n = (f + (1ULL << 61)) >> 62;
    const double r = (double)(long long)(f - (n << 62)) * (1.57079632679489655800e+00 * 0x1p-62);
    q = x < 0.0 ? -(int)n : (int)n;
    // (infinities and NaN have no angle)
    return bits >= 0x7ffULL << 52 ? x - x : x < 0.0 ? -r : r;
}

// sin and cos of x: the nearest multiple of pi/2 is taken off in two fused steps (beyond 2^52 by far_angle), then the series on [-pi/4, pi/4].  Their
// ends are 3e-14 off; the reduction adds 3e-12 at 2^50 and 7e-10 at 2^52, where f32 results keep 6e-8.  Positions times frequencies reach 1e5 rad
// and more, where a product in f32 has lost the angle.
__device__ __forceinline__ void sincos64(double x, float& s, float& c)
{
    double r;
    int m;
    if (fabs(x) < 0x1p52) {
        const double n = rint(x * 0.63661977236758134308);
        r = fma(-n, 1.57079632679489655800e+00, x);
        r = fma(-n, 6.12323399573676603587e-17, r);
        m = (int)(long long)n;
    } else r = far_angle(x, m);
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
    const double so = (m & 1) ? cs : sn, co = (m & 1) ? sn : cs;
    s = (float)((m & 2) ? -so : so);
    c = (float)(((m + 1) & 2) ? -co : co);
}

// N consecutive elements (16 bytes), of which n exist
template <class T, int N, bool VEC> __device__ __forceinline__ bxi4 load_piece(const T* p, int n)
{
    bxi4 r = {0, 0, 0, 0};
    if constexpr (VEC) {
        if (n > 0) r = *reinterpret_cast<const bxi4*>(p);
    } else if (n >= N) {
        r = reinterpret_cast<const BxAny16*>(p)->v;
    } else if (n > 0) {
        T e[N];
#pragma unroll
        for (int j = 0; j < N; ++j) e[j] = j < n ? p[j] : (T)0.0f;
        __builtin_memcpy(&r, e, 16);
    }
    return r;
}
template <class T, int N> __device__ __forceinline__ void floats_of(bxi4 r, float* v)
{
    T e[N];
    __builtin_memcpy(e, &r, 16);
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = (float)e[j];
}
template <class T, int N, bool VEC> __device__ __forceinline__ void store_piece(T* p, const float* v, int n)
{
    T e[N];
#pragma unroll
    for (int j = 0; j < N; ++j) e[j] = (T)v[j];
    if constexpr (VEC) {
        bxi4 r;
        __builtin_memcpy(&r, e, 16);
        if (n > 0) *reinterpret_cast<bxi4*>(p) = r;
    } else if (n >= N) {
        bxi4 r;
        __builtin_memcpy(&r, e, 16);
        reinterpret_cast<BxAny16*>(p)->v = r;
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j)
            if (j < n) p[j] = e[j];
    }
}

// A workgroup serves TPB tokens.  Their angles are formed once for all heads into LDS; then LPR lanes take a head row, N = 8 or 4
// elements of its first stretch and as many of its second stretch each, so that both ends of a rotation pair are in one lane:
//   HALF:        elements [N x, N x + N) and [P + N x, P + N x + N)  -- the pairs N x ..
//   interleaved: elements [2 N x, 2 N x + 2 N)                       -- the pairs N x ..
// What lies behind 2 P is a row of its own kind: plain elements, 2 N a lane.  VEC: the pieces are read and written whole (P and D are
// multiples of N, and of 2 N where they are not rotated); otherwise element by element, with the same arrangement.
template <class T, int LPR, int N, bool HALF, bool VEC>
__global__ __launch_bounds__(256) void rope_kernel(RopeK p, int tpb)
{
    extern __shared__ float angles[];                        // [tpb][P] cos, then sin
    constexpr int RPB = 256 / LPR;
    const int tid = threadIdx.x, P = p.pairs;
    int T_ = p.T;
    if (p.m_dev) { const int live = *p.m_dev; T_ = live < T_ ? live : T_; }
    const int t0 = (int)blockIdx.x * tpb;
    if (t0 >= T_) return;
    const int nt = min(tpb, T_ - t0);
    const int x = tid % LPR, H = p.Hq + p.Hk;
    // this lane's elements: two pieces of N
    const bool turn = N * x < P;
    const int u = 2 * N * x, tail = 2 * P;                   // interleaved, or behind the pairs
    const int px = (P + N - 1) / N;                          // lanes that hold pairs
    const int e0 = turn ? (HALF ? N * x : u) : tail + 2 * N * (x - px), e1 = turn && HALF ? P + N * x : e0 + N;
    // how many of each piece exist
    const int n0 = turn ? (HALF ? min(N, P - N * x) : min(N, 2 * P - e0)) : max(0, min(N, p.D - e0));
    const int n1 = turn ? (HALF ? n0 : max(0, min(N, 2 * P - e1))) : max(0, min(N, p.D - e1));
    // a row's elements are on their way while the angles, or the row before, are worked out
    bxi4 ra, rb;
    const auto fetch = [&](int row) {
        const int t = row / H, hh = row - t * H;
        const long long tok = t0 + t;
        const T* in = hh < p.Hq ? (const T*)p.q + tok * p.qs_t + (long long)hh * p.qs_h : (const T*)p.k + tok * p.ks_t + (long long)(hh - p.Hq) * p.ks_h;
        ra = load_piece<T, N, VEC>(in + e0, n0);
        rb = load_piece<T, N, VEC>(in + e1, n1);
    };
    if (tid / LPR < nt * H) fetch(tid / LPR);
    float *cs = angles, *sn = angles + tpb * P;
    for (int i = tid; i < nt * P; i += 256) {
        const int t = i / P, pr = i - t * P;
        int ax = 0, e = p.sec[0];
        while (pr >= e && ax + 1 < p.axes) e += p.sec[++ax];
        const long long at = (long long)(t0 + t) * p.pos_t + ax;
        const double pos = p.pos_int ? (double)((const int32_t*)p.pos)[at] : (double)((const float*)p.pos)[at];
        sincos64(pos * p.freqs[pr], sn[i], cs[i]);
    }
    __syncthreads();
    for (int row = tid / LPR; row < nt * H; row += RPB) {
        const int t = row / H, hh = row - t * H;
        const bool isq = hh < p.Hq;
        const long long tok = t0 + t;
        T* out = isq ? (T*)p.qo + tok * p.qos_t + (long long)hh * p.qos_h : (T*)p.ko + tok * p.kos_t + (long long)(hh - p.Hq) * p.kos_h;
        const T* w = (const T*)(isq ? p.qw : p.kw);
        float a[N], b[N];
        floats_of<T, N>(ra, a);
        floats_of<T, N>(rb, b);
        if (row + RPB < nt * H) fetch(row + RPB);
        if (p.norm != BX_NORM_NONE) {
            const auto squares = [&]() __attribute__((always_inline)) {
                float sum = 0.0f;
#pragma unroll
                for (int i = 0; i < N; ++i) sum = fmaf(a[i], a[i], fmaf(b[i], b[i], sum));
#pragma unroll
                for (int k = LPR / 2; k >= 1; k >>= 1) sum += __shfl_xor(sum, k, LPR);
                return sum;
            };
            const bool rms = p.norm == BX_NORM_RMS;
            float sum = squares(), eps = p.eps;
            // squares out of f32's range: the head times a power of two, which x / d does not notice (small ones only where eps does not decide)
            if (sum == INFINITY || (sum < 0x1p-80f && eps < (rms ? 0x1p-80f : 0x1p-40f))) {
                const float s = sum == INFINITY ? 0x1p-70f : 0x1p90f;
#pragma unroll
                for (int i = 0; i < N; ++i) { a[i] *= s; b[i] *= s; }
                eps = rms ? eps * s * s : eps * s;
                sum = squares();
            }
            // x / d, by a product with 1 / d and what that leaves of x: as a division rounds it.  (A d that is zero or not finite has no such rest: d = 0
            // there makes it x, which counts for nothing.)
            const float l2 = sqrtf(sum), d = rms ? sqrtf(sum / (float)p.D + eps) : l2 < eps ? eps : l2, f = 1.0f / d;
            const bool safe = d > 0x1p-100f && d < 0x1p100f;
            const float dr = safe ? d : 0.0f, fr = safe ? f : 0.0f;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float ya = a[i] * f, yb = b[i] * f;
                a[i] = fmaf(fmaf(-ya, dr, a[i]), fr, ya);
                b[i] = fmaf(fmaf(-yb, dr, b[i]), fr, yb);
            }
        }
        if (w) {
            float wa[N], wb[N];
            floats_of<T, N>(load_piece<T, N, VEC>(w + e0, n0), wa);
            floats_of<T, N>(load_piece<T, N, VEC>(w + e1, n1), wb);
#pragma unroll
            for (int i = 0; i < N; ++i) { a[i] *= wa[i]; b[i] *= wb[i]; }
        }
        if (turn) {
            const float *c = cs + t * P + N * x, *s = sn + t * P + N * x;
            if constexpr (HALF) {
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const float ci = VEC || i < n0 ? c[i] : 0.0f, si = VEC || i < n0 ? s[i] : 0.0f, v = a[i];
                    a[i] = v * ci - b[i] * si;
                    b[i] = b[i] * ci + v * si;
                }
            } else {
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    float& v0 = i < N / 2 ? a[2 * i] : b[2 * i - N];
                    float& v1 = i < N / 2 ? a[2 * i + 1] : b[2 * i + 1 - N];
                    const bool is = VEC || N * x + i < P;
                    const float ci = is ? c[i] : 0.0f, si = is ? s[i] : 0.0f, v = v0;
                    v0 = v * ci - v1 * si;
                    v1 = v1 * ci + v * si;
                }
            }
        }
        store_piece<T, N, VEC>(out + e0, a, n0);
        store_piece<T, N, VEC>(out + e1, b, n1);
    }
}

template <class T, int LPR, int N>
int rope_launch(hipStream_t s, const RopeK& k, bool vec, int tpb, unsigned grid)
{
    const size_t lds = (size_t)tpb * k.pairs * 8;
    if (k.half) {
        if (vec) rope_kernel<T, LPR, N, true, true><<<grid, 256, lds, s>>>(k, tpb);
        else rope_kernel<T, LPR, N, true, false><<<grid, 256, lds, s>>>(k, tpb);
    } else {
        if (vec) rope_kernel<T, LPR, N, false, true><<<grid, 256, lds, s>>>(k, tpb);
        else rope_kernel<T, LPR, N, false, false><<<grid, 256, lds, s>>>(k, tpb);
    }
    BX_LAUNCH_CHECK();
    return BX_OK;
}

template <class T>
int rope_of(hipStream_t s, int n_cu, const RopeK& k)
{
    constexpr int N = BxElem<T>::CH;
    const auto al = [](const void* p, long long x, long long y) { return (((uintptr_t)p | (uintptr_t)(x * (long long)sizeof(T)) | (uintptr_t)(y * (long long)sizeof(T))) & 15) == 0; };
    const bool vec = k.pairs % N == 0 && (k.D - 2 * k.pairs) % (2 * N) == 0 && (k.Hq == 0 || (al(k.q, k.qs_t, k.qs_h) && al(k.qo, k.qos_t, k.qos_h) && al(k.qw, 0, 0))) &&
                     (k.Hk == 0 || (al(k.k, k.ks_t, k.ks_h) && al(k.ko, k.kos_t, k.kos_h) && al(k.kw, 0, 0)));
    // lanes of a row: its pairs N a lane, then what is not rotated 2 N a lane
    const int lanes = (k.pairs + N - 1) / N + (k.D - 2 * k.pairs + 2 * N - 1) / (2 * N);
    const int lpr = lanes <= 1 ? 1 : lanes <= 2 ? 2 : lanes <= 4 ? 4 : lanes <= 8 ? 8 : lanes <= 16 ? 16 : lanes <= 32 ? 32 : 64;
    // Tokens of a workgroup: about four head rows per lane group, so that the angles' latency is paid once for several rows and
    // neighbouring rows are in flight together; fewer when the tokens would not fill the card, and no more than 48 KB of angles.
    const int H = k.Hq + k.Hk, rpb = 256 / lpr;
    long long tpb = (4LL * rpb + H - 1) / H;
    const long long fill = (k.T + 4LL * n_cu - 1) / (4LL * n_cu);
    if (tpb > fill) tpb = fill;
    if (k.pairs > 0 && tpb > 49152 / (8 * k.pairs)) tpb = 49152 / (8 * k.pairs);
    if (tpb < 1) tpb = 1;
    const unsigned grid = (unsigned)((k.T + tpb - 1) / tpb);
    if (bx_grid_check("bx_qk_norm_rope", grid, 256) != BX_OK) return BX_ERR_ARG;
    switch (lpr) {
        case 1: return rope_launch<T, 1, N>(s, k, vec, (int)tpb, grid);
        case 2: return rope_launch<T, 2, N>(s, k, vec, (int)tpb, grid);
        case 4: return rope_launch<T, 4, N>(s, k, vec, (int)tpb, grid);
        case 8: return rope_launch<T, 8, N>(s, k, vec, (int)tpb, grid);
        case 16: return rope_launch<T, 16, N>(s, k, vec, (int)tpb, grid);
        case 32: return rope_launch<T, 32, N>(s, k, vec, (int)tpb, grid);
        default: return rope_launch<T, 64, N>(s, k, vec, (int)tpb, grid);
    }
}

}  // namespace

int bxk_qk_norm_rope(hipStream_t s, int n_cu, const bx_qk_norm_rope_args& a)
{
    RopeK k = {a.q, a.k, a.pos, a.q_weight, a.k_weight, a.q_out, a.k_out, a.freqs, a.m_dev,
               a.q_stride_t, a.q_stride_h, a.k_stride_t, a.k_stride_h, a.q_out_stride_t, a.q_out_stride_h, a.k_out_stride_t, a.k_out_stride_h,
               a.pos_stride_t, (int)a.T, a.q ? a.Hq : 0, a.k ? a.Hk : 0, a.D, 0, a.axes, {0, 0, 0, 0}, a.norm, a.pairs == BX_PAIRS_HALF,
               a.pos_dtype == BX_POS_I32, a.eps};
    for (int i = 0; i < a.axes; ++i) { k.sec[i] = a.sections[i]; k.pairs += a.sections[i]; }
    if (k.T == 0 || k.Hq + k.Hk == 0) return BX_OK;
    if (a.dtype == BX_TYPE_F32) return rope_of<float>(s, n_cu, k);
    if (a.dtype == BX_TYPE_F16) return rope_of<bx_f16>(s, n_cu, k);
    return rope_of<bx_bf16>(s, n_cu, k);
}
