// k_attn.hip -- attention over keypoints (bx_attention): o_i = sum_j softmax_j(scale q_i . k_j) v_j over the keys j that row i sees,
//   j < k_len,  j <= p_i + right,  j >= p_i - left or j < sinks,      p_i = i + k_len - q_len.
// One pass over the keys with the running maximum and sum of the softmax (f32); scores never reach memory.
//
// A workgroup serves 32 rows per wave of one (batch entry, key head); the query heads that share a key head are rows like any others, so K and V
// are read once for all of them and a single query still fills rows of a matrix instruction.  Both products are taken transposed:
//   S^T = K Q^T : lane l holds row l % 32 of the queries and, in register i, key 8 (i / 4) + 4 (l / 32) + i % 4 of a 32-key block;
//   O^T = V^T P^T: the same lane holds the same row, so maximum, sum and rescaling stay inside a lane (plus one exchange of the two
//                 halves), and the registers of S^T are the second operand as they are, if V's keys are visited in the same order.
// V's first operand needs keys along the registers: halves are read from LDS with the transposing 8-byte load (lane group of 16 = 4 keys x 16
// dimensions), floats one by one.
//
// Few rows, many keys: the key tiles are dealt to `nsplit` workgroups that leave (O, m, l) in the workspace and a second kernel
// joins them in a fixed order.
#include "bx_ops.h"

namespace {

constexpr int BN = 64;               // keys of a tile

struct AttnK {
    const void *q, *k, *v;
    void* o;
    const int32_t *q_lens, *k_lens;
    float* ws;
    long long q_sb, q_st, q_sh, k_sb, k_st, k_sh, v_sb, v_st, v_sh, o_sb, o_st, o_sh;
    int B, Lq, Lk, Hk, G, D, left, right, sinks, nsplit, tiles_r;
    float c;                         // scale * log2(e): the softmax runs in powers of two
};

// what one (row tile, batch entry) has to visit
struct Span {
    int ql, kl, off, R, t_sink, t_lo, t_all;
};

__device__ __forceinline__ Span span_of(const AttnK& p, int b, int r0, int rows)
{
    Span s;
    s.ql = p.Lq; s.kl = p.Lk;
    if (p.q_lens) s.ql = max(0, min(p.Lq, p.q_lens[b]));
    if (p.k_lens) s.kl = max(0, min(p.Lk, p.k_lens[b]));
    s.off = s.kl - s.ql;
    s.R = s.ql * p.G;
    const int i0 = r0 / p.G, i1 = (min(r0 + rows, s.R) - 1) / p.G;
    const int hi = p.right < 0 ? s.kl : max(0, min(s.kl, i1 + s.off + p.right + 1));
    const int lo = p.left < 0 ? 0 : max(0, i0 + s.off - p.left);
    const int t_hi = (hi + BN - 1) / BN;
    s.t_lo = min(lo / BN, t_hi);
    s.t_sink = min((min(p.sinks, hi) + BN - 1) / BN, s.t_lo);
    s.t_all = s.t_sink + t_hi - s.t_lo;
    return s;
}

__device__ __forceinline__ float other_half(float v) { return __shfl_xor(v, 32, 64); }

// The state of a wave's 32 rows and what one tile of 64 keys in LDS does to it.  K rows lie at chunk c ^ kswz(key), V rows at
// c ^ vswz(key): the lanes of one LDS access then meet different banks.
//
// The reference value m of a row is a maximum that may lag: the weights are 2^((s - m) c) and m follows only when a score exceeds it by
// more than 2^8 would allow -- rows of like scores rescale O once instead of every few tiles.  O and l belong to the same m at all times.
template <class T, int DP>
struct Rows {
    static constexpr int CH = BxElem<T>::CH, CPR = DP / CH, ND = DP / 32;
    // f16 weights are held times 2^7: with the 2^8 above they stay below 2^16 and the smallest keep their digits (O and l alike)
    static constexpr float BIAS = __is_same(T, bx_f16) ? 7.0f : 0.0f;
    bxf16 o[ND];
    bxi4 fq[CPR / 2];
    float m, thr, mb, l;
    bool spoilt;                                             // of the wave
    int lane, lr, h;

    static __device__ __forceinline__ int kswz(int key) { return CPR >= 8 ? key & 7 : (key >> 1) & 3; }
    static __device__ __forceinline__ int vswz(int key) { return sizeof(T) == 4 ? 0 : CPR >= 8 ? (key & 3) << 1 : ((key >> 1) & 1) << 1; }

    __device__ __forceinline__ void init(int lane_)
    {
        lane = lane_; lr = lane & 31; h = lane >> 5;
#pragma unroll
        for (int t = 0; t < ND; ++t)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[t][i] = 0.0f;
        k_at = lr * ROW + ((h ^ kswz(lr)) * 16);
        if constexpr (sizeof(T) == 4) v_at = 4 * h * ROW + lr * 4;
        else {
            const int key = 4 * h + ((lane & 15) >> 2), d = 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
            v_at = key * ROW + ((d / 8) ^ vswz(key)) * 16 + (d & 4) * 2;
        }
        m = thr = -INFINITY;
        mb = -BIAS;
        l = 0.0f;
        spoilt = false;
    }

    // LDS addresses, in bytes from the tile's start.  The swizzles are XORs of address bits below a row, so that the chunks of a row are a
    // few lane values away from constant offsets.
    static constexpr int ROW = DP * (int)sizeof(T);
    int k_at, v_at;                                          // set by init
    __device__ __forceinline__ bxi4 kfrag(const bxi4* sk, int k2, int c) const
    {
        constexpr int M = CPR >= 8 ? 3 : 1;
        return *(const bxi4*)((const char*)sk + (k_at ^ ((c & M) * 32)) + (c & ~M) * 32 + k2 * 32 * ROW);
    }
    // V^T operand of 16 keys (halves), in the order of S^T's registers
    __device__ __forceinline__ bxi4 vfrag(const bxi4* sv, int t, int u) const
    {
        typedef short s4 __attribute__((ext_vector_type(4)));
        bxi4 f;
#pragma unroll
        for (int g = 0; g < 2; ++g) {
            const char* a = (const char*)sv + (v_at ^ ((t & 1) * 64)) + (t >> 1) * 128 + (16 * u + 8 * g) * ROW;
            const bxi2 y = __builtin_bit_cast(bxi2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4*)a));
            f[2 * g] = y[0]; f[2 * g + 1] = y[1];
        }
        return f;
    }
    // V^T operand of key 32 k2 + 8 (i / 4) + 4 (l / 32) + i % 4 (floats)
    __device__ __forceinline__ float vfloat(const bxi4* sv, int t, int k2, int i) const
    {
        return *(const float*)((const char*)sv + v_at + t * 128 + (32 * k2 + 8 * (i / 4) + i % 4) * ROW);
    }

    // the weights as second operands: registers of S^T as they are (f32), or rounded to the type of V -- half a step each, as V's own
    // values carry
    struct Weights { bxf16 s[sizeof(T) == 4 ? 2 : 1]; bxi4 f[sizeof(T) == 4 ? 1 : 4]; };

    // acc += V^T P^T for dimensions 32 t ..
    __device__ __forceinline__ bxf16 weigh(const bxi4* sv, const Weights& w, int t, bxf16 acc) const
    {
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int k2 = 0; k2 < 2; ++k2)
#pragma unroll
                for (int i = 0; i < 16; ++i) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(vfloat(sv, t, k2, i), w.s[k2][i], acc, 0, 0, 0);
        } else {
#pragma unroll
            for (int u = 0; u < 4; ++u) acc = bx_mma32<T>(vfrag(sv, t, u), w.f[u], acc);
        }
        return acc;
    }

    // one tile: `masked` says whether sees(k2, i) -- does this lane's row see the key of register i of block k2 -- has to be asked
    template <class See> __device__ __forceinline__ void tile(const bxi4* sk, const bxi4* sv, float c, float slack, bool masked, const See& sees)
    {
        bxf16 s[2];
#pragma unroll
        for (int k2 = 0; k2 < 2; ++k2) {
#pragma unroll
            for (int i = 0; i < 16; ++i) s[k2][i] = 0.0f;
#pragma unroll
            for (int c2 = 0; c2 < CPR / 2; ++c2) s[k2] = bx_mma32<T>(kfrag(sk, k2, c2), fq[c2], s[k2]);
        }
        if (masked) {
#pragma unroll
            for (int k2 = 0; k2 < 2; ++k2)
#pragma unroll
                for (int i = 0; i < 16; ++i) s[k2][i] = sees(k2, i) ? s[k2][i] : -INFINITY;
        }
        float mx = s[0][0];
#pragma unroll
        for (int k2 = 0; k2 < 2; ++k2)
#pragma unroll
            for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[k2][i]);
        mx = fmaxf(mx, other_half(mx));
        if (__any(mx > thr)) {
            const float mn = fmaxf(m, mx);
            // a row that has seen nothing yet has no maximum: its powers are 2^-inf = 0 whatever is subtracted
            const float mc = mn == -INFINITY ? 0.0f : mn * c;
            const float alpha = __builtin_amdgcn_exp2f(fmaf(m, c, -mc));
            m = mn; mb = mc - BIAS; thr = mn + slack;
            l *= alpha;
#pragma unroll
            for (int t = 0; t < ND; ++t)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[t][i] *= alpha;
        }
        float sum = 0.0f;
#pragma unroll
        for (int k2 = 0; k2 < 2; ++k2)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                s[k2][i] = __builtin_amdgcn_exp2f(fmaf(s[k2][i], c, -mb));
                sum += s[k2][i];
            }
        l += sum;
        Weights w;
        if constexpr (sizeof(T) == 4) { w.s[0] = s[0]; w.s[1] = s[1]; }
        else {
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                T e[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) e[j] = (T)s[u / 2][8 * (u % 2) + j];
                __builtin_memcpy(&w.f[u], e, 16);
            }
        }
        // f32 sums a tile by itself first: fewer roundings at the size of O.  So do tiles on a mask's edge, to see whether anything
        // but numbers came out: 0 times an infinity or NaN of a key that a row does not see would be in it (exact_rows).
        if (masked) {
#pragma unroll
            for (int t = 0; t < ND; ++t) {
                bxf16 a;
#pragma unroll
                for (int i = 0; i < 16; ++i) a[i] = 0.0f;
                a = weigh(sv, w, t, a);
                float z = 0.0f;
#pragma unroll
                for (int i = 0; i < 16; ++i) { z = fmaf(a[i], 0.0f, z); o[t][i] += a[i]; }
                spoilt |= __any(z != z);
            }
        } else if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int t = 0; t < ND; ++t) {
                bxf16 a;
#pragma unroll
                for (int i = 0; i < 16; ++i) a[i] = 0.0f;
                a = weigh(sv, w, t, a);
#pragma unroll
                for (int i = 0; i < 16; ++i) o[t][i] += a[i];
            }
        } else {
#pragma unroll
            for (int t = 0; t < ND; ++t) o[t] = weigh(sv, w, t, o[t]);
        }
    }
};

// The 32 rows from w0 on over the key tiles [t0, t1), one row after the other by the whole wave, touching nothing but what a row sees: the
// way of waves that met an infinity or NaN at the edge of a mask.  Lanes are keys for the scores and dimensions for the sums.
template <class T>
__device__ __forceinline__ void exact_rows(const AttnK& p, const Span& sp, const T* kb, const T* vb, int b, int hk, int w0, int lane, int t0, int t1,
                                           int DP, long long part, long long rows)
{
    for (int r = w0; r < min(w0 + 32, sp.R); ++r) {
        const int qi = r / p.G, qg = r - qi * p.G;
        const int hi = p.right < 0 ? sp.kl : min(sp.kl, qi + sp.off + p.right + 1), lo = p.left < 0 ? 0 : qi + sp.off - p.left;
        const T* q = (const T*)p.q + (long long)b * p.q_sb + (long long)qi * p.q_st + (long long)(hk * p.G + qg) * p.q_sh;
        float m = -INFINITY, l = 0.0f, o0 = 0.0f, o1 = 0.0f;
        for (int t = t0; t < t1; ++t) {
            const int j0 = (t < sp.t_sink ? t : sp.t_lo + t - sp.t_sink) * BN, j = j0 + lane;
            const bool see = j < hi && (j >= lo || j < p.sinks);
            float s = 0.0f;
            if (see)
                for (int d = 0; d < p.D; ++d) s = fmaf((float)q[d], (float)kb[(long long)j * p.k_st + d], s);
            float mx = see ? s : -INFINITY;
#pragma unroll
            for (int x = 32; x >= 1; x >>= 1) mx = fmaxf(mx, __shfl_xor(mx, x, 64));
            mx = fmaxf(m, mx);
            const float mc = mx == -INFINITY ? 0.0f : mx * p.c, alpha = __builtin_amdgcn_exp2f(fmaf(m, p.c, -mc));
            const float w = see ? __builtin_amdgcn_exp2f(fmaf(s, p.c, -(mc - Rows<T, 32>::BIAS))) : 0.0f;
            m = mx;
            l = fmaf(l, alpha, bx_wave_sum(w));
            o0 *= alpha; o1 *= alpha;
            unsigned long long seen = __ballot(see);
            while (seen) {
                const int x = __builtin_ctzll(seen);
                seen &= seen - 1;
                const float wx = __shfl(w, x, 64);
                const T* v = vb + (long long)(j0 + x) * p.v_st;
                if (lane < p.D) o0 = fmaf(wx, (float)v[lane], o0);
                if (lane + 64 < p.D) o1 = fmaf(wx, (float)v[lane + 64], o1);
            }
        }
        if (p.nsplit > 1) {
            float* po = p.ws + (part + r) * DP;
            if (lane < DP) po[lane] = o0;
            if (lane + 64 < DP) po[lane + 64] = o1;
            float* ml = p.ws + (long long)p.nsplit * rows * DP + (part + r) * 2;
            if (lane == 0) { ml[0] = m; ml[1] = l; }
        } else {
            const float inv = hi <= 0 ? 0.0f : 1.0f / l;
            T* po = (T*)p.o + (long long)b * p.o_sb + (long long)qi * p.o_st + (long long)(hk * p.G + qg) * p.o_sh;
            if (lane < p.D) po[lane] = (T)(o0 * inv);
            if (lane + 64 < p.D) po[lane + 64] = (T)(o1 * inv);
        }
    }
}

// DIRECT: 16-byte aligned rows and whole chunks go from memory straight into LDS, two buffers deep; others through registers.
constexpr int waves_of(int bytes, int DP, bool direct)
{
    const int w = (DP == 32 ? 4 : DP == 64 ? 3 : 2) - (bytes == 4 ? 1 : 0) - (direct ? 0 : 1);      // without spills in the loop
    return w < 1 ? 1 : w;
}
template <class T, int DP, int NW, bool DIRECT>
__global__ __launch_bounds__(NW * 64, waves_of(sizeof(T), DP, DIRECT)) void attn_kernel(AttnK p)
{
    constexpr int CH = BxElem<T>::CH, CPR = DP / CH, NT = NW * 64, LD = BN * CPR / NT;
    static_assert(BN * CPR % NT == 0, "every thread stages the same number of chunks");
    __shared__ bxi4 sk0[BN * CPR], sv0[BN * CPR], sk1[DIRECT ? BN * CPR : 1], sv1[DIRECT ? BN * CPR : 1];
    using R_ = Rows<T, DP>;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    int id = (int)bx_xcd_order<16>(blockIdx.x, gridDim.x);
    const int split = id % p.nsplit; id /= p.nsplit;
    const int tile = p.tiles_r - 1 - id % p.tiles_r; id /= p.tiles_r;        // the rows that see most first, where the window has no left end
    const int hk = id % p.Hk, b = id / p.Hk;
    const int r0 = tile * NW * 32;
    const Span sp = span_of(p, b, r0, NW * 32);
    if (r0 >= sp.R) return;

    const int per = (sp.t_all + p.nsplit - 1) / p.nsplit;
    const int t0 = min(sp.t_all, split * per), t1 = min(sp.t_all, t0 + per);

    const T* kb = (const T*)p.k + (long long)b * p.k_sb + (long long)hk * p.k_sh;
    const T* vb = (const T*)p.v + (long long)b * p.v_sb + (long long)hk * p.v_sh;

    // this lane's row, and the first and last row of the wave
    R_ w;
    w.init(lane);
    const int h = w.h, w0 = r0 + wave * 32, r = w0 + w.lr;
    const bool live = r < sp.R, wave_live = w0 < sp.R;
    const int row = live ? r : sp.R - 1, qi = row / p.G, qg = row - qi * p.G;
    const int wi0 = w0 / p.G, wi1 = (min(w0 + 32, sp.R) - 1) / p.G;
    const auto hi_of = [&](int i) { return p.right < 0 ? sp.kl : min(sp.kl, i + sp.off + p.right + 1); };
    const auto lo_of = [&](int i) { return p.left < 0 ? 0 : i + sp.off - p.left; };
    const int hi = live ? hi_of(qi) : 0, lo = lo_of(qi);
    const int w_hi0 = hi_of(wi0), w_hi1 = hi_of(wi1), w_lo0 = lo_of(wi0), w_lo1 = lo_of(wi1);
    {
        const T* qr = (const T*)p.q + (long long)b * p.q_sb + (long long)qi * p.q_st + (long long)(hk * p.G + qg) * p.q_sh;
#pragma unroll
        for (int c = 0; c < CPR / 2; ++c) w.fq[c] = bx_load_chunk<T, DIRECT>(qr, (2 * c + h) * CH, p.D);
    }
    const float slack = 8.0f / p.c;

    const auto base_of = [&](int t) { return (t < sp.t_sink ? t : sp.t_lo + t - sp.t_sink) * BN; };
    const auto serve = [&](const bxi4* sk, const bxi4* sv, int t) __attribute__((always_inline)) {
        const int j0 = base_of(t);
        if (!wave_live || j0 >= w_hi1 || (j0 + BN <= w_lo0 && j0 >= p.sinks)) return;
        const bool masked = !(j0 + BN <= w_hi0 && (j0 >= w_lo1 || j0 + BN <= p.sinks));
        const int a_hi = hi - j0 - 4 * h, a_lo = lo - j0 - 4 * h, a_sink = p.sinks - j0 - 4 * h;
        w.tile(sk, sv, p.c, slack, masked, [&](int k2, int i) {
            const int j = 32 * k2 + 8 * (i / 4) + i % 4;
            return j < a_hi && (j >= a_lo || j < a_sink);
        });
    };

    if constexpr (DIRECT) {
        // LDS position e holds chunk (e % CPR) ^ swizzle of key e / CPR.  Keys behind the sequence repeat its last one: no row sees
        // them.  Chunks behind D stay the zeros that they are set to here.
        if (p.D < DP) {
            const bxi4 zero = {0, 0, 0, 0};
            for (int e = tid; e < BN * CPR; e += NT) sk0[e] = sk1[e] = sv0[e] = sv1[e] = zero;
            __syncthreads();
        }
        // A thread's keys of a tile are STEP apart, so its chunks keep their place within a row; the tile's address is the same for
        // all lanes and a lane adds 32 bits to it (the host sees to it that 64 rows stay within those).
        constexpr int STEP = NT / CPR;
        static_assert(STEP % 8 == 0, "the swizzle of a thread's chunks does not depend on the key's step");
        const int key0 = tid / CPR, ck = ((tid % CPR) ^ R_::kswz(key0)) * CH, cv = ((tid % CPR) ^ R_::vswz(key0)) * CH;
        const int wk = p.D < DP ? p.D : DP;
        const unsigned ks = (unsigned)(p.k_st * sizeof(T)), vs = (unsigned)(p.v_st * sizeof(T));
        const unsigned ko = key0 * ks + ck * (unsigned)sizeof(T), vo = key0 * vs + cv * (unsigned)sizeof(T);
        const auto load = [&](bxi4* sk, bxi4* sv, int t) __attribute__((always_inline)) {
            const int j0 = base_of(t);
            const char* kt = (const char*)(kb + (long long)j0 * p.k_st);
            const char* vt = (const char*)(vb + (long long)j0 * p.v_st);
            const bool whole = j0 + BN <= sp.kl;
#pragma unroll
            for (int i = 0; i < LD; ++i) {
                const int e0 = (i * NW + wave) * 64;
                if (whole) {
                    if (ck < wk) bx_load_lds16(kt + (unsigned)(i * STEP) * ks + ko, sk + e0);
                    if (cv < wk) bx_load_lds16(vt + (unsigned)(i * STEP) * vs + vo, sv + e0);
                } else {
                    const unsigned key = min(key0 + i * STEP, sp.kl - 1 - j0);
                    if (ck < wk) bx_load_lds16(kt + (key * ks + ck * (unsigned)sizeof(T)), sk + e0);
                    if (cv < wk) bx_load_lds16(vt + (key * vs + cv * (unsigned)sizeof(T)), sv + e0);
                }
            }
        };
        if (t0 < t1) load(sk0, sv0, t0);
        for (int t = t0; t < t1; ++t) {
            bxi4 *ck_ = (t - t0) & 1 ? sk1 : sk0, *cv_ = (t - t0) & 1 ? sv1 : sv0, *nk_ = (t - t0) & 1 ? sk0 : sk1, *nv_ = (t - t0) & 1 ? sv0 : sv1;
            __syncthreads();
            if (t + 1 < t1) load(nk_, nv_, t + 1);
            serve(ck_, cv_, t);
        }
    } else {
        bxi4 rk[LD], rv[LD];
        const bxi4 zero = {0, 0, 0, 0};
        const auto fetch = [&](int t) {
            const int j0 = base_of(t);
#pragma unroll
            for (int i = 0; i < LD; ++i) {
                const int e = tid + i * NT, key = j0 + e / CPR, d = e % CPR * CH;
                rk[i] = rv[i] = zero;
                if (key < sp.kl) {
                    rk[i] = bx_load_chunk<T, false>(kb + (long long)key * p.k_st, d, p.D);
                    rv[i] = bx_load_chunk<T, false>(vb + (long long)key * p.v_st, d, p.D);
                }
            }
        };
        if (t0 < t1) fetch(t0);
        for (int t = t0; t < t1; ++t) {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < LD; ++i) {
                const int e = tid + i * NT, key = e / CPR, c = e % CPR;
                sk0[key * CPR + (c ^ R_::kswz(key))] = rk[i];
                sv0[key * CPR + (c ^ R_::vswz(key))] = rv[i];
            }
            __syncthreads();
            if (t + 1 < t1) fetch(t + 1);
            serve(sk0, sv0, t);
        }
    }

    const long long rows = (long long)p.B * p.Hk * p.Lq * p.G, part = (long long)split * rows + (long long)(b * p.Hk + hk) * p.Lq * p.G;
    if (w.spoilt) {
        exact_rows<T>(p, sp, kb, vb, b, hk, w0, lane, t0, t1, DP, part, rows);
        return;
    }
    const float l = w.l + other_half(w.l);
    if (!live) return;
    if (p.nsplit > 1) {
        float* po = p.ws + (part + r) * DP;
#pragma unroll
        for (int t = 0; t < R_::ND; ++t)
#pragma unroll
            for (int g = 0; g < 4; ++g)
                *reinterpret_cast<bxf4*>(po + 32 * t + 8 * g + 4 * h) = (bxf4){w.o[t][4 * g], w.o[t][4 * g + 1], w.o[t][4 * g + 2], w.o[t][4 * g + 3]};
        if (h == 0) {
            float* ml = p.ws + (long long)p.nsplit * rows * DP + (part + r) * 2;
            ml[0] = w.m; ml[1] = l;
        }
        return;
    }
    // a row that sees no key is zero; one whose visible scores are all -inf is 0 / 0
    const float inv = hi <= 0 ? 0.0f : 1.0f / l;
    T* po = (T*)p.o + (long long)b * p.o_sb + (long long)qi * p.o_st + (long long)(hk * p.G + qg) * p.o_sh;
#pragma unroll
    for (int t = 0; t < R_::ND; ++t)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int d = 32 * t + 8 * g + 4 * h;
            if (d >= p.D) continue;
            const float v[4] = {w.o[t][4 * g] * inv, w.o[t][4 * g + 1] * inv, w.o[t][4 * g + 2] * inv, w.o[t][4 * g + 3] * inv};
            bx_store4<T>(po + d, v, p.D - d);
        }
}

// joins the parts of a row: weights 2^((m_s - m) c), in the order of the splits.  DP / 4 lanes per row, four dimensions each.
template <class T, int DP>
__global__ __launch_bounds__(256) void attn_join_kernel(AttnK p)
{
    constexpr int LPR = DP / 4, RPB = 256 / LPR;
    const long long rows = (long long)p.B * p.Hk * p.Lq * p.G, at = (long long)blockIdx.x * RPB + threadIdx.x / LPR;
    if (at >= rows) return;
    const int d = threadIdx.x % LPR * 4;
    const int per = p.Lq * p.G, r = (int)(at % per), bh = (int)(at / per), b = bh / p.Hk, hk = bh - b * p.Hk;
    const int qi = r / p.G, qg = r - qi * p.G;
    const int ql = p.q_lens ? max(0, min(p.Lq, p.q_lens[b])) : p.Lq, kl = p.k_lens ? max(0, min(p.Lk, p.k_lens[b])) : p.Lk;
    if (qi >= ql || d >= p.D) return;
    const float* ml = p.ws + (long long)p.nsplit * rows * DP;
    float m = -INFINITY;
    for (int s = 0; s < p.nsplit; ++s) m = fmaxf(m, ml[((long long)s * rows + at) * 2]);
    const float mc = m == -INFINITY ? 0.0f : m * p.c;
    float l = 0.0f, v[4] = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < p.nsplit; ++s) {
        const float w = __builtin_amdgcn_exp2f(fmaf(ml[((long long)s * rows + at) * 2], p.c, -mc));
        l = fmaf(w, ml[((long long)s * rows + at) * 2 + 1], l);
        const bxf4 o = *reinterpret_cast<const bxf4*>(p.ws + ((long long)s * rows + at) * DP + d);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = fmaf(w, o[j], v[j]);
    }
    const bool empty = p.right >= 0 && qi + kl - ql + p.right + 1 <= 0;
    const float inv = empty || kl <= 0 ? 0.0f : 1.0f / l;
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] *= inv;
    T* po = (T*)p.o + (long long)b * p.o_sb + (long long)qi * p.o_st + (long long)(hk * p.G + qg) * p.o_sh;
    bx_store4<T>(po + d, v, p.D - d);
}

int padded(int D) { return D <= 32 ? 32 : D <= 64 ? 64 : 128; }

struct Shape { int DP, tiles_r, nsplit; };

// Rows alone fill the card when there are two workgroups a compute unit; with fewer the keys are split, as long as a part keeps
// four tiles of 64 keys (below that the joining costs more than it saves).
Shape shape_of(int n_cu, const bx_attention_args& a)
{
    Shape s;
    s.DP = padded(a.D);
    const long long R = (long long)a.Lq * (a.Hq / a.Hk);
    s.tiles_r = (int)((R + 127) / 128);
    const long long base = (long long)s.tiles_r * a.Hk * a.B;
    long long keys = a.Lk;
    if (a.left >= 0 && a.right >= 0) {
        const long long span = (long long)a.left + a.right + 1 + (R < 128 ? a.Lq : 128 / (a.Hq / a.Hk) + 1) + a.sinks + 2 * BN;
        keys = span < keys ? span : keys;
    }
    const long long tiles = (keys + BN - 1) / BN;
    long long n = base > 0 ? 2LL * n_cu / base : 1;
    if (n > tiles / 4) n = tiles / 4;
    if (n > 128) n = 128;
    s.nsplit = n < 1 ? 1 : (int)n;
    return s;
}

int64_t bytes_of(const Shape& s, const bx_attention_args& a)
{
    if (s.nsplit <= 1) return 0;
    return (int64_t)s.nsplit * a.B * a.Lq * a.Hq * (s.DP + 2) * 4;
}

template <class T, int DP, bool DIRECT>
int launch(hipStream_t s, const AttnK& k)
{
    const long long grid = (long long)k.tiles_r * k.Hk * k.B * k.nsplit;
    attn_kernel<T, DP, 4, DIRECT><<<(unsigned)grid, 256, 0, s>>>(k);
    BX_LAUNCH_CHECK();
    if (k.nsplit > 1) {
        const long long rows = (long long)k.B * k.Hk * k.Lq * k.G, per = 256 / (DP / 4);
        attn_join_kernel<T, DP><<<(unsigned)((rows + per - 1) / per), 256, 0, s>>>(k);
        BX_LAUNCH_CHECK();
    }
    return BX_OK;
}

template <class T>
int attention_of(hipStream_t s, int n_cu, const bx_attention_args& a)
{
    const Shape sh = shape_of(n_cu, a);
    AttnK k = {a.q, a.k, a.v, a.o, a.q_lens, a.k_lens, (float*)a.workspace,
               a.q_stride_b, a.q_stride_t, a.q_stride_h, a.k_stride_b, a.k_stride_t, a.k_stride_h,
               a.v_stride_b, a.v_stride_t, a.v_stride_h, a.o_stride_b, a.o_stride_t, a.o_stride_h,
               a.B, a.Lq, a.Lk, a.Hk, a.Hq / a.Hk, a.D, a.left, a.right, a.sinks, sh.nsplit, sh.tiles_r,
               (float)((double)a.scale * 1.4426950408889634)};
    const auto al = [](const void* p, long long x, long long y, long long z) {
        return (((uintptr_t)p | (uintptr_t)(x * (long long)sizeof(T)) | (uintptr_t)(y * (long long)sizeof(T)) | (uintptr_t)(z * (long long)sizeof(T))) & 15) == 0;
    };
    const long long far = (1LL << 31) / (BN * (long long)sizeof(T));          // rows further apart: a tile does not fit 32-bit offsets
    const bool direct = a.D % BxElem<T>::CH == 0 && a.k_stride_t < far && a.v_stride_t < far && al(a.q, a.q_stride_b, a.q_stride_t, a.q_stride_h) && al(a.k, a.k_stride_b, a.k_stride_t, a.k_stride_h) &&
                        al(a.v, a.v_stride_b, a.v_stride_t, a.v_stride_h);
    if (sh.DP == 32) return direct ? launch<T, 32, true>(s, k) : launch<T, 32, false>(s, k);
    if (sh.DP == 64) return direct ? launch<T, 64, true>(s, k) : launch<T, 64, false>(s, k);
    return direct ? launch<T, 128, true>(s, k) : launch<T, 128, false>(s, k);
}

}  // namespace

int64_t bxk_attention_workspace(int n_cu, const bx_attention_args& a)
{
    if (a.B == 0 || a.Lq == 0) return 0;
    return bytes_of(shape_of(n_cu, a), a);
}

int bxk_attention(hipStream_t s, int n_cu, const bx_attention_args& a)
{
    if (a.B == 0 || a.Lq == 0) return BX_OK;
    const Shape sh = shape_of(n_cu, a);
    const int64_t need = bytes_of(sh, a);
    if (need > 0 && (!a.workspace || a.workspace_bytes < need)) {
        bx_set_error("bx_attention: workspace of %lld bytes, needs %lld (bx_attention_workspace)", (long long)a.workspace_bytes, (long long)need);
        return BX_ERR_STATE;
    }
    if (((long long)sh.tiles_r * a.Hk * a.B) * sh.nsplit > 0x7fffffffLL || (long long)a.B * a.Lq * a.Hq > 0x7fffffffLL) {
        bx_set_error("bx_attention: too many rows for one launch"); return BX_ERR_ARG;
    }
    if (a.dtype == BX_TYPE_F32) return attention_of<float>(s, n_cu, a);
    if (a.dtype == BX_TYPE_F16) return attention_of<bx_f16>(s, n_cu, a);
    return attention_of<bx_bf16>(s, n_cu, a);
}
