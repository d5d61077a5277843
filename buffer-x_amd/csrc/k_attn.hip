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

template <class T> __device__ __forceinline__ bool bad_chunk(bxi4 c)
{
    bool bad = false;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const unsigned u = (unsigned)c[j];
        if constexpr (sizeof(T) == 4) bad |= (u & 0x7f800000u) == 0x7f800000u;
        else {
            constexpr unsigned e = __is_same(T, bx_f16) ? 0x7c00u : 0x7f80u;
            bad |= (u & e) == e || (u >> 16 & e) == e;
        }
    }
    return bad;
}

__device__ __forceinline__ float other_half(float v) { return __shfl_xor(v, 32, 64); }

template <class T, int DP, int NW, bool ALIGNED>
__global__ __launch_bounds__(NW * 64, 2) void attn_kernel(AttnK p)
{
    constexpr int CH = BxElem<T>::CH, CPR = DP / CH, NT = NW * 64, LD = BN * CPR / NT, ND = DP / 32;
    static_assert(BN * CPR % NT == 0, "every thread stages the same number of chunks");
    __shared__ bxi4 sk[BN * CPR], sv[BN * CPR];
    __shared__ int vbad[2];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, lr = lane & 31, h = lane >> 5;
    int id = blockIdx.x;
    const int split = id % p.nsplit; id /= p.nsplit;
    const int tile = id % p.tiles_r; id /= p.tiles_r;
    const int hk = id % p.Hk, b = id / p.Hk;
    const int r0 = tile * NW * 32;
    const Span sp = span_of(p, b, r0, NW * 32);
    if (r0 >= sp.R) return;

    const int per = (sp.t_all + p.nsplit - 1) / p.nsplit;
    const int t0 = min(sp.t_all, split * per), t1 = min(sp.t_all, t0 + per);

    const T* kb = (const T*)p.k + (long long)b * p.k_sb + (long long)hk * p.k_sh;
    const T* vb = (const T*)p.v + (long long)b * p.v_sb + (long long)hk * p.v_sh;

    // this lane's row, and the first and last row of the wave
    const int w0 = r0 + wave * 32, r = w0 + lr;
    const bool live = r < sp.R, wave_live = w0 < sp.R;
    const int row = live ? r : sp.R - 1, qi = row / p.G, qg = row - qi * p.G;
    const int wi0 = w0 / p.G, wi1 = (min(w0 + 32, sp.R) - 1) / p.G;
    const auto hi_of = [&](int i) { return p.right < 0 ? sp.kl : min(sp.kl, i + sp.off + p.right + 1); };
    const auto lo_of = [&](int i) { return p.left < 0 ? 0 : i + sp.off - p.left; };
    const int hi = hi_of(qi), lo = lo_of(qi);
    const int w_hi0 = hi_of(wi0), w_hi1 = hi_of(wi1), w_lo0 = lo_of(wi0), w_lo1 = lo_of(wi1);
    const int b_hi0 = hi_of(r0 / p.G), b_lo1 = lo_of((min(r0 + NW * 32, sp.R) - 1) / p.G);

    bxi4 fq[CPR / 2];
    {
        const T* qr = (const T*)p.q + (long long)b * p.q_sb + (long long)qi * p.q_st + (long long)(hk * p.G + qg) * p.q_sh;
#pragma unroll
        for (int c = 0; c < CPR / 2; ++c) fq[c] = bx_load_chunk<T, ALIGNED>(qr, (2 * c + h) * CH, p.D);
    }

    bxi4 rk[LD], rv[LD];
    const bxi4 zero = {0, 0, 0, 0};
    const auto base_of = [&](int t) { return (t < sp.t_sink ? t : sp.t_lo + t - sp.t_sink) * BN; };
    // keys behind the sequence read as zero: what lies there may be anything
    const auto fetch = [&](int j0) {
#pragma unroll
        for (int i = 0; i < LD; ++i) {
            const int e = tid + i * NT, key = j0 + e / CPR, d = e % CPR * CH;
            rk[i] = rv[i] = zero;
            if (key < sp.kl) {
                rk[i] = bx_load_chunk<T, ALIGNED>(kb + (long long)key * p.k_st, d, p.D);
                rv[i] = bx_load_chunk<T, ALIGNED>(vb + (long long)key * p.v_st, d, p.D);
            }
        }
    };
    const auto kswz = [](int key) { return CPR >= 8 ? key & 7 : (key >> 1) & 3; };
    const auto vswz = [](int key) { return sizeof(T) == 4 ? 0 : CPR >= 8 ? (key & 3) << 1 : ((key >> 1) & 1) << 1; };

    bxf16 o[ND];
#pragma unroll
    for (int t = 0; t < ND; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[t][i] = 0.0f;
    float m = -INFINITY, l = 0.0f;

    // V^T operand of keys 16 u .. 16 u + 15 of block kb2 and dimensions 32 t .. (halves), in the order of S^T's registers
    const auto vfrag = [&](int t, int kb2, int u) {
        typedef short s4 __attribute__((ext_vector_type(4)));
        bxi4 f;
#pragma unroll
        for (int g = 0; g < 2; ++g) {
            const int key = 32 * kb2 + 16 * u + 8 * g + 4 * h + ((lane & 15) >> 2), d = 32 * t + 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
            const short* a = (const short*)&sv[key * CPR + ((d / 8) ^ vswz(key))] + (d & 4);
            const s4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4*)a);
            const bxi2 y = __builtin_bit_cast(bxi2, x);
            f[2 * g] = y[0]; f[2 * g + 1] = y[1];
        }
        return f;
    };

    if (tid < 2) vbad[tid] = 0;
    if (t0 < t1) fetch(base_of(t0));
    for (int t = t0; t < t1; ++t) {
        const int j0 = base_of(t);
        __syncthreads();
        const bool edge = !(j0 + BN <= b_hi0 && (j0 >= b_lo1 || j0 + BN <= p.sinks));
        bool bad = false;
#pragma unroll
        for (int i = 0; i < LD; ++i) {
            const int e = tid + i * NT, key = e / CPR, c = e % CPR;
            sk[key * CPR + (c ^ kswz(key))] = rk[i];
            sv[key * CPR + (c ^ vswz(key))] = rv[i];
        }
        if (edge) {
#pragma unroll
            for (int i = 0; i < LD; ++i) bad |= bad_chunk<T>(rv[i]);
            if (bad) vbad[t & 1] = 1;
        }
        __syncthreads();
        if (t + 1 < t1) fetch(base_of(t + 1));
        const bool bad_v = vbad[t & 1] != 0;
        if (tid == 0) vbad[(t + 1) & 1] = 0;
        if (!wave_live || j0 >= w_hi1 || (j0 + BN <= w_lo0 && j0 >= p.sinks)) continue;
        const bool masked = !(j0 + BN <= w_hi0 && (j0 >= w_lo1 || j0 + BN <= p.sinks));

        bxf16 s[2];
#pragma unroll
        for (int k2 = 0; k2 < 2; ++k2) {
#pragma unroll
            for (int i = 0; i < 16; ++i) s[k2][i] = 0.0f;
            const int key = 32 * k2 + lr;
#pragma unroll
            for (int c = 0; c < CPR / 2; ++c) s[k2] = bx_mma32<T>(sk[key * CPR + ((2 * c + h) ^ kswz(key))], fq[c], s[k2]);
        }
        const auto sees = [&](int k2, int i) {
            const int j = j0 + 32 * k2 + 8 * (i / 4) + 4 * h + i % 4;
            return live && j < hi && (j >= lo || j < p.sinks);
        };
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
        mx = fmaxf(m, fmaxf(mx, other_half(mx)));
        // a row that has seen nothing yet has no maximum: its powers are 2^-inf = 0 whatever is subtracted
        const float mc = mx == -INFINITY ? 0.0f : mx * p.c;
        const float alpha = __builtin_amdgcn_exp2f(fmaf(m, p.c, -mc));
        m = mx;
        float sum = 0.0f;
        // f16 weights are held times 2^14: the smallest ones then keep their digits (O and l carry the factor alike)
        const float mb = __is_same(T, bx_f16) ? mc - 14.0f : mc;
#pragma unroll
        for (int k2 = 0; k2 < 2; ++k2)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                s[k2][i] = __builtin_amdgcn_exp2f(fmaf(s[k2][i], p.c, -mb));
                sum += s[k2][i];
            }
        l = fmaf(l, alpha, sum);
#pragma unroll
        for (int t2 = 0; t2 < ND; ++t2)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[t2][i] *= alpha;

        if (!(masked && bad_v)) {
            if constexpr (sizeof(T) == 4) {
                const float* fv = (const float*)sv;
#pragma unroll
                for (int k2 = 0; k2 < 2; ++k2)
#pragma unroll
                    for (int i = 0; i < 16; ++i)
#pragma unroll
                        for (int t2 = 0; t2 < ND; ++t2)
                            o[t2] = __builtin_amdgcn_mfma_f32_32x32x2f32(fv[(32 * k2 + 8 * (i / 4) + 4 * h + i % 4) * DP + 32 * t2 + lr], s[k2][i], o[t2], 0, 0, 0);
            } else {
                // the weights are rounded to the type of V: at most half a step of each weight, as V's own values carry
#pragma unroll
                for (int k2 = 0; k2 < 2; ++k2)
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        T e[8];
#pragma unroll
                        for (int j = 0; j < 8; ++j) e[j] = (T)s[k2][8 * u + j];
                        bxi4 fp;
                        __builtin_memcpy(&fp, e, 16);
#pragma unroll
                        for (int t2 = 0; t2 < ND; ++t2) o[t2] = bx_mma32<T>(vfrag(t2, k2, u), fp, o[t2]);
                    }
            }
        } else {
            // A tile that some rows do not see in full, with infinities or NaN in V: 0 times those would leak into rows that do not
            // see them.  The finite part goes through the product as always; NaN, +inf and -inf are counted by products of
            // 0 / 1 matrices over the keys that a row does see, and put in afterwards.  Rare, and taken by whole waves.
#pragma unroll 1
            for (int t2 = 0; t2 < ND; ++t2) {
                bxf16 kind[3];
                bxf16 fin;
#pragma unroll
                for (int i = 0; i < 16; ++i) kind[0][i] = kind[1][i] = kind[2][i] = fin[i] = 0.0f;
#pragma unroll
                for (int k2 = 0; k2 < 2; ++k2)
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const int key = 32 * k2 + 8 * (i / 4) + 4 * h + i % 4, d = 32 * t2 + lr;
                        float v;
                        if constexpr (sizeof(T) == 4) v = ((const float*)sv)[key * DP + d];
                        else v = (float)((const T*)&sv[key * CPR + ((d / CH) ^ vswz(key))])[d % CH];
                        const bool nan = v != v, pinf = v == INFINITY, ninf = v == -INFINITY;
                        const float see = sees(k2, i) ? 1.0f : 0.0f;
                        const float w = sizeof(T) == 4 ? s[k2][i] : (float)(T)s[k2][i];
                        fin = __builtin_amdgcn_mfma_f32_32x32x2f32(nan || pinf || ninf ? 0.0f : v, w, fin, 0, 0, 0);
                        kind[0] = __builtin_amdgcn_mfma_f32_32x32x2f32(nan ? 1.0f : 0.0f, see, kind[0], 0, 0, 0);
                        kind[1] = __builtin_amdgcn_mfma_f32_32x32x2f32(pinf ? 1.0f : 0.0f, see, kind[1], 0, 0, 0);
                        kind[2] = __builtin_amdgcn_mfma_f32_32x32x2f32(ninf ? 1.0f : 0.0f, see, kind[2], 0, 0, 0);
                    }
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    if (kind[1][i] > 0.0f) fin[i] += INFINITY;
                    if (kind[2][i] > 0.0f) fin[i] -= INFINITY;
                    if (kind[0][i] > 0.0f) fin[i] = NAN;
                }
#pragma unroll
                for (int t3 = 0; t3 < ND; ++t3)
                    if (t3 == t2)
#pragma unroll
                        for (int i = 0; i < 16; ++i) o[t3][i] += fin[i];
            }
        }
    }

    l += other_half(l);
    if (!live) return;
    if (p.nsplit > 1) {
        const long long rows = (long long)p.B * p.Hk * p.Lq * p.G, at = (long long)split * rows + (long long)(b * p.Hk + hk) * p.Lq * p.G + r;
        float* po = p.ws + at * DP;
#pragma unroll
        for (int t2 = 0; t2 < ND; ++t2)
#pragma unroll
            for (int g = 0; g < 4; ++g)
                *reinterpret_cast<bxf4*>(po + 32 * t2 + 8 * g + 4 * h) = (bxf4){o[t2][4 * g], o[t2][4 * g + 1], o[t2][4 * g + 2], o[t2][4 * g + 3]};
        if (h == 0) {
            float* ml = p.ws + (long long)p.nsplit * rows * DP + at * 2;
            ml[0] = m; ml[1] = l;
        }
        return;
    }
    // a row that sees no key is zero; one whose visible scores are all -inf is 0 / 0
    const float inv = hi <= 0 ? 0.0f : 1.0f / l;
    T* po = (T*)p.o + (long long)b * p.o_sb + (long long)qi * p.o_st + (long long)(hk * p.G + qg) * p.o_sh;
#pragma unroll
    for (int t2 = 0; t2 < ND; ++t2)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int d = 32 * t2 + 8 * g + 4 * h;
            if (d >= p.D) continue;
            const float v[4] = {o[t2][4 * g] * inv, o[t2][4 * g + 1] * inv, o[t2][4 * g + 2] * inv, o[t2][4 * g + 3] * inv};
            bx_store4<T, ALIGNED>(po + d, v, p.D - d);
        }
}

// joins the parts of a row: weights 2^((m_s - m) c), in the order of the splits.  DP / 4 lanes per row, four dimensions each.
template <class T, int DP, bool ALIGNED>
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
    bx_store4<T, ALIGNED>(po + d, v, p.D - d);
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

template <class T, int DP, bool ALIGNED>
int launch(hipStream_t s, const AttnK& k)
{
    const long long grid = (long long)k.tiles_r * k.Hk * k.B * k.nsplit;
    attn_kernel<T, DP, 4, ALIGNED><<<(unsigned)grid, 256, 0, s>>>(k);
    BX_LAUNCH_CHECK();
    if (k.nsplit > 1) {
        const long long rows = (long long)k.B * k.Hk * k.Lq * k.G, per = 256 / (DP / 4);
        attn_join_kernel<T, DP, ALIGNED><<<(unsigned)((rows + per - 1) / per), 256, 0, s>>>(k);
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
    const bool aligned = al(a.q, a.q_stride_b, a.q_stride_t, a.q_stride_h) && al(a.k, a.k_stride_b, a.k_stride_t, a.k_stride_h) &&
                         al(a.v, a.v_stride_b, a.v_stride_t, a.v_stride_h) && al(a.o, a.o_stride_b, a.o_stride_t, a.o_stride_h);
    if (sh.DP == 32) return aligned ? launch<T, 32, true>(s, k) : launch<T, 32, false>(s, k);
    if (sh.DP == 64) return aligned ? launch<T, 64, true>(s, k) : launch<T, 64, false>(s, k);
    return aligned ? launch<T, 128, true>(s, k) : launch<T, 128, false>(s, k);
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
