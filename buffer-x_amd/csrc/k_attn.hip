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
// (Times of halves that the comments below compare were taken with weights of one number each; two add 3 to 35 % to both sides.)
//
// Few rows, many keys: the key tiles are dealt to `nsplit` workgroups that leave (O, m, l) in the workspace and a second kernel
// joins them in a fixed order.
#include "bx_ops.h"

namespace {

constexpr int BN = 64;               // keys of a tile

// f16 weights are held times 2^7: with the 2^8 that the reference value may lag they stay below 2^16 and the smallest keep their digits.  bf16
// weights are held times 2^-8: none is above 1, so that sums over large values pass the range of f32 no sooner than sum p v would with the largest p
// at 1.  (f32 needs none: sums that are not numbers are formed again by exact_rows, whose weights are at most 1.)
template <class T> __host__ __device__ constexpr float bias_of() { return __is_same(T, bx_f16) ? 7.0f : __is_same(T, bx_bf16) ? -8.0f : 0.0f; }

// Weights are 2^(s c - mb), mb = m c - bias rounded, so that what a row sums is relative to 2^(m c - over), over = m c - mb.  Scores (times scale * log2(e))
// of 2^22 and more are too steep for that: m c and the lag of m are rounded by whole units of the exponent there, and a weight could pass the range of
// its type (below, both together add less than half a unit).  Their weights are 2^((s - m) c), over = 0 (exact_rows).
constexpr float STEEP = 4194304.0f;  // 2^22
template <class T> __device__ __forceinline__ float over_of(float m, float c)
{
    const float mb = fmaf(m, c, -bias_of<T>());
    return fabsf(mb) < STEEP ? fmaf(m, c, -mb) : 0.0f;
}

// n / d for 0 <= n < 2^31 by a multiplication: with l the least for which d <= 2^l, m = floor(2^(31 + l) / d) + 1 is less than 2^32, and n times the
// excess m d - 2^(31 + l) <= d <= 2^l stays below 2^(31 + l), which is what the quotient can bear.  A division takes some twenty
// instructions and a wave does ten before its first tile, which may be its only one (1500 x 140 positions, 2 / 1 heads of 32, f16, 24 keys to
// either side + 1: 32.9 -> 30.2 us; one query over 8192 keys 17.7 -> 17.2).
struct Div {
    unsigned m;
    int s;
    __device__ __forceinline__ int operator()(int n) const { return (int)((unsigned long long)(unsigned)n * m >> s); }
};
Div div_of(int d)
{
    int l = 0;
    while ((1LL << l) < d) ++l;
    return {(unsigned)((1ULL << (31 + l)) / (unsigned)d + 1), 31 + l};
}

struct AttnK {
    const void *q, *k, *v;
    void* o;
    const int32_t *q_lens, *k_lens;
    float* ws;
    long long q_sb, q_st, q_sh, k_sb, k_st, k_sh, v_sb, v_st, v_sh, o_sb, o_st, o_sh;
    int B, Lq, Lk, Hk, G, D, left, right, sinks, nsplit, tiles_r;
    float c;                         // scale * log2(e): the softmax runs in powers of two
    Div by_G, by_Hk, by_nsplit, by_tiles, by_rows;           // by_rows: Lq G
};

// What one (row tile, batch entry) has to visit.  Keys that no row sees are skipped: the rows count what is left, the first `sinks` keys and then
// those from the window's first one on, and key_of is the key that such a count stands for.  So tiles begin where the window begins and the
// first keys cost no tile of their own (32768 positions, 16 / 4 heads of 128, bf16, causal window of 1024 + 4: 341 -> 329 us; 1500 x 140
// positions, 2 / 1 heads of 32, f16, 24 keys to either side + 1: 37.2 -> 33.3 us; the same in f32 103 -> 76 us).
struct Span {
    int ql, kl, off, R, sinks, shift, t_all;
    __device__ __forceinline__ int key_of(int x) const { return x < sinks ? x : x + shift; }
};

__device__ __forceinline__ Span span_of(const AttnK& p, int b, int r0, int rows)
{
    Span s;
    s.ql = p.Lq; s.kl = p.Lk;
    if (p.q_lens) s.ql = max(0, min(p.Lq, p.q_lens[b]));
    if (p.k_lens) s.kl = max(0, min(p.Lk, p.k_lens[b]));
    s.off = s.kl - s.ql;
    s.R = s.ql * p.G;
    const int i0 = p.by_G(r0), i1 = p.by_G(max(0, min(r0 + rows, s.R) - 1));
    const int hi = p.right < 0 ? s.kl : max(0, min(s.kl, i1 + s.off + p.right + 1));
    const int lo = p.left < 0 ? 0 : max(0, i0 + s.off - p.left);
    s.sinks = p.sinks;
    s.shift = max(0, lo - p.sinks);                          // (> 0: every row sees all of the first keys)
    s.t_all = (max(0, hi - s.shift) + BN - 1) / BN;
    return s;
}

// the value of the lane 32 away
__device__ __forceinline__ float other_half(float v)
{
    typedef unsigned u2 __attribute__((ext_vector_type(2)));
    const unsigned x = __builtin_bit_cast(unsigned, v);
    const u2 r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    return __builtin_bit_cast(float, (threadIdx.x & 32) ? r[0] : r[1]);
}

// The state of a wave's 32 rows and what one tile of 64 keys in LDS does to it.  K rows lie at chunk c ^ kswz(key), V rows at
// c ^ vswz(key): the lanes of one LDS access then meet different banks.
//
// The reference value m of a row is a maximum that may lag: m follows only when a score exceeds it by more than 2^8 would allow -- rows of like scores
// rescale O once instead of every few tiles.  O and l belong to the same mb at all times: whatever rescales or joins them takes over_of into
// account, as m c alone is 1e-5 of a weight away from mb where scores are in the hundreds.
//
// NP = 3 (f32 tiles): every operand is the sum of three bf16 numbers, a = a0 + a1 + a2 (8 + 8 + 8 bits, each the nearest to what is left: all 24 bits
// are there).  Six of the nine products are multiplied, the smallest first; the three that are left out are at most 2^-24 of |a b|, the
// rounding of one f32 product, and mostly far less.  Six bf16 matrix instructions take 3/8 of the time of the f32 ones they stand for, and the vector
// unit works beside them, which it does not beside f32 ones: 524 -> 352 us for two clouds of 5000 keypoints, 8 heads of 32.  Infinities leave
// the planes as NaN; a wave whose O is not all numbers redoes its rows in plain f32 (exact_rows).
template <class T, int DP, int NP = 1>
struct Rows {
    static constexpr int CH = BxElem<T>::CH, CPR = DP / CH, ND = DP / 32;
    static constexpr float BIAS = NP == 3 ? bias_of<float>() : bias_of<T>();
    bxf16 o[ND];
    bxi4 fq[NP][CPR / 2];
    float m, mb, l;                                          // m: -inf before the first score
    bool edge;                                               // of the wave
    int lane, lr, h;

    // 16 keys of the same chunk (one cycle of a 16-byte access), and 4 keys of 64 bytes (one cycle of the transposing one), each cover
    // the 64 banks
    static __device__ __forceinline__ int kswz(int key) { return CPR == 4 ? key >> 2 & 3 : CPR == 8 ? key >> 1 & 7 : CPR == 16 ? key & 15 : key & 7; }
    static __device__ __forceinline__ int vswz(int key) { return sizeof(T) == 4 || CPR == 4 ? 0 : CPR == 8 ? (key >> 1 & 1) << 2 : (key & 3) << 2; }

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
        m = -INFINITY;
        mb = -BIAS;
        l = 0.0f;
        edge = false;
    }

    // LDS addresses, in bytes from the tile's start.  The swizzles are XORs of address bits below a row, so that the chunks of a row are a
    // few lane values away from constant offsets.
    static constexpr int ROW = DP * (int)sizeof(T);
    int k_at, v_at;                                          // set by init
    __device__ __forceinline__ bxi4 kfrag(const bxi4* sk, int k2, int c) const
    {
        constexpr int M = CPR == 4 ? 1 : CPR == 16 ? 7 : 3;
        return *(const bxi4*)((const char*)sk + (k_at ^ ((c & M) * 32)) + (c & ~M) * 32 + k2 * 32 * ROW);
    }
    // V^T operand of 16 keys (halves), in the order of S^T's registers
    __device__ __forceinline__ bxi4 vfrag(const bxi4* sv, int t, int u) const
    {
        typedef short s4 __attribute__((ext_vector_type(4)));
        bxi4 f;
#pragma unroll
        for (int g = 0; g < 2; ++g) {
            const char* a = (const char*)sv + (v_at ^ (t * 64)) + (16 * u + 8 * g) * ROW;
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

    // the weights as second operands: registers of S^T as they are (f32), or as the sum of two (halves) or three (f32 by planes) numbers of the
    // operand's type, each the nearest to what the ones before it left.  Two hold 16 bits of bf16 weights and 22 of f16 ones; one alone loses as
    // much as the result's own rounding does (2-norm against 64 bits 2.28e-3 where rounding the result alone is 1.65e-3: 32768 positions of 16 / 4
    // heads of 128, bf16, causal window of 1024 + 4).  The second product costs that case 328 -> 438 us, 1500 x 140 positions of 2 / 1 heads of
    // 32, f16, a band of 49 + 1 32 -> 36 us, one query over 8192 keys 18.2 -> 18.9.
    static constexpr int WP = NP == 3 ? 3 : 2;
    struct Weights { bxf16 s[sizeof(T) == 4 ? 2 : 1]; bxi4 f[WP][sizeof(T) == 4 ? 1 : 4]; };
    static constexpr int PLANE = BN * CPR;                   // chunks of a plane of K or V in LDS

    static __device__ __forceinline__ bxf16 mma_planes(const bxi4* a, bxi4 b0, bxi4 b1, bxi4 b2, bxf16 acc)
    {
        acc = bx_mma32<T>(a[2], b0, acc);
        acc = bx_mma32<T>(a[0], b2, acc);
        acc = bx_mma32<T>(a[1], b1, acc);
        acc = bx_mma32<T>(a[1], b0, acc);
        acc = bx_mma32<T>(a[0], b1, acc);
        return bx_mma32<T>(a[0], b0, acc);
    }

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
            for (int u = 0; u < 4; ++u) {
                if constexpr (NP == 1) {
                    const bxi4 v = vfrag(sv, t, u);
                    acc = bx_mma32<T>(v, w.f[1][u], acc);
                    acc = bx_mma32<T>(v, w.f[0][u], acc);
                }
                else {
                    bxi4 v[NP];
#pragma unroll
                    for (int n = 0; n < NP; ++n) v[n] = vfrag(sv + n * PLANE, t, u);
                    acc = mma_planes(v, w.f[0][u], w.f[1][u], w.f[2][u], acc);
                }
            }
        }
        return acc;
    }

    // S^T of a tile: key(n, k2, c) is the operand of K for chunk pair c of block k2 (of plane n)
    struct Scores { bxf16 s[2]; };
    template <class Key> __device__ __forceinline__ void score(const Key& key, Scores& x) const
    {
#pragma unroll
        for (int k2 = 0; k2 < 2; ++k2) {
#pragma unroll
            for (int i = 0; i < 16; ++i) x.s[k2][i] = 0.0f;
#pragma unroll
            for (int c2 = 0; c2 < CPR / 2; ++c2) {
                if constexpr (NP == 1) x.s[k2] = bx_mma32<T>(key(0, k2, c2), fq[0][c2], x.s[k2]);
                else {
                    bxi4 k[NP];
#pragma unroll
                    for (int n = 0; n < NP; ++n) k[n] = key(n, k2, c2);
                    x.s[k2] = mma_planes(k, fq[0][c2], fq[1][c2], fq[2][c2], x.s[k2]);
                }
            }
        }
    }
    // a tile on the edge of the mask: this lane's row sees the keys [lo, hi) and those before sink, counted from the lane's first key.  Away
    // from the first keys one unsigned comparison tells.
    __device__ __forceinline__ void hide(Scores& x, int lo, int hi, int sink, bool first)
    {
        edge = true;
        if (first) {
#pragma unroll
            for (int k2 = 0; k2 < 2; ++k2)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int j = 32 * k2 + 8 * (i / 4) + i % 4;
                    x.s[k2][i] = j < hi && (j >= lo || j < sink) ? x.s[k2][i] : -INFINITY;
                }
        } else {
            lo = max(lo, -(1 << 20));                        // the distances below stay inside 32 bits
            const unsigned n = (unsigned)max(0, min(hi, 1 << 20) - lo);
#pragma unroll
            for (int k2 = 0; k2 < 2; ++k2)
#pragma unroll
                for (int i = 0; i < 16; ++i) x.s[k2][i] = (unsigned)(32 * k2 + 8 * (i / 4) + i % 4 - lo) < n ? x.s[k2][i] : -INFINITY;
        }
    }
    // the rows' reference values follow where the tile's scores are too far above them -- each row by its own scores, so that its roundings do not
    // go by keys that only the wave's other rows see
    __device__ __forceinline__ void settle(const Scores& x, float c, float slack)
    {
        float mx = x.s[0][0];
#pragma unroll
        for (int k2 = 0; k2 < 2; ++k2)
#pragma unroll
            for (int i = 0; i < 16; ++i) mx = fmaxf(mx, x.s[k2][i]);
        mx = fmaxf(mx, other_half(mx));
        const bool up = mx > m + slack;
        if (__any(up)) {
            const float to = up ? fmaf(mx, c, -BIAS) : mb;
            if (__any(up && fabsf(to) >= STEEP && fabsf(mx) < INFINITY)) { edge = true; o[0][0] = NAN; }      // (for spoilt)
            const float alpha = !up ? 1.0f : m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mb - to);
            m = up ? mx : m;
            mb = to;
            l *= alpha;
#pragma unroll
            for (int t = 0; t < ND; ++t)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[t][i] *= alpha;
        }
    }
    // the weights, and their sum
    __device__ __forceinline__ void weights(Scores& x, float c, Weights& w)
    {
#pragma unroll
        for (int k2 = 0; k2 < 2; ++k2)
#pragma unroll
            for (int i = 0; i < 16; ++i) x.s[k2][i] = __builtin_amdgcn_exp2f(fmaf(x.s[k2][i], c, -mb));
        float sum = 0.0f;
#pragma unroll
        for (int k2 = 0; k2 < 2; ++k2)
#pragma unroll
            for (int i = 0; i < 16; ++i) sum += x.s[k2][i];
        l += sum;
        if constexpr (sizeof(T) == 4) { w.s[0] = x.s[0]; w.s[1] = x.s[1]; }
        else {
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                float e[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) e[j] = x.s[u / 2][8 * (u % 2) + j];
                if constexpr (NP == 3) bx_planes(e, w.f[0][u], w.f[1][u], w.f[2][u]);
                else {
                    // (in pairs: two numbers are rounded by one instruction, and widened again from what it leaves)
                    typedef T t2 __attribute__((ext_vector_type(2)));
                    t2 hi[4], lo[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        unsigned pair = __builtin_bit_cast(unsigned, (t2){(T)e[2 * j], (T)e[2 * j + 1]});
                        asm("" : "+v"(pair));
                        hi[j] = __builtin_bit_cast(t2, pair);
                        lo[j] = (t2){(T)(e[2 * j] - (float)hi[j][0]), (T)(e[2 * j + 1] - (float)hi[j][1])};
                    }
                    __builtin_memcpy(&w.f[0][u], hi, 16);
                    __builtin_memcpy(&w.f[1][u], lo, 16);
                }
            }
        }
    }
    __device__ __forceinline__ void add(const bxi4* sv, const Weights& w)
    {
#pragma unroll
        for (int t = 0; t < ND; ++t) {
            if constexpr (sizeof(T) == 4 || NP == 3) {
                // f32 sums a tile by itself first: fewer roundings at the size of O
                bxf16 a;
#pragma unroll
                for (int i = 0; i < 16; ++i) a[i] = 0.0f;
                a = weigh(sv, w, t, a);
#pragma unroll
                for (int i = 0; i < 16; ++i) o[t][i] += a[i];
            } else o[t] = weigh(sv, w, t, o[t]);
        }
    }
    // Whether a wave's rows have to be summed again (exact_rows): it met the edge of a mask and has anything but numbers in O -- 0 times an infinity
    // or NaN of a key that a row does not see would be in it --, or its scores were too steep, which has put a NaN there.
    __device__ __forceinline__ bool spoilt() const
    {
        float z = 0.0f;
#pragma unroll
        for (int t = 0; t < ND; ++t)
#pragma unroll
            for (int i = 0; i < 16; ++i) z = fmaf(o[t][i], 0.0f, z);
        return (edge || NP == 3) && __any(z != z);
    }
};

// The rows [r0, r1) over the key tiles [t0, t1), one row after the other by the whole wave, in plain f32 and touching nothing but what a row sees:
// the way of waves that met an infinity or NaN at the edge of a mask or scores of 2^22, and of few rows over few keys (attn_short_kernel).  Lanes are keys
// for the scores and dimensions for the sums.  The weights are 2^((s - m) c + over).
template <class T>
__device__ __forceinline__ void exact_rows(const AttnK& p, const Span& sp, const T* kb, const T* vb, int b, int hk, int r0, int r1, int lane, int t0, int t1,
                                           int DP, long long part, long long rows)
{
    constexpr int CH = BxElem<T>::CH;
    for (int r = r0; r < min(r1, sp.R); ++r) {
        const int qi = p.by_G(r), qg = r - qi * p.G;
        const int hi = (p.right < 0 ? sp.kl : min(sp.kl, qi + sp.off + p.right + 1)) - sp.shift, lo = p.left < 0 ? 0 : qi + sp.off - p.left - sp.shift;
        const T* q = (const T*)p.q + (long long)b * p.q_sb + (long long)qi * p.q_st + (long long)(hk * p.G + qg) * p.q_sh;
        float m = -INFINITY, over = 0.0f, l = 0.0f, o0 = 0.0f, o1 = 0.0f;
        for (int t = t0; t < t1; ++t) {
            const int j0 = t * BN, j = j0 + lane;
            const bool see = j < hi && (j >= lo || j < p.sinks);
            const unsigned long long seen = __ballot(see);
            if (!seen) continue;
            const T* k = kb + (long long)min(sp.key_of(j), sp.kl - 1) * p.k_st;
            float s = 0.0f;
            int d = 0;
#pragma unroll 4
            for (; d + CH <= p.D; d += CH) {
                T x[CH], y[CH];
                const bxi4 cx = bx_load_whole<T>(q, d), cy = bx_load_whole<T>(k, d);
                __builtin_memcpy(x, &cx, 16);
                __builtin_memcpy(y, &cy, 16);
#pragma unroll
                for (int i = 0; i < CH; ++i) s = fmaf((float)x[i], (float)y[i], s);
            }
            for (; d < p.D; ++d) s = fmaf((float)q[d], (float)k[d], s);
            float mx = see ? s : -INFINITY;
#pragma unroll
            for (int x = 32; x >= 1; x >>= 1) mx = fmaxf(mx, __shfl_xor(mx, x, 64));
            mx = fmaxf(m, mx);
            const float over_to = over_of<T>(mx, p.c);
            const float alpha = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(fmaf(m - mx, p.c, over_to - over));
            // (rows without a score yet: 2^-inf = 0 whatever is subtracted, and a NaN stays one)
            const float w = see ? __builtin_amdgcn_exp2f(fmaf(mx == -INFINITY ? s : s - mx, p.c, over_to)) : 0.0f;
            m = mx; over = over_to;
            l = fmaf(l, alpha, bx_wave_sum(w));
            o0 *= alpha; o1 *= alpha;
            for (int x0 = 0; x0 < 64; x0 += 8) {
                const unsigned some = (unsigned)(seen >> x0) & 255u;
                if (!some) continue;
                float v0[8], v1[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const T* v = vb + (long long)min(sp.key_of(j0 + x0 + i), sp.kl - 1) * p.v_st;
                    v0[i] = lane < p.D ? (float)v[lane] : 0.0f;
                    v1[i] = lane + 64 < p.D ? (float)v[lane + 64] : 0.0f;
                }
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float wx = __shfl(w, x0 + i, 64);
                    if (some >> i & 1) { o0 = fmaf(wx, v0[i], o0); o1 = fmaf(wx, v1[i], o1); }
                }
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

// Few f32 rows over a tile of keys: a wave per row.  The matrix instructions would multiply 32 rows of 64 keys whatever is there, in 14 000
// cycles: 773 x 4 x 3 rows of 128 over one key 220 -> 25 us, 4 x 3 rows of 128 over 38 keys 20 -> 9 us, 192 x 3 x 18 rows of 128 over 6 keys 56 -> 30
// us; but 1000 x 32 rows of 32 over 16 keys 16 -> 44 us, hence the rule in shape_of.  (Halves, sixteen times as fast there, lose by it.)
__global__ __launch_bounds__(256) void attn_short_kernel(AttnK p)
{
    using T = float;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int id = blockIdx.x;
    int up = p.by_tiles(id);
    const int r = (id - up * p.tiles_r) * 4 + wave; id = up;
    const int b = p.by_Hk(id), hk = id - b * p.Hk;
    const Span sp = span_of(p, b, r, 1);
    if (r >= sp.R) return;
    const T* kb = (const T*)p.k + (long long)b * p.k_sb + (long long)hk * p.k_sh;
    const T* vb = (const T*)p.v + (long long)b * p.v_sb + (long long)hk * p.v_sh;
    exact_rows<T>(p, sp, kb, vb, b, hk, r, r + 1, lane, 0, sp.t_all, 0, 0, 0);
}

template <class T> struct Halves { using type = T; };
template <> struct Halves<float> { using type = bx_bf16; };

// elements [k, k + 8) of a row of n floats
__device__ __forceinline__ void load8(const float* __restrict__ row, int k, int n, float* e)
{
    const bxi4 a = bx_load_chunk<float>(row, k, n), b = bx_load_chunk<float>(row, k + 4, n);
    __builtin_memcpy(e, &a, 16);
    __builtin_memcpy(e + 4, &b, 16);
}

constexpr int waves_of(int bytes, int DP, bool direct)
{
    if (bytes == 4) return DP == 32 ? 3 : DP == 64 ? 2 : 1;
    return DP == 128 ? 2 : (DP == 32 ? 4 : 3) - (direct ? 0 : 1);            // as many as fit without spills
}
template <class T, int DP, int NW, bool DIRECT>
__global__ __launch_bounds__(NW * 64, waves_of(sizeof(T), DP, DIRECT)) void attn_kernel(AttnK p)
{
    constexpr bool F32 = sizeof(T) == 4;
    static_assert(!(F32 && DIRECT), "f32 is taken apart on its way into LDS");
    constexpr int CH = 8, CPR = DP / CH, NT = NW * 64, LD = BN * CPR / NT;   // chunks as they lie in LDS: 8 halves
    static_assert(BN * CPR % NT == 0, "every thread stages the same number of chunks");
    using R_ = Rows<typename Halves<T>::type, DP, F32 ? 3 : 1>;
    __shared__ bxi4 sk0[(F32 ? 3 : 1) * BN * CPR], sv0[(F32 ? 3 : 1) * BN * CPR], sk1[DIRECT ? BN * CPR : 1], sv1[DIRECT ? BN * CPR : 1];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    int id = (int)bx_xcd_order<16>(blockIdx.x, gridDim.x), up = p.by_nsplit(id);
    const int split = id - up * p.nsplit; id = up; up = p.by_tiles(id);
    const int tile = p.tiles_r - 1 - (id - up * p.tiles_r); id = up;        // the rows that see most first, where the window has no left end
    const int b = p.by_Hk(id), hk = id - b * p.Hk;
    const int r0 = tile * NW * 32;
    const Span sp = span_of(p, b, r0, NW * 32);
    if (r0 >= sp.R) return;

    const int per = p.by_nsplit(sp.t_all + p.nsplit - 1);
    const int t0 = min(sp.t_all, split * per), t1 = min(sp.t_all, t0 + per);

    const T* kb = (const T*)p.k + (long long)b * p.k_sb + (long long)hk * p.k_sh;
    const T* vb = (const T*)p.v + (long long)b * p.v_sb + (long long)hk * p.v_sh;

    // this lane's row, and the first and last row of the wave
    R_ w;
    w.init(lane);
    const int h = w.h, w0 = r0 + wave * 32, r = w0 + w.lr;
    const bool live = r < sp.R, wave_live = w0 < sp.R;
    const int row = live ? r : sp.R - 1, qi = p.by_G(row), qg = row - qi * p.G;
    const int wi0 = p.by_G(w0), wi1 = p.by_G(min(w0 + 32, sp.R) - 1);
    const auto hi_of = [&](int i) { return (p.right < 0 ? sp.kl : min(sp.kl, i + sp.off + p.right + 1)) - sp.shift; };
    const auto lo_of = [&](int i) { return p.left < 0 ? 0 : i + sp.off - p.left - sp.shift; };
    const int hi = live ? hi_of(qi) : 0, lo = lo_of(qi);
    const int w_hi0 = wave_live ? hi_of(wi0) : 0, w_hi1 = hi_of(wi1), w_lo0 = lo_of(wi0), w_lo1 = lo_of(wi1);
    {
        const T* qr = (const T*)p.q + (long long)b * p.q_sb + (long long)qi * p.q_st + (long long)(hk * p.G + qg) * p.q_sh;
#pragma unroll
        for (int c = 0; c < CPR / 2; ++c) {
            if constexpr (F32) {
                float e[8];
                load8(qr, (2 * c + h) * CH, p.D, e);
                bx_planes(e, w.fq[0][c], w.fq[1][c], w.fq[2][c]);
            } else w.fq[0][c] = bx_load_chunk<T>(qr, (2 * c + h) * CH, p.D);
        }
    }
    const float slack = 8.0f / p.c;

    const auto hide = [&](typename R_::Scores& x, int t) __attribute__((always_inline)) {
        const int j0 = t * BN;
        // (no branch within the test: where two paths of different length meet behind the products, the compiler leaves too few wait states for
        // their last results; tests/test_mfma_waits.py)
        if ((j0 + BN <= w_hi0) & ((j0 >= w_lo1) | (j0 + BN <= p.sinks))) return;
        w.hide(x, lo - j0 - 4 * h, hi - j0 - 4 * h, p.sinks - j0 - 4 * h, j0 < p.sinks);
    };
    const auto unseen = [&](int t) { const int j0 = t * BN; return !wave_live || j0 >= w_hi1 || (j0 + BN <= w_lo0 && j0 >= p.sinks); };

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
        static_assert(STEP % (CPR == 32 ? 8 : 16) == 0, "the swizzle of a thread's chunks does not depend on the key's step");
        const int key0 = tid / CPR, ck = ((tid % CPR) ^ R_::kswz(key0)) * CH, cv = ((tid % CPR) ^ R_::vswz(key0)) * CH;
        const int wk = p.D < DP ? p.D : DP;
        const unsigned ks = (unsigned)(p.k_st * sizeof(T)), vs = (unsigned)(p.v_st * sizeof(T));
        const unsigned ko = key0 * ks + ck * (unsigned)sizeof(T), vo = key0 * vs + cv * (unsigned)sizeof(T);
        const auto load = [&](const T* base, long long st, unsigned bytes, unsigned off, int c, bxi4* to, int t) __attribute__((always_inline)) {
            const int x0 = t * BN, j0 = sp.key_of(x0);
            if (c < wk) {
                if (j0 + BN <= sp.kl && sp.key_of(x0 + BN - 1) == j0 + BN - 1) {
                    const char* first = (const char*)(base + (long long)j0 * st);
#pragma unroll
                    for (int i = 0; i < LD; ++i) bx_load_lds16(first + ((unsigned)(i * STEP) * bytes + off), to + (i * NW + wave) * 64);
                } else {
#pragma unroll
                    for (int i = 0; i < LD; ++i) bx_load_lds16(base + ((long long)min(sp.key_of(x0 + key0 + i * STEP), sp.kl - 1) * st + c), to + (i * NW + wave) * 64);
                }
            }
        };
        const auto load_k = [&](int t) __attribute__((always_inline)) { load(kb, p.k_st, ks, ko, ck, (t - t0) & 1 ? sk1 : sk0, t); };
        const auto load_v = [&](int t) __attribute__((always_inline)) { load(vb, p.v_st, vs, vo, cv, (t - t0) & 1 ? sv1 : sv0, t); };
        const auto score = [&](typename R_::Scores& x, int t) __attribute__((always_inline)) {
            const bxi4* sk = (t - t0) & 1 ? sk1 : sk0;
            w.score([&](int, int k2, int c) { return w.kfrag(sk, k2, c); }, x);
        };
        if constexpr (DP == 128) {
            // One step: the weights of tile t (the vector unit) while the scores of tile t + 1 are multiplied (the matrix unit), then the sums
            // of tile t.  K runs one tile ahead of V, and both are loaded one step before they are read.
            const auto step = [&](typename R_::Scores& now, typename R_::Scores& next, int t) __attribute__((always_inline)) {
                bx_sync_landed();
                if (t + 2 < t1) load_k(t + 2);
                load_v(t + 1);
                typename R_::Weights u;
                score(next, t + 1);
                w.weights(now, p.c, u);
                w.add((t - t0) & 1 ? sv1 : sv0, u);
                hide(next, t + 1);
                w.settle(next, p.c, slack);
            };
            const auto finish = [&](typename R_::Scores& now) __attribute__((always_inline)) {
                bx_sync_landed();
                typename R_::Weights u;
                w.weights(now, p.c, u);
                w.add((t1 - 1 - t0) & 1 ? sv1 : sv0, u);
            };
            if (t0 < t1) {
                typename R_::Scores a, b2;
                load_k(t0);
                bx_sync_landed();
                if (t0 + 1 < t1) load_k(t0 + 1);
                load_v(t0);
                score(a, t0);
                hide(a, t0);
                w.settle(a, p.c, slack);
                int t = t0;
                for (; t + 2 < t1; t += 2) {
                    step(a, b2, t);
                    step(b2, a, t + 1);
                }
                if (t + 1 < t1) {
                    step(a, b2, t);
                    finish(b2);
                } else finish(a);
            }
        } else {
            // small heads: the vector unit has most of the work, and waves that do not see a tile leave it out
            if (t0 < t1) { load_k(t0); load_v(t0); }
            for (int t = t0; t < t1; ++t) {
                bx_sync_landed();
                if (t + 1 < t1) { load_k(t + 1); load_v(t + 1); }
                if (unseen(t)) continue;
                typename R_::Scores x;
                typename R_::Weights u;
                score(x, t);
                hide(x, t);
                w.settle(x, p.c, slack);
                w.weights(x, p.c, u);
                w.add((t - t0) & 1 ? sv1 : sv0, u);
            }
        }
    } else {
        // through registers: keys behind the sequence become zeros, f32 comes apart into its planes
        constexpr int RW = F32 ? 2 : 1;
        bxi4 rk[LD][RW], rv[LD][RW];
        const auto fetch = [&](int t) {
            const int x0 = t * BN;
            const auto rows = [&](const auto& load) __attribute__((always_inline)) {
#pragma unroll
                for (int i = 0; i < LD; ++i) {
                    const int e = tid + i * NT, key = sp.key_of(x0 + e / CPR), d = e % CPR * CH;
#pragma unroll
                    for (int j = 0; j < RW; ++j) {
                        rk[i][j] = rv[i][j] = (bxi4){0, 0, 0, 0};
                        if (key < sp.kl) {
                            rk[i][j] = load(kb + (long long)key * p.k_st, d + j * BxElem<T>::CH);
                            rv[i][j] = load(vb + (long long)key * p.v_st, d + j * BxElem<T>::CH);
                        }
                    }
                }
            };
            if (p.D == DP) rows([&](const T* row, int k) { return bx_load_whole<T>(row, k); });
            else if (p.D % BxElem<T>::CH == 0) rows([&](const T* row, int k) { return k < p.D ? bx_load_whole<T>(row, k) : (bxi4){0, 0, 0, 0}; });
            else rows([&](const T* row, int k) { return bx_load_chunk<T>(row, k, p.D); });
        };
        const auto put = [&](bxi4* to, const bxi4* r) {
            if constexpr (F32) {
                float e[8];
                __builtin_memcpy(e, r, 32);
                bx_planes(e, to[0], to[R_::PLANE], to[2 * R_::PLANE]);
            } else *to = *r;
        };
        if (t0 < t1) fetch(t0);
        for (int t = t0; t < t1; ++t) {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < LD; ++i) {
                const int e = tid + i * NT, key = e / CPR, c = e % CPR;
                put(&sk0[key * CPR + (c ^ R_::kswz(key))], rk[i]);
                put(&sv0[key * CPR + (c ^ R_::vswz(key))], rv[i]);
            }
            __syncthreads();
            if (t + 1 < t1) fetch(t + 1);
            if (unseen(t)) continue;
            typename R_::Scores x;
            typename R_::Weights u;
            w.score([&](int n, int k2, int c) { return w.kfrag(sk0 + n * R_::PLANE, k2, c); }, x);
            hide(x, t);
            w.settle(x, p.c, slack);
            w.weights(x, p.c, u);
            w.add(sv0, u);
        }
    }

    const long long rows = (long long)p.B * p.Hk * p.Lq * p.G, part = (long long)split * rows + (long long)(b * p.Hk + hk) * p.Lq * p.G;
    if (w.spoilt()) {
        exact_rows<T>(p, sp, kb, vb, b, hk, w0, w0 + 32, lane, t0, t1, DP, part, rows);
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

// Up to 32 rows (single tokens and their like): the waves of a workgroup take the key tiles in turn instead of the rows, each on its own -- K straight
// into the registers of the matrix instruction, V into the wave's piece of LDS -- and meet at the end.  Bound by memory: every wave has its
// 64 keys of K and V in flight at once.
template <class T, int DP>
__global__ __launch_bounds__(256, 2) void attn_rows_kernel(AttnK p)
{
    constexpr int CH = BxElem<T>::CH, CPR = DP / CH, NW = 4, LD = BN * CPR / 64;
    using R_ = Rows<T, DP>;
    __shared__ bxi4 sv_all[NW][BN * CPR];
    __shared__ float sm[NW][32], sl[NW][32];
    static_assert(BN * CPR * 16 >= 32 * DP * 4, "a wave's V holds its O");
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int id = p.by_nsplit(blockIdx.x), split = blockIdx.x - id * p.nsplit;
    const int b = p.by_Hk(id), hk = id - b * p.Hk;
    const Span sp = span_of(p, b, 0, 32);
    if (sp.R <= 0) return;
    const int per = p.by_nsplit(sp.t_all + p.nsplit - 1);
    const int t0 = min(sp.t_all, split * per), t1 = min(sp.t_all, t0 + per);
    const T* kb = (const T*)p.k + (long long)b * p.k_sb + (long long)hk * p.k_sh;
    const T* vb = (const T*)p.v + (long long)b * p.v_sb + (long long)hk * p.v_sh;
    bxi4* sv = sv_all[wave];

    R_ w;
    w.init(lane);
    const int h = w.h, lr = w.lr, row = min(lr, sp.R - 1), qi = p.by_G(row), qg = row - qi * p.G;
    const auto hi_of = [&](int i) { return (p.right < 0 ? sp.kl : min(sp.kl, i + sp.off + p.right + 1)) - sp.shift; };
    const auto lo_of = [&](int i) { return p.left < 0 ? 0 : i + sp.off - p.left - sp.shift; };
    const int hi = lr < sp.R ? hi_of(qi) : 0, lo = lo_of(qi), i1 = p.by_G(sp.R - 1);
    const int w_hi0 = hi_of(0), w_lo1 = lo_of(i1);
    {
        const T* qr = (const T*)p.q + (long long)b * p.q_sb + (long long)qi * p.q_st + (long long)(hk * p.G + qg) * p.q_sh;
#pragma unroll
        for (int c = 0; c < CPR / 2; ++c) w.fq[0][c] = bx_load_chunk<T>(qr, (2 * c + h) * CH, p.D);
    }
    const float slack = 8.0f / p.c;
    if (p.D < DP) {
        const bxi4 zero = {0, 0, 0, 0};
        for (int e = lane; e < BN * CPR; e += 64) sv[e] = zero;
    }
    for (int t = t0 + wave; t < t1; t += NW) {
        const int j0 = t * BN;
        // keys behind the sequence repeat its last one: no row sees them
        bxi4 fk[2][CPR / 2];
#pragma unroll
        for (int k2 = 0; k2 < 2; ++k2) {
            const T* kr = kb + (long long)min(sp.key_of(j0 + 32 * k2 + lr), sp.kl - 1) * p.k_st;
#pragma unroll
            for (int c = 0; c < CPR / 2; ++c) fk[k2][c] = bx_load_chunk<T>(kr, (2 * c + h) * CH, p.D);
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // the last tile's V has been read
#pragma unroll
        for (int i = 0; i < LD; ++i) {
            const int e = i * 64 + lane, key = e / CPR, cv = ((e % CPR) ^ R_::vswz(key)) * CH;
            const T* vr = vb + (long long)min(sp.key_of(j0 + key), sp.kl - 1) * p.v_st + cv;
            if (cv < p.D) bx_load_lds16(vr, sv + i * 64);
        }
        const bool masked = !(j0 + BN <= w_hi0 && (j0 >= w_lo1 || j0 + BN <= p.sinks)) || sp.R < 32;
        typename R_::Scores x;
        typename R_::Weights u;
        w.score([&](int, int k2, int c) { return fk[k2][c]; }, x);
        if (masked) w.hide(x, lo - j0 - 4 * h, hi - j0 - 4 * h, p.sinks - j0 - 4 * h, j0 < p.sinks);
        w.settle(x, p.c, slack);
        w.weights(x, p.c, u);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");     // this wave's V is there
        w.add(sv, u);
    }
    const long long rows = (long long)p.B * p.Hk * p.Lq * p.G, part = (long long)split * rows + (long long)(b * p.Hk + hk) * p.Lq * p.G;
    if (__syncthreads_or(w.spoilt())) {
        if (wave == 0) exact_rows<T>(p, sp, kb, vb, b, hk, 0, 32, lane, t0, t1, DP, part, rows);
        return;
    }
    // every wave lays its rows down in its piece of LDS; then four dimensions of a row a thread, the waves in their order
    float* so = (float*)sv;
#pragma unroll
    for (int t = 0; t < R_::ND; ++t)
#pragma unroll
        for (int g = 0; g < 4; ++g)
            *(bxf4*)&so[lr * DP + (32 * t + 8 * g + 4 * h ^ (lr & 7) * 4)] = (bxf4){w.o[t][4 * g], w.o[t][4 * g + 1], w.o[t][4 * g + 2], w.o[t][4 * g + 3]};
    const float l = w.l + other_half(w.l);
    if (h == 0) { sm[wave][lr] = w.m; sl[wave][lr] = l; }
    __syncthreads();
    for (int e = tid; e < sp.R * (DP / 4); e += 256) {
        const int r = e / (DP / 4), d = e % (DP / 4) * 4;
        if (d >= p.D && p.nsplit == 1) continue;
        const float m = fmaxf(fmaxf(sm[0][r], sm[1][r]), fmaxf(sm[2][r], sm[3][r]));
        const float from = m == -INFINITY ? 0.0f : m, over = over_of<T>(m, p.c);
        float l4 = 0.0f, v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int x = 0; x < NW; ++x) {
            const float f = __builtin_amdgcn_exp2f(fmaf(sm[x][r] - from, p.c, over - over_of<T>(sm[x][r], p.c)));
            const bxf4 o = *(const bxf4*)&((const float*)sv_all[x])[r * DP + (d ^ (r & 7) * 4)];
            l4 = fmaf(f, sl[x][r], l4);
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = fmaf(f, o[j], v[j]);
        }
        if (p.nsplit > 1) {
            *reinterpret_cast<bxf4*>(p.ws + (part + r) * DP + d) = (bxf4){v[0], v[1], v[2], v[3]};
            float* ml = p.ws + (long long)p.nsplit * rows * DP + (part + r) * 2;
            if (d == 0) { ml[0] = m; ml[1] = l4; }
        } else {
            const int oi = p.by_G(r), og = r - oi * p.G;
            const float inv = hi_of(oi) <= 0 ? 0.0f : 1.0f / l4;
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] *= inv;
            bx_store4<T>((T*)p.o + (long long)b * p.o_sb + (long long)oi * p.o_st + (long long)(hk * p.G + og) * p.o_sh + d, v, p.D - d);
        }
    }
}

// joins the parts of a row, each relative to its 2^(m c - over).  DP / 4 lanes have four dimensions each; SG groups of them share the splits of a row and add up
// in their order, so that a single token's many parts are read together instead of one after the other.
template <class T, int DP, int SG>
__global__ __launch_bounds__(256) void attn_join_kernel(AttnK p)
{
    constexpr int LPR = DP / 4, RPB = 256 / LPR / SG;
    __shared__ float sm[RPB][SG], sl[RPB][SG];
    __shared__ bxf4 so[RPB][SG][LPR];
    const long long rows = (long long)p.B * p.Hk * p.Lq * p.G;
    const int x = threadIdx.x % LPR, g = threadIdx.x / LPR % SG, rb = threadIdx.x / LPR / SG, d = x * 4;
    const long long at = (long long)blockIdx.x * RPB + rb;
    const int bh = p.by_rows((int)at), r = (int)at - bh * p.Lq * p.G, b = p.by_Hk(bh), hk = bh - b * p.Hk;    // (fewer than 2^30 rows)
    const int qi = p.by_G(r), qg = r - qi * p.G;
    const bool there = at < rows;
    const int ql = there && p.q_lens ? max(0, min(p.Lq, p.q_lens[b])) : p.Lq, kl = there && p.k_lens ? max(0, min(p.Lk, p.k_lens[b])) : p.Lk;
    const bool live = there && qi < ql;
    const float* ml = p.ws + (long long)p.nsplit * rows * DP;
    // one pass with a running maximum; four parts are on their way at a time
    float m = -INFINITY, l = 0.0f;
    bxf4 v = {0.f, 0.f, 0.f, 0.f};
    const auto take = [&](float ms, float over, float ls, const bxf4& o) {
        const float mn = fmaxf(m, ms), from = mn == -INFINITY ? 0.0f : mn;
        const float a = __builtin_amdgcn_exp2f((m - from) * p.c), w = __builtin_amdgcn_exp2f(fmaf(ms - from, p.c, -over));
        m = mn;
        l = fmaf(l, a, w * ls);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = fmaf(v[j], a, w * o[j]);
    };
    if (live) {
        for (int s0 = g; s0 < p.nsplit; s0 += 4 * SG) {
            float ms[4], ls[4];
            bxf4 o[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const long long i = (long long)min(s0 + j * SG, p.nsplit - 1) * rows + at;
                ms[j] = ml[i * 2]; ls[j] = ml[i * 2 + 1];
                o[j] = *reinterpret_cast<const bxf4*>(p.ws + i * DP + d);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (s0 + j * SG < p.nsplit) take(ms[j], over_of<T>(ms[j], p.c), ls[j], o[j]);
        }
    }
    if constexpr (SG > 1) {
        so[rb][g][x] = v;
        if (x == 0) { sm[rb][g] = m; sl[rb][g] = l; }
        __syncthreads();
        if (g > 0) return;
#pragma unroll
        for (int j = 1; j < SG; ++j) take(sm[rb][j], 0.0f, sl[rb][j], so[rb][j][x]);
    }
    if (!live || d >= p.D) return;
    const bool empty = p.right >= 0 && qi + kl - ql + p.right + 1 <= 0;
    const float inv = empty || kl <= 0 ? 0.0f : 1.0f / l;
    const float y[4] = {v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv};
    bx_store4<T>((T*)p.o + (long long)b * p.o_sb + (long long)qi * p.o_st + (long long)(hk * p.G + qg) * p.o_sh + d, y, p.D - d);
}

int padded(int D) { return D <= 32 ? 32 : D <= 64 ? 64 : 128; }

// waves of a workgroup (32 rows each).  Small heads of halves take two: their tiles are short work and rows come in few (1500 patches of 2 heads
// over 140 positions, f16, band of 24: 36 us, 38 by four waves, 46 by one); four share more of the staging of everything else (two clouds of 5000 keypoints,
// f32: 324 us, 425 by two).
constexpr int group_of(int bytes, int DP) { return bytes == 2 && DP == 32 ? 2 : 4; }

struct Shape { int DP, tiles_r, nsplit; bool rows, brief; };

// whether rows of 16-byte aligned whole chunks let K and V skip the registers
bool direct_of(const bx_attention_args& a)
{
    const int e = a.dtype == BX_TYPE_F32 ? 4 : 2;
    const auto al = [e](const void* p, long long x, long long y, long long z) { return (((uintptr_t)p | (uintptr_t)(x * e) | (uintptr_t)(y * e) | (uintptr_t)(z * e)) & 15) == 0; };
    const long long far = (1LL << 31) / (BN * e);            // rows further apart: a tile does not fit 32-bit offsets
    return a.D * e % 16 == 0 && a.k_stride_t < far && a.v_stride_t < far && al(a.q, a.q_stride_b, a.q_stride_t, a.q_stride_h) &&
           al(a.k, a.k_stride_b, a.k_stride_t, a.k_stride_h) && al(a.v, a.v_stride_b, a.v_stride_t, a.v_stride_h);
}

Shape shape_of(int n_cu, const bx_attention_args& a)
{
    Shape s;
    s.DP = padded(a.D);
    const long long R = (long long)a.Lq * (a.Hq / a.Hk);
    const bool few = R <= 32;                                // (the number of splits goes by the sizes alone: a workspace fits any alignment)
    s.rows = few && direct_of(a);
    s.tiles_r = (int)((R + 32 * group_of(a.dtype == BX_TYPE_F32 ? 4 : 2, s.DP) - 1) / (32 * group_of(a.dtype == BX_TYPE_F32 ? 4 : 2, s.DP)));
    const long long base = (long long)s.tiles_r * a.Hk * a.B;
    long long keys = a.Lk;
    if (a.left >= 0 && a.right >= 0) {
        const long long span = (long long)a.left + a.right + 1 + (R < 128 ? a.Lq : 128 / (a.Hq / a.Hk) + 1) + a.sinks;
        keys = span < keys ? span : keys;
    }
    const long long tiles = (keys + BN - 1) / BN;
    // Rows alone fill the card when every slot for a workgroup (by the waves that fit a SIMD) has one -- three where the mask is a triangle,
    // whose workgroups are of all lengths; with fewer the keys are split, as long as a part keeps eight tiles of 64 keys (four for up to
    // 32 rows, one per wave): below that joining costs more than it saves.
    const int bytes = a.dtype == BX_TYPE_F32 ? 4 : 2;
    const long long slots = (long long)n_cu * (few ? 2 : waves_of(bytes, s.DP, true) * 4 / group_of(bytes, s.DP));
    const long long want = a.left < 0 && a.right >= 0 && !few ? 3 * slots : slots;
    const int least = few ? 4 : 8;
    long long n = base > 0 ? want / base : 1;
    if (n > (tiles + least - 1) / least) n = (tiles + least - 1) / least;
    if (n > 128) n = 128;
    // A few workgroups a compute unit, unevenly: two halves even them out (two clouds of 5000 keypoints f32, 640 workgroups: 352 -> 323 us).
    if (n <= 1 && base < 4LL * n_cu && tiles >= 32) {
        const auto worst = [n_cu](long long g) { return (double)((g + n_cu - 1) / n_cu) * n_cu / (double)g; };
        if (worst(base) - worst(2 * base) > 0.12) n = 2;
    }
    s.nsplit = n < 1 ? 1 : (int)n;
    s.brief = few && bytes == 4 && tiles <= 1 && R * (16 + a.Lk) <= 4 * s.DP;
    if (s.brief) { s.nsplit = 1; s.tiles_r = (int)((R + 3) / 4); }
    return s;
}

int64_t bytes_of(const Shape& s, const bx_attention_args& a)
{
    if (s.nsplit <= 1) return 0;
    return (int64_t)s.nsplit * a.B * a.Lq * a.Hq * (s.DP + 2) * 4;
}

template <class T, int DP>
int launch(hipStream_t s, const AttnK& k, bool brief, bool rows_form, bool direct)
{
    constexpr int G = group_of(sizeof(T), DP);
    const unsigned grid = (unsigned)((long long)k.tiles_r * k.Hk * k.B * k.nsplit);
    if constexpr (sizeof(T) == 4) {
        if (brief) {
            attn_short_kernel<<<grid, 256, 0, s>>>(k);
            BX_LAUNCH_CHECK();
            return BX_OK;
        }
    }
    if (rows_form) attn_rows_kernel<T, DP><<<grid, 256, 0, s>>>(k);
    else if constexpr (sizeof(T) == 4) attn_kernel<T, DP, G, false><<<grid, G * 64, 0, s>>>(k);
    else if (direct) attn_kernel<T, DP, G, true><<<grid, G * 64, 0, s>>>(k);
    else attn_kernel<T, DP, G, false><<<grid, G * 64, 0, s>>>(k);
    BX_LAUNCH_CHECK();
    if (k.nsplit > 1) {
        constexpr int SG = 32 * 8 / (DP / 4) > 8 ? 8 : 32 * 8 / (DP / 4);
        const long long rows = (long long)k.B * k.Hk * k.Lq * k.G, whole = 256 / (DP / 4), shared = whole / SG;
        if (k.nsplit > 8) attn_join_kernel<T, DP, SG><<<(unsigned)((rows + shared - 1) / shared), 256, 0, s>>>(k);
        else attn_join_kernel<T, DP, 1><<<(unsigned)((rows + whole - 1) / whole), 256, 0, s>>>(k);
        BX_LAUNCH_CHECK();
    }
    return BX_OK;
}

template <class T>
int attention_of(hipStream_t s, int n_cu, const bx_attention_args& a)
{
    const Shape sh = shape_of(n_cu, a);
    const AttnK k = {a.q, a.k, a.v, a.o, a.q_lens, a.k_lens, (float*)a.workspace,
                     a.q_stride_b, a.q_stride_t, a.q_stride_h, a.k_stride_b, a.k_stride_t, a.k_stride_h,
                     a.v_stride_b, a.v_stride_t, a.v_stride_h, a.o_stride_b, a.o_stride_t, a.o_stride_h,
                     a.B, a.Lq, a.Lk, a.Hk, a.Hq / a.Hk, a.D, a.left, a.right, a.sinks, sh.nsplit, sh.tiles_r,
                     (float)((double)a.scale * 1.4426950408889634),
                     div_of(a.Hq / a.Hk), div_of(a.Hk), div_of(sh.nsplit), div_of(sh.tiles_r), div_of(a.Lq * (a.Hq / a.Hk))};
    const bool direct = direct_of(a);
    if (sh.DP == 32) return launch<T, 32>(s, k, sh.brief, sh.rows, direct);
    if (sh.DP == 64) return launch<T, 64>(s, k, sh.brief, sh.rows, direct);
    return launch<T, 128>(s, k, sh.brief, sh.rows, direct);
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
    // (joining has less than a workgroup per row)
    if (bx_grid_check("bx_attention", (long long)sh.tiles_r * a.Hk * a.B * sh.nsplit, 256) != BX_OK ||
        (sh.nsplit > 1 && bx_grid_check("bx_attention", (long long)a.B * a.Lq * a.Hq, 256) != BX_OK)) return BX_ERR_ARG;
    if (a.dtype == BX_TYPE_F32) return attention_of<float>(s, n_cu, a);
    if (a.dtype == BX_TYPE_F16) return attention_of<bx_f16>(s, n_cu, a);
    return attention_of<bx_bf16>(s, n_cu, a);
}
