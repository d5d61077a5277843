// k_linear.hip -- y = act(x W^T + b) + r, the dense layer over keypoints (bx_linear).  x [M][K], W [N][K], y [M][N]: the rows of both
// operands run along K, so both are staged as 128-byte slices of rows.  Sums are held in f32, the epilogue (bias, activation, residual)
// runs on the accumulators and the result is rounded once.
#include "bx_ops.h"

namespace {

// Both activations go by |v| and the power 2^(-..) of it, so nothing overflows and small results keep a relative precision.
//   silu: v s (v >= 0) or v h s h (v < 0),  h = exp(-|v| / 2), s = 1 / (1 + h^2): the power instruction ends at 2^-126, its square need not
//   gelu: v (1 - q) or v q,  q = Phi(-|v|) = exp(-v^2 / 2) t h(t),  t = 1 / (1 + 0.2625 |v|): h by the polynomial of degree 8 that fits
//         0.5 erfcx(|v| / sqrt 2) / t with the least relative error (3.4e-8 over 0 .. 14.5 with the coefficients as f32 has them; rounding v^2 in the
//         exponent adds up to v^2 2^-24 of q).  20 instruction slots, where erfc takes over 50: at 67 million outputs that is a third of the time
//         of the product itself.
template <int act> __device__ __forceinline__ float act_of(float v)
{
    if (act == BX_ACT_NONE) return v;
    if (act == BX_ACT_RELU) return v > 0.0f ? v : (v != v ? v : 0.0f);
    if (act == BX_ACT_SILU) {
        const float h = __builtin_amdgcn_exp2f(fabsf(v) * -0.72134752f), s = __builtin_amdgcn_rcpf(fmaf(h, h, 1.0f));
        return v >= 0.0f ? v * s : v * h * s * h;
    }
    const float t = __builtin_amdgcn_rcpf(fmaf(0.2625f, fabsf(v), 1.0f));
    float h = 0.0305265988f;
    h = fmaf(h, t, -0.147754029f);
    h = fmaf(h, t, 0.232594151f);
    h = fmaf(h, t, -0.130927997f);
    h = fmaf(h, t, 0.147445404f);
    h = fmaf(h, t, 0.056567913f);
    h = fmaf(h, t, 0.102634909f);
    h = fmaf(h, t, 0.104164678f);
    h = fmaf(h, t, 0.104748362f);
    const float q = h * t * __builtin_amdgcn_exp2f(v * v * -0.72134752f);
    return v * (v >= 0.0f ? 1.0f - q : q);
}

struct LinearK {
    const void *x, *w, *bias, *residual;
    void* y;
    const int32_t* m_dev;
    long long ldx, ldw, ldr, ldy;
    int M, N, K, act, tiles_n, tiles_m;
};

template <class T>
__device__ __forceinline__ void epilogue4(const LinearK& p, int m, int n, const float* acc)
{
    const int left = p.N - n;
    float v[4], b[4] = {0.f, 0.f, 0.f, 0.f};
    if (p.bias) bx_load4<T>((const T*)p.bias + n, b, left);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float x = acc[j] + b[j];
        v[j] = p.act == BX_ACT_RELU ? act_of<BX_ACT_RELU>(x) : p.act == BX_ACT_GELU ? act_of<BX_ACT_GELU>(x) : p.act == BX_ACT_SILU ? act_of<BX_ACT_SILU>(x) : x;
    }
    if (p.residual) {
        float r[4];
        bx_load4<T>((const T*)p.residual + (long long)m * p.ldr + n, r, left);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] += r[j];
    }
    bx_store4<T>((T*)p.y + (long long)m * p.ldy + n, v, left);
}

// CH consecutive columns (16 bytes) of one row of y, of which `left` exist
template <class T> __device__ __forceinline__ void load_piece(const T* __restrict__ p, float* v, int left)
{
    constexpr int CH = BxElem<T>::CH;
    T e[CH];
    if (left >= CH) { const bxi4 r = reinterpret_cast<const BxAny16*>(p)->v; __builtin_memcpy(e, &r, 16); }
    else {
#pragma unroll
        for (int j = 0; j < CH; ++j) e[j] = j < left ? p[j] : (T)0.0f;
    }
#pragma unroll
    for (int j = 0; j < CH; ++j) v[j] = (float)e[j];
}
template <class T, int ACT> __device__ __forceinline__ void finish_piece(const LinearK& p, int m, int n, float* v, const float* bias)
{
    constexpr int CH = BxElem<T>::CH;
    const int left = p.N - n;
#pragma unroll
    for (int j = 0; j < CH; ++j) v[j] = act_of<ACT>(v[j] + bias[j]);
    if (p.residual) {
        float r[CH];
        load_piece<T>((const T*)p.residual + (long long)m * p.ldr + n, r, left);
#pragma unroll
        for (int j = 0; j < CH; ++j) v[j] += r[j];
    }
    T e[CH];
#pragma unroll
    for (int j = 0; j < CH; ++j) e[j] = (T)v[j];
    T* y = (T*)p.y + (long long)m * p.ldy + n;
    if (left >= CH) { bxi4 r; __builtin_memcpy(&r, e, 16); reinterpret_cast<BxAny16*>(y)->v = r; }
    else {
#pragma unroll
        for (int j = 0; j < CH; ++j)
            if (j < left) y[j] = e[j];
    }
}

// A wave's part of y, from its accumulators (a lane holds 4 columns of a row here and there) to memory: 32 rows at a time are turned over in
// the wave's own piece of LDS, so that whole lanes in a row write 32 TN neighbouring columns.  Without it a store wrote 16 bytes
// of 32 rows each, and 16384 x 4096 bf16 outputs alone took 145 of the layer's 200 us.
template <class T, int TM, int TN, int ACT>
__device__ __forceinline__ void put_rows(const LinearK& p, bxf16 (&acc)[TN][TM], float* lds, int lane, int m0, int n0, int M)
{
    constexpr int CH = BxElem<T>::CH, W = TN * 32, LD = W + 4, LPR = W / CH, RPI = 64 / LPR;      // lanes of a row, rows of a pass
    const int lr = lane & 31, h = lane >> 5, c = lane % LPR * CH, n = n0 + c;
    float bias[CH];
#pragma unroll
    for (int j = 0; j < CH; ++j) bias[j] = 0.0f;
    if (p.bias && n < p.N) load_piece<T>((const T*)p.bias + n, bias, p.N - n);
#pragma unroll
    for (int b = 0; b < TM; ++b) {
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int a = 0; a < TN; ++a)
#pragma unroll
            for (int g = 0; g < 4; ++g)
                *(bxf4*)&lds[lr * LD + a * 32 + 8 * g + 4 * h] = (bxf4){acc[a][b][4 * g], acc[a][b][4 * g + 1], acc[a][b][4 * g + 2], acc[a][b][4 * g + 3]};
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int i = 0; i < 32 / RPI; ++i) {
            const int r = i * RPI + lane / LPR, m = m0 + b * 32 + r;
            float v[CH];
#pragma unroll
            for (int j = 0; j < CH; j += 4) {
                const bxf4 f = *(const bxf4*)&lds[r * LD + c + j];
                v[j] = f[0]; v[j + 1] = f[1]; v[j + 2] = f[2]; v[j + 3] = f[3];
            }
            if (m < M && n < p.N) finish_piece<T, ACT>(p, m, n, v, bias);
        }
    }
}

// One workgroup = a BM x BN tile of y; a wave holds a (BM / WGM) x (BN / WGN) part of it in 32 x 32 accumulators.  The matrix product is
// taken transposed (W rows as the first operand): a lane then holds four consecutive columns of one row of y and stores them together.
// A row slice of 128 bytes is 8 chunks in LDS; chunk c of row r sits at c ^ (r / 2 % 8), so that the 16 lanes that one cycle of LDS serves
// (consecutive rows, same chunk) meet all 64 banks.
//
// DIRECT: rows that are 16-byte aligned go from memory straight into LDS, one slice ahead of the products; what K leaves behind the last
// whole slice, and rows that are not aligned, go through registers, where the elements behind K become zeros.  Rows behind the
// last one repeat it: their products are not stored.
//
// KS > 1: so many groups of waves take the slices of K in turn, each with its own buffers, and meet in LDS at the end -- for outputs that are
// too few to fill the card with tiles, where a workgroup's time is that of its loads one after the other.
//
// ONE: sums of a single slice need one buffer, and more workgroups fit a compute unit.
template <class T, int BM, int BN, int WGM, int WGN, int KS, bool DIRECT, bool ONE>
__global__ __launch_bounds__(KS * WGM * WGN * 64) void linear_tile_kernel(LinearK p)
{
    constexpr int CH = BxElem<T>::CH, BK = 8 * CH, NW = WGM * WGN, NT = NW * 64;
    constexpr int TM = BM / WGM / 32, TN = BN / WGN / 32;
    constexpr int LX = BM * 8 / NT, LW = BN * 8 / NT;
    static_assert(NT % 128 == 0, "a thread's rows are a multiple of 16 apart: its chunks keep their place in a row");
    constexpr int PUT = NW * 32 * (TN * 32 + 4) / 4, SLICES = (ONE ? 1 : 2) * (BM + BN) * 8;
    __shared__ bxi4 lds[PUT > KS * SLICES ? PUT : KS * SLICES];
    const int group = KS > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x / NT) : 0;
    bxi4 *const sx0 = lds + group * SLICES, *const sw0 = sx0 + BM * 8, *const sx1 = ONE ? sx0 : sw0 + BN * 8, *const sw1 = ONE ? sw0 : sx1 + BM * 8;
    const int tid = threadIdx.x % NT, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    // tiles in groups of 8 rows of tiles, down the rows first: the tiles that an XCD works on at a time share rows of x and of W
    const int id = (int)bx_xcd_order<32>(blockIdx.x, gridDim.x), gsize = 8 * p.tiles_n, first = id / gsize * 8, gm = min(8, p.tiles_m - first);
    const int m0 = (first + id % gsize % gm) * BM, n0 = (id % gsize / gm) * BN;
    int M = p.M;
    if (p.m_dev) { const int live = *p.m_dev; M = live < M ? live : M; }
    if (m0 >= M) return;
    const T* x = (const T*)p.x + (long long)m0 * p.ldx;
    const T* w = (const T*)p.w + (long long)n0 * p.ldw;
    const int last_m = M - 1 - m0, last_n = p.N - 1 - n0;

    bxf16 acc[TN][TM];
#pragma unroll
    for (int a = 0; a < TN; ++a)
#pragma unroll
        for (int b = 0; b < TM; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[a][b][i] = 0.0f;

    const int wm = (wave / WGN) * TM * 32, wn = (wave % WGN) * TN * 32, lr = lane & 31, h = lane >> 5;
    // LDS addresses: the swizzle is an XOR of address bits below a row
    const int x_at = (wm + lr) * 128 + ((h ^ (lr >> 1 & 7)) * 16), w_at = (wn + lr) * 128 + ((h ^ (lr >> 1 & 7)) * 16);
    const auto multiply = [&](const bxi4* sx, const bxi4* sw, int pairs) __attribute__((always_inline)) {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            if (c >= pairs) break;
            bxi4 fx[TM], fw[TN];
#pragma unroll
            for (int b = 0; b < TM; ++b) fx[b] = *(const bxi4*)((const char*)sx + (x_at ^ (c * 32)) + b * 32 * 128);
#pragma unroll
            for (int a = 0; a < TN; ++a) fw[a] = *(const bxi4*)((const char*)sw + (w_at ^ (c * 32)) + a * 32 * 128);
#pragma unroll
            for (int a = 0; a < TN; ++a)
#pragma unroll
                for (int b = 0; b < TM; ++b) acc[a][b] = bx_mma32<T>(fw[a], fx[b], acc[a][b]);
        }
    };

    // a slice through registers
    bxi4 rx[LX], rw[LW];
    const auto fetch = [&](int k0) {
        const auto rows = [&](const auto& load) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < LX; ++i) {
                const int e = tid + i * NT;
                rx[i] = load(x + (long long)min(e >> 3, last_m) * p.ldx, k0 + (e & 7) * CH);
            }
#pragma unroll
            for (int i = 0; i < LW; ++i) {
                const int e = tid + i * NT;
                rw[i] = load(w + (long long)min(e >> 3, last_n) * p.ldw, k0 + (e & 7) * CH);
            }
        };
        if (k0 + BK <= p.K) rows([&](const T* row, int k) { return bx_load_whole<T>(row, k); });
        else rows([&](const T* row, int k) { return bx_load_chunk<T>(row, k, p.K); });
    };
    const auto stage = [&](bxi4* sx, bxi4* sw) {
#pragma unroll
        for (int i = 0; i < LX; ++i) { const int e = tid + i * NT, r = e >> 3; sx[r * 8 + ((e & 7) ^ (r >> 1 & 7))] = rx[i]; }
#pragma unroll
        for (int i = 0; i < LW; ++i) { const int e = tid + i * NT, r = e >> 3; sw[r * 8 + ((e & 7) ^ (r >> 1 & 7))] = rw[i]; }
    };

    if constexpr (DIRECT) {
        const int whole = p.K / BK;
        const int c0 = ((tid & 7) ^ (tid >> 4 & 7)) * 16;
        unsigned xo[LX], wo[LW];                             // the host sees to it that a tile's rows lie within 32 bits
#pragma unroll
        for (int i = 0; i < LX; ++i) xo[i] = (unsigned)min((tid + i * NT) >> 3, last_m) * (unsigned)(p.ldx * sizeof(T)) + c0;
#pragma unroll
        for (int i = 0; i < LW; ++i) wo[i] = (unsigned)min((tid + i * NT) >> 3, last_n) * (unsigned)(p.ldw * sizeof(T)) + c0;
        const auto load = [&](bxi4* sx, bxi4* sw, int s) __attribute__((always_inline)) {
            const char *xs = (const char*)x + (long long)s * 128, *ws = (const char*)w + (long long)s * 128;
#pragma unroll
            for (int i = 0; i < LX; ++i) bx_load_lds16(xs + xo[i], sx + i * NT + wave * 64);
#pragma unroll
            for (int i = 0; i < LW; ++i) bx_load_lds16(ws + wo[i], sw + i * NT + wave * 64);
        };
        if (group < whole) load(sx0, sw0, group);
        for (int s = group, i = 0; i < (whole + KS - 1) / KS; s += KS, ++i) {
            bx_sync_landed();
            const bool odd = i & 1;
            if (s + KS < whole) load(odd ? sx0 : sx1, odd ? sw0 : sw1, s + KS);
            if (KS == 1 || s < whole) multiply(odd ? sx1 : sx0, odd ? sw1 : sw0, 4);
        }
        if (whole * BK < p.K) {
            if (group == 0) fetch(whole * BK);
            __syncthreads();
            if (group == 0) stage(sx0, sw0);
            __syncthreads();
            if (group == 0) multiply(sx0, sw0, (p.K - whole * BK + 2 * CH - 1) / (2 * CH));
        }
    } else {
        const int steps = (p.K + BK - 1) / BK;
        if (group < steps) { fetch(group * BK); stage(sx0, sw0); }
        for (int s = group, i = 0; i < (steps + KS - 1) / KS; s += KS, ++i) {
            __syncthreads();
            const bool odd = i & 1;
            if (s + KS < steps) fetch((s + KS) * BK);
            if (KS == 1 || s < steps) multiply(odd ? sx1 : sx0, odd ? sw1 : sw0, ONE ? (p.K + 2 * CH - 1) / (2 * CH) : 4);
            if (s + KS < steps) stage(odd ? sx0 : sx1, odd ? sw0 : sw1);
        }
    }
    if constexpr (KS > 1) {
        // the groups' sums, added in their order
        constexpr int A = TN * TM * 4;
        static_assert((KS - 1) * NW * 64 * A <= KS * SLICES, "the groups' sums fit the buffers");
        __syncthreads();
        bxf4* sums = (bxf4*)lds;
        if (group > 0) {
#pragma unroll
            for (int j = 0; j < A; ++j) {
                const bxf16& f = acc[j / 4 / TM][j / 4 % TM];
                sums[(((group - 1) * NW + wave) * A + j) * 64 + lane] = (bxf4){f[j % 4 * 4], f[j % 4 * 4 + 1], f[j % 4 * 4 + 2], f[j % 4 * 4 + 3]};
            }
        }
        __syncthreads();
        if (group == 0) {
#pragma unroll 1
            for (int g = 0; g < KS - 1; ++g)
#pragma unroll
                for (int j = 0; j < A; ++j) {
                    bxf16& f = acc[j / 4 / TM][j / 4 % TM];
                    const bxf4 v = sums[((g * NW + wave) * A + j) * 64 + lane];
#pragma unroll
                    for (int i = 0; i < 4; ++i) f[j % 4 * 4 + i] += v[i];
                }
        }
        __syncthreads();
        if (group > 0) return;
    }

    if (KS == 1) __syncthreads();
    float* mine = (float*)lds + wave * 32 * (TN * 32 + 4);
    if (p.act == BX_ACT_NONE) put_rows<T, TM, TN, BX_ACT_NONE>(p, acc, mine, lane, m0 + wm, n0 + wn, M);
    else if (p.act == BX_ACT_RELU) put_rows<T, TM, TN, BX_ACT_RELU>(p, acc, mine, lane, m0 + wm, n0 + wn, M);
    else if (p.act == BX_ACT_GELU) put_rows<T, TM, TN, BX_ACT_GELU>(p, acc, mine, lane, m0 + wm, n0 + wn, M);
    else put_rows<T, TM, TN, BX_ACT_SILU>(p, acc, mine, lane, m0 + wm, n0 + wn, M);
}

// f32 by bf16 planes: every operand is the sum of three bf16 numbers, a = a0 + a1 + a2 (8 + 8 + 8 bits, each the nearest to what is left: all 24
// bits are there), taken apart on the way into LDS.  Six of the nine products are multiplied, the smallest first; the three left out are
// at most 2^-24 of |a b|, the rounding of one f32 product, and mostly far less (|a1| <= 2^-8 |a|, |a2| <= 2^-17 |a|).  The six bf16 matrix instructions take 3/8 of the time of the f32 ones.
// An infinity leaves the planes as NaN: results that are not finite are summed again, in plain f32.
template <int BM, int BN, int WGM, int WGN>
__global__ __launch_bounds__(WGM * WGN * 64) void linear_planes_kernel(LinearK p)
{
    using T = float;
    constexpr int NW = WGM * WGN, NT = NW * 64, BK = 32, TM = BM / WGM / 32, TN = BN / WGN / 32;
    constexpr int LX = BM * 4 / NT, LW = BN * 4 / NT, PX = BM * 4, PW = BN * 4, BUF = 3 * (PX + PW);      // pieces of 8 elements: a thread's, a plane's
    constexpr int PUT = NW * 32 * (TN * 32 + 4) / 4;
    __shared__ bxi4 lds[PUT > 2 * BUF ? PUT : 2 * BUF];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int id = (int)bx_xcd_order<32>(blockIdx.x, gridDim.x), gsize = 8 * p.tiles_n, first = id / gsize * 8, gm = min(8, p.tiles_m - first);
    const int m0 = (first + id % gsize % gm) * BM, n0 = (id % gsize / gm) * BN;
    int M = p.M;
    if (p.m_dev) { const int live = *p.m_dev; M = live < M ? live : M; }
    if (m0 >= M) return;
    const T* x = (const T*)p.x + (long long)m0 * p.ldx;
    const T* w = (const T*)p.w + (long long)n0 * p.ldw;
    const int last_m = M - 1 - m0, last_n = p.N - 1 - n0;

    bxf16 acc[TN][TM];
#pragma unroll
    for (int a = 0; a < TN; ++a)
#pragma unroll
        for (int b = 0; b < TM; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[a][b][i] = 0.0f;
    const int wm = (wave / WGN) * TM * 32, wn = (wave % WGN) * TN * 32, lr = lane & 31, h = lane >> 5;
    // rows of 64 bytes: four of them cover the banks, chunk c of row r sits at c ^ (r / 4 % 4)
    const int x_at = (wm + lr) * 64 + ((h ^ (lr >> 2 & 3)) * 16), w_at = 3 * PX * 16 + (wn + lr) * 64 + ((h ^ (lr >> 2 & 3)) * 16);

    bxi4 rx[LX][2], rw[LW][2];
    const auto fetch = [&](int k0) {
        const auto rows = [&](const auto& load) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < LX; ++i) {
                const int e = tid + i * NT;
                const T* row = x + (long long)min(e >> 2, last_m) * p.ldx;
#pragma unroll
                for (int j = 0; j < 2; ++j) rx[i][j] = load(row, k0 + (e & 3) * 8 + j * 4);
            }
#pragma unroll
            for (int i = 0; i < LW; ++i) {
                const int e = tid + i * NT;
                const T* row = w + (long long)min(e >> 2, last_n) * p.ldw;
#pragma unroll
                for (int j = 0; j < 2; ++j) rw[i][j] = load(row, k0 + (e & 3) * 8 + j * 4);
            }
        };
        if (k0 + BK <= p.K) rows([&](const T* row, int k) { return bx_load_whole<T>(row, k); });
        else rows([&](const T* row, int k) { return bx_load_chunk<T>(row, k, p.K); });
    };
    const auto put = [&](bxi4* plane, int stride, int e, const bxi4* r) {
        float f[8];
        __builtin_memcpy(f, r, 32);
        bxi4* to = plane + (e >> 2) * 4 + ((e & 3) ^ (e >> 4 & 3));
        bx_planes(f, to[0], to[stride], to[2 * stride]);
    };
    const auto stage = [&](bxi4* buf) {
#pragma unroll
        for (int i = 0; i < LX; ++i) put(buf, PX, tid + i * NT, rx[i]);
#pragma unroll
        for (int i = 0; i < LW; ++i) put(buf + 3 * PX, PW, tid + i * NT, rw[i]);
    };
    const auto multiply = [&](const bxi4* buf) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            bxi4 fx[TM][3], fw[TN][3];
#pragma unroll
            for (int n = 0; n < 3; ++n) {
#pragma unroll
                for (int b = 0; b < TM; ++b) fx[b][n] = *(const bxi4*)((const char*)buf + (x_at ^ (c * 32)) + n * PX * 16 + b * 32 * 64);
#pragma unroll
                for (int a = 0; a < TN; ++a) fw[a][n] = *(const bxi4*)((const char*)buf + (w_at ^ (c * 32)) + n * PW * 16 + a * 32 * 64);
            }
            constexpr int PA[6] = {2, 0, 1, 1, 0, 0}, PB[6] = {0, 2, 1, 0, 1, 0};
#pragma unroll
            for (int q = 0; q < 6; ++q)
#pragma unroll
                for (int a = 0; a < TN; ++a)
#pragma unroll
                    for (int b = 0; b < TM; ++b) acc[a][b] = bx_mma32<bx_bf16>(fw[a][PA[q]], fx[b][PB[q]], acc[a][b]);
        }
    };
    const int steps = (p.K + BK - 1) / BK;
    if (steps > 0) { fetch(0); stage(lds); }
    for (int s = 0; s < steps; ++s) {
        __syncthreads();
        if (s + 1 < steps) fetch((s + 1) * BK);
        multiply(lds + (s & 1) * BUF);
        if (s + 1 < steps) stage(lds + (~s & 1) * BUF);
    }

    bool odd = false;
#pragma unroll
    for (int a = 0; a < TN; ++a)
#pragma unroll
        for (int b = 0; b < TM; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i) odd |= !(fabsf(acc[a][b][i]) < INFINITY);
    if (__any(odd)) {
#pragma unroll
        for (int a = 0; a < TN; ++a)
#pragma unroll
            for (int b = 0; b < TM; ++b)
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (!(fabsf(acc[a][b][i]) < INFINITY)) {
                        const T* xr = x + (long long)min(wm + b * 32 + lr, last_m) * p.ldx;
                        const T* wr = w + (long long)min(wn + a * 32 + 8 * (i / 4) + 4 * h + i % 4, last_n) * p.ldw;
                        float sum = 0.0f;
                        for (int k = 0; k < p.K; ++k) sum = fmaf(xr[k], wr[k], sum);
                        acc[a][b][i] = sum;
                    }
    }
    __syncthreads();
    float* mine = (float*)lds + wave * 32 * (TN * 32 + 4);
    if (p.act == BX_ACT_NONE) put_rows<T, TM, TN, BX_ACT_NONE>(p, acc, mine, lane, m0 + wm, n0 + wn, M);
    else if (p.act == BX_ACT_RELU) put_rows<T, TM, TN, BX_ACT_RELU>(p, acc, mine, lane, m0 + wm, n0 + wn, M);
    else if (p.act == BX_ACT_GELU) put_rows<T, TM, TN, BX_ACT_GELU>(p, acc, mine, lane, m0 + wm, n0 + wn, M);
    else put_rows<T, TM, TN, BX_ACT_SILU>(p, acc, mine, lane, m0 + wm, n0 + wn, M);
}

// Few rows: one workgroup = 16 columns of y x 16 rows, its NW waves split K and meet in LDS.  Operands go from memory to the matrix
// units directly: a wave reads 64 bytes of 16 rows of W per step, and W is read once per 16 rows of x.
template <class T, int NW>
__global__ __launch_bounds__(NW * 64) void linear_rows_kernel(LinearK p)
{
    constexpr int CH = BxElem<T>::CH, BK = 4 * CH, U = 4;
    __shared__ float part[NW][16][17];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, lr = lane & 15, q = lane >> 4;
    const int n0 = (int)(blockIdx.x % p.tiles_n) * 16, m0 = (int)(blockIdx.x / p.tiles_n) * 16;
    int M = p.M;
    if (p.m_dev) { const int live = *p.m_dev; M = live < M ? live : M; }
    if (m0 >= M) return;
    // rows that do not exist repeat the last one: their products are not stored
    const T* xr = (const T*)p.x + (long long)min(m0 + lr, M - 1) * p.ldx;
    const T* wr = (const T*)p.w + (long long)min(n0 + lr, p.N - 1) * p.ldw;
    bxf4 acc = {0.f, 0.f, 0.f, 0.f};
    const int steps = (p.K + BK - 1) / BK;
    for (int s0 = wave; s0 < steps; s0 += NW * U) {
        bxi4 fx[U], fw[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int k = (s0 + u * NW) * BK + q * CH;
            if ((s0 + u * NW + 1) * BK <= p.K) { fw[u] = bx_load_whole<T>(wr, k); fx[u] = bx_load_whole<T>(xr, k); }
            else { fw[u] = bx_load_chunk<T>(wr, k, p.K); fx[u] = bx_load_chunk<T>(xr, k, p.K); }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) acc = bx_mma16<T>(fw[u], fx[u], acc);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) part[wave][lr][4 * q + i] = acc[i];
    __syncthreads();
    // lane (row, column group): four consecutive columns
    if (tid < 64) {
        const int m = m0 + lr, n = n0 + 4 * q;
        float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < NW; ++w)
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] += part[w][lr][4 * q + i];
        if (m < M && n < p.N) epilogue4<T>(p, m, n, v);
    }
}

template <class T, int BM, int BN, int WGM, int WGN, int KS = 1>
int launch_tile(hipStream_t s, LinearK k, bool aligned)
{
    k.tiles_n = (k.N + BN - 1) / BN;
    k.tiles_m = (k.M + BM - 1) / BM;
    const long long tiles = (long long)k.tiles_n * k.tiles_m;
    if (bx_grid_check("bx_linear", tiles, KS * WGM * WGN * 64) != BX_OK) return BX_ERR_ARG;
    const long long far = (1LL << 31) / (256 * (long long)sizeof(T));
    const bool direct = aligned && k.ldx < far && k.ldw < far;
    constexpr int threads = KS * WGM * WGN * 64;
    if constexpr (KS == 1 && BN <= 64) {
        if (k.K <= 8 * BxElem<T>::CH) {
            if (direct) linear_tile_kernel<T, BM, BN, WGM, WGN, 1, true, true><<<(unsigned)tiles, threads, 0, s>>>(k);
            else linear_tile_kernel<T, BM, BN, WGM, WGN, 1, false, true><<<(unsigned)tiles, threads, 0, s>>>(k);
            BX_LAUNCH_CHECK();
            return BX_OK;
        }
    }
    if (direct) linear_tile_kernel<T, BM, BN, WGM, WGN, KS, true, false><<<(unsigned)tiles, threads, 0, s>>>(k);
    else linear_tile_kernel<T, BM, BN, WGM, WGN, KS, false, false><<<(unsigned)tiles, threads, 0, s>>>(k);
    BX_LAUNCH_CHECK();
    return BX_OK;
}

template <int BM, int BN, int WGM, int WGN>
int launch_planes(hipStream_t s, LinearK k)
{
    k.tiles_n = (k.N + BN - 1) / BN;
    k.tiles_m = (k.M + BM - 1) / BM;
    const long long tiles = (long long)k.tiles_n * k.tiles_m;
    if (bx_grid_check("bx_linear", tiles, WGM * WGN * 64) != BX_OK) return BX_ERR_ARG;
    linear_planes_kernel<BM, BN, WGM, WGN><<<(unsigned)tiles, WGM * WGN * 64, 0, s>>>(k);
    BX_LAUNCH_CHECK();
    return BX_OK;
}

template <class T>
int linear_of(hipStream_t s, int n_cu, const bx_linear_args& a)
{
    LinearK k = {a.x, a.w, a.bias, a.residual, a.y, a.m_dev, a.ldx, a.ldw, a.ldr, a.ldy, (int)a.M, (int)a.N, (int)a.K, a.act, 0, 0};
    const auto al16 = [](const void* p, long long ld) { return ((uintptr_t)p & 15) == 0 && (ld * (long long)sizeof(T)) % 16 == 0; };
    const bool aligned = al16(a.x, a.ldx) && al16(a.w, a.ldw);
    const auto tiles = [&](int bm, int bn) { return (long long)((k.M + bm - 1) / bm) * ((k.N + bn - 1) / bn); };
    // Few rows, or an output that 16 x 16 pieces fill the card with once: these read W (or x) straight from memory.  1 x 1024 x 1024 bf16:
    // 4.2 us, 6.3 by the tiles below; 1000 x 32 by K = 512 f32: 6.0, 10.2; where there are more pieces they read too much again: 100 x 4096
    // by K = 2048 bf16 28 us, 9.0 by tiles.
    const long long pieces = tiles(16, 16);
    if (k.M <= 16 || pieces <= n_cu) {
        if (bx_grid_check("bx_linear", pieces, 512) != BX_OK) return BX_ERR_ARG;
        k.tiles_n = (k.N + 15) / 16;
        linear_rows_kernel<T, 8><<<(unsigned)pieces, 512, 0, s>>>(k);
        BX_LAUNCH_CHECK();
        return BX_OK;
    }
    // Tiles that do not fill the card once: smaller ones with the slices of K dealt to four or two groups of waves.  32 x 4096 by K = 2048
    // bf16 8.6 us (11.6 whole), 100 x 4096 9.0 (18.5), 300 x 4096 16.4 (19.7); f32 300 x 1024 by 1024 16.7 (25.6).
    if (k.K > 16 * BxElem<T>::CH) {
        if (k.M <= 32 && tiles(32, 64) <= n_cu) return launch_tile<T, 32, 64, 1, 2, 4>(s, k, aligned);
        if (tiles(64, 32) <= n_cu) return launch_tile<T, 64, 32, 2, 1, 4>(s, k, aligned);
        if (tiles(64, 64) <= n_cu) return launch_tile<T, 64, 64, 2, 2, 2>(s, k, aligned);
    }
    // Up to 32 columns leave half of the other tiles empty: 587689 x 32 by 16 f16 15 us (21 by 64 x 64).
    if (k.N <= 32) return launch_tile<T, 128, 32, 4, 1>(s, k, aligned);
    if constexpr (sizeof(T) == 2) {
        // Large outputs want 256 x 256 (16384 x 4096 by K = 1024 bf16 with gelu: 174 us; 175 by 128 x 128, 192 by 64 x 128).  Rows that are not
        // aligned go through registers, which larger tiles save most of: 16384 x 4096 by 1023 165 us (240 by 128 x 128, 366 by 64 x 64),
        // 8000 x 2000 by 700 36 us (66), 30000 x 500 by 501 30 us (37, 56); 100000 x 300 by 65 36 us by 128 x 128 (43, 40 by 64 x 64).
        if (aligned) {
            if (k.N > 128 && tiles(256, 256) >= 2 * n_cu) return launch_tile<T, 256, 256, 4, 4>(s, k, aligned);
            if (k.N > 64 && tiles(64, 128) >= 4 * n_cu && k.K >= 256) return launch_tile<T, 64, 128, 2, 2>(s, k, aligned);
        } else {
            if (k.N > 128 && tiles(256, 256) >= n_cu - n_cu / 8 && k.K >= 192) return launch_tile<T, 256, 256, 4, 4>(s, k, aligned);
            if (k.N > 64 && tiles(128, 128) >= n_cu - n_cu / 4) return launch_tile<T, 128, 128, 4, 2>(s, k, aligned);
        }
    } else if (k.K >= 128) {
        // f32 by planes: 8192 x 4096 by 1024 361 us (442 by 64 x 128, 532 on the f32 units), 10000 x 1024 by 1024 150 us (177), 10000 x 256 by
        // 256 20.4 us (23.3).  Shorter sums are bound by memory either way (700000 x 64 by 32: 62 us both).
        if (k.N > 128 && tiles(128, 256) >= 3 * n_cu) return launch_planes<128, 256, 2, 4>(s, k);
        if (k.N > 64 && tiles(64, 128) >= 4 * n_cu) return launch_planes<64, 128, 2, 2>(s, k);
        return launch_planes<64, 64, 2, 2>(s, k);
    }
    return launch_tile<T, 64, 64, 2, 2>(s, k, aligned);
}

}  // namespace

int bxk_linear(hipStream_t s, int n_cu, const bx_linear_args& a)
{
    if (a.M == 0 || a.N == 0) return BX_OK;
    if (a.dtype == BX_TYPE_F32) return linear_of<float>(s, n_cu, a);
    if (a.dtype == BX_TYPE_F16) return linear_of<bx_f16>(s, n_cu, a);
    return linear_of<bx_bf16>(s, n_cu, a);
}
