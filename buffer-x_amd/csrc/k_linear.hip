// k_linear.hip -- y = act(x W^T + b) + r, the dense layer over keypoints (bx_linear).  x [M][K], W [N][K], y [M][N]: the rows of both
// operands run along K, so both are staged as 128-byte slices of rows.  Sums are held in f32, the epilogue (bias, activation, residual)
// runs on the accumulators and the result is rounded once.
#include "bx_ops.h"

namespace {

__device__ __forceinline__ float act_of(float v, int act)
{
    if (act == BX_ACT_RELU) return v > 0.0f ? v : (v != v ? v : 0.0f);
    // erfc keeps the relative precision that 1 + erf loses for negative arguments
    if (act == BX_ACT_GELU) return 0.5f * v * erfcf(-v * 0.70710678118654752f);
    if (act == BX_ACT_SILU) return v / (1.0f + expf(-v));
    return v;
}

struct LinearK {
    const void *x, *w, *bias, *residual;
    void* y;
    const int32_t* m_dev;
    long long ldx, ldw, ldr, ldy;
    int M, N, K, act, tiles_n;
};

template <class T>
__device__ __forceinline__ void epilogue4(const LinearK& p, int m, int n, const float* acc)
{
    const int left = p.N - n;
    float v[4], b[4] = {0.f, 0.f, 0.f, 0.f};
    if (p.bias) bx_load4<T>((const T*)p.bias + n, b, left);
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = act_of(acc[j] + b[j], p.act);
    if (p.residual) {
        float r[4];
        bx_load4<T>((const T*)p.residual + (long long)m * p.ldr + n, r, left);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] += r[j];
    }
    bx_store4<T>((T*)p.y + (long long)m * p.ldy + n, v, left);
}

// One workgroup = a BM x BN tile of y; a wave holds a (BM / WGM) x (BN / WGN) part of it in 32 x 32 accumulators.  The matrix product is
// taken transposed (W rows as the first operand): a lane then holds four consecutive columns of one row of y and stores them together.
// A row slice of 128 bytes is 8 chunks in LDS; chunk c of row r sits at c ^ (r & 7), so that the 8 lanes of a 128-byte LDS access
// (consecutive rows, same chunk) meet 8 different bank groups.
template <class T, int BM, int BN, int WGM, int WGN, bool ALIGNED>
__global__ __launch_bounds__(WGM * WGN * 64) void linear_tile_kernel(LinearK p)
{
    constexpr int CH = BxElem<T>::CH, BK = 8 * CH, NT = WGM * WGN * 64;
    constexpr int TM = BM / WGM / 32, TN = BN / WGN / 32;
    constexpr int LX = BM * 8 / NT, LW = BN * 8 / NT;
    __shared__ bxi4 sx[2][BM * 8], sw[2][BN * 8];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int m0 = (int)(blockIdx.x / p.tiles_n) * BM, n0 = (int)(blockIdx.x % p.tiles_n) * BN;
    int M = p.M;
    if (p.m_dev) { const int live = *p.m_dev; M = live < M ? live : M; }
    if (m0 >= M) return;
    const T* x = (const T*)p.x;
    const T* w = (const T*)p.w;
    bxi4 rx[LX], rw[LW];
    const bxi4 zero = {0, 0, 0, 0};

    auto fetch = [&](int k0) {
#pragma unroll
        for (int i = 0; i < LX; ++i) {
            const int id = tid + i * NT, r = id >> 3, c = id & 7;
            rx[i] = m0 + r < M ? bx_load_chunk<T, ALIGNED>(x + (long long)(m0 + r) * p.ldx, k0 + c * CH, p.K) : zero;
        }
#pragma unroll
        for (int i = 0; i < LW; ++i) {
            const int id = tid + i * NT, r = id >> 3, c = id & 7;
            rw[i] = n0 + r < p.N ? bx_load_chunk<T, ALIGNED>(w + (long long)(n0 + r) * p.ldw, k0 + c * CH, p.K) : zero;
        }
    };
    auto stage = [&](int buf) {
#pragma unroll
        for (int i = 0; i < LX; ++i) { const int id = tid + i * NT, r = id >> 3; sx[buf][r * 8 + ((id & 7) ^ (r & 7))] = rx[i]; }
#pragma unroll
        for (int i = 0; i < LW; ++i) { const int id = tid + i * NT, r = id >> 3; sw[buf][r * 8 + ((id & 7) ^ (r & 7))] = rw[i]; }
    };

    bxf16 acc[TN][TM];
#pragma unroll
    for (int a = 0; a < TN; ++a)
#pragma unroll
        for (int b = 0; b < TM; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[a][b][i] = 0.0f;

    const int wm = (wave / WGN) * TM * 32, wn = (wave % WGN) * TN * 32, lr = lane & 31, h = lane >> 5;
    const int steps = (p.K + BK - 1) / BK;
    if (steps > 0) { fetch(0); stage(0); }
    for (int s = 0; s < steps; ++s) {
        __syncthreads();
        if (s + 1 < steps) fetch((s + 1) * BK);
        const bxi4 *bx = sx[s & 1], *bw = sw[s & 1];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            bxi4 fx[TM], fw[TN];
#pragma unroll
            for (int b = 0; b < TM; ++b) { const int r = wm + b * 32 + lr; fx[b] = bx[r * 8 + ((2 * c + h) ^ (r & 7))]; }
#pragma unroll
            for (int a = 0; a < TN; ++a) { const int r = wn + a * 32 + lr; fw[a] = bw[r * 8 + ((2 * c + h) ^ (r & 7))]; }
#pragma unroll
            for (int a = 0; a < TN; ++a)
#pragma unroll
                for (int b = 0; b < TM; ++b) acc[a][b] = bx_mma32<T>(fw[a], fx[b], acc[a][b]);
        }
        if (s + 1 < steps) stage((s + 1) & 1);
    }

#pragma unroll
    for (int b = 0; b < TM; ++b) {
        const int m = m0 + wm + b * 32 + lr;
        if (m >= M) continue;
#pragma unroll
        for (int a = 0; a < TN; ++a)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int n = n0 + wn + a * 32 + 8 * g + 4 * h;
                if (n >= p.N) continue;
                const float v[4] = {acc[a][b][4 * g], acc[a][b][4 * g + 1], acc[a][b][4 * g + 2], acc[a][b][4 * g + 3]};
                epilogue4<T>(p, m, n, v);
            }
    }
}

// Few rows: one workgroup = 16 columns of y x 16 rows, its NW waves split K and meet in LDS.  Operands go from memory to the matrix
// units directly: a wave reads 64 bytes of 16 rows of W per step, and W is read once per 16 rows of x.
template <class T, int NW, bool ALIGNED>
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
            fw[u] = bx_load_chunk<T, ALIGNED>(wr, k, p.K);
            fx[u] = bx_load_chunk<T, ALIGNED>(xr, k, p.K);
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

template <class T, int BM, int BN, int WGM, int WGN>
int launch_tile(hipStream_t s, LinearK k, bool aligned)
{
    k.tiles_n = (k.N + BN - 1) / BN;
    const long long tiles = (long long)k.tiles_n * ((k.M + BM - 1) / BM);
    if (tiles > 0x7fffffffLL) { bx_set_error("bx_linear: %lld tiles exceed one launch", tiles); return BX_ERR_ARG; }
    if (aligned) linear_tile_kernel<T, BM, BN, WGM, WGN, true><<<(unsigned)tiles, WGM * WGN * 64, 0, s>>>(k);
    else linear_tile_kernel<T, BM, BN, WGM, WGN, false><<<(unsigned)tiles, WGM * WGN * 64, 0, s>>>(k);
    BX_LAUNCH_CHECK();
    return BX_OK;
}

template <class T>
int linear_of(hipStream_t s, int n_cu, const bx_linear_args& a)
{
    LinearK k = {a.x, a.w, a.bias, a.residual, a.y, a.m_dev, a.ldx, a.ldw, a.ldr, a.ldy, (int)a.M, (int)a.N, (int)a.K, a.act, 0};
    const auto al16 = [](const void* p, long long ld) { return ((uintptr_t)p & 15) == 0 && (ld * (long long)sizeof(T)) % 16 == 0; };
    const bool aligned = al16(a.x, a.ldx) && al16(a.w, a.ldw);
    const long long tiles64 = (long long)((k.M + 63) / 64) * ((k.N + 63) / 64);
    if (k.M <= 32 || (tiles64 < n_cu / 2 && k.K >= 256)) {
        k.tiles_n = (k.N + 15) / 16;
        const long long g = (long long)k.tiles_n * ((k.M + 15) / 16);
        if (aligned) linear_rows_kernel<T, 8, true><<<(unsigned)g, 512, 0, s>>>(k);
        else linear_rows_kernel<T, 8, false><<<(unsigned)g, 512, 0, s>>>(k);
        BX_LAUNCH_CHECK();
        return BX_OK;
    }
    if ((long long)((k.M + 127) / 128) * ((k.N + 127) / 128) >= 2 * n_cu) return launch_tile<T, 128, 128, 2, 2>(s, k, aligned);
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
