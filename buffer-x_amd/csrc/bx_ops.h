// bx_ops.h -- what the dense operators over keypoints share (k_linear.hip, k_rope.hip, k_attn.hip): element types, 16-byte chunks and the
// matrix instructions that consume them.  A chunk is 16 bytes of one row: 4 floats or 8 halves.  Every kernel feeds the matrix units
// one chunk per lane and operand, so the three element types share one code path:
//   f16 / bf16: one v_mfma_f32_32x32x16 (16x16x32) per chunk;
//   f32:        four v_mfma_f32_32x32x2 (16x16x4), step j taking element j of both operands' chunks -- the products of a sum are
//               visited in another order than by k, the same one on both sides.
#pragma once
#include "bx_common.h"

typedef float bxf4 __attribute__((ext_vector_type(4)));
typedef float bxf16 __attribute__((ext_vector_type(16)));
typedef int bxi4 __attribute__((ext_vector_type(4)));
typedef int bxi2 __attribute__((ext_vector_type(2)));
typedef _Float16 bxh8 __attribute__((ext_vector_type(8)));
typedef __bf16 bxb8 __attribute__((ext_vector_type(8)));
typedef __bf16 bx_bf16;
typedef _Float16 bx_f16;

// 16 bytes at any element boundary (gfx950 loads and stores them unaligned in one instruction)
struct __attribute__((packed, aligned(2))) BxAny16 { bxi4 v; };

template <class T> struct BxElem {
    static constexpr int CH = 16 / (int)sizeof(T);      // elements per chunk
};

template <class T> __device__ __forceinline__ bxf16 bx_mma32(bxi4 a, bxi4 b, bxf16 c)
{
    if constexpr (sizeof(T) == 4) {
        const bxf4 x = __builtin_bit_cast(bxf4, a), y = __builtin_bit_cast(bxf4, b);
#pragma unroll
        for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(x[j], y[j], c, 0, 0, 0);
        return c;
    } else if constexpr (__is_same(T, bx_f16)) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(bxh8, a), __builtin_bit_cast(bxh8, b), c, 0, 0, 0);
    } else {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bxb8, a), __builtin_bit_cast(bxb8, b), c, 0, 0, 0);
    }
}

template <class T> __device__ __forceinline__ bxf4 bx_mma16(bxi4 a, bxi4 b, bxf4 c)
{
    if constexpr (sizeof(T) == 4) {
        const bxf4 x = __builtin_bit_cast(bxf4, a), y = __builtin_bit_cast(bxf4, b);
#pragma unroll
        for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(x[j], y[j], c, 0, 0, 0);
        return c;
    } else if constexpr (__is_same(T, bx_f16)) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(bxh8, a), __builtin_bit_cast(bxh8, b), c, 0, 0, 0);
    } else {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bxb8, a), __builtin_bit_cast(bxb8, b), c, 0, 0, 0);
    }
}

// eight floats as the sum of three bf16 operands: each plane holds the nearest bf16 to what the ones before it left
__device__ __forceinline__ void bx_planes(const float* e, bxi4& p0, bxi4& p1, bxi4& p2)
{
    bx_bf16 a[8], b[8], c[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        a[j] = (bx_bf16)e[j];
        const float r = e[j] - (float)a[j];
        b[j] = (bx_bf16)r;
        c[j] = (bx_bf16)(r - (float)b[j]);
    }
    __builtin_memcpy(&p0, a, 16);
    __builtin_memcpy(&p1, b, 16);
    __builtin_memcpy(&p2, c, 16);
}

// elements [k, k + CH) of a row, all of which exist
template <class T> __device__ __forceinline__ bxi4 bx_load_whole(const T* __restrict__ row, int k) { return reinterpret_cast<const BxAny16*>(row + k)->v; }

// elements [k, k + CH) of a row of `n` elements as one chunk; what lies at or behind n is zero and is not read: the last chunk of a row is
// loaded from where it still fits and shifted into place, rows shorter than a chunk go element by element
template <class T> __device__ __forceinline__ bxi4 bx_load_chunk(const T* __restrict__ row, int k, int n)
{
    constexpr int CH = BxElem<T>::CH;
    if (n < CH) {
        T e[CH];
#pragma unroll
        for (int j = 0; j < CH; ++j) e[j] = k + j < n ? row[k + j] : (T)0.0f;
        bxi4 r;
        __builtin_memcpy(&r, e, 16);
        return r;
    }
    if (k >= n) return (bxi4){0, 0, 0, 0};
    const int a = min(k, n - CH);
    bxi4 v = reinterpret_cast<const BxAny16*>(row + a)->v;
    if (k > a) {
        typedef unsigned long long u2 __attribute__((ext_vector_type(2)));
        u2 w = __builtin_bit_cast(u2, v);
        const int s = (k - a) * (int)sizeof(T) * 8;          // 16 .. 112 bits
        w[0] = s >= 64 ? w[1] >> (s - 64) : (w[0] >> s | w[1] << (64 - s));
        w[1] = s >= 64 ? 0 : w[1] >> s;
        v = __builtin_bit_cast(bxi4, w);
    }
    return v;
}

// four consecutive elements of one row, of which n exist.  Results are rounded once to T (nearest, ties to even).
struct __attribute__((packed, aligned(2))) BxAny8 { bxi2 v; };
template <class T> __device__ __forceinline__ void bx_store4(T* __restrict__ p, const float* v, int n)
{
    T e[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) e[j] = (T)v[j];
    if (n >= 4) {
        if constexpr (sizeof(T) == 4) { bxi4 r; __builtin_memcpy(&r, e, 16); reinterpret_cast<BxAny16*>(p)->v = r; }
        else { bxi2 r; __builtin_memcpy(&r, e, 8); reinterpret_cast<BxAny8*>(p)->v = r; }
        return;
    }
#pragma unroll
    for (int j = 0; j < 3; ++j)
        if (j < n) p[j] = e[j];
}

template <class T> __device__ __forceinline__ void bx_load4(const T* __restrict__ p, float* v, int n)
{
    T e[4];
    if (n >= 4) {
        if constexpr (sizeof(T) == 4) { const bxi4 r = reinterpret_cast<const BxAny16*>(p)->v; __builtin_memcpy(e, &r, 16); }
        else { const bxi2 r = reinterpret_cast<const BxAny8*>(p)->v; __builtin_memcpy(e, &r, 8); }
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) e[j] = j < n ? p[j] : (T)0.0f;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = (float)e[j];
}

// 16 bytes per lane from memory straight into LDS, at lds + 16 lane (lds is the same for the whole wave)
__device__ __forceinline__ void bx_load_lds16(const void* g, void* lds)
{
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)g, (__attribute__((address_space(3))) void*)lds, 16, 0, 0);
}

// a barrier behind which every wave's loads into LDS have landed
__device__ __forceinline__ void bx_sync_landed()
{
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
}

// Workgroups go to the eight XCDs in turn.  This order gives each XCD runs of C neighbours of the logical order instead, whose operands
// its L2 then reads once; what does not fill whole rounds keeps its place.
template <unsigned C> __device__ __forceinline__ unsigned bx_xcd_order(unsigned id, unsigned n)
{
    const unsigned full = n / (8 * C) * (8 * C);
    if (id >= full) return id;
    const unsigned x = id & 7, j = id >> 3;
    return j / C * (8 * C) + x * C + j % C;
}

// a launch has fewer than 2^32 threads
inline int bx_grid_check(const char* what, long long groups, int threads)
{
    if (groups * threads < 1LL << 32) return BX_OK;
    bx_set_error("%s: %lld workgroups exceed one launch", what, groups);
    return BX_ERR_ARG;
}

int bxk_linear(hipStream_t s, int n_cu, const bx_linear_args& a);
int bxk_qk_norm_rope(hipStream_t s, int n_cu, const bx_qk_norm_rope_args& a);
int64_t bxk_attention_workspace(int n_cu, const bx_attention_args& a);
int bxk_attention(hipStream_t s, int n_cu, const bx_attention_args& a);
