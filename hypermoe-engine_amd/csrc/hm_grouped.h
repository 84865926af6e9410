// hm_grouped.h -- what the kernels of 16-bit products share: grouped products of experts with SwiGLU and
// their gradients (hm_grouped.hip), and projections with low-rank adapters (hm_adapter.hip).
//
// A product is C(m, n) = sum_k X(m, k) W(n, k), both operands FP16 or BF16, sums FP32.  An operand's values
// lie with k contiguous ("k-major": rows of x, a projection's matrix) or with m or n contiguous (a matrix
// read transposed; both operands of a weight's gradient, whose k are the rows).
//
// v_mfma_f32_16x16x32: lane l supplies 8 consecutive k, from 8 (l / 16), of row l % 16 of A and of column
// l % 16 of B; its 4 results are column l % 16, rows 4 (l / 16) + v.  W is A and X is B: a lane's results
// are then 4 consecutive outputs of one row.
#pragma once

#include "hm_fp8_product.h"

typedef __bf16 v8b __attribute__((ext_vector_type(8)));

template <typename T>
struct Elem16;
template <>
struct Elem16<hm_f16> {
    typedef v8h v8;
    static __device__ __forceinline__ v4f mfma(v8 a, v8 b, v4f c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    }
};
template <>
struct Elem16<hm_bf16> {
    typedef v8b v8;
    static __device__ __forceinline__ v4f mfma(v8 a, v8 b, v4f c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    }
};

enum GKind {
    G_MATMUL,       // y = acc
    G_SWIGLU,       // z = silu(g) u, g and u two products; pre = g | u if wanted
    G_SWIGLU_GRAD,  // acc = dz; dpre and z from pre
    G_WEIGHT_GRAD,  // y = (y +) acc, one matrix a group, k the group's rows
    G_ADAPTER       // y = acc + mid up_a^T
};

struct GProduct {
    const void* x;             // [x_rows x K] (weight gradient: dy [rows x M])
    const void* w;             // groups matrices [N x K] or [K x N] (weight gradient: x [rows x N])
    void* y;
    const int32_t* offsets;    // groups + 1; nullptr: one group of all rows
    const int32_t* perm;       // SwiGLU: row of x of each grouped row, or nullptr
    int64_t rows, x_rows;
    int64_t M;                 // weight gradient: rows of a result matrix
    int64_t K, N;              // inner dimension (not of the weight gradient), output columns
    int64_t w_group;           // elements from one group's matrix to the next
    int groups;
    bool accumulate;
    const void* pre_in;        // SwiGLU gradient: [rows x 2N]
    void* pre_out;             // SwiGLU: [rows x 2N] or nullptr
    void* z;                   // SwiGLU gradient: [rows x N] or nullptr
    // adapters
    const int32_t* ids;        // [rows]; outside 0 .. adapters - 1: none
    const void* mid;           // [rows x rank]
    const void* up;            // adapters matrices [N x rank] or [rank x N]
    int adapters;
    int rank;
    bool wide;                 // results are aligned to 4 elements
};

// The SwiGLU's gradient for one value: dz, gate and up to the gradients of both, and z.
__device__ __forceinline__ void swiglu_grad(float dz, float g, float u, float* dg, float* du, float* z) {
    // s = 1 / (1 + e^-g) on the exponential and reciprocal units, a unit in the last place each; the exponent g log2 e is
    // rounded to FP32 before, which is |g| 2^-24 of e^-g, so for negative g |g| / 2 units of s besides (10 at -20, 40 at
    // -80).  Below g = -87, where it is under 2e-38, s is 0, and g s too
    const float s = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(g * -1.44269504088896f));
    const float a = g * s;
    *du = dz * a;
    *dg = dz * u * (s + a * (1.0f - s));
    *z = a * u;
}

template <typename T>
struct __attribute__((packed, aligned(2))) Loose8 {  // 16 bytes aligned to an element
    T v[8];
};
template <>
struct __attribute__((packed, aligned(4))) Loose8<float> {
    float v[8];
};
// n values (8 at most) from and to rows of any alignment
template <typename T>
__device__ __forceinline__ void load8(const T* p, int n, float (&f)[8]) {
    if (n >= 8) {
        const Loose8<T> w = *reinterpret_cast<const Loose8<T>*>(p);
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = (float)w.v[i];
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = i < n ? (float)p[i] : 0.0f;
    }
}
template <typename T>
__device__ __forceinline__ void store8(T* p, int n, const float (&f)[8]) {
    if (n >= 8) {
        Loose8<T> w;
#pragma unroll
        for (int i = 0; i < 8; ++i) w.v[i] = (T)f[i];
        *reinterpret_cast<Loose8<T>*>(p) = w;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < n) p[i] = (T)f[i];
    }
}

// 16 bytes from a place aligned to 2.
typedef uint64_t u64x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ u64x2 load16(const void* p) {
    typedef uint64_t loose __attribute__((ext_vector_type(2), aligned(2)));
    return *(const __attribute__((address_space(1))) loose*)p;   // (never the LDS: no flat load)
}

// 8 values to a place aligned to their element, past the L2's other contents (a result is larger than the L2 by far, and
// what the L2 holds is read again: weight gradients of 128 groups, 805 MB of results, 435 us without the hint, 303 with).
__device__ __forceinline__ void stream16(void* p, u64x2 v) {
    typedef uint64_t loose __attribute__((ext_vector_type(2), aligned(2)));
    __builtin_nontemporal_store(v, (__attribute__((address_space(1))) loose*)p);
}
template <typename T>
__device__ __forceinline__ u64x2 pack8(const float (&f)[8]) {
    Loose8<T> w;
#pragma unroll
    for (int i = 0; i < 8; ++i) w.v[i] = (T)f[i];
    return __builtin_bit_cast(u64x2, w);
}
template <typename T>
__device__ __forceinline__ void stream8(T* p, const float (&f)[8]) {
    if constexpr (sizeof(T) == 2) stream16(p, pack8<T>(f));
    else store8(p, 8, f);
}
// The value of the lane 8 further in its 16 (DPP row_ror:8).
__device__ __forceinline__ u64x2 other8(u64x2 v) {
    typedef int i32x4 __attribute__((ext_vector_type(4)));
    i32x4 w = __builtin_bit_cast(i32x4, v);
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = __builtin_amdgcn_update_dpp(0, w[i], 0x128, 0xF, 0xF, false);
    return __builtin_bit_cast(u64x2, w);
}

// n values (8 at most) of a row as a fragment's 8, zeros behind them.
template <typename T>
__device__ __forceinline__ typename Elem16<T>::v8 load_frag8(const T* p, int64_t n) {
    typedef typename Elem16<T>::v8 v8;
    typedef short v8s __attribute__((ext_vector_type(8)));
    typedef const __attribute__((address_space(1))) short* global_t;
    if (n >= 8) return __builtin_bit_cast(v8, load16(p));
    v8s w = {};
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (i < n) w[i] = ((global_t)p)[i];
    return __builtin_bit_cast(v8, w);
}

// A fragment's 8 values of k from the LDS, `next4` bytes from one 4 of them to the next: ds_read_b64_tr_b16, in
// which lane i of 16 gives the place of 4 consecutive values of row i / 4 and gets the values of 4 rows in column i.
typedef short v4s __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) v4s* lds_v4s;
template <typename V>
__device__ __forceinline__ V read_transposed(const uint8_t* at, int next4) {
    const v4s a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s)at);
    const v4s b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s)(at + next4));
    return __builtin_bit_cast(V, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
}

// The minimum over the wave, in every lane.
__device__ __forceinline__ int wave_min(int v) {
    v = min(v, __builtin_amdgcn_update_dpp(0, v, 0xB1, 0xF, 0xF, false));
    v = min(v, __builtin_amdgcn_update_dpp(0, v, 0x4E, 0xF, 0xF, false));
    v = min(v, __builtin_amdgcn_update_dpp(0, v, 0x141, 0xF, 0xF, false));
    v = min(v, __builtin_amdgcn_update_dpp(0, v, 0x140, 0xF, 0xF, false));
    return min(min(__builtin_amdgcn_readlane(v, 0), __builtin_amdgcn_readlane(v, 16)),
               min(__builtin_amdgcn_readlane(v, 32), __builtin_amdgcn_readlane(v, 48)));
}

// Whether two arrays of so many bytes share memory.
static inline bool hm_overlap(const void* a, int64_t na, const void* b, int64_t nb) {
    const uint64_t pa = reinterpret_cast<uintptr_t>(a), pb = reinterpret_cast<uintptr_t>(b);
    return a && b && (pa < pb ? pb - pa < (uint64_t)na : pa - pb < (uint64_t)nb);
}

int hm_g_launch_generic(GKind kind, bool w_kmajor, int32_t dtype, int32_t y_dtype, const GProduct& p, hipStream_t s);
// The tile kernels (hm_grouped_tile.h).  form 256: tiles of 256 x 256 results, 128: of 128 x 256, 64: of 128 x 128,
// these three for operands aligned to 16 bytes throughout; 32: of 128 x 128 for others.
int hm_g_launch_tiles_f16(GKind kind, int form, bool w_kmajor, bool f32, const GProduct& p, hipStream_t s);
int hm_g_launch_tiles_bf16(GKind kind, int form, bool w_kmajor, bool f32, const GProduct& p, hipStream_t s);
// The kernel for few rows (hm_grouped_stream.hip): x w^T, SwiGLU or adapters, 16 mt rows a workgroup (1, 2, 4; 8 for
// adapters).
int hm_g_launch_stream(GKind kind, int mt, int32_t dtype, bool f32, const GProduct& p, hipStream_t s);
// The kernel that a product's sizes and alignment ask for (hm_grouped.hip).
int hm_g_launch(GKind kind, bool w_kmajor, int32_t dtype, int32_t y_dtype, const GProduct& p, hipStream_t s);
