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
};

// The SwiGLU's gradient for one value: dz, gate and up to the gradients of both, and z.
__device__ __forceinline__ void swiglu_grad(float dz, float g, float u, float* dg, float* du, float* z) {
    // s = 1 / (1 + e^-g) on the exponential and reciprocal units, within two units in the last place; e^-g
    // is infinite below g = -88.7, s then 0, and g s too
    const float s = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(g * -1.44269504088896f));
    const float a = g * s;
    *du = dz * a;
    *dg = dz * u * (s + a * (1.0f - s));
    *z = a * u;
}

// Whether two arrays of so many bytes share memory.
static inline bool hm_overlap(const void* a, int64_t na, const void* b, int64_t nb) {
    const uint64_t pa = reinterpret_cast<uintptr_t>(a), pb = reinterpret_cast<uintptr_t>(b);
    return a && b && (pa < pb ? pb - pa < (uint64_t)na : pa - pb < (uint64_t)nb);
}

int hm_g_launch_generic(GKind kind, bool w_kmajor, int32_t dtype, int32_t y_dtype, const GProduct& p, hipStream_t s);
