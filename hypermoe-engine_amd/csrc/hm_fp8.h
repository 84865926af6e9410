// hm_fp8.h -- what the FP8 and row kernels share: element types, and the block-scaled e4m3 format.
//
// Format.  A matrix [rows x width] is rows of hm_fp8_pitch(width) bytes (width rounded up to 128),
// e4m3 (OCP: bias 7, largest 448, 0x7f NaN), zeros past the width.  Every block of `block_rows` rows
// (1 or 128) x 128 columns has one float scale, scale[row / block_rows][column / 128]:
//   amax  = max(|x|, 2^-100) over the block
//   scale = amax / 448
//   byte  = the e4m3 value nearest to 448 x / amax, ties to even
// 2^-100 keeps the scale, its reciprocal and the operands below inside the normal floats.  A block
// that holds an infinity or a NaN becomes NaN throughout (bytes 0x7f, scale NaN), so it shows in every
// product that reads it.
#pragma once

#include "hm_device.h"

constexpr int kF8Block = 128;       // values per scale along a row
constexpr float kF8Top = 448.0f;    // largest e4m3 value
constexpr float kF8Tiny = 0x1p-100f;

__host__ __device__ __forceinline__ int64_t hm_f8_blocks(int64_t width) {
    return (width + kF8Block - 1) / kF8Block;
}
__host__ __device__ __forceinline__ int64_t hm_f8_pitch(int64_t width) {
    return hm_f8_blocks(width) * kF8Block;
}

// Element types of the operators' 16- and 32-bit operands (HM_DTYPE_FP32, _FP16, _BF16).  Sums are
// floats everywhere; a store to 16 bits rounds once, to nearest even.
typedef _Float16 hm_f16;
typedef __bf16 hm_bf16;
static inline bool hm_row_dtype(int32_t dtype) {
    return dtype == HM_DTYPE_FP32 || dtype == HM_DTYPE_FP16 || dtype == HM_DTYPE_BF16;
}
static inline size_t hm_row_dtype_size(int32_t dtype) { return dtype == HM_DTYPE_FP32 ? 4 : 2; }

// N elements of T as one memory operation of up to 16 bytes.
template <typename T, int N>
struct alignas(sizeof(T) * N) hm_pack {
    T v[N];
};

// One block's quantisation: q = a y, then one step of the residual, which is the correctly rounded
// a / b (y the rounded 1 / b) wherever a / b lies between two e4m3 values, so 16-bit inputs are always
// cut exactly as the formula says (their quotients do land there).  a = 448/512 x and b = amax / 512
// cannot overflow.
struct hm_f8_scaler {
    float b, y, scale;
    bool finite;
};
__device__ __forceinline__ hm_f8_scaler hm_f8_scaler_of(float amax) {
    hm_f8_scaler s;
    s.finite = amax <= 3.402823466e38f;   // false for infinity and NaN
    const float m = fmaxf(amax, kF8Tiny);
    s.b = m * 0x1p-9f;
    s.y = __fdiv_rn(1.0f, s.b);
    s.scale = s.finite ? __fdiv_rn(m, kF8Top) : __builtin_nanf("");
    return s;
}
__device__ __forceinline__ float hm_f8_scaled(const hm_f8_scaler& s, float x) {
    const float a = x * 0.875f;
    const float q = a * s.y;
    return __builtin_fmaf(__builtin_fmaf(-q, s.b, a), s.y, q);
}
// Four values as four bytes (the lowest address first).
__device__ __forceinline__ uint32_t hm_f8_pack4(const hm_f8_scaler& s, float x0, float x1, float x2,
                                                float x3) {
    int w = 0;
    w = __builtin_amdgcn_cvt_pk_fp8_f32(hm_f8_scaled(s, x0), hm_f8_scaled(s, x1), w, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(hm_f8_scaled(s, x2), hm_f8_scaled(s, x3), w, true);
    return s.finite ? (uint32_t)w : 0x7f7f7f7fu;
}
// |x| into a running maximum that keeps a NaN (as a value above every finite one).
__device__ __forceinline__ float hm_f8_amax(float amax, float x) {
    const float m = fabsf(x);
    return m <= amax ? amax : (m == m ? m : __builtin_inff());
}

// One hm_fp8_experts call (hm_fp8_gemm.hip): its two stages, for the block to time them apart.
struct hm_f8_experts_call {
    const hm_layer* layer;
    const void* x;
    int32_t x_dtype;
    int64_t tokens;
    const int32_t* offsets;
    const int32_t* perm_tokens;
    int64_t pairs;
    void* y;
    int32_t y_dtype;
    void* workspace;
    size_t workspace_bytes;
};
int hm_f8_experts_gate_up(const hm_f8_experts_call& c, hipStream_t s);
int hm_f8_experts_down(const hm_f8_experts_call& c, hipStream_t s);
