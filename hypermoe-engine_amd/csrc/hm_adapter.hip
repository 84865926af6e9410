// hm_adapter.hip -- low-rank adapters of many requests beside a shared projection:
//   mid[t] = s_a x[t] A_a^T,  y[t] = x[t] W^T + mid[t] B_a^T,  a = ids[t]
// the input's gradient by the same entry point with the matrices transposed, and the adapters' gradients
//   d_a = sum over the rows t of adapter a of  left[t]^T right[t].
#include "hm_grouped.h"

#include <limits.h>

namespace {

constexpr int kThreads = 256;

// mid of one row: a wave for every fourth rank (k-major), or 256 threads over k and ranks.
template <typename T, bool KM>
__global__ __launch_bounds__(kThreads) void adapter_mid_kernel(const T* __restrict__ x, const T* __restrict__ down,
                                                               const float* __restrict__ scale,
                                                               const int32_t* __restrict__ ids, int adapters,
                                                               int rank, int64_t K, T* __restrict__ mid) {
    const int64_t row = blockIdx.x;
    const int a = ids[row];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const bool has = a >= 0 && a < adapters;
    const T* xr = x + row * K;
    const T* d = down + (int64_t)(has ? a : 0) * rank * K;
    const float s = has ? scale[a] : 0.0f;
    for (int r = wave; r < rank; r += kThreads / 64) {
        float v = 0.0f;
        if (has)
            for (int64_t k = lane; k < K; k += 64)
                v = __builtin_fmaf((float)xr[k], (float)(KM ? d[r * K + k] : d[k * rank + r]), v);
#pragma unroll
        for (int m = 32; m >= 1; m >>= 1) v += __shfl_xor(v, m, 64);
        if (lane == 0) mid[row * rank + r] = has ? (T)(s * v) : (T)0.0f;
    }
}

template <typename T>
int launch_mid(const void* x, bool km, const void* down, const float* scale, const int32_t* ids, int adapters,
               int rank, int64_t rows, int64_t K, void* mid, hipStream_t s) {
    auto run = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3((unsigned)rows), dim3(kThreads), 0, s, static_cast<const T*>(x),
                           static_cast<const T*>(down), scale, ids, adapters, rank, K, static_cast<T*>(mid));
    };
    if (km) run(adapter_mid_kernel<T, true>);
    else run(adapter_mid_kernel<T, false>);
    HM_LAUNCHED();
    return HM_OK;
}

bool type16(int32_t dtype) { return dtype == HM_DTYPE_FP16 || dtype == HM_DTYPE_BF16; }
bool aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }
constexpr int64_t kMaxRows = ((int64_t)1 << 31) / kThreads - 1, kMaxDim = (int64_t)1 << 26,
                  kMaxMatrix = (int64_t)1 << 40, kMaxAdapters = 65535;

}  // namespace

extern "C" {

int hm_adapter_matmul(const void* x, int32_t dtype, const void* w, int32_t w_transposed, const void* down,
                      const void* up, const float* scale, const int32_t* ids, int64_t adapters, int64_t rank,
                      int64_t rows, int64_t inner, int64_t cols, void* mid, void* y, void* stream) {
    HM_REQUIRE(type16(dtype) && (w_transposed == 0 || w_transposed == 1));
    HM_REQUIRE(adapters >= 1 && rank >= 1 && rank <= HM_ADAPTER_MAX_RANK && rows >= 0 && inner >= 1 && cols >= 1);
    if (rows > kMaxRows || inner > kMaxDim || cols > kMaxDim || inner * cols > kMaxMatrix || adapters > kMaxAdapters) return HM_ERR_OVERFLOW;
    if (rows == 0) return HM_OK;
    HM_REQUIRE(x && w && down && up && scale && ids && mid && y && aligned(x, 2) && aligned(w, 2) &&
               aligned(down, 2) && aligned(up, 2) && aligned(scale, 4) && aligned(ids, 4) && aligned(mid, 2) &&
               aligned(y, 2));
    const int64_t ny = 2 * rows * cols, nm = 2 * rows * rank, nx = 2 * rows * inner, nw = 2 * inner * cols,
                  nd = 2 * adapters * rank * inner, nu = 2 * adapters * rank * cols;
    HM_REQUIRE(!hm_overlap(y, ny, x, nx) && !hm_overlap(y, ny, w, nw) && !hm_overlap(y, ny, down, nd) &&
               !hm_overlap(y, ny, up, nu) && !hm_overlap(y, ny, mid, nm) && !hm_overlap(mid, nm, x, nx) &&
               !hm_overlap(mid, nm, w, nw) && !hm_overlap(mid, nm, down, nd) && !hm_overlap(mid, nm, up, nu));
    const hipStream_t s = hm_stream(stream);
    const int rc = dtype == HM_DTYPE_FP16
                       ? launch_mid<hm_f16>(x, !w_transposed, down, scale, ids, (int)adapters, (int)rank, rows,
                                            inner, mid, s)
                       : launch_mid<hm_bf16>(x, !w_transposed, down, scale, ids, (int)adapters, (int)rank, rows,
                                             inner, mid, s);
    if (rc) return rc;
    GProduct p = {};
    p.x = x;
    p.w = w;
    p.y = y;
    p.rows = p.x_rows = rows;
    p.K = inner;
    p.N = cols;
    p.groups = 1;
    p.ids = ids;
    p.mid = mid;
    p.up = up;
    p.adapters = (int)adapters;
    p.rank = (int)rank;
    return hm_g_launch_generic(G_ADAPTER, !w_transposed, dtype, dtype, p, s);
}

size_t hm_adapter_weight_grad_workspace_bytes(int64_t adapters, int64_t rows, int64_t left_cols,
                                              int64_t right_cols) {
    (void)adapters, (void)rows, (void)left_cols, (void)right_cols;
    return 0;
}

int hm_adapter_weight_grad(const void* left, const void* right, int32_t dtype, const int32_t* ids,
                           int64_t adapters, int64_t rows, int64_t left_cols, int64_t right_cols, void* dw,
                           int32_t dw_dtype, int32_t accumulate, void* workspace, size_t workspace_bytes,
                           void* stream) {
    HM_REQUIRE(type16(dtype) && (dw_dtype == dtype || dw_dtype == HM_DTYPE_FP32) &&
               (accumulate == 0 || accumulate == 1));
    HM_REQUIRE(adapters >= 1 && rows >= 0 && left_cols >= 1 && right_cols >= 1);
    if (rows > kMaxRows || adapters > kMaxAdapters || left_cols > kMaxDim || right_cols > kMaxDim ||
        left_cols * right_cols > kMaxMatrix) return HM_ERR_OVERFLOW;
    HM_REQUIRE((rows == 0 || (left && right && ids)) && dw && aligned(left, 2) && aligned(right, 2) &&
               aligned(ids, 4) && aligned(dw, dw_dtype == HM_DTYPE_FP32 ? 4 : 2));
    const int64_t nw = adapters * left_cols * right_cols * (dw_dtype == HM_DTYPE_FP32 ? 4 : 2);
    HM_REQUIRE(!hm_overlap(dw, nw, left, 2 * rows * left_cols) && !hm_overlap(dw, nw, right, 2 * rows * right_cols));
    if (workspace_bytes < hm_adapter_weight_grad_workspace_bytes(adapters, rows, left_cols, right_cols))
        return HM_ERR_INVALID;
    GProduct p = {};
    p.x = left;
    p.w = right;
    p.y = dw;
    p.ids = ids;
    p.rows = rows;
    p.M = left_cols;
    p.N = right_cols;
    p.groups = (int)adapters;
    p.accumulate = accumulate;
    return hm_g_launch_generic(G_WEIGHT_GRAD, false, dtype, dw_dtype, p, hm_stream(stream));
}

}  // extern "C"
