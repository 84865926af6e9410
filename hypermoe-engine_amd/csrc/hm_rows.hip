// hm_rows.hip -- token rows to expert order and back with the routing weights applied, and the
// gradients of both, for FP32, FP16 and BF16 rows.
//
// With slot(t, r) the grouped row of token t's r-th expert and w its weight:
//   dispatch       rows[slot(t,r)] = w x[t]                   dw = <g[slot(t,r)], x[t]>,
//                                                             dx[t] = sum_r w g[slot(t,r)]
//   combine        out[t] = res[t] + sum_r w y[slot(t,r)]     dw = <g[t], y[slot(t,r)]>,
//                                                             dy[slot(t,r)] = w g[t]
// so there are two movements, each the other's gradient: `spread` writes a token's row to its slots and
// takes the dot products in the same pass; `join` sums a token's slots and takes theirs in a second pass
// over the same rows.  A pair with a slot outside [0, rows) is one that no expert took: it is written
// nowhere, adds nothing and has weight gradient 0.
//
// Bound by the rows' bytes (one read or write each; the products are a few operations a value).  A
// workgroup owns a token, or without dot products a column chunk of it, so every sum has one owner
// and a fixed order (ranks ascending): no atomics, the same bits every run.  4096 tokens, top-8, 2048
// wide, BF16: dispatch 26 us (151 MB), join 26 to 47 (168 MB; the least where the rows are still in the
// caches), with dot products 49, combine's gradient with both results 49 (285 MB): 4.2 to 5.8 TB/s where a
// large copy reaches 4.8.
#include "hm_fp8.h"

#include <limits.h>

namespace {

constexpr int kRThreads = 256;
constexpr int kRanks = 8;   // ranks walked at once: their row loads are in flight together

// V consecutive values of a row: 16 bytes where the rows are aligned to that, else 2 values (4096 tokens,
// top-8, BF16, forward and backward: 2048 wide 155 us, 2046 226; by single values 336), else one.
template <typename T, int V>
struct Chunk {
    float v[V];
    __device__ __forceinline__ void load(const T* p) {
        const hm_pack<T, V> w = *reinterpret_cast<const hm_pack<T, V>*>(p);
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = (float)w.v[i];
    }
    __device__ __forceinline__ void store(T* p) const {
        hm_pack<T, V> w;
#pragma unroll
        for (int i = 0; i < V; ++i) w.v[i] = (T)v[i];
        *reinterpret_cast<hm_pack<T, V>*>(p) = w;
    }
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = 0.0f;
    }
};

// Sums of kRanks values over the workgroup, in a fixed order (lanes, then waves); dots[r] for
// r < ranks goes to `to`.  Every thread calls it.
__device__ __forceinline__ void reduce_dots(float (&dots)[kRanks], int ranks, float* to) {
    __shared__ float s[kRThreads / 64][kRanks];
#pragma unroll
    for (int r = 0; r < kRanks; ++r) {
        float v = dots[r];
#pragma unroll
        for (int m = 32; m >= 1; m >>= 1) v += __shfl_xor(v, m, 64);
        if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6][r] = v;
    }
    __syncthreads();
    if ((int)threadIdx.x < ranks) {
        float v = s[0][threadIdx.x];
#pragma unroll
        for (int w = 1; w < kRThreads / 64; ++w) v += s[w][threadIdx.x];
        to[threadIdx.x] = v;
    }
    __syncthreads();
}

// rows[slot(t,r)] = w src[t]; DOT: dots[t,r] = <src[t], other[slot(t,r)]>.
template <typename T, int V, bool DOT>
__global__ __launch_bounds__(kRThreads) void rows_spread_kernel(
    const T* __restrict__ src, const T* __restrict__ other, const int32_t* __restrict__ slots,
    const float* __restrict__ weights, int top_k, int64_t rows, int64_t width, T* __restrict__ out,
    float* __restrict__ dots) {
    const int64_t t = blockIdx.x;
    const int32_t* ts = slots + t * top_k;
    const int64_t step = (int64_t)gridDim.y * kRThreads * V;
    const int64_t c0 = ((int64_t)blockIdx.y * kRThreads + threadIdx.x) * V;
    for (int r0 = 0; r0 < top_k; r0 += kRanks) {
        const int n = min(kRanks, top_k - r0);
        float d[kRanks];
#pragma unroll
        for (int i = 0; i < kRanks; ++i) d[i] = 0.0f;
        for (int64_t c = c0; c < width; c += step) {
            Chunk<T, V> x;
            x.load(src + t * width + c);
#pragma unroll
            for (int i = 0; i < kRanks; ++i) {
                if (i >= n) break;
                const int64_t slot = ts[r0 + i];
                if (slot < 0 || slot >= rows) continue;
                Chunk<T, V> y;
                if constexpr (DOT) {
                    y.load(other + slot * width + c);
#pragma unroll
                    for (int j = 0; j < V; ++j) d[i] = __builtin_fmaf(x.v[j], y.v[j], d[i]);
                }
                if (weights) {
                    const float w = weights[t * top_k + r0 + i];
#pragma unroll
                    for (int j = 0; j < V; ++j) y.v[j] = w * x.v[j];
                } else {
                    y = x;
                }
                y.store(out + slot * width + c);
            }
        }
        if constexpr (DOT) reduce_dots(d, n, dots + t * top_k + r0);
    }
}

// dst[t] = (residual[t]) + sum_r w src[slot(t,r)]; DOT: dots[t,r] = <other[t], src[slot(t,r)]>.
template <typename T, int V, bool DOT>
__global__ __launch_bounds__(kRThreads) void rows_join_kernel(
    const T* __restrict__ src, const T* __restrict__ other, const int32_t* __restrict__ slots,
    const float* __restrict__ weights, const T* residual, int top_k, int64_t rows, int64_t width,
    T* dst, float* __restrict__ dots) {  // (residual may be dst)
    const int64_t t = blockIdx.x;
    const int32_t* ts = slots + t * top_k;
    const int64_t step = (int64_t)gridDim.y * kRThreads * V;
    const int64_t c0 = ((int64_t)blockIdx.y * kRThreads + threadIdx.x) * V;
    for (int64_t c = c0; c < width; c += step) {
        Chunk<T, V> acc;
        acc.zero();
        for (int r = 0; r < top_k; ++r) {
            const int64_t slot = ts[r];
            if (slot < 0 || slot >= rows) continue;
            Chunk<T, V> y;
            y.load(src + slot * width + c);
            const float w = weights ? weights[t * top_k + r] : 1.0f;
#pragma unroll
            for (int j = 0; j < V; ++j) acc.v[j] = __builtin_fmaf(w, y.v[j], acc.v[j]);
        }
        if (residual) {
            Chunk<T, V> y;
            y.load(residual + t * width + c);
#pragma unroll
            for (int j = 0; j < V; ++j) acc.v[j] = y.v[j] + acc.v[j];
        }
        acc.store(dst + t * width + c);
    }
    if constexpr (DOT) {
        for (int r0 = 0; r0 < top_k; r0 += kRanks) {
            const int n = min(kRanks, top_k - r0);
            float d[kRanks];
#pragma unroll
            for (int i = 0; i < kRanks; ++i) d[i] = 0.0f;
            for (int64_t c = c0; c < width; c += step) {
                Chunk<T, V> x;
                x.load(other + t * width + c);
#pragma unroll
                for (int i = 0; i < kRanks; ++i) {
                    if (i >= n) break;
                    const int64_t slot = ts[r0 + i];
                    if (slot < 0 || slot >= rows) continue;
                    Chunk<T, V> y;
                    y.load(src + slot * width + c);
#pragma unroll
                    for (int j = 0; j < V; ++j) d[i] = __builtin_fmaf(x.v[j], y.v[j], d[i]);
                }
            }
            reduce_dots(d, n, dots + t * top_k + r0);
        }
    }
}

// What the four entry points ask of their sizes.
int check_rows(const int32_t* slots, const float* weights, int64_t tokens, int32_t top_k,
               int64_t rows, int64_t width, int32_t dtype) {
    HM_REQUIRE(slots && hm_row_dtype(dtype));
    HM_REQUIRE(tokens >= 0 && top_k > 0 && rows >= 0 && width > 0);
    HM_REQUIRE((uintptr_t)slots % 4 == 0 && (uintptr_t)weights % 4 == 0);
    if (tokens > INT_MAX / kRThreads || top_k > 65535 || rows > INT_MAX || width > INT_MAX)
        return HM_ERR_OVERFLOW;
    return HM_OK;
}

bool aligned(const void* p, uintptr_t to) { return (uintptr_t)p % to == 0; }

dim3 rows_grid(int64_t tokens, int64_t width, int v, bool whole_rows) {
    const int64_t chunks = (width + (int64_t)kRThreads * v - 1) / ((int64_t)kRThreads * v);
    return dim3((unsigned)tokens, whole_rows ? 1u : (unsigned)(chunks > 64 ? 64 : chunks));
}

template <typename T>
int spread(const void* src, const void* other, const int32_t* slots, const float* weights,
           int64_t tokens, int32_t top_k, int64_t rows, int64_t width, void* out, float* dots,
           hipStream_t s) {
    constexpr int V = 16 / sizeof(T);
    const bool vec = width % V == 0 && aligned(src, 16) && aligned(other, 16) && aligned(out, 16);
    constexpr uintptr_t P = 2 * sizeof(T);
    const bool pairs = width % 2 == 0 && aligned(src, P) && aligned(other, P) && aligned(out, P);
    auto run = [&](auto kernel, int v) {
        hipLaunchKernelGGL(kernel, rows_grid(tokens, width, v, dots != nullptr), dim3(kRThreads), 0, s,
                           static_cast<const T*>(src), static_cast<const T*>(other), slots, weights,
                           (int)top_k, rows, width, static_cast<T*>(out), dots);
    };
    if (dots)
        vec ? run(rows_spread_kernel<T, V, true>, V)
        : pairs ? run(rows_spread_kernel<T, 2, true>, 2) : run(rows_spread_kernel<T, 1, true>, 1);
    else
        vec ? run(rows_spread_kernel<T, V, false>, V)
        : pairs ? run(rows_spread_kernel<T, 2, false>, 2) : run(rows_spread_kernel<T, 1, false>, 1);
    HM_LAUNCHED();
    return HM_OK;
}

template <typename T>
int join(const void* src, const void* other, const int32_t* slots, const float* weights,
         const void* residual, int64_t tokens, int32_t top_k, int64_t rows, int64_t width, void* dst,
         float* dots, hipStream_t s) {
    constexpr int V = 16 / sizeof(T);
    const bool vec = width % V == 0 && aligned(src, 16) && aligned(other, 16) &&
                     aligned(residual, 16) && aligned(dst, 16);
    constexpr uintptr_t P = 2 * sizeof(T);
    const bool pairs = width % 2 == 0 && aligned(src, P) && aligned(other, P) &&
                       aligned(residual, P) && aligned(dst, P);
    auto run = [&](auto kernel, int v) {
        hipLaunchKernelGGL(kernel, rows_grid(tokens, width, v, dots != nullptr), dim3(kRThreads), 0, s,
                           static_cast<const T*>(src), static_cast<const T*>(other), slots, weights,
                           static_cast<const T*>(residual), (int)top_k, rows, width,
                           static_cast<T*>(dst), dots);
    };
    if (dots)
        vec ? run(rows_join_kernel<T, V, true>, V)
        : pairs ? run(rows_join_kernel<T, 2, true>, 2) : run(rows_join_kernel<T, 1, true>, 1);
    else
        vec ? run(rows_join_kernel<T, V, false>, V)
        : pairs ? run(rows_join_kernel<T, 2, false>, 2) : run(rows_join_kernel<T, 1, false>, 1);
    HM_LAUNCHED();
    return HM_OK;
}

#define HM_BY_DTYPE(dtype, fn, ...)                                    \
    ((dtype) == HM_DTYPE_FP32   ? fn<float>(__VA_ARGS__)               \
     : (dtype) == HM_DTYPE_FP16 ? fn<hm_f16>(__VA_ARGS__)              \
                                : fn<hm_bf16>(__VA_ARGS__))

}  // namespace

extern "C" {

int hm_dispatch_rows(const void* x, const int32_t* slots, const float* weights, int64_t tokens,
                     int32_t top_k, int64_t rows, int64_t width, int32_t dtype, void* out,
                     void* stream) {
    const int rc = check_rows(slots, weights, tokens, top_k, rows, width, dtype);
    if (rc) return rc;
    HM_REQUIRE(x && (out || rows == 0) && x != out);
    const size_t size = hm_row_dtype_size(dtype);
    HM_REQUIRE(aligned(x, size) && aligned(out, size));
    if (tokens == 0 || rows == 0) return HM_OK;
    return HM_BY_DTYPE(dtype, spread, x, nullptr, slots, weights, tokens, top_k, rows, width, out,
                       nullptr, hm_stream(stream));
}

int hm_dispatch_rows_grad(const void* dout, const void* x, const int32_t* slots,
                          const float* weights, int64_t tokens, int32_t top_k, int64_t rows,
                          int64_t width, int32_t dtype, void* dx, float* dweights, void* stream) {
    const int rc = check_rows(slots, weights, tokens, top_k, rows, width, dtype);
    if (rc) return rc;
    HM_REQUIRE((dout || rows == 0) && dx && dout != dx && x != dx);
    HM_REQUIRE(!dweights || (x && weights));  // without weights there is no gradient of theirs
    const size_t size = hm_row_dtype_size(dtype);
    HM_REQUIRE(aligned(dout, size) && aligned(x, size) && aligned(dx, size) && aligned(dweights, 4));
    if (tokens == 0) return HM_OK;
    return HM_BY_DTYPE(dtype, join, dout, dweights ? x : nullptr, slots, weights, nullptr, tokens,
                       top_k, rows, width, dx, dweights, hm_stream(stream));
}

int hm_combine_rows(const void* y, const int32_t* slots, const float* weights, const void* residual,
                    int64_t tokens, int32_t top_k, int64_t rows, int64_t width, int32_t dtype,
                    void* out, void* stream) {
    const int rc = check_rows(slots, weights, tokens, top_k, rows, width, dtype);
    if (rc) return rc;
    HM_REQUIRE((y || rows == 0) && out && y != out);
    const size_t size = hm_row_dtype_size(dtype);
    HM_REQUIRE(aligned(y, size) && aligned(residual, size) && aligned(out, size));
    if (tokens == 0) return HM_OK;
    return HM_BY_DTYPE(dtype, join, y, nullptr, slots, weights, residual, tokens, top_k, rows, width,
                       out, nullptr, hm_stream(stream));
}

int hm_combine_rows_grad(const void* dout, const void* y, const int32_t* slots, const float* weights,
                         int64_t tokens, int32_t top_k, int64_t rows, int64_t width, int32_t dtype,
                         void* dy, float* dweights, void* stream) {
    const int rc = check_rows(slots, weights, tokens, top_k, rows, width, dtype);
    if (rc) return rc;
    HM_REQUIRE(dout && (dy || rows == 0) && dout != dy && (!y || y != dy));
    HM_REQUIRE(!dweights || ((y || rows == 0) && weights));
    const size_t size = hm_row_dtype_size(dtype);
    HM_REQUIRE(aligned(dout, size) && aligned(y, size) && aligned(dy, size) && aligned(dweights, 4));
    if (tokens == 0 || (rows == 0 && !dweights)) return HM_OK;
    return HM_BY_DTYPE(dtype, spread, dout, dweights ? y : nullptr, slots, weights, tokens, top_k,
                       rows, width, dy, dweights, hm_stream(stream));
}

}  // extern "C"
