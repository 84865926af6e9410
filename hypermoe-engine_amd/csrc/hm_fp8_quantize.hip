// hm_fp8_quantize.hip -- rows and weight blocks to block-scaled e4m3 (hm_fp8.h).
//
// Memory bound: every value is read once and stays in registers between its block's maximum and its
// conversion.
//   rows, contiguous columns   16 lanes hold one block, 8 values each; the maximum goes over the lanes
//                              by DPP, the 8 bytes of a lane are one store
//   blocks of 128 rows         one workgroup a block, 4 rows x 8 columns a lane
//   contiguous rows            (a transposed operand) 128 x 128 a workgroup, transposed as bytes, in the
//                              LDS
// 65536 x 4096 BF16 (0.8 GB): rows 164 us, 4.9 TB/s, blocks 144, contiguous rows 171 and 155; a copy
// of that size reaches 4.8.  4096 x 2048: 7.5 us, of which 3 are the launch's own.  Off 16 bytes value by
// value but for 16-bit rows: contiguous rows from an odd element 354 and 341, FP32 rows 457 (aligned 228).
#include "hm_fp8.h"

#include <limits.h>

namespace {

constexpr int kQThreads = 256;

// 8 consecutive values from p (VEC: 16-byte loads), zeros from column `left` on.  Unaligned 16-bit values
// come as the words that hold them, shifted by half a word where p is odd (65536 x 4095 of rows of 4096:
// 206 us against 342 value by value).
template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T* __restrict__ p, int64_t left, float (&v)[8]) {
    if (VEC && left >= 8) {
        constexpr int N = 16 / sizeof(T);
#pragma unroll
        for (int i = 0; i < 8 / N; ++i) {
            const hm_pack<T, N> w = reinterpret_cast<const hm_pack<T, N>*>(p)[i];
#pragma unroll
            for (int j = 0; j < N; ++j) v[i * N + j] = (float)w.v[j];
        }
    } else if (sizeof(T) == 2 && left >= 8) {
        const uint32_t* d = reinterpret_cast<const uint32_t*>((uintptr_t)p & ~(uintptr_t)3);
        const bool odd = ((uintptr_t)p & 2) != 0;
        const uint32_t w[5] = {d[0], d[1], d[2], d[3], d[odd ? 4 : 3]};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t u = __builtin_amdgcn_alignbit(w[i + 1], w[i], odd ? 16 : 0);
            hm_pack<T, 2> pair;
            __builtin_memcpy(&pair, &u, 4);
            v[2 * i] = (float)pair.v[0];
            v[2 * i + 1] = (float)pair.v[1];
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i < left ? (float)p[i] : 0.0f;
    }
}

template <typename T, bool VEC>
__device__ __forceinline__ void quantize_rows(const T* __restrict__ x, int64_t rows, int64_t width,
                                              int64_t stride, uint8_t* __restrict__ q,
                                              float* __restrict__ scale, int64_t block) {
    const int64_t nb = hm_f8_blocks(width);
    const int64_t g = block * (kQThreads / 16) + (threadIdx.x >> 4);
    const bool live = g < rows * nb;
    const int64_t gg = live ? g : 0;
    const int64_t r = gg / nb, kb = gg - r * nb;
    const int c = 8 * (threadIdx.x & 15);
    const int64_t k = kb * kF8Block + c;
    float v[8];
    load8<T, VEC>(x + r * stride + k, width - k, v);
    float amax = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) amax = hm_f8_amax(amax, v[i]);
    amax = hm_row16_max(amax);
    const hm_f8_scaler s = hm_f8_scaler_of(amax);
    if (!live) return;
    uint2 w;
    w.x = hm_f8_pack4(s, v[0], v[1], v[2], v[3]);
    w.y = hm_f8_pack4(s, v[4], v[5], v[6], v[7]);
    *reinterpret_cast<uint2*>(q + (r * nb + kb) * kF8Block + c) = w;
    if ((threadIdx.x & 15) == 0) scale[r * nb + kb] = s.scale;
}

template <typename T, bool VEC>
__global__ __launch_bounds__(kQThreads) void f8_quantize_rows_kernel(
    const T* __restrict__ x, int64_t rows, int64_t width, int64_t stride, uint8_t* __restrict__ q,
    float* __restrict__ scale) {
    quantize_rows<T, VEC>(x, rows, width, stride, q, scale, (int64_t)blockIdx.y * gridDim.x + blockIdx.x);
}

// The rows of an expert batch, and (workgroup 0) the table of its m-tiles: entry 0 their number, then
// {expert, first row, rows} of each, experts ascending.  A launch of its own would cost as much as the
// quantisation.  Offsets outside [0, pairs] are cut to it, tiles past `cap` dropped.
constexpr int kMaxTableExperts = 1024;

template <typename T, bool VEC>
__global__ __launch_bounds__(kQThreads) void f8_prepare_kernel(
    const T* __restrict__ x, int64_t rows, int64_t width, uint8_t* __restrict__ q,
    float* __restrict__ scale, const int32_t* __restrict__ offsets, int experts, int pairs, int bm,
    int cap, int4* __restrict__ table) {
    if (blockIdx.x > 0) {
        quantize_rows<T, VEC>(x, rows, width, width, q, scale, (int64_t)blockIdx.x - 1);
        return;
    }
    __shared__ int s_first[kMaxTableExperts + 1];   // an expert's first tile
    const int tid = threadIdx.x, lane = tid & 63;
    auto bounds = [&](int e, int* lo) __attribute__((always_inline)) {
        *lo = max(0, min(offsets[e], pairs));
        return max(0, min(offsets[e + 1], pairs) - *lo);
    };
    if (tid < 64) {
        int base = 0;
        for (int c0 = 0; c0 < experts; c0 += 64) {
            const int e = c0 + lane;
            int lo;
            const int n = e < experts ? (bounds(e, &lo) + bm - 1) / bm : 0;
            int incl = n;
#pragma unroll
            for (int s = 1; s < 64; s <<= 1) {
                const int o = __shfl_up(incl, s, 64);
                if (lane >= s) incl += o;
            }
            if (e < experts) s_first[e] = min(base + incl - n, cap);
            base = min(base + __shfl(incl, 63, 64), cap);
        }
        if (lane == 0) {
            s_first[experts] = base;
            table[0] = make_int4(base, 0, 0, 0);
        }
    }
    __syncthreads();
    const int total = s_first[experts];
    for (int t = tid; t < total; t += kQThreads) {
        int a = 0, b = experts;                     // s_first[a] <= t < s_first[b]
        while (b - a > 1) {
            const int m = (a + b) / 2;
            if (s_first[m] <= t) a = m;
            else b = m;
        }
        int lo;
        const int n = bounds(a, &lo), at = (t - s_first[a]) * bm;
        table[1 + t] = make_int4(a, lo + at, min(bm, n - at), 0);
    }
}

// The maximum over a workgroup of `waves` waves; every thread gets it.
__device__ __forceinline__ float block_max(float v, float* s_max, int waves) {
    v = hm_wave_max_dpp(v);
    if ((threadIdx.x & 63) == 0) s_max[threadIdx.x >> 6] = v;
    __syncthreads();
    float m = s_max[0];
    for (int i = 1; i < waves; ++i) m = fmaxf(m, s_max[i]);
    return m;
}

// Block (blockIdx.y, blockIdx.x) of 128 rows x 128 columns, columns contiguous.
template <typename T, bool VEC>
__global__ __launch_bounds__(512) void f8_quantize_blocks_kernel(
    const T* __restrict__ x, int64_t rows, int64_t width, int64_t stride, uint8_t* __restrict__ q,
    float* __restrict__ scale) {
    __shared__ float s_max[8];
    const int64_t nb = hm_f8_blocks(width);
    const int64_t kb = blockIdx.x, rb = blockIdx.y;
    const int c = 8 * (threadIdx.x & 15);
    const int64_t k = kb * kF8Block + c;
    const int64_t r0 = rb * kF8Block + (threadIdx.x >> 4);
    float v[4][8];
    float amax = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int64_t r = r0 + 32 * i;
        if (r < rows) {
            load8<T, VEC>(x + r * stride + k, width - k, v[i]);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[i][j] = 0.0f;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) amax = hm_f8_amax(amax, v[i][j]);
    }
    const hm_f8_scaler s = hm_f8_scaler_of(block_max(amax, s_max, 8));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int64_t r = r0 + 32 * i;
        if (r >= rows) break;
        uint2 w;
        w.x = hm_f8_pack4(s, v[i][0], v[i][1], v[i][2], v[i][3]);
        w.y = hm_f8_pack4(s, v[i][4], v[i][5], v[i][6], v[i][7]);
        *reinterpret_cast<uint2*>(q + (r * nb + kb) * kF8Block + c) = w;
    }
    if (threadIdx.x == 0) scale[rb * nb + kb] = s.scale;
}

// Contiguous rows: x[k ld + r].  A workgroup takes 128 rows x 128 columns.  A load is V values of one k
// (16 bytes where x is aligned, else one), 128 / V lanes side by side; a thread holds V rows x KT
// consecutive k, so that its bytes of a row are words.  They change owner in the LDS, from where whole
// 128-byte rows are stored: lanes that store their own words, or a row's 32 bytes, write the same lines
// from several waves (2.0 TB/s at 65536 x 4096 BF16 against 4.7).
template <typename T, int V, bool BLOCK>
__global__ __launch_bounds__(512) void f8_quantize_transposed_kernel(
    const T* __restrict__ x, int64_t rows, int64_t width, int64_t ld, uint8_t* __restrict__ q,
    float* __restrict__ scale) {
    constexpr int LK = kF8Block / V, KT = kF8Block * LK / 512, WORDS = KT / 4;
    constexpr int PARTS = 512 / LK;            // threads of a row
    constexpr int ROW = kF8Block / 4 + 1;      // words of a row in the LDS, and one against conflicts
    __shared__ uint32_t s_q[kF8Block * ROW];
    __shared__ float s_max[BLOCK ? 8 : PARTS * kF8Block];
    const int tid = threadIdx.x, part = tid / LK, rl = V * (tid % LK);
    const int64_t nb = hm_f8_blocks(width);
    const int64_t kb = blockIdx.x, row0 = (int64_t)blockIdx.y * kF8Block;
    const int64_t k0 = kb * kF8Block + part * KT, r0 = row0 + rl;
    float v[KT][V];
    float amax[V];
#pragma unroll
    for (int j = 0; j < V; ++j) amax[j] = 0.0f;
#pragma unroll
    for (int i = 0; i < KT; ++i) {
        const T* p = x + (k0 + i) * ld + r0;
        if (k0 + i < width && r0 + V <= rows) {
            const hm_pack<T, V> w = *reinterpret_cast<const hm_pack<T, V>*>(p);
#pragma unroll
            for (int j = 0; j < V; ++j) v[i][j] = (float)w.v[j];
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j) v[i][j] = k0 + i < width && r0 + j < rows ? (float)p[j] : 0.0f;
        }
    }
#pragma unroll
    for (int i = 0; i < KT; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) amax[j] = hm_f8_amax(amax[j], v[i][j]);
    if constexpr (BLOCK) {
#pragma unroll
        for (int j = 1; j < V; ++j) amax[0] = fmaxf(amax[0], amax[j]);
        amax[0] = block_max(amax[0], s_max, 8);
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j) s_max[part * kF8Block + rl + j] = amax[j];
        __syncthreads();
        if (tid < kF8Block) {
            float m = s_max[tid];
#pragma unroll
            for (int i = 1; i < PARTS; ++i) m = fmaxf(m, s_max[i * kF8Block + tid]);
            s_max[tid] = m;
            if (row0 + tid < rows) scale[(row0 + tid) * nb + kb] = hm_f8_scaler_of(m).scale;
        }
        __syncthreads();
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const hm_f8_scaler s = hm_f8_scaler_of(BLOCK ? amax[0] : s_max[rl + j]);
#pragma unroll
        for (int i = 0; i < WORDS; ++i)
            s_q[(rl + j) * ROW + part * WORDS + i] =
                hm_f8_pack4(s, v[4 * i][j], v[4 * i + 1][j], v[4 * i + 2][j], v[4 * i + 3][j]);
        if (BLOCK && tid == 0 && j == 0) scale[blockIdx.y * nb + kb] = s.scale;
    }
    __syncthreads();
#pragma unroll
    for (int h = 0; h < 2; ++h) {               // 8 lanes a row
        const int r = 64 * h + tid / 8, w = 4 * (tid % 8);
        if (row0 + r >= rows) break;
        const uint32_t* from = s_q + r * ROW + w;
        *reinterpret_cast<uint4*>(q + ((row0 + r) * nb + kb) * kF8Block + 4 * w) =
            make_uint4(from[0], from[1], from[2], from[3]);
    }
}

template <typename T>
int launch_quantize(const T* x, int64_t rows, int64_t width, int64_t row_stride, int64_t col_stride,
                    int32_t block_rows, uint8_t* q, float* scale, hipStream_t s) {
    const int64_t nb = hm_f8_blocks(width);
    if (col_stride == 1) {
        const bool vec = (uintptr_t)x % 16 == 0 && row_stride % (16 / (int64_t)sizeof(T)) == 0;
        if (block_rows == 1) {
            // a grid's first dimension holds 2^31 - 1 lanes, its second 65535 times that
            if (rows > ((int64_t)1 << 42) / nb) return HM_ERR_OVERFLOW;
            const int64_t groups = (rows * nb + kQThreads / 16 - 1) / (kQThreads / 16);
            const int64_t deep = (groups + INT_MAX / kQThreads - 1) / (INT_MAX / kQThreads);
            hipLaunchKernelGGL((vec ? f8_quantize_rows_kernel<T, true> : f8_quantize_rows_kernel<T, false>),
                               dim3((unsigned)((groups + deep - 1) / deep), (unsigned)deep), dim3(kQThreads),
                               0, s, x, rows, width, row_stride, q, scale);
        } else {
            const int64_t rb = hm_f8_blocks(rows);
            if (rb > 65535 || nb > INT_MAX / 512) return HM_ERR_OVERFLOW;
            hipLaunchKernelGGL((vec ? f8_quantize_blocks_kernel<T, true> : f8_quantize_blocks_kernel<T, false>),
                               dim3((unsigned)nb, (unsigned)rb), dim3(512), 0, s, x, rows, width,
                               row_stride, q, scale);
        }
    } else {
        constexpr int V = 16 / sizeof(T);
        const int64_t rb = hm_f8_blocks(rows);
        if (rb > 65535 || nb > INT_MAX / 512) return HM_ERR_OVERFLOW;
        const bool vec = (uintptr_t)x % 16 == 0 && col_stride % V == 0;
        auto run = [&](auto kernel) {
            hipLaunchKernelGGL(kernel, dim3((unsigned)nb, (unsigned)rb), dim3(512), 0, s, x, rows, width,
                               col_stride, q, scale);
        };
        if (block_rows == 1)
            vec ? run(f8_quantize_transposed_kernel<T, V, false>) : run(f8_quantize_transposed_kernel<T, 1, false>);
        else
            vec ? run(f8_quantize_transposed_kernel<T, V, true>) : run(f8_quantize_transposed_kernel<T, 1, true>);
    }
    HM_LAUNCHED();
    return HM_OK;
}

template <typename T>
int launch_prepare(const T* x, int64_t rows, int64_t width, uint8_t* q, float* scale,
                   const int32_t* offsets, int experts, int pairs, int bm, int cap, int4* table,
                   hipStream_t s) {
    const bool vec = (uintptr_t)x % 16 == 0 && width % (16 / (int64_t)sizeof(T)) == 0;
    const int64_t grid = (rows * hm_f8_blocks(width) + kQThreads / 16 - 1) / (kQThreads / 16) + 1;
    if (grid > INT_MAX / kQThreads) return HM_ERR_OVERFLOW;
    hipLaunchKernelGGL((vec ? f8_prepare_kernel<T, true> : f8_prepare_kernel<T, false>),
                       dim3((unsigned)grid), dim3(kQThreads), 0, s, x, rows, width, q, scale, offsets,
                       experts, pairs, bm, cap, table);
    HM_LAUNCHED();
    return HM_OK;
}

}  // namespace

// x [rows x width] to FP8, and the m-tile table of a batch of at most kMaxTableExperts experts.
int hm_f8_launch_prepare(const void* x, int32_t dtype, int64_t rows, int64_t width, uint8_t* q,
                         float* scale, const int32_t* offsets, int experts, int pairs, int bm, int cap,
                         int4* table, hipStream_t s) {
    switch (dtype) {
    case HM_DTYPE_FP32:
        return launch_prepare(static_cast<const float*>(x), rows, width, q, scale, offsets, experts,
                              pairs, bm, cap, table, s);
    case HM_DTYPE_FP16:
        return launch_prepare(static_cast<const hm_f16*>(x), rows, width, q, scale, offsets, experts,
                              pairs, bm, cap, table, s);
    default:
        return launch_prepare(static_cast<const hm_bf16*>(x), rows, width, q, scale, offsets, experts,
                              pairs, bm, cap, table, s);
    }
}

extern "C" {

int64_t hm_fp8_pitch(int64_t width) { return width > 0 ? hm_f8_pitch(width) : 0; }

int hm_fp8_quantize(const void* x, int32_t dtype, int64_t rows, int64_t width, int64_t row_stride,
                    int64_t col_stride, int32_t block_rows, uint8_t* q, float* scale, void* stream) {
    HM_REQUIRE(x && q && scale && rows >= 0 && width > 0);
    HM_REQUIRE(hm_row_dtype(dtype) && (block_rows == 1 || block_rows == kF8Block));
    HM_REQUIRE((uintptr_t)x % hm_row_dtype_size(dtype) == 0 && (uintptr_t)q % 16 == 0 &&
               (uintptr_t)scale % 4 == 0);
    HM_REQUIRE(row_stride > 0 && col_stride > 0 && (row_stride == 1 || col_stride == 1));
    if (rows == 0) return HM_OK;
    if (rows > (int64_t)1 << 40 || width > (int64_t)1 << 31 ||
        rows > INT64_MAX / 8 / row_stride || width > INT64_MAX / 8 / col_stride)
        return HM_ERR_OVERFLOW;
    hipStream_t s = hm_stream(stream);
    switch (dtype) {
    case HM_DTYPE_FP32:
        return launch_quantize(static_cast<const float*>(x), rows, width, row_stride, col_stride,
                               block_rows, q, scale, s);
    case HM_DTYPE_FP16:
        return launch_quantize(static_cast<const hm_f16*>(x), rows, width, row_stride, col_stride,
                               block_rows, q, scale, s);
    default:
        return launch_quantize(static_cast<const hm_bf16*>(x), rows, width, row_stride, col_stride,
                               block_rows, q, scale, s);
    }
}

}  // extern "C"
