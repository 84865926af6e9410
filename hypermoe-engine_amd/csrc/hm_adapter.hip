// hm_adapter.hip -- low-rank adapters of many requests beside a shared projection:
//   mid[t] = s_a x[t] A_a^T,  y[t] = x[t] W^T + mid[t] B_a^T,  a = ids[t]
// the input's gradient by the same entry point with the matrices transposed, and the adapters' gradients
//   d_a = sum over the rows t of adapter a of  left[t]^T right[t].
// mid is held in the operands' 16 bits: it is an operand of the second product's matrix instructions and of B's gradient,
// and half a step of it (BF16 2^-8) is that much of the adapter's part of y alone, beside y's own rounding.
#include "hm_grouped.h"

#include <limits.h>

#include <algorithm>
#include <type_traits>

namespace {

constexpr int kThreads = 256;

// ---- mid
// Few rows, each perhaps with an adapter of its own: a wave takes one rank of one row (k-major), or a workgroup 16
// ranks of one row, k in 16 parts.  Bound by latency: 32 rows, rank 16 of 2048, 4.3 us.
template <typename T, bool KM>
__global__ __launch_bounds__(kThreads) void adapter_mid_rows_kernel(const T* __restrict__ x,
                                                                    const T* __restrict__ down,
                                                                    const float* __restrict__ scale,
                                                                    const int32_t* __restrict__ ids, int adapters,
                                                                    int rank, int64_t K, T* __restrict__ mid) {
    const int64_t row = blockIdx.x;
    const int a = ids[row];
    const bool has = a >= 0 && a < adapters;
    const T* xr = x + row * K;
    const T* d = down + (int64_t)(has ? a : 0) * rank * K;
    if constexpr (KM) {
        const int lane = threadIdx.x & 63, r = (int)blockIdx.y * (kThreads / 64) + (threadIdx.x >> 6);
        if (r >= rank) return;
        float v = 0.0f;
        if (has) {
            const T* dr = d + (int64_t)r * K;
#pragma unroll 4
            for (int64_t k = 8 * lane; k < K; k += 512) {
                float p[8], q[8];
                load8(xr + k, (int)min(K - k, (int64_t)8), p);
                load8(dr + k, (int)min(K - k, (int64_t)8), q);
#pragma unroll
                for (int i = 0; i < 8; ++i) v = __builtin_fmaf(p[i], q[i], v);
            }
        }
#pragma unroll
        for (int m = 32; m >= 1; m >>= 1) v += __shfl_xor(v, m, 64);
        if (lane == 0) mid[row * rank + r] = has ? (T)(scale[a] * v) : (T)0.0f;
    } else {
        __shared__ float s_part[16][17];
        const int c = threadIdx.x & 15, part = threadIdx.x >> 4, r = (int)blockIdx.y * 16 + c;
        float v = 0.0f;
        if (has && r < rank) {
#pragma unroll 8
            for (int64_t k = part; k < K; k += 16) v = __builtin_fmaf((float)xr[k], (float)d[k * rank + r], v);
        }
        s_part[part][c] = v;
        __syncthreads();
        if (part == 0 && r < rank) {
            for (int i = 1; i < 16; ++i) v += s_part[i][c];
            mid[row * rank + r] = has ? (T)(scale[a] * v) : (T)0.0f;
        }
    }
}

// More rows: a workgroup takes 16 rows and 16 RF ranks, its 8 waves k in parts of 64, straight from memory into
// fragments (x is read once; the adapters' matrices, read by every workgroup, stay in the L2 and bound it); once for
// each adapter that the rows name, its own rows kept.  The waves' sums meet in the LDS in wave order.
constexpr int kMidWaves = 8;

template <typename T, bool KM, int RF>
__global__ __launch_bounds__(64 * kMidWaves, 2) void adapter_mid_tile_kernel(const T* __restrict__ x,
                                                                          const T* __restrict__ down,
                                                                          const float* __restrict__ scale,
                                                                          const int32_t* __restrict__ ids,
                                                                          int adapters, int rank, int64_t rows,
                                                                          int64_t K, T* __restrict__ mid) {
    typedef typename Elem16<T>::v8 v8;
    constexpr int kPart = 64 * kMidWaves;
    __shared__ v4f s_part[kMidWaves][RF][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int i16 = lane & 15, g = lane >> 4;
    const int64_t row0 = (int64_t)blockIdx.x * 16, row = row0 + i16;
    const int r0 = (int)blockIdx.y * 16 * RF;
    int mine = row < rows ? ids[row] : -1;
    if (mine >= adapters) mine = -1;
    const T* xr = x + min(row, rows - 1) * K;
    // rows without adapter
    for (int q = threadIdx.x; q < 16 * 16 * RF; q += 64 * kMidWaves) {
        const int r = r0 + q % (16 * RF), m = q / (16 * RF);
        if (row0 + m >= rows || r >= rank) continue;
        const int id = ids[row0 + m];
        if (id < 0 || id >= adapters) mid[(row0 + m) * rank + r] = (T)0.0f;
    }
    int cur = -1;
    while (true) {
        cur = wave_min(mine > cur ? mine : INT_MAX);
        if (cur == INT_MAX) break;
        const T* d = down + (int64_t)cur * rank * K;
        v4f acc[RF] = {};
        int64_t k0 = 64 * wave;
        // U parts at a time, all their loads in flight; `whole`: within K
        auto parts = [&](auto u_, bool whole) __attribute__((always_inline)) {
            constexpr int U = decltype(u_)::value;
            v8 xf[U][2], df[U][2][RF];
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int64_t k = k0 + kPart * u + 32 * h + 8 * g, n = whole ? 8 : K - k;
                    xf[u][h] = load_frag8<T>(xr + k, n);
#pragma unroll
                    for (int f = 0; f < RF; ++f) {
                        const int r = min(r0 + 16 * f + i16, rank - 1);   // (ranks past the last are dropped)
                        if constexpr (KM) {
                            df[u][h][f] = load_frag8<T>(d + (int64_t)r * K + k, n);
                        } else {
                            Loose8<T> w;
#pragma unroll
                            for (int i = 0; i < 8; ++i) w.v[i] = whole || i < n ? d[(k + i) * rank + r] : (T)0.0f;
                            df[u][h][f] = __builtin_bit_cast(v8, w);
                        }
                    }
                }
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int f = 0; f < RF; ++f) acc[f] = Elem16<T>::mfma(df[u][h][f], xf[u][h], acc[f]);
            k0 += kPart * U;
        };
        constexpr int U = KM ? 4 : 2;
        while (k0 + kPart * (U - 1) + 64 <= K) parts(std::integral_constant<int, U>{}, true);
        while (k0 < K) parts(std::integral_constant<int, 1>{}, false);
#pragma unroll
        for (int f = 0; f < RF; ++f) s_part[wave][f][lane] = acc[f];
        __syncthreads();
        // entry (f, lane): row i16, ranks 4 g .. of fragment f; a wave each
        if (wave < RF) {
            v4f v = s_part[0][wave][lane];
#pragma unroll
            for (int w = 1; w < kMidWaves; ++w) v += s_part[w][wave][lane];
            if (mine == cur) {
                const float s = scale[cur];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int r = r0 + 16 * wave + 4 * g + j;
                    if (r < rank) mid[row * rank + r] = (T)(s * v[j]);
                }
            }
        }
        __syncthreads();
    }
}

constexpr int64_t kMidRows = 256;   // rows up to which mid is taken row by row

template <typename T>
int launch_mid(const void* x_, bool km, const void* down_, const float* scale, const int32_t* ids, int adapters,
               int rank, int64_t rows, int64_t K, void* mid_, hipStream_t s) {
    const T *x = static_cast<const T*>(x_), *down = static_cast<const T*>(down_);
    T* mid = static_cast<T*>(mid_);
    if (rows <= kMidRows) {
        const dim3 grid((unsigned)rows, (unsigned)((rank + (km ? 3 : 15)) / (km ? 4 : 16)));
        auto run = [&](auto kernel) {
            hipLaunchKernelGGL(kernel, grid, dim3(kThreads), 0, s, x, down, scale, ids, adapters, rank, K, mid);
        };
        if (km) run(adapter_mid_rows_kernel<T, true>);
        else run(adapter_mid_rows_kernel<T, false>);
    } else {
        const int rf = rank <= 16 ? 1 : rank <= 32 ? 2 : 4;
        const dim3 grid((unsigned)((rows + 15) / 16), (unsigned)((rank + 16 * rf - 1) / (16 * rf)));
        auto run = [&](auto kernel) {
            hipLaunchKernelGGL(kernel, grid, dim3(64 * kMidWaves), 0, s, x, down, scale, ids, adapters, rank, rows, K, mid);
        };
        if (rf == 1) km ? run(adapter_mid_tile_kernel<T, true, 1>) : run(adapter_mid_tile_kernel<T, false, 1>);
        else if (rf == 2) km ? run(adapter_mid_tile_kernel<T, true, 2>) : run(adapter_mid_tile_kernel<T, false, 2>);
        else km ? run(adapter_mid_tile_kernel<T, true, 4>) : run(adapter_mid_tile_kernel<T, false, 4>);
    }
    HM_LAUNCHED();
    return HM_OK;
}

// ---- the matrices' gradients
// A workgroup takes a 64 x 64 tile of the gradients over one part of the rows, for every gridDim.y-th adapter in turn:
// it collects the rows that are the adapter's, up to 256 at a time (in ascending order, so sums have one order), loads those rows' columns, and takes
// them 64 at a time through the LDS, where they are read transposed.  Parts meet in a second kernel; a part without rows
// of an adapter is a flag and no more.  LDS rows are 64 columns of one row, 128 bytes, piece c at c ^ s(row): the 8 rows
// that the LDS serves at once lie on all of its banks.
// Bound by round trips: the ids, the rows, and the parts' sums: 2048 rows, 4 adapters, [16 x 2048] 10.8 us and the sums 4.2.
constexpr int kGT = 64;
constexpr int kScan = 1024;   // ids that a wave looks at at once
constexpr int kRound = 256;   // rows that are loaded at once

// EVEN: L and R are multiples of 8, so every piece is whole or absent and loads have no branches.  (The kernel runs
// through its code about once, so the time goes with the code's length: instructions come from the L2.)
template <typename T, typename O, bool EVEN>
__global__ __launch_bounds__(kThreads) void adapter_grad_kernel(const T* __restrict__ left, const T* __restrict__ right,
                                                                const int32_t* __restrict__ ids, int64_t rows,
                                                                int64_t L, int64_t R, int64_t part_rows,
                                                                float* __restrict__ parts, int32_t* __restrict__ flags,
                                                                O* __restrict__ dw, int adapters, int accumulate) {
    typedef typename Elem16<T>::v8 v8;
    __shared__ __attribute__((aligned(16))) uint8_t s_l[kGT * 128], s_r[kGT * 128];
    __shared__ int s_list[4][2 * kRound];   // (each wave its own)
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int wm = wave >> 1, wn = wave & 1, i16 = lane & 15, g = lane >> 4;
    const int64_t ntr = (R + kGT - 1) / kGT;
    const int64_t l0 = (int64_t)blockIdx.x / ntr * kGT, c0 = (int64_t)blockIdx.x % ntr * kGT;
    const int64_t beg = (int64_t)blockIdx.z * part_rows, end = min(beg + part_rows, rows);
    auto swz = [](int r) { return (r & 2) | ((r & 8) >> 1); };
    const int trow = 8 * g + (i16 >> 2), tc = i16 & 3;
    const int at0 = trow * 128 + 8 * (tc & 1), pc = tc >> 1;
    v4f acc[2][2] = {};
    int head = 0, count = 0;
    bool any = false;
    auto round = [&](int n) __attribute__((always_inline)) {   // the first n of the list
        constexpr int S = kRound / kGT;
        v8 v[S][2][2];
#pragma unroll
        for (int s = 0; s < S; ++s) {
            if (kGT * s >= n) break;
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int q = t + kThreads * u, k = kGT * s + (q >> 3), col = 8 * (q & 7);
                const int64_t row = k < n ? s_list[wave][(head + k) & (2 * kRound - 1)] : -1;
                if constexpr (EVEN) {
                    const bool il = row >= 0 && l0 + col < L, ir = row >= 0 && c0 + col < R;
                    const u64x2 vl = load16(left + (il ? row * L + l0 + col : 0));
                    const u64x2 vr = load16(right + (ir ? row * R + c0 + col : 0));
                    v[s][0][u] = __builtin_bit_cast(v8, il ? vl : u64x2{});
                    v[s][1][u] = __builtin_bit_cast(v8, ir ? vr : u64x2{});
                } else {
                    const T *pl = left + row * L + l0 + col, *pr = right + row * R + c0 + col;
                    v[s][0][u] = load_frag8<T>(pl, row >= 0 ? min(L - l0 - col, (int64_t)8) : 0);
                    v[s][1][u] = load_frag8<T>(pr, row >= 0 ? min(R - c0 - col, (int64_t)8) : 0);
                }
            }
        }
#pragma unroll
        for (int s = 0; s < S; ++s) {
            if (kGT * s >= n) break;
            __syncthreads();
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int q = t + kThreads * u, k = q >> 3, at = k * 128 + 16 * ((q & 7) ^ swz(k));
                *reinterpret_cast<v8*>(s_l + at) = v[s][0][u];
                *reinterpret_cast<v8*>(s_r + at) = v[s][1][u];
            }
            __syncthreads();
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if (kGT * s + 32 * h >= n) break;
                v8 a[2], b[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int at = at0 + 32 * h * 128;
                    b[i] = read_transposed<v8>(s_l + at + 16 * ((4 * wm + 2 * i + pc) ^ swz(trow)), 4 * 128);
                    a[i] = read_transposed<v8>(s_r + at + 16 * ((4 * wn + 2 * i + pc) ^ swz(trow)), 4 * 128);
                }
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int j = 0; j < 2; ++j) acc[i][j] = Elem16<T>::mfma(a[j], b[i], acc[i][j]);
            }
        }
        head += n;
        count -= n;
        any = true;
    };
    int id[kScan / 64];
    int64_t loaded = -1;   // the first row whose ids are in registers
    for (int adapter = blockIdx.y; adapter < adapters; adapter += gridDim.y) {
        int64_t p0 = beg;
        int i = 0;         // of the ids from p0 on, the next 64
        any = false;
        for (bool more = true; more;) {
            while (count < kRound) {
                if (i == kScan / 64) {
                    i = 0;
                    p0 += kScan;
                }
                if (p0 + 64 * i >= end) {
                    more = false;
                    break;
                }
                if (loaded != p0) {
#pragma unroll
                    for (int q = 0; q < kScan / 64; ++q) {
                        const int64_t r = p0 + 64 * q + lane;
                        id[q] = r < end ? ids[r] : -1;
                    }
                    loaded = p0;
                }
                int here = -1;
#pragma unroll
                for (int q = 0; q < kScan / 64; ++q) here = q == i ? id[q] : here;
                const uint64_t m = __ballot(here == adapter);
                if (here == adapter)
                    s_list[wave][(head + count + __popcll(m & ((1ull << lane) - 1))) & (2 * kRound - 1)] =
                        (int)(p0 + 64 * i + lane);
                count += __popcll(m);
                ++i;
            }
            if (count > 0) round(min(count, kRound));
        }
        if (flags) {
            if (blockIdx.x == 0 && t == 0) flags[(int64_t)blockIdx.z * adapters + adapter] = any;
            if (!any) continue;
        }
        // lane: row 16 i + i16 of the wave's 32, columns 4 g .. of its 16 j
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int64_t l = l0 + 32 * wm + 16 * i + i16;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int64_t c = c0 + 32 * wn + 16 * j + 4 * g, at = ((int64_t)adapter * L + l) * R + c;
                v4f v = acc[i][j];
                acc[i][j] = v4f{};
                if (l >= L) continue;
                if (parts) {
                    store4(parts + (int64_t)blockIdx.z * adapters * L * R + at - c, c, R, v, false);
                } else {
                    if (accumulate) {
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            if (c + k < R) v[k] += (float)dw[at + k];
                    }
                    store4(dw + at - c, c, R, v, false);
                }
            }
        }
    }
}

// The parts' sums, in their order; blockIdx.y: the adapter.
template <typename O>
__global__ __launch_bounds__(kThreads) void adapter_grad_join_kernel(const float* __restrict__ parts,
                                                                     const int32_t* __restrict__ flags, int n,
                                                                     int64_t size, O* __restrict__ dw,
                                                                     int accumulate) {
    const int a = blockIdx.y, lane = threadIdx.x & 63;
    uint64_t has = __ballot(lane < n && flags[(int64_t)min(lane, n - 1) * gridDim.y + a]);   // n <= 64
    for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < size; i += (int64_t)gridDim.x * kThreads) {
        const int64_t at = a * size + i;
        float v = accumulate ? (float)dw[at] : 0.0f;
        float sum = 0.0f;
        for (uint64_t m = has; m; m &= m - 1) sum += parts[(__ffsll((long long)m) - 1) * gridDim.y * size + at];
        dw[at] = (O)(sum + v);
    }
}

// Parts that the rows are cut into: so many that about 512 workgroups share the work, 256 rows a part at least, and their
// sums within 1 GB (each part holds every adapter's; with so many adapters those fill the chip, in turn, by themselves).
constexpr int64_t kPartsBytes = (int64_t)1 << 30;
int grad_parts(int64_t adapters, int64_t rows, int64_t L, int64_t R) {
    const int64_t tiles = ((L + kGT - 1) / kGT) * ((R + kGT - 1) / kGT);
    const int64_t most = std::min((int64_t)64, kPartsBytes / (4 * adapters * (L * R + 1)));
    return (int)std::max((int64_t)1, std::min(std::min((int64_t)512 / tiles, (rows + 255) / 256), most));
}

template <typename T, typename O>
int launch_grad(const void* left, const void* right, const int32_t* ids, int64_t adapters, int64_t rows, int64_t L,
                int64_t R, void* dw, int accumulate, void* workspace, hipStream_t s) {
    const int n = grad_parts(adapters, rows, L, R);
    const int64_t tiles = ((L + kGT - 1) / kGT) * ((R + kGT - 1) / kGT), size = adapters * L * R;
    if (tiles > INT_MAX / kThreads) return HM_ERR_OVERFLOW;
    float* parts = n > 1 ? static_cast<float*>(workspace) : nullptr;
    int32_t* flags = n > 1 ? reinterpret_cast<int32_t*>(parts + n * size) : nullptr;
    const int64_t share = std::max((int64_t)1, std::min(adapters, 1024 / (tiles * n)));
    auto run = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3((unsigned)tiles, (unsigned)share, (unsigned)n), dim3(kThreads), 0, s,
                           static_cast<const T*>(left), static_cast<const T*>(right), ids, rows, L, R, (rows + n - 1) / n,
                           parts, flags, static_cast<O*>(dw), (int)adapters, accumulate);
    };
    if (L % 8 == 0 && R % 8 == 0) run(adapter_grad_kernel<T, O, true>);
    else run(adapter_grad_kernel<T, O, false>);
    HM_LAUNCHED();
    if (n > 1) {
        const int64_t each = L * R;
        hipLaunchKernelGGL((adapter_grad_join_kernel<O>),
                           dim3((unsigned)std::min((each + kThreads - 1) / kThreads, (int64_t)4096), (unsigned)adapters),
                           dim3(kThreads), 0, s, parts, flags, n, each, static_cast<O*>(dw), accumulate);
        HM_LAUNCHED();
    }
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
               !hm_overlap(mid, nm, w, nw) && !hm_overlap(mid, nm, down, nd) && !hm_overlap(mid, nm, up, nu) &&
               !hm_overlap(y, ny, scale, 4 * adapters) && !hm_overlap(mid, nm, scale, 4 * adapters) &&
               !hm_overlap(y, ny, ids, 4 * rows) && !hm_overlap(mid, nm, ids, 4 * rows));
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
    return hm_g_launch(G_ADAPTER, !w_transposed, dtype, dtype, p, s);
}

size_t hm_adapter_weight_grad_workspace_bytes(int64_t adapters, int64_t rows, int64_t left_cols,
                                              int64_t right_cols) {
    if (adapters < 1 || adapters > kMaxAdapters || rows < 0 || left_cols < 1 || right_cols < 1 ||
        left_cols > kMaxDim || right_cols > kMaxDim || left_cols * right_cols > kMaxMatrix)
        return 0;
    const int n = grad_parts(adapters, rows, left_cols, right_cols);
    // the parts' sums, then a flag for each part and adapter
    return n > 1 ? (size_t)n * adapters * (left_cols * right_cols + 1) * 4 : 0;
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
    HM_REQUIRE(!hm_overlap(dw, nw, left, 2 * rows * left_cols) && !hm_overlap(dw, nw, right, 2 * rows * right_cols) &&
               !hm_overlap(dw, nw, ids, 4 * rows));
    const size_t need = hm_adapter_weight_grad_workspace_bytes(adapters, rows, left_cols, right_cols);
    HM_REQUIRE(workspace_bytes >= need && (!need || (workspace && aligned(workspace, 4))));
    HM_REQUIRE(!need || (!hm_overlap(workspace, need, dw, nw) && !hm_overlap(workspace, need, left, 2 * rows * left_cols) &&
                         !hm_overlap(workspace, need, right, 2 * rows * right_cols) &&
                         !hm_overlap(workspace, need, ids, 4 * rows)));
    const hipStream_t s = hm_stream(stream);
    auto run = [&](auto launcher) {
        return launcher(left, right, ids, adapters, rows, left_cols, right_cols, dw, accumulate, workspace, s);
    };
    if (dtype == HM_DTYPE_FP16)
        return dw_dtype == HM_DTYPE_FP32 ? run(launch_grad<hm_f16, float>) : run(launch_grad<hm_f16, hm_f16>);
    return dw_dtype == HM_DTYPE_FP32 ? run(launch_grad<hm_bf16, float>) : run(launch_grad<hm_bf16, hm_bf16>);
}

}  // extern "C"
