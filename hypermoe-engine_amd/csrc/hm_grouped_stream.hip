// hm_grouped_stream.hip -- 16-bit products of few rows (hm_grouped.h): y = x w^T of groups, gate and up with SwiGLU,
// and a projection with adapters, for decode batches.
//
// Every weight is read for a handful of rows, so the kernel is a stream of weights.  A workgroup of 8 waves owns 8 / KP
// times 16 columns of up to 16 MT rows of one group; KP waves share the k of 16 columns by 64 in turn, straight from
// memory into fragments (128 bytes of each of 16 rows of w), no LDS and no barrier before their sums meet, in wave
// order.  x's rows come from the caches.
// Bound by the weights' bytes: 16 tokens, top-8 of 128 experts, 2048 x 768 matrices, 50 us (260 MB, 5.2 TB/s; all eight
// waves on 16 columns 83).  At one token by latency: gate and up 13.4 us (50 MB).
#include "hm_grouped.h"

#include <limits.h>

#include <algorithm>
#include <type_traits>

namespace {

constexpr int kWaves = 8;

template <typename T, typename O, GKind KIND, int MT, int KP>
__global__ __launch_bounds__(64 * kWaves) void g_stream_kernel(GProduct p) {
    typedef typename Elem16<T>::v8 v8;
    constexpr bool GU = KIND == G_SWIGLU;
    constexpr int NP = GU ? 2 : 1;
    __shared__ v4f s_part[kWaves][MT * NP][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int i16 = lane & 15, g = lane >> 4;
    const int part = wave % KP;
    constexpr int CG = kWaves / KP;
    const int64_t N = p.N, K = p.K, n0 = ((int64_t)blockIdx.x * CG + wave / KP) * 16;
    const int64_t m = (int64_t)blockIdx.y + (int64_t)blockIdx.z * gridDim.y;
    Tile t;
    if (p.offsets) {
        if (!locate(p.offsets, p.groups, p.rows, 16 * MT, m, &t)) return;
    } else {
        t.e = 0;
        t.row0 = m * 16 * MT;
        t.nrows = min((int64_t)16 * MT, p.rows - t.row0);
        if (t.nrows <= 0) return;
    }
    // rows past the last repeat it (their results are dropped), columns past the last too
    const T* xr[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        int64_t row = t.row0 + min((int64_t)16 * i + i16, t.nrows - 1);
        if (GU && p.perm) {
            const int v = p.perm[row];
            row = v >= 0 && v < p.x_rows ? v : 0;
        }
        xr[i] = static_cast<const T*>(p.x) + row * K + 8 * g;
    }
    const T* wr = static_cast<const T*>(p.w) + (int64_t)t.e * p.w_group + min(n0 + i16, N - 1) * K + 8 * g;
    v4f acc[MT][NP] = {};
    int64_t k0 = 64 * part;
    // U parts at a time, all their loads in flight
    auto parts = [&](auto u_) __attribute__((always_inline)) {
        constexpr int U = decltype(u_)::value;
        v8 a[U][NP][2], b[U][MT][2];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int64_t k = k0 + 64 * KP * u + 32 * h;
#pragma unroll
                for (int q = 0; q < NP; ++q) a[u][q][h] = load_frag8<T>(wr + q * N * K + k, 8);
#pragma unroll
                for (int i = 0; i < MT; ++i) b[u][i][h] = load_frag8<T>(xr[i] + k, 8);
            }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 0; i < MT; ++i)
#pragma unroll
                    for (int q = 0; q < NP; ++q) acc[i][q] = Elem16<T>::mfma(a[u][q][h], b[u][i][h], acc[i][q]);
        k0 += 64 * KP * U;
    };
    constexpr int U = MT <= 2 ? 4 : MT == 4 ? 2 : 1;
    while (k0 + 64 * KP * (U - 1) + 64 <= K) parts(std::integral_constant<int, U>{});
    while (k0 + 64 <= K) parts(std::integral_constant<int, 1>{});
    if (k0 < K) {  // the last of k
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int64_t n = K - k0 - 32 * h - 8 * g;
            v8 a[NP];
#pragma unroll
            for (int q = 0; q < NP; ++q) a[q] = load_frag8<T>(wr + q * N * K + k0 + 32 * h, n);
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                const v8 b = load_frag8<T>(xr[i] + k0 + 32 * h, n);
#pragma unroll
                for (int q = 0; q < NP; ++q) acc[i][q] = Elem16<T>::mfma(a[q], b, acc[i][q]);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int q = 0; q < NP; ++q) s_part[wave][i * NP + q][lane] = acc[i][q];
    __syncthreads();
    // entry (i, lane): row 16 i + i16, columns 4 g .. of the 16 columns whose waves begin with `w0`
    auto total = [&](int w0, int q, int l) __attribute__((always_inline)) {
        v4f v = s_part[w0][q][l];
#pragma unroll
        for (int w = 1; w < KP; ++w) v += s_part[w0 + w][q][l];
        return v;
    };
    const int64_t c0 = (int64_t)blockIdx.x * CG * 16;
    if constexpr (KIND == G_ADAPTER) {
        // one result a thread: its row's mid times the column's row of the row's adapter
        const T* mid = static_cast<const T*>(p.mid);
        for (int q = threadIdx.x; q < 256 * MT * CG; q += 64 * kWaves) {
            const int c = q % (16 * CG), r = q / (16 * CG);
            if (r >= t.nrows || c0 + c >= N) continue;
            const int64_t row = t.row0 + r;
            float v = 0.0f;
#pragma unroll
            for (int w = 0; w < KP; ++w)
                v += s_part[(c >> 4) * KP + w][r >> 4][16 * ((c & 15) >> 2) + (r & 15)][c & 3];
            const int a = p.ids[row];
            if (a >= 0 && a < p.adapters) {
                const T* u = static_cast<const T*>(p.up) + ((int64_t)a * N + c0 + c) * p.rank;
                for (int k = 0; k < p.rank; k += 8) {
                    float x8[8], u8[8];
                    load8(mid + row * p.rank + k, p.rank - k, x8);
                    load8(u + k, p.rank - k, u8);
#pragma unroll
                    for (int i = 0; i < 8; ++i) v = __builtin_fmaf(x8[i], u8[i], v);
                }
            }
            static_cast<T*>(p.y)[row * N + c0 + c] = (T)v;
        }
    } else {
        for (int q = threadIdx.x; q < 64 * MT * CG; q += 64 * kWaves) {
            const int cg = q / (64 * MT), i = q / 64 % MT, l = q & 63, r = 16 * i + (l & 15);
            const int64_t row = t.row0 + r, c = c0 + 16 * cg + 4 * (l >> 4);
            if (r >= t.nrows || c >= N) continue;
            const bool wide = N % 4 == 0 && p.wide;
            const v4f v = total(cg * KP, i * NP, l);
            if constexpr (GU) {
                const v4f u = total(cg * KP, i * NP + 1, l);
                v4f z;
#pragma unroll
                for (int j = 0; j < 4; ++j) z[j] = fast_silu(v[j]) * u[j];
                store4(static_cast<T*>(p.y) + row * N, c, N, z, wide);
                if (p.pre_out) {
                    T* pre = static_cast<T*>(p.pre_out) + row * 2 * N;
                    store4(pre, c, N, v, wide);
                    store4(pre + N, c, N, u, wide);
                }
            } else {
                store4(static_cast<O*>(p.y) + row * N, c, N, v, wide);
            }
        }
    }
}

template <typename T, typename O, GKind KIND>
int launch(int mt, const GProduct& p, hipStream_t s) {
    const int64_t m = p.offsets ? p.rows / (16 * mt) + std::min((int64_t)p.groups, p.rows)
                                : (p.rows + 16 * mt - 1) / (16 * mt);
    const int64_t deep = (m + 65534) / 65535;
    // few workgroups: all 8 waves on 16 columns; otherwise two, which then have more in flight each
    const int kp = m * ((p.N + 15) / 16) <= 2048 || mt == 8 ? 8 : 2;
    const int64_t n = (p.N + 128 / kp - 1) / (128 / kp);
    if (n > INT_MAX / (64 * kWaves) || deep > 65535) return HM_ERR_OVERFLOW;
    const dim3 grid((unsigned)n, (unsigned)((m + deep - 1) / deep), (unsigned)deep);
    auto run = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(64 * kWaves), 0, s, p); };
    if (mt == 1) kp == 8 ? run(g_stream_kernel<T, O, KIND, 1, 8>) : run(g_stream_kernel<T, O, KIND, 1, 2>);
    else if (mt == 2) kp == 8 ? run(g_stream_kernel<T, O, KIND, 2, 8>) : run(g_stream_kernel<T, O, KIND, 2, 2>);
    else if (mt == 4) kp == 8 ? run(g_stream_kernel<T, O, KIND, 4, 8>) : run(g_stream_kernel<T, O, KIND, 4, 2>);
    else if constexpr (KIND == G_ADAPTER) run(g_stream_kernel<T, O, KIND, 8, 8>);
    HM_LAUNCHED();
    return HM_OK;
}

template <typename T>
int launch_kind(GKind kind, int mt, bool f32, const GProduct& p, hipStream_t s) {
    if (kind == G_SWIGLU) return launch<T, T, G_SWIGLU>(mt, p, s);
    if (kind == G_ADAPTER) return launch<T, T, G_ADAPTER>(mt, p, s);
    return f32 ? launch<T, float, G_MATMUL>(mt, p, s) : launch<T, T, G_MATMUL>(mt, p, s);
}

}  // namespace

int hm_g_launch_stream(GKind kind, int mt, int32_t dtype, bool f32, const GProduct& p, hipStream_t s) {
    return dtype == HM_DTYPE_FP16 ? launch_kind<hm_f16>(kind, mt, f32, p, s)
                                  : launch_kind<hm_bf16>(kind, mt, f32, p, s);
}
