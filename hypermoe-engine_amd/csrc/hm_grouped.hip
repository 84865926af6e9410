// hm_grouped.hip -- grouped products of 16-bit experts: y = x w^T and x w, gate and up with SwiGLU, the
// SwiGLU's gradient behind the down matrix's, and the weights' gradients; entry points, the choice of a kernel, and the
// kernel for operands of any size and alignment: 64 x 64 results a workgroup, 32 of k a step, through registers into the
// LDS.  Bound by a step's round trip: 16 groups of 512 rows, 1001 x 1333, 190 us, 115 TFLOP/s.
#include "hm_grouped.h"
#include "hm_lds_dma.h"

#include <limits.h>

#include <algorithm>

namespace {

constexpr int kBT = 64;        // tile edge
constexpr int kBK = 32;        // k a step
constexpr int kPitch = 40;     // values from one row of a staged operand to the next (16-byte pieces)
constexpr int kThreads = 256;

// One thread's 8 values of an operand tile [64 x 32]: k-major row t / 4, k 8 (t % 4) ..; else k t / 8, rows
// 8 (t % 8) .. .  `at(r, k)` is the place of a value, -1 a row that counts as zeros.
template <typename T, bool KM>
struct Stage {
    T v[8];
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = (T)0.0f;
    }
    // k-major: `row` the row's first value (nullptr: zeros), k of K
    __device__ __forceinline__ void load_k(const T* row, int64_t k, int64_t K) {
        zero();
        if (!row || k >= K) return;
        if (k + 8 <= K) {
            const Loose8<T> w = *reinterpret_cast<const Loose8<T>*>(row + k);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = w.v[i];
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (k + i < K) v[i] = row[k + i];
        }
    }
    __device__ __forceinline__ void store(T* s) const {
        const int t = threadIdx.x;
        if (KM) {
            hm_pack<T, 8> w;
#pragma unroll
            for (int i = 0; i < 8; ++i) w.v[i] = v[i];
            *reinterpret_cast<hm_pack<T, 8>*>(s + (t >> 2) * kPitch + 8 * (t & 3)) = w;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) s[(8 * (t & 7) + i) * kPitch + (t >> 3)] = v[i];
        }
    }
};

template <typename T, typename O, GKind KIND, bool WK>
__global__ __launch_bounds__(kThreads) void grouped_generic_kernel(GProduct p) {
    typedef typename Elem16<T>::v8 v8;
    constexpr bool XK = KIND != G_WEIGHT_GRAD;     // x k-major
    constexpr bool GU = KIND == G_SWIGLU;
    constexpr int TN = GU ? kBT / 2 : kBT;
    __shared__ __attribute__((aligned(16))) T s_x[kBT * kPitch];
    __shared__ __attribute__((aligned(16))) T s_w[kBT * kPitch];
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const int wm = wave >> 1, wn = wave & 1, i16 = lane & 15, g = lane >> 4;
    const T* x = static_cast<const T*>(p.x);
    const T* w = static_cast<const T*>(p.w);

    int64_t row0, nrows, n0, K;
    int e;
    if (KIND == G_WEIGHT_GRAD) {
        const int64_t ntn = (p.N + kBT - 1) / kBT;
        e = blockIdx.y;
        row0 = (int64_t)blockIdx.x / ntn * kBT;
        n0 = (int64_t)blockIdx.x % ntn * kBT;
        nrows = min((int64_t)kBT, p.M - row0);
    } else {
        n0 = (int64_t)blockIdx.x * TN;
        Tile tile;
        if (p.offsets) {
            if (!locate(p.offsets, p.groups, p.rows, kBT, (int64_t)blockIdx.y + (int64_t)blockIdx.z * gridDim.y,
                        &tile))
                return;
        } else {
            tile.e = 0;
            tile.row0 = ((int64_t)blockIdx.y + (int64_t)blockIdx.z * gridDim.y) * kBT;
            tile.nrows = min((int64_t)kBT, p.rows - tile.row0);
            if (tile.nrows <= 0) return;
        }
        e = tile.e;
        row0 = tile.row0;
        nrows = tile.nrows;
    }
    // the rows that are summed over, for the weight gradient
    int64_t kbeg = 0, kend = p.K;
    if (KIND == G_WEIGHT_GRAD) {
        kbeg = max(0, p.offsets[e]);
        kend = min((int64_t)p.offsets[e + 1], p.rows);
    }
    w += KIND == G_WEIGHT_GRAD ? 0 : (int64_t)e * p.w_group;

    v4f acc[2][2] = {};
    int at[2];   // the adapters of the lane's rows
    // `own`: of an adapter's step, whose rows alone take it: the others' operand is zeros, but 0 times an infinity or a NaN
    // of the adapter's matrix is NaN
    auto step = [&](int own) __attribute__((always_inline)) {
        __syncthreads();
        v8 a[2], b[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            a[i] = *reinterpret_cast<const v8*>(s_w + (32 * wn + 16 * i + i16) * kPitch + 8 * g);
            b[i] = *reinterpret_cast<const v8*>(s_x + (32 * wm + 16 * i + i16) * kPitch + 8 * g);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const v4f r = Elem16<T>::mfma(a[j], b[i], acc[i][j]);
                acc[i][j] = own < 0 || at[i] == own ? r : acc[i][j];
            }
        __syncthreads();
    };
    // the row of x of tile row r
    auto x_row = [&](int r) __attribute__((always_inline)) -> const T* {
        if (r >= nrows) return nullptr;
        if (KIND == G_SWIGLU && p.perm) {
            const int v = p.perm[row0 + r];
            return x + (v >= 0 && v < p.x_rows ? (int64_t)v : 0) * p.K;
        }
        return x + (row0 + r) * p.K;
    };
    // row r of the staged w: output column, of gate and then up for each wave
    auto w_col = [&](int r, bool* up) __attribute__((always_inline)) -> int64_t {
        *up = false;
        if (!GU) return n0 + r;
        *up = (r >> 4) & 1;
        return n0 + (r >> 5) * 16 + (r & 15);
    };

    if constexpr (KIND == G_WEIGHT_GRAD) {
        for (int64_t k0 = kbeg; k0 < kend; k0 += kBK) {
            const int64_t k = k0 + (t >> 3);
            const bool mine = k < kend;
            Stage<T, false> sx, sw;
            sx.load_k(mine ? x + k * p.M : nullptr, row0 + 8 * (t & 7), p.M);
            sw.load_k(mine ? w + k * p.N : nullptr, n0 + 8 * (t & 7), p.N);
            sx.store(s_x);
            sw.store(s_w);
            step(-1);
        }
    } else {
        bool up;
        const T* xr = x_row(t >> 2);
        const int64_t wc = w_col(t >> 2, &up);
        for (int64_t k0 = 0; k0 < p.K; k0 += kBK) {
            Stage<T, true> sx;
            Stage<T, WK> sw;
            sx.load_k(xr, k0 + 8 * (t & 3), p.K);
            if constexpr (WK) {
                sw.load_k(wc < p.N ? w + (wc + (up ? p.N : 0)) * p.K : nullptr, k0 + 8 * (t & 3), p.K);
            } else {
                const int64_t k = k0 + (t >> 3);
                sw.load_k(k < p.K ? w + k * p.N : nullptr, n0 + 8 * (t & 7), p.N);
            }
            sx.store(s_x);
            sw.store(s_w);
            step(-1);
        }
        if constexpr (KIND == G_ADAPTER) {
            const T* mid = static_cast<const T*>(p.mid);
            const int mine = lane < nrows ? p.ids[row0 + lane] : -1;
#pragma unroll
            for (int i = 0; i < 2; ++i) at[i] = __shfl(mine, 32 * wm + 16 * i + i16, 64);
            int cur = -1;
            while (true) {
                // the next adapter of these rows (the same in every wave)
                int next = mine > cur && mine < p.adapters ? mine : INT_MAX;
#pragma unroll
                for (int m = 32; m >= 1; m >>= 1) next = min(next, __shfl_xor(next, m, 64));
                if (next == INT_MAX) break;
                cur = next;
                const T* upm = static_cast<const T*>(p.up) + (int64_t)cur * p.N * p.rank;
                const int r = t >> 2;
                const bool take = __shfl(mine, r & 63, 64) == cur && r < nrows;
                for (int k0 = 0; k0 < p.rank; k0 += kBK) {
                    Stage<T, true> sx;
                    Stage<T, WK> sw;
                    sx.load_k(take ? mid + (row0 + r) * p.rank : nullptr, k0 + 8 * (t & 3), p.rank);
                    if constexpr (WK) {
                        sw.load_k(wc < p.N ? upm + wc * p.rank : nullptr, k0 + 8 * (t & 3), p.rank);
                    } else {
                        const int k = k0 + (t >> 3);
                        sw.load_k(k < p.rank ? upm + (int64_t)k * p.N : nullptr, n0 + 8 * (t & 7), p.N);
                    }
                    sx.store(s_x);
                    sw.store(s_w);
                    step(cur);
                }
            }
        }
    }

#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int r = 32 * wm + 16 * i + i16;
        if (r >= nrows) continue;
        const int64_t row = row0 + r;
#pragma unroll
        for (int j = 0; j < (GU ? 1 : 2); ++j)
#pragma unroll
            for (int v = 0; v < 4; ++v) {
                const int64_t c = n0 + (GU ? 16 * wn : 32 * wn + 16 * j) + 4 * g + v;
                if (c >= p.N) continue;
                if constexpr (KIND == G_SWIGLU) {
                    const float gate = acc[i][0][v], upv = acc[i][1][v];
                    static_cast<T*>(p.y)[row * p.N + c] = (T)(fast_silu(gate) * upv);
                    if (p.pre_out) {
                        T* pre = static_cast<T*>(p.pre_out) + row * 2 * p.N + c;
                        pre[0] = (T)gate;
                        pre[p.N] = (T)upv;
                    }
                } else if constexpr (KIND == G_SWIGLU_GRAD) {
                    const T* pre = static_cast<const T*>(p.pre_in) + row * 2 * p.N + c;
                    float dg, du, z;
                    swiglu_grad(acc[i][j][v], (float)pre[0], (float)pre[p.N], &dg, &du, &z);
                    T* d = static_cast<T*>(p.y) + row * 2 * p.N + c;
                    d[0] = (T)dg;
                    d[p.N] = (T)du;
                    if (p.z) static_cast<T*>(p.z)[row * p.N + c] = (T)z;
                } else if constexpr (KIND == G_WEIGHT_GRAD) {
                    O* y = static_cast<O*>(p.y) + ((int64_t)e * p.M + row) * p.N + c;
                    *y = (O)(acc[i][j][v] + (p.accumulate ? (float)*y : 0.0f));
                } else {
                    static_cast<O*>(p.y)[row * p.N + c] = (O)acc[i][j][v];
                }
            }
    }
}

template <typename T, typename O, GKind KIND, bool WK>
int launch(const GProduct& p, hipStream_t s) {
    dim3 grid;
    if (KIND == G_WEIGHT_GRAD) {
        const int64_t tiles = ((p.M + kBT - 1) / kBT) * ((p.N + kBT - 1) / kBT);
        if (tiles > INT_MAX / kThreads) return HM_ERR_OVERFLOW;
        grid = dim3((unsigned)tiles, (unsigned)p.groups);
    } else {
        const int tn = KIND == G_SWIGLU ? kBT / 2 : kBT;
        const int64_t n = (p.N + tn - 1) / tn;
        const int64_t m = p.offsets ? p.rows / kBT + std::min((int64_t)p.groups, p.rows) : (p.rows + kBT - 1) / kBT;
        const int64_t deep = (m + 65534) / 65535;
        if (n > INT_MAX / kThreads || deep > 65535) return HM_ERR_OVERFLOW;
        grid = dim3((unsigned)n, (unsigned)((m + deep - 1) / deep), (unsigned)deep);
    }
    hipLaunchKernelGGL((grouped_generic_kernel<T, O, KIND, WK>), grid, dim3(kThreads), 0, s, p);
    HM_LAUNCHED();
    return HM_OK;
}

template <typename T>
int launch_kind(GKind kind, bool wk, bool f32, const GProduct& p, hipStream_t s) {
    switch (kind) {
    case G_SWIGLU: return launch<T, T, G_SWIGLU, true>(p, s);
    case G_SWIGLU_GRAD: return launch<T, T, G_SWIGLU_GRAD, false>(p, s);
    case G_WEIGHT_GRAD:
        return f32 ? launch<T, float, G_WEIGHT_GRAD, false>(p, s) : launch<T, T, G_WEIGHT_GRAD, false>(p, s);
    case G_ADAPTER: return wk ? launch<T, T, G_ADAPTER, true>(p, s) : launch<T, T, G_ADAPTER, false>(p, s);
    default: break;
    }
    if (wk) return f32 ? launch<T, float, G_MATMUL, true>(p, s) : launch<T, T, G_MATMUL, true>(p, s);
    return f32 ? launch<T, float, G_MATMUL, false>(p, s) : launch<T, T, G_MATMUL, false>(p, s);
}

bool type16(int32_t dtype) { return dtype == HM_DTYPE_FP16 || dtype == HM_DTYPE_BF16; }
bool aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }
bool result_type(int32_t y, int32_t dtype) { return y == dtype || y == HM_DTYPE_FP32; }

constexpr int64_t kMaxRows = ((int64_t)1 << 31) - 1, kMaxDim = (int64_t)1 << 26,
                  kMaxMatrix = (int64_t)1 << 40;

// Sizes that every grouped call shares.
int check_sizes(int64_t groups, int64_t rows, int64_t a, int64_t b) {
    HM_REQUIRE(groups >= 1 && groups <= HM_GROUPED_MAX_GROUPS && rows >= 0 && a >= 1 && b >= 1);
    if (rows > kMaxRows || a > kMaxDim || b > kMaxDim || a * b > kMaxMatrix) return HM_ERR_OVERFLOW;
    return HM_OK;
}

}  // namespace

int hm_g_launch_generic(GKind kind, bool w_kmajor, int32_t dtype, int32_t y_dtype, const GProduct& p,
                        hipStream_t s) {
    const bool f32 = y_dtype == HM_DTYPE_FP32;
    return dtype == HM_DTYPE_FP16 ? launch_kind<hm_f16>(kind, w_kmajor, f32, p, s)
                                  : launch_kind<hm_bf16>(kind, w_kmajor, f32, p, s);
}

// Whether a product fits the tile kernels: offsets from a tile's first row (x's first row where rows are gathered)
// stay below HM_BUF_RANGE.
static bool tile_ok(GKind kind, bool w_kmajor, const GProduct& p) {
    const int64_t top = HM_BUF_RANGE;
    const int64_t wide = (int64_t)1 << 24;   // columns, of which a stage has 64 rows
    if (p.rows > INT_MAX - 256) return false;
    if (kind == G_WEIGHT_GRAD) return p.M <= wide && p.N <= wide;
    if (p.K > (int64_t)1 << 22 || (!w_kmajor && p.N > wide)) return false;
    return kind != G_SWIGLU || ((p.N + 256) * p.K * 2 < top && (!p.perm || p.x_rows * p.K * 2 < top));
}

// Whether everything that a tile moves in 16 bytes is aligned to that.
static bool dma_ok(GKind kind, bool w_kmajor, const GProduct& p) {
    if (!aligned(p.x, 16) || !aligned(p.w, 16)) return false;
    if (kind == G_WEIGHT_GRAD) return p.M % 8 == 0 && p.N % 8 == 0;
    if (p.K % 8 || (!w_kmajor && p.N % 8)) return false;
    return kind != G_ADAPTER || (p.rank % 8 == 0 && aligned(p.mid, 16) && aligned(p.up, 16));
}

// Which kernel: rows << 16 of a stream workgroup, the form of a tile, 0: the generic kernel.
static int pick(GKind kind, bool w_kmajor, const GProduct& p) {
    const bool nt = w_kmajor && kind != G_WEIGHT_GRAD;
    const int64_t groups = p.offsets ? p.groups : 1, each = (p.rows + groups - 1) / groups;
    if (nt && (each <= 16 || p.rows <= 64)) return (p.rows <= 16 || each <= 4 ? 1 : p.rows <= 32 || each <= 8 ? 2 : 4) << 16;
    // Adapters of up to 128 rows: the stream kernel takes an adapter for each row as easily as one for all (the host does
    // not know which), tiles take a stage more for every adapter: 128 rows, 2048 x 2048, rank 16, one adapter 31 us
    // against 29 on tiles, one a row 33 against 184; rank 64 65 and 31, 72 and 192.  Beyond, rows of one adapter are
    // taken to lie side by side: 256 rows, rank 16, one adapter 30 (streamed 31), one a row 186 (35); 512 rows 31 (58)
    // and 249 (123).
    if (kind == G_ADAPTER && nt && p.rows <= 128) return 8 << 16;
    if (!tile_ok(kind, w_kmajor, p)) return 0;
    const bool wg = kind == G_WEIGHT_GRAD;
    const int64_t m128 = wg ? p.groups * ((p.M + 127) / 128) : p.rows / 128 + groups;
    // Off 16 bytes (128 x 128 tiles through registers against the generic kernel's 64 x 64): 16 groups of 512 rows,
    // 1001 x 1333, 70 us and 190, but 8 of 100, 1001 x 777, transposed 44 and 36: few tiles leave most of the chip idle.
    if (!dma_ok(kind, w_kmajor, p)) return nt || m128 * ((p.N + 127) / 128) >= 128 ? 32 : 0;
    // 128 x 128 where larger tiles are fewer than the chip's CUs: 2048 x 2048 x 2048 27 us, 128 x 256 34, 256 x 256 48.
    const int wide = kind == G_SWIGLU ? 128 : 256;   // (gate and up share a tile)
    if (m128 * ((p.N + wide - 1) / wide) < 256) return 64;
    // 256 x 256 from 384 rows a group on: 8 groups of 4096 rows, 2048 x 1536, 195 us against 219 of 128 x 256; but 128
    // of 256 rows on average, uneven, 182 and 157: half of the second tile of a group is empty.  Gate and up from 256 on
    // (those groups 289 and 297; even groups 32 x 272 rows 87 and 90, 32 x 512 93 and 96, but 64 x 256 131 and 120, and
    // below it 64 x 240 140 and 125).  The SwiGLU's gradient not at all: its results take more time than the matrix
    // instructions, and 128 x 256 tiles spread them better (8 groups of 4096 rows, 2048 x 768, 171 us and 157).
    if (kind == G_SWIGLU_GRAD) return 128;
    return wg || each >= (kind == G_SWIGLU ? 256 : 384) ? 256 : 128;
}

int hm_g_launch(GKind kind, bool w_kmajor, int32_t dtype, int32_t y_dtype, const GProduct& p_, hipStream_t s) {
    GProduct p = p_;
    const bool f32 = y_dtype == HM_DTYPE_FP32;
    p.wide = aligned(p.y, f32 ? 16 : 8) && aligned(p.pre_out, 8);
    const int form = pick(kind, w_kmajor, p);
    if (!form) return hm_g_launch_generic(kind, w_kmajor, dtype, y_dtype, p, s);
    if (form >> 16) return hm_g_launch_stream(kind, form >> 16, dtype, f32, p, s);
    return dtype == HM_DTYPE_FP16 ? hm_g_launch_tiles_f16(kind, form, w_kmajor, f32, p, s)
                                  : hm_g_launch_tiles_bf16(kind, form, w_kmajor, f32, p, s);
}

extern "C" {

int hm_grouped_matmul(const void* x, int32_t dtype, const void* w, int32_t w_transposed,
                      const int32_t* offsets, int64_t groups, int64_t rows, int64_t inner, int64_t cols,
                      void* y, int32_t y_dtype, void* stream) {
    HM_REQUIRE(type16(dtype) && result_type(y_dtype, dtype) && (w_transposed == 0 || w_transposed == 1));
    if (const int rc = check_sizes(groups, rows, inner, cols)) return rc;
    if (rows == 0) return HM_OK;
    HM_REQUIRE(x && w && offsets && y && aligned(x, 2) && aligned(w, 2) && aligned(offsets, 4) &&
               aligned(y, y_dtype == HM_DTYPE_FP32 ? 4 : 2));
    const int64_t ny = rows * cols * (y_dtype == HM_DTYPE_FP32 ? 4 : 2);
    HM_REQUIRE(!hm_overlap(y, ny, x, 2 * rows * inner) && !hm_overlap(y, ny, w, 2 * groups * inner * cols) &&
               !hm_overlap(y, ny, offsets, 4 * (groups + 1)));
    GProduct p = {};
    p.x = x;
    p.w = w;
    p.y = y;
    p.offsets = offsets;
    p.rows = p.x_rows = rows;
    p.K = inner;
    p.N = cols;
    p.w_group = inner * cols;
    p.groups = (int)groups;
    return hm_g_launch(G_MATMUL, !w_transposed, dtype, y_dtype, p, hm_stream(stream));
}

int hm_grouped_swiglu(const void* x, int32_t dtype, int64_t x_rows, const int32_t* perm_tokens, const void* w,
                      const int32_t* offsets, int64_t groups, int64_t rows, int64_t hidden,
                      int64_t intermediate, void* z, void* pre, void* stream) {
    HM_REQUIRE(type16(dtype));
    if (const int rc = check_sizes(groups, rows, hidden, intermediate)) return rc;
    HM_REQUIRE(perm_tokens ? x_rows >= 1 || rows == 0 : x_rows == rows);
    if (x_rows > kMaxRows) return HM_ERR_OVERFLOW;
    if (rows == 0) return HM_OK;
    HM_REQUIRE(x && w && offsets && z && aligned(x, 2) && aligned(w, 2) && aligned(offsets, 4) &&
               aligned(perm_tokens, 4) && aligned(z, 2) && aligned(pre, 2));
    const int64_t nz = 2 * rows * intermediate, nx = 2 * x_rows * hidden, nw = 4 * groups * hidden * intermediate,
                  no = 4 * (groups + 1);
    HM_REQUIRE(!hm_overlap(z, nz, x, nx) && !hm_overlap(z, nz, w, nw) && !hm_overlap(z, nz, perm_tokens, 4 * rows) &&
               !hm_overlap(pre, 2 * nz, x, nx) && !hm_overlap(pre, 2 * nz, w, nw) &&
               !hm_overlap(pre, 2 * nz, perm_tokens, 4 * rows) && !hm_overlap(z, nz, pre, 2 * nz) &&
               !hm_overlap(z, nz, offsets, no) && !hm_overlap(pre, 2 * nz, offsets, no));
    GProduct p = {};
    p.x = x;
    p.w = w;
    p.y = z;
    p.pre_out = pre;
    p.offsets = offsets;
    p.perm = perm_tokens;
    p.rows = rows;
    p.x_rows = x_rows;
    p.K = hidden;
    p.N = intermediate;
    p.w_group = 2 * hidden * intermediate;
    p.groups = (int)groups;
    return hm_g_launch(G_SWIGLU, true, dtype, dtype, p, hm_stream(stream));
}

int hm_grouped_swiglu_grad(const void* dy, int32_t dtype, const void* w, const void* pre,
                           const int32_t* offsets, int64_t groups, int64_t rows, int64_t hidden,
                           int64_t intermediate, void* dpre, void* z, void* stream) {
    HM_REQUIRE(type16(dtype));
    if (const int rc = check_sizes(groups, rows, hidden, intermediate)) return rc;
    if (rows == 0) return HM_OK;
    HM_REQUIRE(dy && w && pre && offsets && dpre && aligned(dy, 2) && aligned(w, 2) && aligned(pre, 2) &&
               aligned(offsets, 4) && aligned(dpre, 2) && aligned(z, 2));
    const int64_t nz = 2 * rows * intermediate, ny = 2 * rows * hidden, nw = 2 * groups * hidden * intermediate,
                  no = 4 * (groups + 1);
    HM_REQUIRE(!hm_overlap(dpre, 2 * nz, dy, ny) && !hm_overlap(dpre, 2 * nz, w, nw) &&
               !hm_overlap(dpre, 2 * nz, pre, 2 * nz) && !hm_overlap(z, nz, dy, ny) && !hm_overlap(z, nz, w, nw) &&
               !hm_overlap(z, nz, pre, 2 * nz) && !hm_overlap(z, nz, dpre, 2 * nz) &&
               !hm_overlap(dpre, 2 * nz, offsets, no) && !hm_overlap(z, nz, offsets, no));
    GProduct p = {};
    p.x = dy;
    p.w = w;
    p.y = dpre;
    p.pre_in = pre;
    p.z = z;
    p.offsets = offsets;
    p.rows = p.x_rows = rows;
    p.K = hidden;
    p.N = intermediate;
    p.w_group = hidden * intermediate;
    p.groups = (int)groups;
    return hm_g_launch(G_SWIGLU_GRAD, false, dtype, dtype, p, hm_stream(stream));
}

size_t hm_grouped_weight_grad_workspace_bytes(int64_t groups, int64_t rows, int64_t cols, int64_t inner) {
    (void)groups, (void)rows, (void)cols, (void)inner;
    return 0;
}

int hm_grouped_weight_grad(const void* dy, const void* x, int32_t dtype, const int32_t* offsets, int64_t groups,
                           int64_t rows, int64_t cols, int64_t inner, void* dw, int32_t dw_dtype,
                           int32_t accumulate, void* workspace, size_t workspace_bytes, void* stream) {
    HM_REQUIRE(type16(dtype) && result_type(dw_dtype, dtype) && (accumulate == 0 || accumulate == 1));
    if (const int rc = check_sizes(groups, rows, cols, inner)) return rc;
    HM_REQUIRE((rows == 0 || (dy && x)) && offsets && dw && aligned(dy, 2) && aligned(x, 2) &&
               aligned(offsets, 4) && aligned(dw, dw_dtype == HM_DTYPE_FP32 ? 4 : 2));
    const int64_t nw = groups * cols * inner * (dw_dtype == HM_DTYPE_FP32 ? 4 : 2);
    HM_REQUIRE(!hm_overlap(dw, nw, dy, 2 * rows * cols) && !hm_overlap(dw, nw, x, 2 * rows * inner) &&
               !hm_overlap(dw, nw, offsets, 4 * (groups + 1)));
    if (workspace_bytes < hm_grouped_weight_grad_workspace_bytes(groups, rows, cols, inner)) return HM_ERR_INVALID;
    GProduct p = {};
    p.x = dy;
    p.w = x;
    p.y = dw;
    p.offsets = offsets;
    p.rows = rows;
    p.M = cols;
    p.N = inner;
    p.groups = (int)groups;
    p.accumulate = accumulate;
    return hm_g_launch(G_WEIGHT_GRAD, false, dtype, dw_dtype, p, hm_stream(stream));
}

int hm_debug_grouped_form(int32_t kind, int64_t groups, int64_t rows, int64_t inner, int64_t cols, int32_t rank,
                          int32_t aligned16) {
    if (kind < 0 || kind > 6 || check_sizes(groups, rows, inner, cols) || rows == 0) return -1;
    static const GKind kinds[7] = {G_MATMUL, G_MATMUL, G_SWIGLU, G_SWIGLU_GRAD, G_WEIGHT_GRAD, G_ADAPTER, G_ADAPTER};
    const void* at = reinterpret_cast<const void*>((uintptr_t)(aligned16 ? 1 << 20 : (1 << 20) + 2));
    GProduct p = {};
    p.x = p.w = p.mid = p.up = at;
    p.offsets = kind < 5 ? static_cast<const int32_t*>(at) : nullptr;
    p.rows = p.x_rows = rows;
    p.groups = (int)groups;
    p.K = inner;
    p.M = cols;   // weight gradient: [cols x inner]
    p.N = kind == 4 ? inner : cols;
    p.rank = rank;
    return pick(kinds[kind], kind == 0 || kind == 2 || kind == 5, p);
}

}  // extern "C"
