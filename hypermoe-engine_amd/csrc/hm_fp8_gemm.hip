// hm_fp8_gemm.hip -- products of block-scaled e4m3 matrices (hm_fp8.h) and the FP8 experts.
//
//   y[m, n] = sum over blocks b of 128 of  xs[m, b] ws[n, b] P(m, n, b),
//   P(m, n, b) = sum_{k in block b} x[m, k] w[n, k]
// with x [M x K] scaled by rows and w [N x K] by 128 x 128 blocks or by rows.  One
// v_mfma_f32_16x16x128_f8f6f4 is 16 x 16 of the P of one block; one fused multiply-add by the block's
// scale joins it to the FP32 sum.
//
// Operand layout of the instruction: lane l supplies 32 bytes of row l % 16 of A and of column l % 16
// of B, the same K positions of both, so which 32 of the 128 a lane group l / 16 holds is free as long
// as both operands agree (16-byte pieces g and g + 4).  Its 4 results are column l % 16, rows
// 4 (l / 16) + v.  The weights are A and the rows of x are B: a lane's results are then four
// consecutive outputs of one row, under one scale of x.
#include "hm_fp8.h"

#include <limits.h>

namespace {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v8i __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));

typedef __bf16 v2b __attribute__((ext_vector_type(2)));
typedef __bf16 v8b __attribute__((ext_vector_type(8)));

__device__ __forceinline__ v4f mfma_f8(v8i a, v8i b, v4f c) {
    // formats 0, 0: e4m3; no block exponents
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, 0, 0, 0, 0);
}

// The lane's 32 bytes of a 128-byte block of one row: pieces g and g + 4.
__device__ __forceinline__ v8i join_frag(v4i lo, v4i hi) {
    return v8i{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
}
__device__ __forceinline__ v8i load_frag(const uint8_t* block, int g) {
    return join_frag(*reinterpret_cast<const v4i*>(block + 16 * g),
                     *reinterpret_cast<const v4i*>(block + 16 * (g + 4)));
}

// The FP8 instruction aligns each eight consecutive products to the largest of them and drops what
// lies more than 13 bits below it (measured: 2^16 + 2^2 is 2^16 inside a group of eight and exact
// across groups), 1.3e-5 to 2.4e-5 of a sum's norm: under a sixth of FP16's rounding step and a
// hundredth of BF16's, but 300 times FP32's.  Where that shows, the operands are widened to bf16
// (exact) for v_mfma_f32_16x16x32_bf16, whose sums are FP32 (1e-8), at half the rate: Frag<true>.
template <bool PREC>
struct Frag;
template <>
struct Frag<false> {
    v8i v;
    __device__ __forceinline__ void set(v8i f) { v = f; }
};
template <>
struct Frag<true> {
    v8b v[4];
    __device__ __forceinline__ void set(v8i f) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v2b w[4];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                w[2 * h] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)f[2 * i + h], 1.0f, false);
                w[2 * h + 1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)f[2 * i + h], 1.0f, true);
            }
            v[i] = v8b{w[0][0], w[0][1], w[1][0], w[1][1], w[2][0], w[2][1], w[3][0], w[3][1]};
        }
    }
};
// P of one block.
__device__ __forceinline__ v4f block_product(const Frag<false>& a, const Frag<false>& b) {
    return mfma_f8(a.v, b.v, v4f{});
}
__device__ __forceinline__ v4f block_product(const Frag<true>& a, const Frag<true>& b) {
    v4f c = {};
#pragma unroll
    for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.v[i], b.v[i], c, 0, 0, 0);
    return c;
}

// Four consecutive outputs of a row, columns n .. n + 3 (those below cols).
template <typename T>
__device__ __forceinline__ void store4(T* y, int64_t n, int64_t cols, v4f v, bool wide) {
    if (wide && n + 4 <= cols) {
        hm_pack<T, 4> w;
#pragma unroll
        for (int i = 0; i < 4; ++i) w.v[i] = (T)v[i];
        *reinterpret_cast<hm_pack<T, 4>*>(y + n) = w;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (n + i < cols) y[n + i] = (T)v[i];
    }
}

// A product's operands.  Grouped: expert e's rows are offsets[e] .. offsets[e + 1], row g of a group
// reads row perm[g] of x (or g itself), and its matrix starts at w + e w_expert.
struct Product {
    const uint8_t* x;
    const float* xs;
    const uint8_t* w;
    const float* ws;
    int64_t w_expert, ws_expert;  // bytes, scales from one expert's matrix to the next one's
    const int32_t* perm;
    const int32_t* offsets;
    int64_t rows, x_rows;         // output rows, rows of x
    int64_t K, N;
    int experts;
    bool wide;                    // y's rows take 4-element stores
};

// The m-tile `tile` of `bm` rows, experts in ascending order: its expert, first row and row count.
struct Tile {
    int e;
    int64_t row0, nrows;
};
// Every lane of the wave must be active.  False past the last tile; rows stays inside [0, rows).
__device__ __forceinline__ bool locate(const int32_t* __restrict__ offsets, int experts, int64_t rows,
                                       int bm, int64_t tile, Tile* t) {
    const int lane = threadIdx.x & 63;
    int64_t base = 0;
    for (int c0 = 0; c0 < experts; c0 += 64) {
        const int e = c0 + lane;
        const int n = e < experts ? offsets[e + 1] - offsets[e] : 0;
        const int64_t tiles = (n + bm - 1) / bm;
        int64_t incl = tiles;
#pragma unroll
        for (int sft = 1; sft < 64; sft <<= 1) {
            const int64_t o = __shfl_up(incl, sft, 64);
            if (lane >= sft) incl += o;
        }
        const int64_t total = __shfl(incl, 63, 64);
        if (tile < base + total) {
            const int first = __ffsll((long long)__ballot(base + incl > tile)) - 1;
            const int64_t in = tile - base - __shfl(incl - tiles, first, 64);
            t->e = c0 + first;
            t->row0 = offsets[t->e] + in * bm;
            t->nrows = min((int64_t)bm, min((int64_t)offsets[t->e + 1], rows) - t->row0);
            return t->row0 >= 0 && t->nrows > 0;
        }
        base += total;
    }
    return false;
}

constexpr int kSWaves = 8;

// Weights streamed from memory: a workgroup of 8 waves owns 16 MT rows x 16 outputs (GU: 16 gate and
// 16 up outputs, z = silu(g) u), its waves split K by blocks and their sums meet in the LDS in wave
// order.  BROW: w has a scale for each of its rows.
template <int MT, bool GU, bool BROW, typename T>
__global__ __launch_bounds__(64 * kSWaves) void f8_stream_kernel(Product p, T* __restrict__ y) {
    constexpr int NP = GU ? 2 : 1;
    __shared__ __attribute__((aligned(16))) v4f s_part[kSWaves][NP * MT][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int j = lane & 15, g = lane >> 4;
    Tile t = {0, (int64_t)blockIdx.y * 16 * MT, 0};
    if (p.offsets) {
        if (!locate(p.offsets, p.experts, p.rows, 16 * MT, blockIdx.y, &t)) return;
    } else {
        t.nrows = min((int64_t)16 * MT, p.rows - t.row0);
    }
    const int64_t nb = hm_f8_blocks(p.K), pitch = nb * kF8Block;
    const int64_t n0 = 16 * (int64_t)blockIdx.x;
    // rows past the matrix re-read its last
    const int64_t wn = min(n0 + j, p.N - 1);
    const uint8_t* w[NP];
    const float* ws[NP];
#pragma unroll
    for (int q = 0; q < NP; ++q) {
        w[q] = p.w + t.e * p.w_expert + q * p.N * pitch + wn * pitch;
        ws[q] = p.ws + t.e * p.ws_expert + q * hm_f8_blocks(p.N) * nb;
        if (!BROW) ws[q] += n0 / kF8Block * nb;
    }
    const uint8_t* x[MT];
    const float* xs[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        const int64_t r = t.row0 + min((int64_t)(16 * m + j), t.nrows - 1);
        int64_t xr = p.perm ? p.perm[r] : r;
        if (xr < 0 || xr >= p.x_rows) xr = 0;
        x[m] = p.x + xr * pitch;
        xs[m] = p.xs + xr * nb;
    }
    v4f acc[NP][MT];
#pragma unroll
    for (int q = 0; q < NP; ++q)
#pragma unroll
        for (int m = 0; m < MT; ++m) acc[q][m] = v4f{};
    for (int64_t b = wave; b < nb; b += kSWaves) {
        Frag<true> fw[NP];
#pragma unroll
        for (int q = 0; q < NP; ++q) fw[q].set(load_frag(w[q] + b * kF8Block, g));
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            Frag<true> fx;
            fx.set(load_frag(x[m] + b * kF8Block, g));
            const float sx = xs[m][b];
#pragma unroll
            for (int q = 0; q < NP; ++q) {
                const v4f part = block_product(fw[q], fx);
#pragma unroll
                for (int v = 0; v < 4; ++v) {
                    const float sw = BROW ? ws[q][min(n0 + 4 * g + v, p.N - 1) * nb + b] : ws[q][b];
                    acc[q][m][v] = __builtin_fmaf(part[v], sx * sw, acc[q][m][v]);
                }
            }
        }
    }
#pragma unroll
    for (int q = 0; q < NP; ++q)
#pragma unroll
        for (int m = 0; m < MT; ++m) s_part[wave][q * MT + m][lane] = acc[q][m];
    __syncthreads();
    for (int m = wave; m < MT; m += kSWaves) {
        if (16 * m + j >= t.nrows) continue;
        v4f r[NP];
#pragma unroll
        for (int q = 0; q < NP; ++q) {
            r[q] = s_part[0][q * MT + m][lane];
#pragma unroll
            for (int i = 1; i < kSWaves; ++i) r[q] += s_part[i][q * MT + m][lane];
        }
        if constexpr (GU) {
#pragma unroll
            for (int v = 0; v < 4; ++v) r[0][v] = hm_silu(r[0][v]) * r[NP - 1][v];
        }
        store4(y + (t.row0 + 16 * m + j) * p.N, n0 + 4 * g, p.N, r[0], p.wide);
    }
}

template <bool GU, bool BROW, typename T>
int launch_stream(const Product& p, int64_t m_tiles16, T* y, hipStream_t s) {
    // m_tiles16: an upper bound of the 16-row tiles
    const int64_t cols = (p.N + 15) / 16;
    const int mt = p.rows <= 16 ? 1 : 4;
    const int64_t rows_tiles = p.offsets ? (mt == 1 ? m_tiles16 : (p.rows + 63) / 64 + min((int64_t)p.experts, p.rows))
                                         : (p.rows + 16 * mt - 1) / (16 * mt);
    if (rows_tiles > 65535 || cols > INT_MAX / 512) return HM_ERR_OVERFLOW;
    const dim3 grid((unsigned)cols, (unsigned)rows_tiles);
    if (mt == 1)
        hipLaunchKernelGGL((f8_stream_kernel<1, GU, BROW, T>), grid, dim3(64 * kSWaves), 0, s, p, y);
    else
        hipLaunchKernelGGL((f8_stream_kernel<4, GU, BROW, T>), grid, dim3(64 * kSWaves), 0, s, p, y);
    HM_LAUNCHED();
    return HM_OK;
}

template <typename T>
int matmul(Product& p, int32_t w_block_rows, void* y, hipStream_t s) {
    p.wide = p.N % 4 == 0 && (uintptr_t)y % (4 * sizeof(T)) == 0;
    T* out = static_cast<T*>(y);
    return w_block_rows == 1 ? launch_stream<false, true>(p, 0, out, s)
                             : launch_stream<false, false>(p, 0, out, s);
}

constexpr size_t kAlign = 256;
size_t align_up(size_t v) { return (v + kAlign - 1) & ~(kAlign - 1); }

// The experts' workspace: the quantised rows of x, z in floats, and its bytes and scales.
struct ExpertsPlan {
    uint8_t* xq;
    float* xs;
    float* z;
    uint8_t* zq;
    float* zs;
};
size_t plan_experts(const hm_layer* L, int64_t tokens, int64_t pairs, char* base, ExpertsPlan* p) {
    size_t used = 0;
    auto take = [&](size_t bytes) {
        char* at = base ? base + used : nullptr;
        used += align_up(bytes);
        return at;
    };
    const int64_t H = L->hidden, I = L->intermediate;
    ExpertsPlan q;
    q.xq = reinterpret_cast<uint8_t*>(take((size_t)tokens * hm_f8_pitch(H)));
    q.xs = reinterpret_cast<float*>(take((size_t)tokens * hm_f8_blocks(H) * sizeof(float)));
    q.z = reinterpret_cast<float*>(take((size_t)pairs * I * sizeof(float)));
    q.zq = reinterpret_cast<uint8_t*>(take((size_t)pairs * hm_f8_pitch(I)));
    q.zs = reinterpret_cast<float*>(take((size_t)pairs * hm_f8_blocks(I) * sizeof(float)));
    if (p) *p = q;
    return used;
}

bool layer_ok(const hm_layer* L) {
    return L && L->dtype == HM_DTYPE_FP8 && L->packed && L->scale && L->experts > 0 &&
           L->hidden > 0 && L->intermediate > 0 && (uintptr_t)L->packed % 16 == 0 &&
           (uintptr_t)L->scale % 4 == 0;
}

}  // namespace

extern "C" {

int hm_fp8_matmul(const uint8_t* xq, const float* xs, const uint8_t* wq, const float* ws,
                  int32_t w_block_rows, int64_t rows, int64_t inner, int64_t cols, void* y,
                  int32_t y_dtype, void* stream) {
    HM_REQUIRE(xq && xs && wq && ws && y && rows >= 0 && inner > 0 && cols > 0);
    HM_REQUIRE(hm_row_dtype(y_dtype) && (w_block_rows == 1 || w_block_rows == kF8Block));
    HM_REQUIRE((uintptr_t)xq % 16 == 0 && (uintptr_t)wq % 16 == 0 && (uintptr_t)xs % 4 == 0 &&
               (uintptr_t)ws % 4 == 0 && (uintptr_t)y % hm_row_dtype_size(y_dtype) == 0);
    HM_REQUIRE(static_cast<const void*>(xq) != y && static_cast<const void*>(wq) != y);
    if (rows == 0) return HM_OK;
    if (rows > INT_MAX || cols > INT_MAX || inner > INT_MAX) return HM_ERR_OVERFLOW;
    Product p = {xq, xs, wq, ws, 0, 0, nullptr, nullptr, rows, rows, inner, cols, 1, false};
    hipStream_t s = hm_stream(stream);
    switch (y_dtype) {
    case HM_DTYPE_FP32: return matmul<float>(p, w_block_rows, y, s);
    case HM_DTYPE_FP16: return matmul<hm_f16>(p, w_block_rows, y, s);
    default: return matmul<hm_bf16>(p, w_block_rows, y, s);
    }
}

size_t hm_fp8_experts_workspace_bytes(const hm_layer* layer, int64_t tokens, int64_t pairs) {
    if (!layer || layer->dtype != HM_DTYPE_FP8 || layer->hidden <= 0 || layer->intermediate <= 0 ||
        tokens <= 0 || pairs <= 0)
        return 0;
    return plan_experts(layer, tokens, pairs, nullptr, nullptr) + kAlign;
}

int hm_fp8_experts(const hm_layer* layer, const void* x, int32_t x_dtype, int64_t tokens,
                   const int32_t* offsets, const int32_t* perm_tokens, int64_t pairs, void* y,
                   int32_t y_dtype, void* workspace, size_t workspace_bytes, void* stream) {
    HM_REQUIRE(layer_ok(layer) && x && offsets && perm_tokens && y && tokens >= 0 && pairs >= 0);
    HM_REQUIRE(hm_row_dtype(x_dtype) && hm_row_dtype(y_dtype));
    HM_REQUIRE((uintptr_t)x % hm_row_dtype_size(x_dtype) == 0 &&
               (uintptr_t)y % hm_row_dtype_size(y_dtype) == 0);
    if (pairs == 0 || tokens == 0) return HM_OK;
    if (layer->experts > 1024) return HM_ERR_UNSUPPORTED;
    if (pairs > INT_MAX || tokens > INT_MAX || layer->hidden > 1 << 24 ||
        layer->intermediate > 1 << 24)
        return HM_ERR_OVERFLOW;
    HM_REQUIRE(workspace);
    char* base = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(workspace) + kAlign - 1) &
                                         ~(uintptr_t)(kAlign - 1));
    ExpertsPlan ws;
    const size_t need = plan_experts(layer, tokens, pairs, base, &ws);
    HM_REQUIRE(workspace_bytes >= need + (size_t)(base - static_cast<char*>(workspace)));
    const int64_t H = layer->hidden, I = layer->intermediate, E = layer->experts;
    const int64_t ph = hm_f8_pitch(H), pi = hm_f8_pitch(I);
    const int64_t hb = hm_f8_blocks(H), ib = hm_f8_blocks(I);
    const int64_t per = 2 * I * ph + H * pi;
    const uint8_t* packed = static_cast<const uint8_t*>(layer->packed);
    hipStream_t s = hm_stream(stream);
    int rc = hm_fp8_quantize(x, x_dtype, tokens, H, H, 1, 1, ws.xq, ws.xs, stream);
    if (rc) return rc;
    Product gu = {ws.xq, ws.xs, packed, layer->scale, per, 3 * hb * ib, perm_tokens, offsets,
                  pairs, tokens, H, I, (int)E, I % 4 == 0};
    if ((rc = launch_stream<true, false>(gu, pairs, ws.z, s))) return rc;
    rc = hm_fp8_quantize(ws.z, HM_DTYPE_FP32, pairs, I, I, 1, 1, ws.zq, ws.zs, stream);
    if (rc) return rc;
    Product dn = {ws.zq, ws.zs, packed + 2 * I * ph, layer->scale + 2 * hb * ib, per, 3 * hb * ib,
                  nullptr, offsets, pairs, pairs, I, H, (int)E, false};
    dn.wide = H % 4 == 0 && (uintptr_t)y % (4 * hm_row_dtype_size(y_dtype)) == 0;
    switch (y_dtype) {
    case HM_DTYPE_FP32: return launch_stream<false, false>(dn, pairs, static_cast<float*>(y), s);
    case HM_DTYPE_FP16: return launch_stream<false, false>(dn, pairs, static_cast<hm_f16*>(y), s);
    default: return launch_stream<false, false>(dn, pairs, static_cast<hm_bf16*>(y), s);
    }
}

}  // extern "C"
