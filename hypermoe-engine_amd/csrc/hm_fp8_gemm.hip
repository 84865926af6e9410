// hm_fp8_gemm.hip -- products of block-scaled e4m3 matrices and the FP8 experts: the entry points, and
// the kernel for few rows, which streams the weights (hm_fp8_product.h, hm_fp8_tile.hip).
#include "hm_fp8_product.h"

#include <limits.h>

#include <algorithm>

namespace {

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

// Which kernel takes one matrix product: the one of least time, estimated as a start plus steps (blocks
// of K) x rounds of workgroups x the measured time of a step, alone on its CU while the tiles do not
// fill the chip and with all CUs busy beyond that (us).  Tiles of 64 x 128 and, for FP8 instructions,
// 128 x 128 sit two to a CU.  2048 x 2048 x K: 64 x 128 tiles 54 us at K = 8192, 128 x 256 58, 256 x 256
// 93; 4096 x 4096: 104, 72 and 63 at K = 4096.  The stream kernel has no ring to fill: 16 rows of
// 2048 x 2048 7 us against 8 for the smallest tile, 333 x 1000 x 777 (FP32) 7.3 against 10.5.
struct Form {
    int bm, bn, per_cu;
    double alone, shared;
};
constexpr Form kFast[] = {{256, 256, 1, 1.35, 1.71}, {128, 256, 1, 0.79, 0.99},
                          {128, 128, 2, 0.58, 1.14}, {64, 128, 2, 0.41, 0.85}};
constexpr Form kExact[] = {{128, 256, 1, 1.9, 2.1}, {128, 128, 1, 1.3, 1.4}, {64, 128, 2, 0.85, 1.24}};
constexpr int kCus = 256;

// nullptr: the stream kernel
const Form* choose_form(const Product& p, bool exact) {
    const double steps = (double)hm_f8_blocks(p.K);
    const double groups = (double)((p.N + 15) / 16) * (double)((p.rows + 63) / 64);
    double best = 4.7 + steps / 16 * (groups <= kCus ? 4.0 : groups / (2 * kCus) * 12.0);
    const Form* form = nullptr;
    if (!hm_f8_tile_ok(p, false)) return nullptr;
    const Form* forms = exact ? kExact : kFast;
    for (int i = 0; i < (exact ? 3 : 4); ++i) {
        const Form& f = forms[i];
        const int64_t tiles = ((p.rows + f.bm - 1) / f.bm) * ((p.N + f.bn - 1) / f.bn);
        const int64_t rounds = (tiles + kCus * f.per_cu - 1) / (kCus * f.per_cu);
        const double t = 4.0 + steps * (tiles <= kCus ? f.alone : rounds * f.shared);
        if (t < best) {
            best = t;
            form = &f;
        }
    }
    return form;
}

template <typename T>
int matmul(Product& p, int32_t w_block_rows, void* y, int32_t dtype, hipStream_t s) {
    if (const Form* f = choose_form(p, dtype == HM_DTYPE_FP32)) {
        p.wide = p.N * sizeof(T) % 16 == 0 && (uintptr_t)y % 16 == 0;
        return hm_f8_launch_tiles(f->bm, f->bn, w_block_rows == 1, p, nullptr,
                                  (p.rows + f->bm - 1) / f->bm, y, dtype, s);
    }
    p.wide = p.N % 4 == 0 && (uintptr_t)y % (4 * sizeof(T)) == 0;
    T* out = static_cast<T*>(y);
    return w_block_rows == 1 ? launch_stream<false, true>(p, 0, out, s)
                             : launch_stream<false, false>(p, 0, out, s);
}

constexpr size_t kAlign = 256;
size_t align_up(size_t v) { return (v + kAlign - 1) & ~(kAlign - 1); }

// The experts' workspace.  Tiles: the quantised rows of x, the bytes and scales of z, the m-tile table.
// Streamed: z in floats besides.
struct ExpertsPlan {
    uint8_t* xq;
    float* xs;
    float* z;
    uint8_t* zq;
    float* zs;
    int4* table;
};

// Few rows stream (a token or two: 21 and 27 us against 24 and 26 for tiles); others take tiles of 64 rows, or
// 128 where an expert has that many on average (128 experts top-8, 2048 tokens: 194 us against 211; 1024:
// 168 against 160).
constexpr int64_t kStreamPairs = 8;
struct ExpertsForm {
    bool tiles;
    int bm;
    int cap;      // upper bound of the m-tiles
};
Product gate_up(const hm_layer* L, int64_t tokens, int64_t pairs) {
    return Product{nullptr, nullptr, nullptr, nullptr, 0, 0, reinterpret_cast<const int32_t*>(4), nullptr, pairs,
                   tokens, L->hidden, L->intermediate, (int)L->experts, false};
}
ExpertsForm experts_form(const hm_layer* L, int64_t tokens, int64_t pairs) {
    ExpertsForm f;
    const Product gu = gate_up(L, tokens, pairs);
    const Product dn = {nullptr, nullptr, nullptr, nullptr, 0, 0, nullptr, nullptr, pairs, pairs,
                        L->intermediate, L->hidden, (int)L->experts, false};
    f.tiles = pairs > kStreamPairs && hm_f8_tile_ok(gu, true) && hm_f8_tile_ok(dn, false);
    f.bm = pairs >= 128 * L->experts ? 128 : 64;
    f.cap = (int)(pairs / f.bm + std::min(L->experts, pairs));
    return f;
}

size_t plan_experts(const hm_layer* L, int64_t tokens, int64_t pairs, char* base, ExpertsPlan* p) {
    size_t used = 0;
    auto take = [&](size_t bytes) {
        char* at = base ? base + used : nullptr;
        used += align_up(bytes);
        return at;
    };
    const ExpertsForm f = experts_form(L, tokens, pairs);
    const int64_t H = L->hidden, I = L->intermediate;
    ExpertsPlan q;
    q.xq = reinterpret_cast<uint8_t*>(take((size_t)tokens * hm_f8_pitch(H)));
    q.xs = reinterpret_cast<float*>(take((size_t)tokens * hm_f8_blocks(H) * sizeof(float)));
    q.z = f.tiles ? nullptr : reinterpret_cast<float*>(take((size_t)pairs * I * sizeof(float)));
    q.zq = reinterpret_cast<uint8_t*>(take((size_t)pairs * hm_f8_pitch(I)));
    q.zs = reinterpret_cast<float*>(take((size_t)pairs * hm_f8_blocks(I) * sizeof(float)));
    q.table = f.tiles ? reinterpret_cast<int4*>(take(((size_t)f.cap + 1) * sizeof(int4))) : nullptr;
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
    case HM_DTYPE_FP32: return matmul<float>(p, w_block_rows, y, y_dtype, s);
    case HM_DTYPE_FP16: return matmul<hm_f16>(p, w_block_rows, y, y_dtype, s);
    default: return matmul<hm_bf16>(p, w_block_rows, y, y_dtype, s);
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
    const ExpertsForm form = experts_form(layer, tokens, pairs);
    int rc;
    Product gu = {ws.xq, ws.xs, packed, layer->scale, per, 3 * hb * ib, perm_tokens, offsets,
                  pairs, tokens, H, I, (int)E, I % 4 == 0};
    Product dn = {ws.zq, ws.zs, packed + 2 * I * ph, layer->scale + 2 * hb * ib, per, 3 * hb * ib,
                  nullptr, offsets, pairs, pairs, I, H, (int)E, false};
    const size_t ysize = hm_row_dtype_size(y_dtype);
    if (form.tiles) {
        rc = hm_f8_launch_prepare(x, x_dtype, tokens, H, ws.xq, ws.xs, offsets, (int)E, (int)pairs,
                                  form.bm, form.cap, ws.table, s);
        if (rc) return rc;
        // z goes to 8 bits, so what the FP8 instruction drops can move a byte of it by a step (1.4e-3 of
        // a BF16 result, whose own rounding is 1.7e-3): only where its rate counts and y is BF16
        const bool exact = y_dtype != HM_DTYPE_BF16 || pairs < 128 * E;
        rc = hm_f8_launch_gateup_tiles(form.bm, exact, gu, ws.table, form.cap, ws.zq, ws.zs, s);
        if (rc) return rc;
        dn.wide = H * ysize % 16 == 0 && (uintptr_t)y % 16 == 0;
        return hm_f8_launch_tiles(form.bm, 256, false, dn, ws.table, form.cap, y, y_dtype, s);
    }
    rc = hm_fp8_quantize(x, x_dtype, tokens, H, H, 1, 1, ws.xq, ws.xs, stream);
    if (rc) return rc;
    if ((rc = launch_stream<true, false>(gu, pairs, ws.z, s))) return rc;
    rc = hm_fp8_quantize(ws.z, HM_DTYPE_FP32, pairs, I, I, 1, 1, ws.zq, ws.zs, stream);
    if (rc) return rc;
    dn.wide = H % 4 == 0 && (uintptr_t)y % (4 * ysize) == 0;
    switch (y_dtype) {
    case HM_DTYPE_FP32: return launch_stream<false, false>(dn, pairs, static_cast<float*>(y), s);
    case HM_DTYPE_FP16: return launch_stream<false, false>(dn, pairs, static_cast<hm_f16*>(y), s);
    default: return launch_stream<false, false>(dn, pairs, static_cast<hm_bf16*>(y), s);
    }
}

}  // extern "C"
