// hm_fp8_gemm.hip -- products of block-scaled e4m3 matrices and the FP8 experts: the entry points, and
// the kernel for few rows, which streams the weights (hm_fp8_product.h, hm_fp8_tile.hip).
#include "hm_fp8_product.h"

#include <limits.h>

#include <algorithm>

namespace {

constexpr int kSWaves = 8;

// Weights streamed from memory: a workgroup of 8 waves owns 16 MT rows x 16 outputs (GU: 16 gate and
// 16 up outputs, z = silu(g) u), its waves split K by blocks and their sums meet in the LDS in wave
// order.  BROW: w has a scale for each of its rows.  Bound by latency: one row of 2048 x 2048 3.8 us,
// 333 x 1000 x 777 (FP32) 8.0: eight blocks of K for eight waves, each of which widens five fragments for
// four products, and 294 workgroups on 256 CUs.
template <int MT, bool GU, bool BROW, typename T>
__global__ __launch_bounds__(64 * kSWaves) void f8_stream_kernel(Product p, T* __restrict__ y) {
    constexpr int NP = GU ? 2 : 1;
    __shared__ __attribute__((aligned(16))) v4f s_part[kSWaves][NP * MT][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int j = lane & 15, g = lane >> 4;
    const int64_t tile = (int64_t)blockIdx.z * gridDim.y + blockIdx.y;
    Tile t = {0, tile * 16 * MT, 0};
    if (p.offsets) {
        if (!locate(p.offsets, p.experts, p.rows, 16 * MT, tile, &t)) return;
    } else {
        t.nrows = min((int64_t)16 * MT, p.rows - t.row0);
        if (t.nrows <= 0) return;
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

constexpr int kCus = 256;

// Rows of a stream workgroup, in 16s: as few as leave no CU more than one workgroup (64 x 2048 x 4096: 32
// rows 9.8 us, 64 15, 16 11; 32 x 2048 x 4096: 16 rows 7.5, 64 10.8).
int stream_mt(int64_t rows, int64_t cols) {
    const int64_t groups = (cols + 15) / 16;
    for (int mt = 1; mt < 4; mt *= 2)
        if (rows <= 16 * mt || groups * ((rows + 16 * mt - 1) / (16 * mt)) <= kCus) return mt;
    return 4;
}

template <bool GU, bool BROW, typename T>
int launch_stream(const Product& p, int64_t m_tiles16, T* y, hipStream_t s) {
    // m_tiles16: an upper bound of the 16-row tiles
    const int64_t cols = (p.N + 15) / 16;
    const int mt = p.offsets ? (p.rows <= 16 ? 1 : 4) : stream_mt(p.rows, p.N);
    const int64_t rows_tiles = p.offsets ? (mt == 1 ? m_tiles16 : (p.rows + 63) / 64 + min((int64_t)p.experts, p.rows))
                                         : (p.rows + 16 * mt - 1) / (16 * mt);
    // (a grid's second and third dimensions hold 65535 each)
    const int64_t deep = (rows_tiles + 65534) / 65535;
    if (deep > 65535 || cols > INT_MAX / 512) return HM_ERR_OVERFLOW;
    const dim3 grid((unsigned)cols, (unsigned)((rows_tiles + deep - 1) / deep), (unsigned)deep);
    auto run = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(64 * kSWaves), 0, s, p, y); };
    if (mt == 1) run(f8_stream_kernel<1, GU, BROW, T>);
    else if (mt == 4) run(f8_stream_kernel<4, GU, BROW, T>);
    else if constexpr (!GU) run(f8_stream_kernel<2, GU, BROW, T>);   // (groups take 1 or 4)
    HM_LAUNCHED();
    return HM_OK;
}

// ---- Experts of a few rows (64 at most): two launches, each quantising what it multiplies.
// A decode step reads every chosen expert's weights for a row or two; the rest is latency.  A workgroup
// of 8 waves owns 8 / KP x 16 outputs (GU: gate and up) of up to 16 rows of one expert.  Its weights are
// sent for first (KP waves split K, two blocks each in flight), then its rows are cut to 8 bits into the
// LDS, 16 lanes a block, so that nothing is launched before or between the products; the waves' sums
// meet in the LDS in wave order.  One token, top-8 of 128 experts of 2048 x 768: 13.6 us as called,
// under the tracer gate/up 8.9 us (25 MB) and down 6.2 (13 MB); by quantisation and tiles 19.4.
struct Decode {
    const void* x;
    const uint8_t* w;
    const float* ws;
    const int32_t* perm;       // rows of x, nullptr: the grouped rows themselves
    const int32_t* offsets;
    void* y;
    int64_t w_expert;
    int ws_expert, experts, pairs, x_rows, K, N;
    bool vec, wide;            // x takes 16-byte loads, y 4-element stores
};

// The 16-row tile `tile`, as locate() does; in a batch whose groups have at most 16 rows each it is the
// tile-th expert with rows, found by ballots (128 experts a round, their offsets in one round trip).
__device__ __forceinline__ bool locate16(const int32_t* __restrict__ offsets, int experts, int pairs,
                                         int tile, Tile* t) {
    const int lane = threadIdx.x & 63;
    int base = 0;
    for (int c0 = 0; c0 < experts; c0 += 128) {
        int lo[2], hi[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int e = min(c0 + 64 * h + lane, experts - 1);
            lo[h] = offsets[e];
            hi[h] = offsets[e + 1];
            if (c0 + 64 * h + lane >= experts) hi[h] = lo[h];
        }
        if (__ballot(hi[0] - lo[0] > 16 || hi[1] - lo[1] > 16))
            return locate(offsets, experts, pairs, 16, tile, t);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            unsigned long long m = __ballot(hi[h] > lo[h]);
            const int here = __popcll(m);
            if (tile < base + here) {
                for (int i = base; i < tile; ++i) m &= m - 1;
                const int l = __builtin_amdgcn_readfirstlane(__ffsll((long long)m) - 1);
                t->e = c0 + 64 * h + l;
                t->row0 = __builtin_amdgcn_readlane(lo[h], l);
                t->nrows = min(__builtin_amdgcn_readlane(hi[h], l), pairs) - t->row0;
                return t->row0 >= 0 && t->nrows > 0;
            }
            base += here;
        }
    }
    return false;
}

// Bytes of LDS of a decode workgroup for `rows` rows: each row's bytes (and 16, against bank conflicts),
// then the scales.
__host__ __device__ __forceinline__ int decode_stride(int K) { return (int)hm_f8_pitch(K) + 16; }
__host__ __device__ __forceinline__ int decode_lds(int rows, int K) {
    return rows * (decode_stride(K) + 4 * (int)hm_f8_blocks(K));
}

template <typename XT, bool GU, int KP, typename T>
__global__ __launch_bounds__(64 * kSWaves, 4) void f8_decode_kernel(Decode p) {
    constexpr int NP = GU ? 2 : 1, D = 2;   // D blocks in flight
    extern __shared__ __attribute__((aligned(16))) uint8_t s_x[];
    __shared__ __attribute__((aligned(16))) v4f s_part[kSWaves][NP][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int j = lane & 15, g = lane >> 4;
    const int part = wave % KP;
    const int n0 = 16 * ((int)blockIdx.x * (kSWaves / KP) + wave / KP);
    // (the batch's rows of x, beside the offsets rather than after them)
    const int rows_of = p.perm ? p.perm[min(lane, p.pairs - 1)] : 0;
    Tile t;
    if (!locate16(p.offsets, p.experts, p.pairs, blockIdx.y, &t)) return;
    const int nb = (int)hm_f8_blocks(p.K), stride = decode_stride(p.K), nrows = (int)t.nrows;
    const int64_t pitch = (int64_t)nb * kF8Block;
    const uint8_t* w[NP];
    const float* ws[NP];
#pragma unroll
    for (int q = 0; q < NP; ++q) {  // columns past the last re-read it
        w[q] = p.w + t.e * p.w_expert + ((int64_t)q * p.N + min(n0 + j, p.N - 1)) * pitch;
        ws[q] = p.ws + (int64_t)t.e * p.ws_expert +
                (q * (int)hm_f8_blocks(p.N) + min(n0, p.N - 1) / kF8Block) * nb;
    }
    v8i raw[D][NP];
    float sw[D][NP];
    auto load_w = [&](int b0) __attribute__((always_inline)) {
#pragma unroll
        for (int d = 0; d < D; ++d) {
            const int b = min(b0 + d * KP, nb - 1);   // (past the last block: read again, not used)
#pragma unroll
            for (int q = 0; q < NP; ++q) {
                raw[d][q] = load_frag(w[q] + b * kF8Block, g);
                sw[d][q] = ws[q][b];
            }
        }
    };
    // unit u of the rows: block u % nb of row u / nb, 8 values a lane.  The first round's loads go out
    // before the weights', which arrive later and in order.
    const int units = nrows * nb;
    float v[8];
    auto load_unit = [&](int u) __attribute__((always_inline)) {
        const int r = u / nb, k = (u - r * nb) * kF8Block + 8 * j;
        int xr = p.perm ? __shfl(rows_of, (int)t.row0 + r, 64) : (int)t.row0 + r;
        if (xr < 0 || xr >= p.x_rows) xr = 0;
        const XT* x = static_cast<const XT*>(p.x) + (int64_t)xr * p.K + k;
        if (p.vec && k + 8 <= p.K) {
            constexpr int N = 16 / sizeof(XT);
#pragma unroll
            for (int i = 0; i < 8 / N; ++i) {
                const hm_pack<XT, N> pk = reinterpret_cast<const hm_pack<XT, N>*>(x)[i];
#pragma unroll
                for (int q = 0; q < N; ++q) v[i * N + q] = (float)pk.v[q];
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = k + i < p.K ? (float)x[i] : 0.0f;
        }
    };
    float* s_scale = reinterpret_cast<float*>(s_x + nrows * stride);
    auto store_unit = [&](int u) __attribute__((always_inline)) {
        const int r = u / nb, k = (u - r * nb) * kF8Block + 8 * j;
        float amax = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) amax = hm_f8_amax(amax, v[i]);
        const hm_f8_scaler s = hm_f8_scaler_of(hm_row16_max(amax));
        uint2 bytes;
        bytes.x = hm_f8_pack4(s, v[0], v[1], v[2], v[3]);
        bytes.y = hm_f8_pack4(s, v[4], v[5], v[6], v[7]);
        *reinterpret_cast<uint2*>(s_x + r * stride + k) = bytes;
        if (j == 0) s_scale[u] = s.scale;
    };
    // (past the last unit: that one again, the same bytes)
    const int u0 = min((int)(threadIdx.x >> 4), units - 1);
    load_unit(u0);
    __builtin_amdgcn_sched_barrier(0);
    load_w(part);
    __builtin_amdgcn_sched_barrier(0);
    store_unit(u0);
    for (int u = 32 + (int)(threadIdx.x >> 4); u - (int)(threadIdx.x >> 4) < units; u += 32) {
        load_unit(min(u, units - 1));
        store_unit(min(u, units - 1));
    }
    __syncthreads();
    const int row = min(j, nrows - 1);
    const uint8_t* x = s_x + row * stride;
    v4f acc[NP] = {};
    for (int b0 = part; b0 < nb; b0 += D * KP) {
        if (b0 != part) load_w(b0);
#pragma unroll
        for (int d = 0; d < D; ++d) {
            const int b = b0 + d * KP;
            if (b >= nb) break;
            Frag<true> fx, fw;
            fx.set(load_frag(x + b * kF8Block, g));
            const float sx = s_scale[row * nb + b];
#pragma unroll
            for (int q = 0; q < NP; ++q) {
                fw.set(raw[d][q]);
                const v4f r4 = block_product(fw, fx);
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[q][i] = __builtin_fmaf(r4[i], sx * sw[d][q], acc[q][i]);
            }
        }
    }
#pragma unroll
    for (int q = 0; q < NP; ++q) s_part[wave][q][lane] = acc[q];
    __syncthreads();
    if (part || n0 >= p.N || j >= nrows) return;
#pragma unroll
    for (int q = 0; q < NP; ++q)
#pragma unroll
        for (int i = 1; i < KP; ++i) acc[q] += s_part[wave + i][q][lane];
    if constexpr (GU) {
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[0][i] = fast_silu(acc[0][i]) * acc[NP - 1][i];
    }
    store4(static_cast<T*>(p.y) + (t.row0 + j) * p.N, n0 + 4 * g, p.N, acc[0], p.wide);
}

template <typename XT, bool GU, typename T>
int launch_decode(const Decode& p, hipStream_t s) {
    // parts of two blocks each
    const int64_t nb = hm_f8_blocks(p.K);
    auto run = [&](auto kernel, int kp) {
        const int cols = 16 * kSWaves / kp;
        hipLaunchKernelGGL(kernel, dim3((unsigned)((p.N + cols - 1) / cols), (unsigned)p.pairs),
                           dim3(64 * kSWaves), decode_lds(std::min(p.pairs, 16), p.K), s, p);
    };
    if (nb > 8) run(f8_decode_kernel<XT, GU, 8, T>, 8);
    else if (nb > 4) run(f8_decode_kernel<XT, GU, 4, T>, 4);
    else run(f8_decode_kernel<XT, GU, 2, T>, 2);
    HM_LAUNCHED();
    return HM_OK;
}

// Which kernel takes one matrix product: the one of least time, estimated as a start plus steps (blocks
// of K) x rounds of workgroups x the measured time of a step (us): of a workgroup alone on the chip, of
// one on every CU (between them by the share of CUs at work: clocks and L2 are shared), and of two on
// every CU where the form's LDS lets them.  The constants fit 14 shapes of K = 1024 and 4096 within 20 %.
// 2048 x 2048 x 4096: 64 x 128 tiles 29 us, 128 x 128 34, 128 x 256 34, 256 x 256 50; 4096 x 4096: 111, 88,
// 76 and 66.  The stream kernel has no ring to fill: 16 rows of 2048 x 2048 7 us against 8 for the smallest
// tile, 333 x 777 x 4096 (FP32) 21 against 28, 16 x 2048 x 256 2.9 against 4.1 (kernel alone), 32 x 8192 x
// 4096 17.4 against 14.5; but it reads w again for every 64 rows: 4096 x 4096 x 256 76 us against 12.
struct Form {
    int bm, bn, per_cu, min_blocks;
    double alone, every, shared;
};
constexpr Form kFast[] = {{256, 256, 1, 1, 1.43, 1.95, 1.95}, {128, 256, 1, 2, 0.92, 1.1, 1.1},
                          {128, 128, 2, 1, 0.58, 0.95, 1.3}, {64, 128, 2, 2, 0.44, 0.47, 0.82}};
constexpr Form kExact[] = {{128, 256, 1, 2, 1.9, 2.1, 2.1}, {128, 128, 1, 1, 1.2, 1.2, 1.2},
                           {64, 128, 2, 2, 0.8, 0.84, 1.27}};

// nullptr: the stream kernel
const Form* choose_form(const Product& p, bool exact) {
    const double steps = (double)hm_f8_blocks(p.K);
    const int mt = stream_mt(p.rows, p.N);
    const double groups = (double)((p.N + 15) / 16) * (double)((p.rows + 16 * mt - 1) / (16 * mt));
    const double each = steps / 16 * (mt == 1 ? 1.3 : mt == 2 ? 3.2 : 6.0);
    double best = groups <= kCus ? 3.0 + each : 4.7 + each * groups / kCus;
    const Form* form = nullptr;
    if (!hm_f8_tile_ok(p, false)) return nullptr;
    const Form* forms = exact ? kExact : kFast;
    for (int i = 0; i < (exact ? 3 : 4); ++i) {
        const Form& f = forms[i];
        if (steps < f.min_blocks) continue;
        const int64_t tiles = ((p.rows + f.bm - 1) / f.bm) * ((p.N + f.bn - 1) / f.bn);
        const int64_t rounds = (tiles + kCus * f.per_cu - 1) / (kCus * f.per_cu);
        // (a tile whose lower half has no rows takes 0.7 of a step)
        const double t = 4.0 + steps * (p.rows <= f.bm / 2 ? 0.7 : 1.0) *
                                   (tiles <= kCus ? f.alone + (f.every - f.alone) * tiles / kCus
                                                  : rounds * f.shared);
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
// Decode: z in floats.  Shapes without either (short or very large dimensions): all but the table.
struct ExpertsPlan {
    uint8_t* xq;
    float* xs;
    float* z;
    uint8_t* zq;
    float* zs;
    int4* table;
};

// The decode kernels take up to kDecodePairs rows, or four times as many where they go to experts of up to 8
// on average and kDecodeBytes of weights at most: beyond, the weights' stream hides the tiles' extra
// launch (16 tokens, top-2 of 8 experts of 2048 x 768, 38 MB: 16.7 us against 24.5 by tiles; top-8 of 128:
// 3 tokens, 113 MB, 31.1 against 32.3; 4 tokens 37.8 against 36.4; 32 tokens, top-2 of 4, 26.3 against
// 24.7).  Others take tiles of 64 rows, or 128 where an expert has that many on average (128 experts
// top-8, 2048 tokens: 194 us against 211; 1024: 168 against 160), or, with the FP8 instruction, 256 from
// 384 rows an expert (6144 tokens: 367 us against 395; 4096: 315 against 293; 8 experts top-2 of 4096 x
// 2048, 16384 tokens: 932 us, 1.77 PFLOP/s, against 1079).  The decode kernels keep 16 rows in 64 KiB of LDS
// (decode_lds), so that two workgroups share a CU: H and I up to 3840.
constexpr int64_t kDecodePairs = 16, kDecodeBytes = (int64_t)1 << 27;
bool decode_rows(const hm_layer* L, int64_t pairs) {
    if (pairs <= kDecodePairs) return true;
    return pairs <= 4 * kDecodePairs && pairs <= 8 * L->experts &&
           std::min(pairs, L->experts) * 3 * L->hidden <= kDecodeBytes / L->intermediate;
}
enum class Experts { kDecode, kTiles, kStream };
struct ExpertsForm {
    Experts kind;
    int bm;
    int cap;      // upper bound of the m-tiles
};
ExpertsForm experts_form(const hm_layer* L, int64_t tokens, int64_t pairs, bool exact) {
    ExpertsForm f = {Experts::kStream, 64, 0};
    const int64_t H = L->hidden, I = L->intermediate;
    static const int32_t gathered = 0;
    Product gu = {}, dn = {};
    gu.rows = dn.rows = dn.x_rows = pairs;
    gu.x_rows = tokens;
    gu.K = dn.N = H;
    gu.N = dn.K = I;
    gu.perm = &gathered;
    if (decode_rows(L, pairs) && decode_lds(16, (int)std::max(H, I)) <= 65536) {
        f.kind = Experts::kDecode;
    } else if (hm_f8_tile_ok(gu, true) && hm_f8_tile_ok(dn, false) && I > kF8Block) {
        f.kind = Experts::kTiles;
        if (pairs >= 128 * L->experts) f.bm = !exact && pairs >= 384 * L->experts ? 256 : 128;
        f.cap = (int)(pairs / f.bm + std::min(L->experts, pairs));
    }
    return f;
}

size_t plan_experts(const hm_layer* L, int64_t tokens, int64_t pairs, char* base, ExpertsPlan* p) {
    size_t used = 0;
    auto take = [&](size_t bytes) {
        char* at = base ? base + used : nullptr;
        used += align_up(bytes);
        return at;
    };
    const ExpertsForm f = experts_form(L, tokens, pairs, true);  // of the two the one with more m-tiles
    const int64_t H = L->hidden, I = L->intermediate;
    ExpertsPlan q;
    q.table = nullptr;
    q.z = nullptr;
    q.xq = q.zq = nullptr;
    q.xs = q.zs = nullptr;
    if (f.kind != Experts::kTiles) q.z = reinterpret_cast<float*>(take((size_t)pairs * I * sizeof(float)));
    if (f.kind != Experts::kDecode) {
        q.xq = reinterpret_cast<uint8_t*>(take((size_t)tokens * hm_f8_pitch(H)));
        q.xs = reinterpret_cast<float*>(take((size_t)tokens * hm_f8_blocks(H) * sizeof(float)));
        q.zq = reinterpret_cast<uint8_t*>(take((size_t)pairs * hm_f8_pitch(I)));
        q.zs = reinterpret_cast<float*>(take((size_t)pairs * hm_f8_blocks(I) * sizeof(float)));
    }
    if (f.kind == Experts::kTiles) q.table = reinterpret_cast<int4*>(take(((size_t)f.cap + 1) * sizeof(int4)));
    if (p) *p = q;
    return used;
}

bool layer_ok(const hm_layer* L) {
    return L && L->dtype == HM_DTYPE_FP8 && L->packed && L->scale && L->experts > 0 &&
           L->hidden > 0 && L->intermediate > 0 && (uintptr_t)L->packed % 16 == 0 &&
           (uintptr_t)L->scale % 4 == 0;
}

}  // namespace

namespace {

// z goes to 8 bits, so what the FP8 instruction drops can move a byte of it by a step (1.4e-3 of a BF16
// result, whose own rounding is 1.7e-3): taken only where its rate counts and y is BF16.
bool exact_z(const hm_f8_experts_call& c) {
    return c.y_dtype != HM_DTYPE_BF16 || c.pairs < 128 * c.layer->experts;
}

// The checks of an experts call, its form and its workspace.  *empty: nothing to do.
int check_experts(const hm_f8_experts_call& c, ExpertsForm* form, ExpertsPlan* plan, bool* empty) {
    const hm_layer* L = c.layer;
    HM_REQUIRE(layer_ok(L) && c.x && c.offsets && c.perm_tokens && c.y && c.tokens >= 0 && c.pairs >= 0);
    HM_REQUIRE(hm_row_dtype(c.x_dtype) && hm_row_dtype(c.y_dtype));
    HM_REQUIRE((uintptr_t)c.x % hm_row_dtype_size(c.x_dtype) == 0 &&
               (uintptr_t)c.y % hm_row_dtype_size(c.y_dtype) == 0 && (uintptr_t)c.offsets % 4 == 0 &&
               (uintptr_t)c.perm_tokens % 4 == 0);
    *empty = c.pairs == 0 || c.tokens == 0;
    if (*empty) return HM_OK;
    if (L->experts > 1024) return HM_ERR_UNSUPPORTED;
    if (c.pairs > INT_MAX || c.tokens > INT_MAX || L->hidden > 1 << 24 || L->intermediate > 1 << 24)
        return HM_ERR_OVERFLOW;
    HM_REQUIRE(c.workspace);
    char* base = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(c.workspace) + kAlign - 1) &
                                         ~(uintptr_t)(kAlign - 1));
    const size_t need = plan_experts(L, c.tokens, c.pairs, base, plan);
    HM_REQUIRE(c.workspace_bytes >= need + (size_t)(base - static_cast<char*>(c.workspace)));
    *form = experts_form(L, c.tokens, c.pairs, exact_z(c));
    return HM_OK;
}

struct LayerDims {
    int64_t H, I, E, ph, pi, hb, ib, per, scales;
    explicit LayerDims(const hm_layer* L)
        : H(L->hidden), I(L->intermediate), E(L->experts), ph(hm_f8_pitch(H)), pi(hm_f8_pitch(I)),
          hb(hm_f8_blocks(H)), ib(hm_f8_blocks(I)), per(2 * I * ph + H * pi), scales(3 * hb * ib) {}
};

}  // namespace

// z of every grouped row, in the form that the down projection reads.
int hm_f8_experts_gate_up(const hm_f8_experts_call& c, hipStream_t s) {
    ExpertsForm form;
    ExpertsPlan ws;
    bool empty;
    int rc = check_experts(c, &form, &ws, &empty);
    if (rc || empty) return rc;
    const hm_layer* L = c.layer;
    const LayerDims d(L);
    const uint8_t* packed = static_cast<const uint8_t*>(L->packed);
    if (form.kind == Experts::kDecode) {
        const bool vec = (uintptr_t)c.x % 16 == 0 && d.H * hm_row_dtype_size(c.x_dtype) % 16 == 0;
        const Decode p = {c.x, packed, L->scale, c.perm_tokens, c.offsets, ws.z, d.per, (int)d.scales,
                          (int)d.E, (int)c.pairs, (int)c.tokens, (int)d.H, (int)d.I, vec, d.I % 4 == 0};
        return c.x_dtype == HM_DTYPE_FP32   ? launch_decode<float, true, float>(p, s)
               : c.x_dtype == HM_DTYPE_FP16 ? launch_decode<hm_f16, true, float>(p, s)
                                            : launch_decode<hm_bf16, true, float>(p, s);
    }
    const Product gu = {ws.xq, ws.xs, packed, L->scale, d.per, d.scales, c.perm_tokens, c.offsets,
                        c.pairs, c.tokens, d.H, d.I, (int)d.E, d.I % 4 == 0};
    if (form.kind == Experts::kTiles) {
        rc = hm_f8_launch_prepare(c.x, c.x_dtype, c.tokens, d.H, ws.xq, ws.xs, c.offsets, (int)d.E,
                                  (int)c.pairs, form.bm, form.cap, ws.table, s);
        if (rc) return rc;
        return hm_f8_launch_gateup_tiles(form.bm, exact_z(c), gu, ws.table, form.cap, ws.zq, ws.zs, s);
    }
    rc = hm_fp8_quantize(c.x, c.x_dtype, c.tokens, d.H, d.H, 1, 1, ws.xq, ws.xs, s);
    if (rc) return rc;
    if ((rc = launch_stream<true, false>(gu, c.pairs, ws.z, s))) return rc;
    return hm_fp8_quantize(ws.z, HM_DTYPE_FP32, c.pairs, d.I, d.I, 1, 1, ws.zq, ws.zs, s);
}

int hm_f8_experts_down(const hm_f8_experts_call& c, hipStream_t s) {
    ExpertsForm form;
    ExpertsPlan ws;
    bool empty;
    const int rc = check_experts(c, &form, &ws, &empty);
    if (rc || empty) return rc;
    const hm_layer* L = c.layer;
    const LayerDims d(L);
    const uint8_t* packed = static_cast<const uint8_t*>(L->packed) + 2 * d.I * d.ph;
    const float* scale = L->scale + 2 * d.hb * d.ib;
    const size_t ysize = hm_row_dtype_size(c.y_dtype);
    if (form.kind == Experts::kDecode) {
        const Decode p = {ws.z, packed, scale, nullptr, c.offsets, c.y, d.per, (int)d.scales, (int)d.E,
                          (int)c.pairs, (int)c.pairs, (int)d.I, (int)d.H, d.I % 4 == 0,
                          d.H % 4 == 0 && (uintptr_t)c.y % (4 * ysize) == 0};
        return c.y_dtype == HM_DTYPE_FP32   ? launch_decode<float, false, float>(p, s)
               : c.y_dtype == HM_DTYPE_FP16 ? launch_decode<float, false, hm_f16>(p, s)
                                            : launch_decode<float, false, hm_bf16>(p, s);
    }
    Product dn = {ws.zq, ws.zs, packed, scale, d.per, d.scales, nullptr, c.offsets, c.pairs, c.pairs,
                  d.I, d.H, (int)d.E, false};
    if (form.kind == Experts::kTiles) {
        dn.wide = d.H * ysize % 16 == 0 && (uintptr_t)c.y % 16 == 0;
        return hm_f8_launch_tiles(form.bm, 256, false, dn, ws.table, form.cap, c.y, c.y_dtype, s);
    }
    dn.wide = d.H % 4 == 0 && (uintptr_t)c.y % (4 * ysize) == 0;
    switch (c.y_dtype) {
    case HM_DTYPE_FP32: return launch_stream<false, false>(dn, c.pairs, static_cast<float*>(c.y), s);
    case HM_DTYPE_FP16: return launch_stream<false, false>(dn, c.pairs, static_cast<hm_f16*>(c.y), s);
    default: return launch_stream<false, false>(dn, c.pairs, static_cast<hm_bf16*>(c.y), s);
    }
}

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
    if (!layer || layer->dtype != HM_DTYPE_FP8 || layer->experts <= 0 || layer->hidden <= 0 ||
        layer->intermediate <= 0 || tokens <= 0 || pairs <= 0)
        return 0;
    return plan_experts(layer, tokens, pairs, nullptr, nullptr) + kAlign;
}

int hm_fp8_experts(const hm_layer* layer, const void* x, int32_t x_dtype, int64_t tokens,
                   const int32_t* offsets, const int32_t* perm_tokens, int64_t pairs, void* y,
                   int32_t y_dtype, void* workspace, size_t workspace_bytes, void* stream) {
    const hm_f8_experts_call c = {layer, x, x_dtype, tokens, offsets, perm_tokens, pairs, y, y_dtype,
                                  workspace, workspace_bytes};
    const int rc = hm_f8_experts_gate_up(c, hm_stream(stream));
    return rc ? rc : hm_f8_experts_down(c, hm_stream(stream));
}

int hm_debug_fp8_matmul_form(int64_t rows, int64_t inner, int64_t cols, int32_t y_dtype) {
    if (rows <= 0 || inner <= 0 || cols <= 0 || !hm_row_dtype(y_dtype)) return -1;
    Product p = {};
    p.rows = p.x_rows = rows;
    p.K = inner;
    p.N = cols;
    const Form* f = choose_form(p, y_dtype == HM_DTYPE_FP32);
    return f ? f->bm << 16 | f->bn : 0;
}

int hm_debug_fp8_experts_form(const hm_layer* layer, int64_t tokens, int64_t pairs, int32_t y_dtype) {
    if (!layer || layer->dtype != HM_DTYPE_FP8 || layer->experts <= 0 || layer->hidden <= 0 ||
        layer->intermediate <= 0 || tokens <= 0 || pairs <= 0 || !hm_row_dtype(y_dtype))
        return -1;
    hm_f8_experts_call c = {};
    c.layer = layer;
    c.pairs = pairs;
    c.y_dtype = y_dtype;
    const bool exact = exact_z(c);
    const ExpertsForm f = experts_form(layer, tokens, pairs, exact);
    if (f.kind != Experts::kTiles) return f.kind == Experts::kDecode ? 16 : 0;
    return exact ? f.bm << 16 : f.bm;
}

int hm_fp8_pack_layer(const void* payload, int32_t dtype, int64_t experts, int64_t hidden,
                      int64_t intermediate, void* packed, float* scale, void* stream) {
    HM_REQUIRE(payload && packed && scale && payload != packed && experts > 0 && hidden > 0 &&
               intermediate > 0 && hm_row_dtype(dtype));
    HM_REQUIRE((uintptr_t)payload % hm_row_dtype_size(dtype) == 0 && (uintptr_t)packed % 16 == 0 &&
               (uintptr_t)scale % 4 == 0);
    if (hidden > 1 << 24 || intermediate > 1 << 24 || experts > 1 << 20) return HM_ERR_OVERFLOW;
    const int64_t H = hidden, I = intermediate, blocks = hm_f8_blocks(H) * hm_f8_blocks(I);
    uint8_t* q = static_cast<uint8_t*>(packed);
    const char* src = static_cast<const char*>(payload);
    const size_t matrix = (size_t)H * I * hm_row_dtype_size(dtype);
    for (int64_t e = 0; e < experts; ++e) {
        for (int p = 0; p < 3; ++p) {
            // [K x N] row-major: output n's inner dimension runs at stride N
            const int64_t K = p < 2 ? H : I, N = p < 2 ? I : H;
            const int rc = hm_fp8_quantize(src, dtype, N, K, N == 1 ? K : 1, N == 1 ? 1 : N, kF8Block, q,
                                           scale, stream);
            if (rc) return rc;
            src += matrix;
            q += N * hm_f8_pitch(K);
            scale += blocks;
        }
    }
    return HM_OK;
}

}  // extern "C"
