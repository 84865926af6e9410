// hm_fp8_product.h -- what the product kernels of block-scaled e4m3 matrices share.
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
#pragma once

#include "hm_fp8.h"

typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v8i __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));

typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));

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

// The FP8 instruction aligns each eight consecutive products, by the sums of their exponents, to the
// largest of them and cuts what lies more than 13 bits below it (measured: 2^16 + 2^2 is 2^16 inside a group
// of eight and exact across groups): at most 2^-10 of sum |x w|.  Of a result's norm that is 1.5e-5 for
// normally distributed operands, under a tenth of FP16's rounding and a hundredth of BF16's, and 5.1e-5 for
// bytes spread evenly over the format, but 150 to 400 times FP32's sums.  Where that shows, the operands
// are widened to fp16 (exact) for v_mfma_f32_16x16x32_f16, whose sums are FP32 (1.1e-7 over 4096 columns),
// at half the rate: Frag<true>.
template <bool PREC>
struct Frag;
template <>
struct Frag<false> {
    v8i v;
    __device__ __forceinline__ void set(v8i f) { v = f; }
};
template <>
struct Frag<true> {
    v8h v[4];
    __device__ __forceinline__ void set(v8i f) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v2h w[4];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                w[2 * h] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((unsigned)f[2 * i + h], 1.0f, false);
                w[2 * h + 1] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((unsigned)f[2 * i + h], 1.0f, true);
            }
            v[i] = v8h{w[0][0], w[0][1], w[1][0], w[1][1], w[2][0], w[2][1], w[3][0], w[3][1]};
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
    for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x32_f16(a.v[i], b.v[i], c, 0, 0, 0);
    return c;
}

// g / (1 + e^-g) on the exponential and reciprocal units, a unit in the last place each, and for negative g |g| / 2 units
// of the exponent's rounding (below g = -87, where it is under 3e-37 in size, 0).
__device__ __forceinline__ float fast_silu(float g) {
    return g * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(g * -1.44269504088896f));
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
// Every lane of the wave must be active.  False past the last tile; offsets are cut to [0, rows] before anything
// is counted, so that a last one of 2^31 - 1 does not take a count past 31 bits.
__device__ __forceinline__ bool locate(const int32_t* __restrict__ offsets, int experts, int64_t rows,
                                       int bm, int64_t tile, Tile* t) {
    const int lane = threadIdx.x & 63, top = (int)min(rows, (int64_t)0x7fffffff);
    int64_t base = 0;
    for (int c0 = 0; c0 < experts; c0 += 64) {
        const int e = min(c0 + lane, experts - 1);
        const int from = offsets[e], to = offsets[e + 1];   // (both in one round trip: no branch between them)
        const int lo = max(0, min(from, top)), hi = max(lo, min(to, top));
        const int64_t tiles = c0 + lane < experts ? ((uint32_t)(hi - lo) + (uint32_t)bm - 1) / (uint32_t)bm : 0;
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
            t->row0 = max(0, offsets[t->e]) + in * bm;
            t->nrows = min((int64_t)bm, min((int64_t)offsets[t->e + 1], rows) - t->row0);
            return t->nrows > 0;
        }
        base += total;
    }
    return false;
}

// The tile kernels (hm_fp8_tile.hip).  table: the m-tiles of a grouped product (entry 0: their number
// in x; then {expert, first row, rows}) and m_tiles an upper bound of them, or nullptr and the m-tiles of
// one matrix.  bm: rows of x per tile, 64, 128 or (16-bit results) 256; bn: 128 or 256 rows of w.  Rings of
// three stages (64 x 128, 64 x 256, 128 x 256) need two blocks of K, gathered rows three: a stage of the
// next tile is the first to go out in the last two steps, gathered rows are fetched one step before.
bool hm_f8_tile_ok(const Product& p, bool gu);
int hm_f8_launch_tiles(int bm, int bn, bool brow, const Product& p, const int4* table, int64_t m_tiles,
                       void* y, int32_t dtype, hipStream_t s);
int hm_f8_launch_gateup_tiles(int bm, bool prec, const Product& p, const int4* table, int64_t m_tiles,
                              uint8_t* zq, float* zs, hipStream_t s);
// hm_fp8_quantize.hip
int hm_f8_launch_prepare(const void* x, int32_t dtype, int64_t rows, int64_t width, uint8_t* q,
                         float* scale, const int32_t* offsets, int experts, int pairs, int bm, int cap,
                         int4* table, hipStream_t s);
