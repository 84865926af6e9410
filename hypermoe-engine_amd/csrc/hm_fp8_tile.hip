// hm_fp8_tile.hip -- tiles of the block-scaled FP8 product (hm_fp8_product.h) through an LDS ring: one
// matrix, or the experts' groups; plain, or gate and up with SwiGLU and the quantisation of z.
//
// Persistent workgroups of 8 waves, 2 (rows of x) x 4 (rows of w); a wave owns 16 XF x 16 WF outputs
// (tile BM = 32 XF rows of x, BN = 64 WF of w).  A stage is one block of 128 of K: (BM + BN) rows of 128
// bytes, moved to the LDS by DMA, and the stage's scales (one float a row, whatever block it covers).
// Stages of consecutive tiles form one stream, so a tile's first stages load while its predecessor ends.
//   LDS   row r's 16-byte piece c sits at position c ^ s(r): a fragment read takes rows of one piece
//         by 16 lanes, and s separates those 16 (eight values and the row's parity), for w with the
//         row order below.  No bank conflicts.
//   w     fragment j's row i is w row 4 SH (i / 4) + 4 j + i % 4 of the wave's, so that a lane ends
//         with 4 SH consecutive outputs of one row (SH: fragments side by side).
//   order tiles are cut into 8 contiguous ranges, one per XCD (workgroup i runs on XCD i % 8); n-tiles
//         of an m-tile lie together, for one matrix in groups of m-tiles, so what is read by several
//         workgroups at once is in one L2.
// Epilogue of gate/up (GU): z = silu(g) u for one block of 128 columns; its maximum over the block goes
// over lanes, then through the LDS over the four waves of a row; the bytes and scale are stored.
//
// Bound by the matrix instructions and the clock they leave: 4096 x 4096 x 4096 to BF16 65 us, 2.1
// PFLOP/s (the library's product with one scale for all: 2.5 to 2.6), matrix pipes 55 % busy at 1.73 GHz,
// waves waiting for operands 30 % and for an issue slot 35 % of their time.  FP32 results 139 us.  128
// experts top-8 of 2048 x 768, 4096 tokens, to BF16: gate/up 182 us (206 GFLOP; 634 MB read where weights and
// rows are 411, because m-tiles of an expert read them again), down 105.  Results off 16 bytes are stored
// value by value: 4096 x 4096 x 2048 to BF16 41 us, 2044 to 2047 columns 62; to FP32 75, and 95 where odd.
#include "hm_fp8_product.h"
#include "hm_lds_dma.h"

#include <limits.h>

#include <algorithm>
#include <type_traits>

namespace {

constexpr int kXcds = 8;
constexpr int kTThreads = 512;

struct TileAt {
    int e, row0, nrows, n0;
};

__device__ __forceinline__ int uni(int v) { return __builtin_amdgcn_readfirstlane(v); }
template <typename P>
__device__ __forceinline__ P* uni(P* p) {
    const uint64_t v = reinterpret_cast<uint64_t>(p);
    return reinterpret_cast<P*>(((uint64_t)(uint32_t)uni((int)(v >> 32)) << 32) | (uint32_t)uni((int)v));
}

// Tile j: n-tiles of an m-tile lie together, for one matrix in groups of m-tiles, so many that the tiles
// which an XCD has at once cover about as many rows of x as of w (4096 x 4096 x 4096 by groups of 4 and 8:
// 64 x 128 tiles 105.5 and 100 us, 256 x 256 63.4 and 64).  (Per lane.)
template <int BM, int TN>
__device__ __forceinline__ TileAt tile_at(const Product& p, const int4* __restrict__ table, int j, int mt,
                                          int ntn) {
    constexpr int SUPER = BM == 256 ? 4 : 8;
    TileAt t;
    if (table) {
        const int m = j / ntn;
        const int4 e = table[1 + m];
        t.e = e.x;
        t.row0 = e.y;
        t.nrows = e.z;
        t.n0 = (j - m * ntn) * TN;
    } else {
        const int grp = j / (SUPER * ntn), first = grp * SUPER;
        const int gm = min(mt - first, SUPER), r = j - first * ntn;
        t.e = 0;
        t.row0 = (first + r % gm) * BM;
        t.nrows = min(BM, (int)p.rows - t.row0);
        t.n0 = r / gm * TN;
    }
    return t;
}

// A tile's results.  The lane holds column run c0 .. c0 + 4 SH - 1 of the rows 16 i + i16 (from wm 16 XF).
template <int XF, int WF, typename T>
__device__ __forceinline__ void store_y(const Product& p, const TileAt& t, const v4f (&acc)[XF][WF], T* y,
                                        int r0, int c0) {
    constexpr int VN = 16 / sizeof(T);
    const int N = (int)p.N;
#pragma unroll
    for (int i = 0; i < XF; ++i) {
        const int r = r0 + 16 * i;
        if (r >= t.nrows) continue;
        T* to = y + (int64_t)(t.row0 + r) * N + c0;
        if (p.wide && c0 + 4 * WF <= N) {
#pragma unroll
            for (int q = 0; q < 4 * WF; q += VN) {
                hm_pack<T, VN> w;
#pragma unroll
                for (int v = 0; v < VN; ++v) w.v[v] = (T)acc[i][(q + v) / 4][(q + v) % 4];
                *reinterpret_cast<hm_pack<T, VN>*>(to + q) = w;
            }
        } else {
#pragma unroll
            for (int q = 0; q < 4 * WF; ++q)
                if (c0 + q < N) to[q] = (T)acc[i][q / 4][q % 4];
        }
    }
}
// Maximum over the lanes of one column, l % 16 (the four lane groups).
__device__ __forceinline__ float column_max(float v) {
    const unsigned u = __float_as_uint(v);
    const auto a = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    const unsigned w = __float_as_uint(fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1])));
    const auto b = __builtin_amdgcn_permlane16_swap(w, w, false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
// z = silu(gate) up and its quantisation (one block of 128 columns; s_amax: a maximum for each of the
// four waves of a row).  Every wave of the workgroup calls it.  The matrix instructions stand still
// meanwhile, so it is kept short: z carries FP32 noise of a few units in the last place, and the scale
// and the bytes' quotients go by one reciprocal instead of divisions.
template <int XF, int WF, int BM>
__device__ __forceinline__ void store_z(const Product& p, const TileAt& t, v4f (&acc)[XF][WF],
                                        float (&s_amax)[4][BM], uint8_t* zq, float* zs, int r0, int c0,
                                        int wn, int g) {
    constexpr int SH = WF / 2;
    const int N = (int)p.N, nbn = (int)hm_f8_blocks(p.N);
    const bool whole = t.n0 + kF8Block <= N;
#pragma unroll
    for (int i = 0; i < XF; ++i) {
        float amax = 0.0f, bad = 0.0f;
#pragma unroll
        for (int q = 0; q < SH; ++q)
#pragma unroll
            for (int v = 0; v < 4; ++v) {
                float z = fast_silu(acc[i][q][v]) * acc[i][SH + q][v];
                if (!whole) z = c0 + 4 * q + v < N ? z : 0.0f;
                acc[i][q][v] = z;
                amax = fmaxf(amax, fabsf(z));
                bad = __builtin_fmaf(z, 0.0f, bad);  // NaN from an infinity or a NaN
            }
        amax = column_max(bad == 0.0f ? amax : __builtin_inff());
        if (g == 0) s_amax[wn][r0 + 16 * i] = amax;
    }
    lds_barrier();
#pragma unroll
    for (int i = 0; i < XF; ++i) {
        const int r = r0 + 16 * i;
        const float amax = fmaxf(fmaxf(s_amax[0][r], s_amax[1][r]), fmaxf(s_amax[2][r], s_amax[3][r]));
        if (r >= t.nrows) continue;
        const bool finite = amax < __builtin_inff();
        const float m = fmaxf(amax, kF8Tiny);
        const float inv = 0.875f * __builtin_amdgcn_rcpf(m * 0x1p-9f);  // 448 / m; 1 / m may be subnormal, 0 here
        uint32_t w[SH];
#pragma unroll
        for (int q = 0; q < SH; ++q) {
            int b = __builtin_amdgcn_cvt_pk_fp8_f32(acc[i][q][0] * inv, acc[i][q][1] * inv, 0, false);
            b = __builtin_amdgcn_cvt_pk_fp8_f32(acc[i][q][2] * inv, acc[i][q][3] * inv, b, true);
            w[q] = finite ? (uint32_t)b : 0x7f7f7f7fu;
        }
        const int64_t row = t.row0 + r;
        hm_pack<uint32_t, SH> out;
#pragma unroll
        for (int q = 0; q < SH; ++q) out.v[q] = w[q];
        *reinterpret_cast<hm_pack<uint32_t, SH>*>(zq + row * (nbn * kF8Block) + c0) = out;
        if (wn == 0 && g == 0)
            zs[row * nbn + t.n0 / kF8Block] = finite ? m * (1.0f / kF8Top) : __builtin_nanf("");
    }
}

template <int XF, int WF, int NS, bool GU, bool BROW, bool PREC, typename T>
__global__ __launch_bounds__(kTThreads) void f8_tile_kernel(Product p, const int4* __restrict__ table,
                                                            T* __restrict__ y, uint8_t* __restrict__ zq,
                                                            float* __restrict__ zs) {
    constexpr int BM = 32 * XF, BN = 64 * WF, ROWS = BM + BN;
    constexpr int LPW = ROWS / 64;             // a wave's 1 KB (8-row) DMAs per stage
    constexpr int XL = BM / 64;                // the first of them are rows of x
    constexpr int SH = GU ? WF / 2 : WF;
    constexpr int SB = 2 + (SH == 4 ? 2 : SH == 2 ? 1 : 0);  // where i / 4 sits in a w row
    constexpr int TN = GU ? BN / 2 : BN;       // output columns per tile
    constexpr int STAGE = ROWS * kF8Block;
    constexpr int XA = XF >= 4 ? 2 : 1;        // fragments of x read ahead
    constexpr bool GATHER = GU;                // rows of x by perm, else consecutive
    // store instructions that a wave issues at least for a whole tile
    constexpr int STORES = GU ? XF : XF * 4 * WF * (int)sizeof(T) / 16;
    static_assert((NS - 2) * (LPW + 1) + STORES < 64, "vmcnt range");
    static_assert(BM % 64 == 0 && (!GU || TN == kF8Block), "tile shape");
    __shared__ __attribute__((aligned(1024))) uint8_t ring[NS * STAGE];
    __shared__ __attribute__((aligned(16))) float s_sc[NS][ROWS];
    __shared__ __attribute__((aligned(16))) int32_t s_rt[GATHER ? 2 : 1][GATHER ? BM : 64];  // x rows of a tile
    __shared__ float s_amax[GU ? 4 : 1][GU ? BM : 1];

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave >> 2, wn = wave & 3;
    const int i16 = lane & 15, g = lane >> 4;
    const int nb = (int)hm_f8_blocks(p.K);
    const uint32_t pitch = (uint32_t)nb * kF8Block;
    const int N = (int)p.N, nbn = (int)hm_f8_blocks(p.N);
    const int ntn = (N + TN - 1) / TN;
    const int mt = table ? table[0].x : (int)((p.rows + BM - 1) / BM);
    const int total = mt * ntn;
    const int per = (total + kXcds - 1) / kXcds;
    const int step = gridDim.x / kXcds;
    const int jbeg = (blockIdx.x % kXcds) * per + blockIdx.x / kXcds;
    const int jend = min((int)(blockIdx.x % kXcds + 1) * per, total);
    if (jbeg >= jend) return;

    // The workgroup's tiles, one a lane, 64 at a time: a tile's place is a lane read, not a memory access
    // and divisions at the head of every tile.
    const int ntiles = (jend - jbeg + step - 1) / step;
    TileAt mine;
    auto list = [&](int first) __attribute__((always_inline)) {
        mine = tile_at<BM, TN>(p, table, min(jbeg + (first + lane) * step, jend - 1), mt, ntn);
    };
    auto info = [&](int i) __attribute__((always_inline)) {
        if ((i & 63) == 0) list(i);
        const int l = i & 63;
        return TileAt{__builtin_amdgcn_readlane(mine.e, l), __builtin_amdgcn_readlane(mine.row0, l),
                      __builtin_amdgcn_readlane(mine.nrows, l), __builtin_amdgcn_readlane(mine.n0, l)};
    };

    // ---- sources.  Lane l of DMA c of a wave: row 8 (wave + 8 c) + l / 8, position l % 8.
    const int lr = lane >> 3, pos = lane & 7;
    uint32_t voff[LPW];
    uint32_t soff;
    const uint8_t *xbase, *wbase;
    const float* sbase;
    const int sgrp = wave % LPW;               // this wave's 64 of the stage's ROWS scales
    // the x row (of the product's x) of tile row r
    auto make_src = [&](const TileAt& t, int m) __attribute__((always_inline)) {
        xbase = p.x + (GATHER ? 0 : (int64_t)t.row0 * pitch);
        wbase = p.w + (int64_t)t.e * p.w_expert;
        auto x_row = [&](int r) __attribute__((always_inline)) {
            if constexpr (!GATHER) return min(r, t.nrows - 1);
            const int v = s_rt[m][r];
            return v >= 0 && v < (int)p.x_rows ? v : 0;
        };
        // row r of the tile's w rows, of the expert's matrices (up follows gate)
        auto w_row = [&](int r) __attribute__((always_inline)) {
            if (GU && r >= TN) return N + min(t.n0 + r - TN, N - 1);
            return min(t.n0 + r, N - 1);
        };
#pragma unroll
        for (int c = 0; c < LPW; ++c) {
            const int r = 8 * (wave + 8 * c) + lr;
            if (c < XL) {
                voff[c] = (uint32_t)x_row(r) * pitch + 16 * (pos ^ ((r >> 1) & 7));
            } else {
                const int wr = r - BM;
                const int s = ((wr >> 1) & 1) | (((wr >> SB) & 3) << 1);
                voff[c] = (uint32_t)w_row(wr) * pitch + 16 * (pos ^ s);
            }
        }
        const int sr = 64 * sgrp + lane;
        if (64 * sgrp < BM) {
            sbase = p.xs + (GATHER ? 0 : (int64_t)t.row0 * nb);
            soff = (uint32_t)x_row(sr) * nb * 4;
        } else {
            sbase = p.ws + (int64_t)t.e * p.ws_expert;
            const int wr = w_row(sr - BM);
            if (BROW) soff = (uint32_t)wr * nb * 4;
            else if (GU && wr >= N) soff = (uint32_t)(nbn + (wr - N) / kF8Block) * nb * 4;
            else soff = (uint32_t)(wr / kF8Block) * nb * 4;
        }
    };
    // load c (0 .. LPW) of stage ks into a slot
    auto issue = [&](int slot, int ks, int c) __attribute__((always_inline)) {
        if (c < LPW)
            dma16_off(uni((c < XL ? xbase : wbase) + ks * kF8Block), voff[c],
                      ring + slot * STAGE + 1024 * wave + 8192 * c);
        else
            dma4_off(uni(sbase + ks), soff, &s_sc[slot][64 * sgrp]);
    };
    // the x rows of a gathered tile (rows past its last repeat that one)
    auto fetch_rows = [&](const TileAt& t, int m) __attribute__((always_inline)) {
        const int r = 64 * (wave % XL) + lane;
        dma4_off(uni(p.perm + t.row0), 4u * (uint32_t)min(r, t.nrows - 1), &s_rt[m][64 * (wave % XL)]);
    };

    // ---- fragments
    const int xrd = (wm * 16 * XF + i16) * kF8Block + 16 * (g ^ ((i16 >> 1) & 7));
    const int wrd = (BM + wn * 16 * SH + 4 * SH * (i16 >> 2) + (i16 & 3)) * kF8Block +
                    16 * (g ^ (((i16 >> 1) & 1) | ((i16 >> 2) << 1)));
    auto read = [&](const uint8_t* at, int off) __attribute__((always_inline)) {
        return join_frag(*reinterpret_cast<const v4i*>(at + off), *reinterpret_cast<const v4i*>(at + (off ^ 64)));
    };
    v4f acc[XF][WF];

    // The stage in `slot`, and between its matrix instructions the loads of stage `ks` into `to`: issued
    // at once they would hold the wave, since the vector memory unit takes one in 16 cycles.  A
    // multiply-add takes the result of the matrix instruction before the last.
    auto compute = [&](int slot, int to, int ks) __attribute__((always_inline)) {
        const uint8_t* st = ring + slot * STAGE;
        v8i raw[XA + 1];
        float sx[XA + 1];
        auto read_x = [&](int i) __attribute__((always_inline)) {
            raw[i % (XA + 1)] = read(st + i * 16 * kF8Block, xrd);
            sx[i % (XA + 1)] = s_sc[slot][wm * 16 * XF + 16 * i + i16];
        };
        // in the order of their use: the first instruction waits for four of the reads
        read_x(0);
        v8i wraw[WF];
#pragma unroll
        for (int j = 0; j < WF; ++j) {
            wraw[j] = read(st + (j / SH) * TN * kF8Block + (j % SH) * 4 * kF8Block, wrd);
            __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int i = 1; i < XA && i < XF; ++i) read_x(i);
        Frag<PREC> fw[WF];
        float sw1[2];
        v4f swv[WF];
        const float* sc = s_sc[slot] + BM + wn * 16 * SH;
        if constexpr (BROW) {
#pragma unroll
            for (int j = 0; j < WF; ++j) swv[j] = *reinterpret_cast<const v4f*>(sc + 4 * SH * g + 4 * j);
        } else {
            sw1[0] = sc[0];
            sw1[1] = GU ? sc[TN] : 0.0f;
        }
        constexpr int LAG = 2, NT = XF * WF, NI = LPW + 1;
        constexpr int EVERY = NT / NI > 1 ? 2 : 1;
        static_assert(NI * EVERY <= NT + EVERY - 1, "a slot for every load");
        v4f part[LAG + 1];
        float sxi[2];
        Frag<PREC> fx;
#pragma unroll
        for (int t = 0; t < NT + LAG; ++t) {
            if (t < NT) {
                const int i = t / WF, j = t % WF;
                if (j == 0) {
                    fx.set(raw[i % (XA + 1)]);
                    sxi[i & 1] = sx[i % (XA + 1)];
                    if (i + XA < XF) read_x(i + XA);
                }
                if (i == 0) fw[j].set(wraw[j]);
                part[t % (LAG + 1)] = block_product(fw[j], fx);
                if (t % EVERY == 0 && t / EVERY < NI) issue(to, ks, t / EVERY);
                __builtin_amdgcn_sched_barrier(0);
            }
            if (t >= LAG) {
                const int u = t - LAG, i = u / WF, j = u % WF;
#pragma unroll
                for (int v = 0; v < 4; ++v)
                    acc[i][j][v] = __builtin_fmaf(part[u % (LAG + 1)][v],
                                                  sxi[i & 1] * (BROW ? swv[j][v] : sw1[GU ? j / SH : 0]),
                                                  acc[i][j][v]);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    auto issue_all = [&](int to, int ks) __attribute__((always_inline)) {
#pragma unroll
        for (int c = 0; c <= LPW; ++c) issue(to, ks, c);
    };

    // ---- the stream
    TileAt cur = info(0);
    int m = 0;
    if constexpr (GATHER) {
        fetch_rows(cur, 0);
        wait_vmcnt<0>();
        lds_barrier();
    }
    make_src(cur, 0);
#pragma unroll
    for (int s = 0; s < NS - 1; ++s) issue_all(s, s);
#pragma unroll
    for (int i = 0; i < XF; ++i)
#pragma unroll
        for (int k = 0; k < WF; ++k) acc[i][k] = v4f{};
    int tile = 0, slot = 0, ks = 0, stored = 0;
    bool has_next = ntiles > 1;
    TileAt nxt = cur;
    if (has_next) nxt = info(1);
    while (true) {
        // this wave's loads of the stage have landed (at most the NS - 2 stages after it are in
        // flight), then every wave's; and every wave has read the slot that is refilled below
        // (after a whole tile's stores, which are younger, they may be in flight too)
        if (stored) wait_vmcnt<(NS - 2) * (LPW + 1) + STORES>();
        else wait_vmcnt<(NS - 2) * (LPW + 1)>();
        stored = 0;
        lds_barrier();
        int ahead = ks + NS - 1;
        if constexpr (GATHER) {
            if (ks == 0 && has_next) fetch_rows(nxt, m ^ 1);
        }
        if (ahead >= nb) {
            if (ahead == nb && has_next) make_src(nxt, m ^ 1);
            // (the stream's end loads stages once more that nothing reads, so that loads and waits have
            // no conditions)
            ahead -= nb;
        }
        const int to = slot == 0 ? NS - 1 : slot - 1;
        // a wave whose rows all lie past the tile's last only loads
        if (wm * 16 * XF < cur.nrows) compute(slot, to, ahead);
        else issue_all(to, ahead);
        slot = slot == NS - 1 ? 0 : slot + 1;
        if (++ks < nb) continue;
        const int r0 = wm * 16 * XF + i16, c0 = cur.n0 + wn * 16 * SH + 4 * SH * g;
        if constexpr (GU) store_z<XF, WF, BM>(p, cur, acc, s_amax, zq, zs, r0, c0, wn, g);
        else store_y<XF, WF, T>(p, cur, acc, y, r0, c0);
        stored = cur.nrows >= (wm + 1) * 16 * XF && (GU || (p.wide && cur.n0 + TN <= N));
        if (!has_next) break;
#pragma unroll
        for (int i = 0; i < XF; ++i)
#pragma unroll
            for (int k = 0; k < WF; ++k) acc[i][k] = v4f{};
        ks = 0;
        m ^= 1;
        cur = nxt;
        has_next = ++tile + 1 < ntiles;
        if (has_next) nxt = info(tile + 1);
    }
    wait_vmcnt<0>();  // the LDS is not given back under a load
}

int cu_count() {
    static int cached[64];
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) dev = 0;
    if (cached[dev] == 0) {
        int cus = 0;
        if (hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || cus < kXcds)
            cus = 256;
        cached[dev] = cus;
    }
    return cached[dev];
}

// per_cu workgroups share a CU (their LDS)
template <int XF, int WF, int NS, bool GU, bool BROW, bool PREC, typename T>
int launch(const Product& p, const int4* table, int64_t m_tiles, T* y, uint8_t* zq, float* zs,
           hipStream_t s) {
    constexpr int TN = GU ? 32 * WF : 64 * WF;
    constexpr size_t lds = (size_t)NS * (32 * XF + 64 * WF) * (kF8Block + 4);
    const int64_t tiles = m_tiles * ((p.N + TN - 1) / TN);
    if (tiles > INT_MAX / 2) return HM_ERR_OVERFLOW;
    const int64_t slots = (int64_t)cu_count() / kXcds * (lds > 76 * 1024 ? 1 : 2);
    const int64_t grid = kXcds * std::min((tiles + kXcds - 1) / kXcds, slots);
    hipLaunchKernelGGL((f8_tile_kernel<XF, WF, NS, GU, BROW, PREC, T>), dim3((unsigned)grid),
                       dim3(kTThreads), 0, s, p, table, y, zq, zs);
    HM_LAUNCHED();
    return HM_OK;
}

template <bool BROW, bool PREC, typename T>
int launch_plain(int bm, int bn, const Product& p, const int4* table, int64_t m_tiles, void* y,
                 hipStream_t s) {
    T* out = static_cast<T*>(y);
    if constexpr (!PREC) {
        if (bm == 256) return launch<8, 4, 2, false, BROW, PREC, T>(p, table, m_tiles, out, nullptr, nullptr, s);
    }
    if constexpr (!BROW) {  // the experts' down projection
        if (bm == 64 && bn == 256)
            return launch<2, 4, 3, false, BROW, PREC, T>(p, table, m_tiles, out, nullptr, nullptr, s);
    }
    if (bn == 256) return launch<4, 4, 3, false, BROW, PREC, T>(p, table, m_tiles, out, nullptr, nullptr, s);
    return bm == 128 ? launch<4, 2, 2, false, BROW, PREC, T>(p, table, m_tiles, out, nullptr, nullptr, s)
                     : launch<2, 2, 3, false, BROW, PREC, T>(p, table, m_tiles, out, nullptr, nullptr, s);
}

}  // namespace

bool hm_f8_tile_ok(const Product& p, bool gu) {
    const uint64_t pitch = (uint64_t)hm_f8_pitch(p.K), top = (uint64_t)1 << 32;
    return (!gu || p.K > 2 * kF8Block) && p.rows < (int64_t)1 << 30 && p.N < (int64_t)1 << 28 &&
           (uint64_t)(gu ? 2 * p.N : p.N) * pitch < top && (!p.perm || (uint64_t)p.x_rows * pitch < top) &&
           256 * pitch < top;
}

int hm_f8_launch_tiles(int bm, int bn, bool brow, const Product& p, const int4* table, int64_t m_tiles,
                       void* y, int32_t dtype, hipStream_t s) {
    if (dtype == HM_DTYPE_FP32)
        return brow ? launch_plain<true, true, float>(bm, bn, p, table, m_tiles, y, s)
                    : launch_plain<false, true, float>(bm, bn, p, table, m_tiles, y, s);
    if (dtype == HM_DTYPE_FP16)
        return brow ? launch_plain<true, false, hm_f16>(bm, bn, p, table, m_tiles, y, s)
                    : launch_plain<false, false, hm_f16>(bm, bn, p, table, m_tiles, y, s);
    return brow ? launch_plain<true, false, hm_bf16>(bm, bn, p, table, m_tiles, y, s)
                : launch_plain<false, false, hm_bf16>(bm, bn, p, table, m_tiles, y, s);
}

int hm_f8_launch_gateup_tiles(int bm, bool prec, const Product& p, const int4* table, int64_t m_tiles,
                              uint8_t* zq, float* zs, hipStream_t s) {
    float* none = nullptr;
    if (prec)
        return bm == 128 ? launch<4, 4, 3, true, false, true, float>(p, table, m_tiles, none, zq, zs, s)
                         : launch<2, 4, 3, true, false, true, float>(p, table, m_tiles, none, zq, zs, s);
    // (the FP8 instruction from 128 rows an expert on, which have no 64-row tiles)
    return bm == 256 ? launch<8, 4, 2, true, false, false, float>(p, table, m_tiles, none, zq, zs, s)
                     : launch<4, 4, 3, true, false, false, float>(p, table, m_tiles, none, zq, zs, s);
}
