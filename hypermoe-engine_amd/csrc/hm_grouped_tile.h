// hm_grouped_tile.h -- tiles of the 16-bit products (hm_grouped.h) through an LDS ring; one source for each type
// (hm_grouped_tile_f16.hip, hm_grouped_tile_bf16.hip).
//
// Persistent workgroups of WMC (rows of x) x WNC (columns) waves; a wave owns 16 XF x 16 WF results, a tile is BM = 16 XF
// WMC rows x BN = 16 WF WNC columns.  A stage is KB = 64 of k of both operands, 128 (BM + BN) bytes, moved to the LDS by
// DMA (operands off 16 bytes: through registers); the stages of consecutive tiles form one stream, so a tile's first
// stages load while its predecessor ends.  A stage is two steps of 32 k.  A step multiplies fragments that the step before
// read from the LDS, so no matrix instruction waits for the LDS; between the two steps lies the one barrier of a stage:
// the next stage has landed, and this one, which every wave now has in registers, is refilled.
//   k-major operand   LDS row r is 64 k of one row; its 16-byte piece c sits at position c ^ s(r), and s
//                     separates the 16 rows that a read takes of one piece.
//   other operands    LDS row k is BM or BN consecutive values; piece c sits at c ^ s(k).  Read by
//                     ds_read_b64_tr_b16: 16 lanes read 4 rows of k x 16 values and get them transposed.  The LDS
//                     serves 32 lanes, 8 rows, at once; s spreads those over all of its banks.
//   w                 fragment j's row i is column 32 (j / 2) + 8 (i / 4) + 4 (j % 2) + i % 4 of the wave's, so that a
//                     lane ends with 8 consecutive results of a row from two fragments, and four lanes with 32.  In
//                     the transposed form j % 2 is (j + i / 4) % 2, or half of the banks would stand idle.
//   order             tiles are cut into 8 ranges, one per XCD (workgroup i runs on XCD i % 8), whose workgroups take them
//                     in turn; within a group m-tiles by kSuper, so what is read by several workgroups at once is in
//                     one L2 (128 groups of 256 rows, 2048 x 1536: 279 us; each workgroup a range of its own: 418).
//
// Between memory and the matrix instructions where groups are of some 256 rows (their weights are read for few products),
// bound by the matrix instructions and the clock that they leave otherwise: 8192 x 8192 x 8192 to BF16 780 us, 1.41
// PFLOP/s (the library's product 1.45); 8 groups of 4096 rows, gate and up of 2048 x 768 with SwiGLU 165 us, 1.25 PFLOP/s;
// 128 groups of 256 rows 218 us, 4 TB/s (165 at the rate of reads, 137 by operations; without the results 204), and their
// weight gradients (805 MB of results) 281 to 293 us (without the results 192).  Off 16 bytes, 16 groups of 512 rows, 1001 x
// 1333: 70 us, 310 TFLOP/s, where a stage waits for the one that the registers hold.
#pragma once

#include "hm_grouped.h"
#include "hm_lds_dma.h"

#include <limits.h>

#include <algorithm>
#include <type_traits>

namespace {

constexpr int kXcds = 8;
constexpr int kSuper = 4;
constexpr int KB = 64;

__device__ __forceinline__ int uni(int v) { return __builtin_amdgcn_readfirstlane(v); }
template <typename P>
__device__ __forceinline__ P* uni(P* p) {
    const uint64_t v = reinterpret_cast<uint64_t>(p);
    return reinterpret_cast<P*>(((uint64_t)(uint32_t)uni((int)(v >> 32)) << 32) | (uint32_t)uni((int)v));
}

struct TileAt {
    int e;              // group
    int row0, nrows;    // rows of the tile (weight gradient: of the result)
    int n0;
    int k0, kn;         // weight gradient: the group's rows
    int nb;             // stages of k
};

template <int WMC, int WNC, int XF, int WF, int NS, bool DMA, GKind KIND, bool WK, typename T, typename O>
__global__ __launch_bounds__(64 * WMC * WNC, 2) void g_tile_kernel(GProduct p) {
    typedef typename Elem16<T>::v8 v8;
    constexpr bool WG = KIND == G_WEIGHT_GRAD, XK = !WG, GU = KIND == G_SWIGLU;
    constexpr int NW = WMC * WNC, BM = 16 * XF * WMC, BN = 16 * WF * WNC, SH = GU ? WF / 2 : WF, TN = GU ? BN / 2 : BN;
    constexpr int ROW = 2 * KB, RPB = 1024 / ROW, PCS = KB / 8;   // a k-major row's bytes, rows in 1 KB, pieces
    constexpr int STAGE = ROW * (BM + BN), WOFF = ROW * BM;
    constexpr int XL = BM / RPB / NW, LPW = (BM + BN) / RPB / NW;   // a wave's 1 KB loads a stage, of x first
    static_assert(RPB * NW <= 64, "ids");
    static_assert(DMA || NW == 4, "fetch() takes the swizzles to be the same for every c");
    static_assert(XF % 2 == 0 && (SH == 2 || SH == 4 || SH == 8) && BM % (RPB * NW) == 0 && BN % (RPB * NW) == 0, "tile");
    __shared__ __attribute__((aligned(1024))) uint8_t ring[NS * STAGE];
    __shared__ int s_pre[HM_GROUPED_MAX_GROUPS], s_cost[HM_GROUPED_MAX_GROUPS];  // m-tiles, cost to a group's end

    // (the barriers are hand-written: without this the compiler may take the ring, whose address would leave the
    // function nowhere where there is no DMA, to be out of their reach)
    asm volatile("" : : "s"((unsigned)(uintptr_t)(lds_ptr_t)ring) : "memory");
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / WNC, wn = wave % WNC, i16 = lane & 15, g = lane >> 4;
    const int N = (int)p.N, K = (int)p.K;
    const int ntn = (N + TN - 1) / TN;
    const T* xp = static_cast<const T*>(p.x);
    const T* wp = static_cast<const T*>(p.w);

    // ---- tiles: an XCD takes a range of them of an eighth of the cost, its workgroups every step-th tile of that.
    // A tile costs its rows, 16 at a time (weight gradient: its stages), and COST besides.
    constexpr int COST = WG ? 6 * 64 / KB : 3 * BM / 64;
    const int mtw = (int)((p.M + BM - 1) / BM);       // weight gradient: m-tiles
    int total, cost = 0;
    if (p.offsets) {
        // 4 groups a thread; a group's rows are cut to 0 .. rows, and none where its offsets descend
        const int e0 = 4 * threadIdx.x;
        int cnt[4], cst[4], sum = 0, csum = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            cnt[i] = cst[i] = 0;
            if (e0 + i < p.groups) {
                const int lo = max(0, p.offsets[e0 + i]);
                const int n = max(0, (int)min((int64_t)p.offsets[e0 + i + 1], p.rows) - lo);
                cnt[i] = (n + BM - 1) / BM;
                cst[i] = WG ? (n + KB - 1) / KB + COST : (n + 15) / 16 + cnt[i] * COST;
            }
            sum += cnt[i];
            csum += cst[i];
        }
        int incl = sum, cincl = csum;
#pragma unroll
        for (int m = 1; m < 64; m <<= 1) {
            const int o = __shfl_up(incl, m, 64), co = __shfl_up(cincl, m, 64);
            if (lane >= m) incl += o, cincl += co;
        }
        int* s_wave = reinterpret_cast<int*>(ring);
        if (lane == 63) s_wave[wave] = incl, s_wave[NW + wave] = cincl;
        __syncthreads();
        int base = incl - sum, cbase = cincl - csum;
        for (int i = 0; i < wave; ++i) base += s_wave[i], cbase += s_wave[NW + i];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            base += cnt[i];
            cbase += cst[i];
            if (e0 + i < p.groups) s_pre[e0 + i] = base, s_cost[e0 + i] = cbase;
        }
        __syncthreads();
        total = uni(WG ? p.groups * mtw * ntn : s_pre[p.groups - 1] * ntn);
        cost = uni(s_cost[p.groups - 1]);
    } else {
        total = (int)((p.rows + BM - 1) / BM) * ntn;
    }
    auto before = [&](const int* pre, int e) __attribute__((always_inline)) { return e ? uni(pre[e - 1]) : 0; };
    // how many of an ascending array are at most v / scale
    auto below = [&](const int* pre, int64_t scale, int64_t v) __attribute__((always_inline)) {
        int e = 0;
        for (int c = 0; c < p.groups; c += 64)
            e += __popcll(__ballot(c + lane < p.groups && pre[min(c + lane, p.groups - 1)] * scale <= v));
        return min(uni(e), p.groups - 1);
    };
    auto share = [&](int x) __attribute__((always_inline)) {
        if (!p.offsets) return (int)(((int64_t)total * x) >> 3);
        if (x == kXcds) return total;
        const int64_t v = (int64_t)cost * x;
        const int e = below(s_cost, kXcds, v);
        const int first = WG ? e * mtw * ntn : before(s_pre, e) * ntn;
        const int tiles = WG ? mtw * ntn : (uni(s_pre[e]) - before(s_pre, e)) * ntn;
        const int c0 = before(s_cost, e), c1 = uni(s_cost[e]);
        return uni(first + min(tiles, (int)((float)(v - (int64_t)c0 * kXcds) * tiles / ((float)(c1 - c0) * kXcds))));
    };
    const int step = gridDim.x / kXcds;
    const int jbeg = uni(share(blockIdx.x % kXcds)) + blockIdx.x / kXcds;
    const int jend = uni(share(blockIdx.x % kXcds + 1));
    if (jbeg >= jend) return;

    // Tile j (the same in every lane).
    auto tile_at = [&](int j) __attribute__((always_inline)) {
        TileAt t;
        int mt, jl = j;
        if constexpr (WG) {
            mt = mtw;
            t.e = j / (mt * ntn);
            jl = j - t.e * mt * ntn;
            const int lo = max(0, p.offsets[t.e]);
            const int hi = (int)min((int64_t)p.offsets[t.e + 1], p.rows);
            t.k0 = uni(lo);
            t.kn = uni(max(0, hi - lo));
            t.nb = max(1, (t.kn + KB - 1) / KB);
        } else if (p.offsets) {
            t.e = below(s_pre, 1, j / ntn);
            mt = uni(s_pre[t.e]) - before(s_pre, t.e);
            jl = j - before(s_pre, t.e) * ntn;
        } else {
            t.e = 0;
            mt = (int)((p.rows + BM - 1) / BM);
        }
        const int grp = jl / (kSuper * ntn), first = grp * kSuper;
        const int gm = max(1, min(mt - first, kSuper)), r = jl - first * ntn;
        const int m = first + r % gm;
        t.n0 = r / gm * TN;
        if constexpr (WG) {
            t.row0 = m * BM;
            t.nrows = min(BM, (int)p.M - t.row0);
        } else {
            const int lo = p.offsets ? uni(max(0, p.offsets[t.e])) : 0;
            const int hi = p.offsets ? uni((int)min((int64_t)p.offsets[t.e + 1], p.rows)) : (int)p.rows;
            t.row0 = lo + m * BM;
            t.nrows = min(BM, hi - t.row0);
            if (m < 0 || r < 0) t.row0 = lo, t.nrows = 0, t.n0 = N;   // (offsets of no batch: counts past 32 bits)
            t.k0 = 0;
            t.kn = K;
            t.nb = (K + KB - 1) / KB;
        }
        t.row0 = uni(t.row0);
        t.nrows = uni(t.nrows);
        t.n0 = uni(t.n0);
        return t;
    };

    // ---- the producer: the next stage that is loaded
    TileAt pt;
    int pj = jbeg, pks = 0;   // (its tile, its stage)
    uint32_t voff[LPW];
    const uint8_t *xbase, *wbase;
    int left = 0;              // k from the stage's first on
    int xcols = 0, wcols = 0;  // without DMA, operands that are not k-major: columns from this lane's on
    auto x_swz = [](int r) __attribute__((always_inline)) {
        if constexpr (XK) return (r >> 1) & 7;
        return ((r & 3) << 1) | (r & 8);
    };
    auto w_swz = [](int r) __attribute__((always_inline)) {
        if constexpr (WK) return ((r >> 1) & 1) | (((r >> 3) & 3) << 1);
        return (r & 1) | ((r & 2) << 1) | (r & 8);
    };
    // byte offset of the row of x that tile row r reads (from xbase)
    auto x_off = [&](const TileAt& t, int r) __attribute__((always_inline)) -> uint32_t {
        if (r >= t.nrows) return HM_BUF_RANGE;
        int row = r;
        if constexpr (GU) {
            if (p.perm) {
                row = p.perm[t.row0 + r];
                if (row < 0 || row >= (int)p.x_rows) row = 0;
            }
        }
        return (uint32_t)row * (uint32_t)K * 2;
    };
    // of the row of the group's matrix that row r of the staged w is (from wbase, the matrix's row n0)
    auto w_off = [&](const TileAt& t, int r) __attribute__((always_inline)) -> uint32_t {
        const bool up = GU && r >= TN;
        const int n = up ? r - TN : r;
        if (t.n0 + n >= N) return HM_BUF_RANGE;
        return (uint32_t)(up ? N + n : n) * (uint32_t)K * 2;
    };
    // where the stage is the last of k: what lies past it counts as zeros in both operands
    auto cut = [&]() __attribute__((always_inline)) {
        left = uni(pt.kn - pks * KB);
        if (left >= KB || (!DMA && XK && WK)) return;
        int l = lane;
        asm volatile("" : "+v"(l));
#pragma unroll
        for (int c = 0; c < LPW; ++c) {
            const bool isx = c < XL;
            const int b = wave + NW * (isx ? c : c - XL);
            int k;
            if ((isx && XK) || (!isx && WK)) {
                if (!DMA) continue;   // (these count what is left of a piece)
                const int r = RPB * b + l / PCS;
                k = 8 * (l % PCS ^ (isx ? x_swz(r) : w_swz(r)));
            } else {
                const int pcs = isx ? BM / 8 : BN / 8;
                k = b * (64 / pcs) + l / pcs;
            }
            if (k >= left) voff[c] = HM_BUF_RANGE;
        }
    };
    // ---- adapters: behind a tile's stages of k, for each adapter that its rows name (ascending) the stages of its
    // rank: mid, with the rows of other adapters as zeros, and the adapter's matrix.  A lane knows the adapters of the
    // tile's rows lane + 64 i.
    constexpr int IDS = KIND == G_ADAPTER ? (BM + 63) / 64 : 1;
    int ids[IDS];
    int low = -1;              // the adapter whose stages are loaded, -1: k's; INT_MAX: past the last tile
    int lows = 0;              // its stage
    auto read_ids = [&]() __attribute__((always_inline)) {
        int l = lane;
        asm volatile("" : "+v"(l));
#pragma unroll
        for (int i = 0; i < IDS; ++i) {
            const int r = 64 * i + l;
            ids[i] = r < pt.nrows ? p.ids[pt.row0 + r] : -1;
        }
        low = -1;
    };
    auto next_low = [&]() __attribute__((always_inline)) {
        if (low == INT_MAX) return false;
        if (low >= 0 && (lows + 1) * KB < p.rank) {
            ++lows;
            xbase += 2 * KB;
            wbase = uni(wbase + (WK ? 2 * KB : 2 * (int64_t)KB * N));
        } else {
            int v = INT_MAX;
#pragma unroll
            for (int i = 0; i < IDS; ++i) v = min(v, ids[i] > low && ids[i] < p.adapters ? ids[i] : INT_MAX);
            v = wave_min(v);
            if (v == INT_MAX) return false;
            low = v;
            lows = 0;
            xbase = uni(static_cast<const uint8_t*>(p.mid) + (int64_t)pt.row0 * p.rank * 2);
            wbase = uni(static_cast<const uint8_t*>(p.up) +
                        2 * ((int64_t)low * N * p.rank + (WK ? (int64_t)pt.n0 * p.rank : (int64_t)pt.n0)));
        }
        left = uni(p.rank - lows * KB);
        int l = lane;
        asm volatile("" : "+v"(l));
#pragma unroll
        for (int c = 0; c < LPW; ++c) {
            const bool isx = c < XL;
            const int b = wave + NW * (isx ? c : c - XL);
            if (isx || WK) {
                const int r = RPB * b + l / PCS, pc = l % PCS ^ (isx ? x_swz(r) : w_swz(r));
                const bool mine = isx ? __shfl(ids[RPB * NW * c / 64 % IDS], r & 63, 64) == low : pt.n0 + r < N;
                voff[c] = mine && (!DMA || 8 * pc < left) ? (uint32_t)r * (uint32_t)p.rank * 2 + 16 * pc : HM_BUF_RANGE;
            } else {
                const int r = b * (512 / BN) + l / (BN / 8), col = 8 * ((l % (BN / 8)) ^ w_swz(r));
                voff[c] = r < left && pt.n0 + col < N ? (uint32_t)r * (uint32_t)N * 2 + 2 * (uint32_t)col : HM_BUF_RANGE;
            }
        }
        pt.nb = 0;   // (each of these stages asks for the next one)
        return true;
    };
    auto make_src = [&]() __attribute__((always_inline)) {
        const TileAt& t = pt;
        int l = lane;
        asm volatile("" : "+v"(l));
        if constexpr (WG) {
            xbase = uni(reinterpret_cast<const uint8_t*>(xp + (int64_t)t.k0 * p.M + t.row0));
            wbase = uni(reinterpret_cast<const uint8_t*>(wp + (int64_t)t.k0 * N + t.n0));
        } else {
            xbase = uni(reinterpret_cast<const uint8_t*>(xp + (GU && p.perm ? 0 : (int64_t)t.row0 * K)));
            wbase = uni(reinterpret_cast<const uint8_t*>(wp + (int64_t)t.e * p.w_group +
                                                         (WK ? (int64_t)t.n0 * K : (int64_t)t.n0)));
        }
#pragma unroll
        for (int c = 0; c < LPW; ++c) {
            const bool isx = c < XL;
            const int b = wave + NW * (isx ? c : c - XL);
            if ((isx && XK) || (!isx && WK)) {
                const int r = RPB * b + l / PCS;
                const uint32_t row = isx ? x_off(t, r) : w_off(t, r);
                voff[c] = row + 16 * (l % PCS ^ (isx ? x_swz(r) : w_swz(r)));
            } else {
                const int pcs = isx ? BM / 8 : BN / 8;   // pieces a row
                const int ld = isx ? (int)p.M : N;
                const int r = b * (64 / pcs) + l / pcs;
                const int col = 8 * ((l % pcs) ^ (isx ? x_swz(r) : w_swz(r)));
                (isx ? xcols : wcols) = ld - (isx ? t.row0 : t.n0) - col;   // (the same for every c)
                voff[c] = (isx ? t.row0 : t.n0) + col < ld ? (uint32_t)r * (uint32_t)ld * 2 + 2 * (uint32_t)col
                                                          : HM_BUF_RANGE;
            }
        }
        cut();
        if constexpr (KIND == G_ADAPTER) read_ids();
    };
    // bytes from one stage's values to the next one's
    const int64_t xstep = XK ? 2 * KB : 2 * (int64_t)KB * p.M;
    const int64_t wstep = WK ? 2 * KB : 2 * (int64_t)KB * N;
    // load c of the producer's stage into a slot
    hm_buf xbuf, wbuf;
    v8 regs[DMA ? 1 : LPW];
    auto issue = [&](int slot, int c) __attribute__((always_inline)) {
        const bool isx = c < XL;
        const int b = wave + NW * (isx ? c : c - XL);
        uint8_t* to = ring + slot * STAGE + (isx ? 0 : WOFF) + 1024 * b;
        if constexpr (DMA) dma16_buf(isx ? xbuf : wbuf, voff[c], to);
        else *reinterpret_cast<v8*>(to + 16 * lane) = regs[c];
    };
    // Without DMA (operands off 16 bytes): the stage goes through registers, loaded one step ahead of the write.  A
    // piece that ends past its row's last value is loaded so far before that it ends there, and shifted.
    auto fetch = [&]() __attribute__((always_inline)) {
        if (left <= 0 || low == INT_MAX) {
#pragma unroll
            for (int c = 0; c < LPW; ++c) regs[c] = v8{};
            return;
        }
        int l = lane;
        asm volatile("" : "+v"(l));
        // values of a row, and from the stage's first piece on; whether every piece is whole
        const int xrow = XK ? (low >= 0 ? p.rank : K) : (int)p.M, wrow = WK ? (low >= 0 ? p.rank : K) : N;
        const int xleft = XK ? left : (int)p.M - pt.row0, wleft = WK ? left : N - pt.n0;
        const bool whole = xleft >= (XK ? KB : BM) && wleft >= (WK ? KB : BN);
        auto load = [&](auto kind) __attribute__((always_inline)) {
#pragma unroll
            for (int c = 0; c < LPW; ++c) {
                const bool isx = c < XL;
                const int r = 8 * (wave + NW * (isx ? c : c - XL)) + (l >> 3);
                const uint8_t* base = isx ? xbase : wbase;
                const bool in = voff[c] < HM_BUF_RANGE;
                int n = (isx && XK) || (!isx && WK) ? left - 8 * ((l & 7) ^ (isx ? x_swz(r) : w_swz(r)))
                        : isx                       ? xcols
                                                    : wcols;
                if constexpr (decltype(kind)::value == 2) {   // rows of fewer than 8 values
                    regs[c] = load_frag8<T>(reinterpret_cast<const T*>(base + voff[c]), in ? n : 0);
                    continue;
                }
                const bool some = in && n > 0;
                uint32_t off = some ? voff[c] : 0;
                u64x2 v;
                if constexpr (decltype(kind)::value == 0) {
                    v = load16(base + off);
                } else {
                    const uint32_t back = 16 * (8 - min(8, some ? n : isx ? xleft : wleft));   // bits
                    v = load16(base + (int64_t)off - back / 8);
                    if (back >= 64) v = u64x2{v[1] >> (back & 63), 0};
                    else if (back) v = u64x2{v[0] >> back | v[1] << (64 - back), v[1] >> back};
                }
                regs[c] = __builtin_bit_cast(v8, some ? v : u64x2{});
            }
        };
        if (xrow < 8 || wrow < 8) load(std::integral_constant<int, 2>{});
        else if (whole) load(std::integral_constant<int, 0>{});
        else load(std::integral_constant<int, 1>{});
    };
    // The descriptors of the producer's stage, ahead of its loads: a scalar register that the vector unit wrote may
    // be read by a memory instruction five wait states later, and the compiler does not look into theirs.
    auto describe = [&]() __attribute__((always_inline)) {
        if constexpr (!DMA) return;
        xbuf = make_buf(xbase);
        wbuf = make_buf(wbase);
        asm volatile("s_nop 4" : "+s"(xbuf), "+s"(wbuf));
    };
    uint32_t last = 0;         // bit s: the stage in slot s is its tile's last
    // to the stage after the one that went to `slot`
    auto advance = [&](int slot) __attribute__((always_inline)) {
        last &= ~(1u << slot);
        // (readfirstlane: the compiler does not see by itself that these are the same in every lane)
        pks = uni(pks + 1);
        if (pks < uni(pt.nb)) {
            xbase = uni(xbase + xstep);
            wbase = uni(wbase + wstep);
            cut();
            return;
        }
        if constexpr (KIND == G_ADAPTER) {
            if (next_low()) return;
        }
        last |= 1u << slot;
        pks = 0;
        if (uni(pj) + step < jend) {
            pj += step;
            pt = tile_at(pj);
            make_src();
        } else {   // past the last tile: stages of nothing, so that loads and waits have no conditions
            pt.nb = INT_MAX;
            pt.kn = INT_MAX;
            low = INT_MAX;
#pragma unroll
            for (int c = 0; c < LPW; ++c) voff[c] = HM_BUF_RANGE;
        }
    };

    // ---- fragments
    // k-major: one 16-byte read; otherwise two transposing reads of 8 bytes, in which lane i16 gives the place of 4
    // values of row i16 / 4 and gets the values of column i16
    int xrd, wrd[WK ? 1 : WF];
    const int trow = 8 * g + (i16 >> 2), tc = i16 & 3;
    if constexpr (XK) xrd = (wm * 16 * XF + i16) * ROW + 16 * (g ^ x_swz(i16));
    else xrd = trow * 2 * BM + 16 * ((wm * 2 * XF + (tc >> 1)) ^ x_swz(trow)) + 8 * (tc & 1);
    if constexpr (WK) {
        const int r = 8 * (i16 >> 2) + (i16 & 3);
        wrd[0] = WOFF + (wn * 16 * SH + r) * ROW + 16 * (g ^ w_swz(r));
    } else {
        const int at = WOFF + trow * 2 * BN + 16 * ((wn * 2 * WF + tc) ^ w_swz(trow)) + 8 * (tc & 1);
#pragma unroll
        for (int j = 0; j < WF; ++j) wrd[j] = at ^ (64 * (j >> 1)) ^ (8 * (j & 1));
    }
    auto read_x = [&](const uint8_t* st, int h, int i) __attribute__((always_inline)) {
        if constexpr (XK) {
            return *reinterpret_cast<const v8*>(st + (xrd ^ (64 * h)) + i * 16 * ROW);
        } else {
            const uint8_t* at = st + (xrd ^ (32 * i)) + 32 * h * 2 * BM;
            return read_transposed<v8>(at, 4 * 2 * BM);
        }
    };
    auto read_w = [&](const uint8_t* st, int h, int j) __attribute__((always_inline)) {
        if constexpr (WK) {
            return *reinterpret_cast<const v8*>(st + (wrd[0] ^ (64 * h)) +
                                                ((j / SH) * TN + 32 * ((j % SH) >> 1) + 4 * (j & 1)) * ROW);
        } else {
            const uint8_t* at = st + wrd[j] + 32 * h * 2 * BN;
            return read_transposed<v8>(at, 4 * 2 * BN);
        }
    };

    v4f acc[XF][WF];
    struct Frags {
        v8 x[XF], w[WF];
    };
    // One step: the products of `f`, and among them the reads of the next step's fragments (half h of the stage at
    // st) and, if LOAD, the loads of the producer's stage.
    constexpr int NT = XF * WF, NR = XF + WF;
    constexpr int RS = std::max(1, NT * 3 / 4 / NR), DS = std::max(1, NT / 2 / LPW);
    auto mma = [&](const Frags& f, Frags& n, const uint8_t* st, int h, bool load, int slot) __attribute__((always_inline)) {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const int i = t / WF, j = t % WF;
            acc[i][j] = Elem16<T>::mfma(f.w[j], f.x[i], acc[i][j]);
            if (t % RS == 0 && t / RS < NR) {
                // x 0, all of w, the rest of x: the order of their use
                const int q = t / RS;
                if (q == 0) n.x[0] = read_x(st, h, 0);
                else if (q <= WF) n.w[q - 1] = read_w(st, h, q - 1);
                else n.x[q - WF] = read_x(st, h, q - WF);
            }
            if (load && t % DS == 0 && t / DS < LPW) issue(slot, t / DS);
            __builtin_amdgcn_sched_barrier(0);
        }
    };

    // ---- results
    // (lanes are taken anew, or the compiler keeps every address of it through the main loop and spills)
    // WHOLE: all rows and columns of this wave are results, so nothing is asked and loads go out together.
    auto results = [&](const TileAt& t, auto whole_) __attribute__((always_inline)) {
        constexpr bool WHOLE = decltype(whole_)::value;
        int l = lane;
        asm volatile("" : "+v"(l));
        const int gg = l >> 4;
        const bool odd = !WK && (gg & 1);   // transposed reads: the two fragments of 8 columns in the other order
        const int c0 = t.n0 + wn * 16 * SH + 8 * gg;
        const int r0 = wm * 16 * XF + (l & 15);
        const int64_t at0 = (WG ? (int64_t)t.e * p.M + t.row0 : (int64_t)t.row0) + r0;
        // PAIR: a lane's two pieces of a row are 32 values apart, and four lanes' pieces 64 bytes.  Lanes i and i + 8 trade
        // one, so that a store takes 8 whole rows of 128 bytes instead of 16 halves.
        constexpr bool PAIR = WHOLE && SH == 4 && sizeof(O) == 2;
        const bool high = l & 8;
        auto put = [&](auto* to, int64_t ld, int n, int q, const float (&f)[8], u64x2& kept) __attribute__((always_inline)) {
            typedef std::remove_pointer_t<decltype(to)> E;
            if constexpr (!WHOLE) {
                store8(to, n, f);
            } else if constexpr (!PAIR) {
                stream8(to, f);
            } else if (q == 0) {
                kept = pack8<E>(f);
            } else {
                // (`to` is this row's second piece, `ld` what lies between rows)
                const u64x2 second = pack8<E>(f), got = other8(high ? kept : second);
                stream16(to + (high ? -8 * ld : -32), high ? got : kept);
                stream16(to + (high ? 0 : 8 * ld - 32), high ? second : got);
            }
        };
#pragma unroll
        for (int i = 0; i < XF; ++i) {
            if (!WHOLE && r0 + 16 * i >= t.nrows) continue;
            const int64_t row = at0 + 16 * i;
            u64x2 k0, k1, k2;
#pragma unroll
            for (int q = 0; q < SH; q += 2) {
                const int c = c0 + 16 * q, n = WHOLE ? 8 : N - c;
                if (n <= 0) continue;
                float a[8], b[8], d[8];
#pragma unroll
                for (int v = 0; v < 4; ++v) {
                    a[v] = odd ? acc[i][q + 1][v] : acc[i][q][v];
                    a[4 + v] = odd ? acc[i][q][v] : acc[i][q + 1][v];
                }
                if constexpr (GU) {
#pragma unroll
                    for (int v = 0; v < 8; ++v) {
                        b[v] = acc[i][SH + q + v / 4][v % 4];
                        d[v] = fast_silu(a[v]) * b[v];
                    }
                    put(static_cast<T*>(p.y) + row * N + c, N, n, q, d, k0);
                    if (p.pre_out) {
                        T* pre = static_cast<T*>(p.pre_out) + row * 2 * N + c;
                        put(pre, 2 * N, n, q, a, k1);
                        put(pre + N, 2 * N, n, q, b, k2);
                    }
                } else if constexpr (KIND == G_SWIGLU_GRAD) {
                    const T* pre = static_cast<const T*>(p.pre_in) + row * 2 * N + c;
                    load8(pre, n, b);
                    load8(pre + N, n, d);
                    float z[8];
#pragma unroll
                    for (int v = 0; v < 8; ++v) swiglu_grad(a[v], b[v], d[v], &a[v], &d[v], &z[v]);
                    T* to = static_cast<T*>(p.y) + row * 2 * N + c;
                    put(to, 2 * N, n, q, a, k0);
                    put(to + N, 2 * N, n, q, d, k1);
                    if (p.z) put(static_cast<T*>(p.z) + row * N + c, N, n, q, z, k2);
                } else {
                    O* y = static_cast<O*>(p.y) + row * N + c;
                    if (WG && p.accumulate) {
                        load8(y, n, b);
#pragma unroll
                        for (int v = 0; v < 8; ++v) a[v] += b[v];
                    }
                    put(y, N, n, q, a, k0);
                }
            }
        }
    };
    // ---- adapters: a tile in which an infinity or a NaN of an adapter's matrix met rows of others.  Their mid is 0 in that
    // adapter's stages, but 0 times either is NaN.  Only where the tile names such an adapter (one whose matrix is finite,
    // or a result that its own row makes infinite, harms no other row), and for rows of other adapters only: their
    // results anew, 16 rows at a time, fragments straight from memory, in the stages' order of k and with each row's own
    // adapter alone, so the bits are those that the tile leaves without it.  4096 rows, 2048 x 2048, rank 64, an adapter
    // of NaN that every tile names: 0.74 ms instead of 0.083 (transposed 2.1 instead of 0.086), all of x NaN 0.12.  (Result
    // by result it was 62 ms, for either.)
    auto rescue = [&](const TileAt& t) __attribute__((always_inline)) {
        if constexpr (KIND != G_ADAPTER) return;
        wait_vmcnt<0>();       // (the tile's results, some of which are written again)
        int l = lane;
        asm volatile("" : "+v"(l));
        const int gg = l >> 4, li = l & 15;
        const T* up = static_cast<const T*>(p.up);
        const int c0 = t.n0 + wn * 16 * SH, nc = min(16 * SH, N - c0);   // this wave's columns
        if (nc <= 0) return;
        int named[IDS];
#pragma unroll
        for (int i = 0; i < IDS; ++i) {
            const int r = 64 * i + l;
            named[i] = r < t.nrows ? p.ids[t.row0 + r] : -1;
        }
        int bad = -1;          // an adapter with such values in these columns
        bool more = false;     // there are others
#pragma unroll 1
        for (int cur = -1; !more;) {
            int v = INT_MAX;
#pragma unroll
            for (int i = 0; i < IDS; ++i) v = min(v, named[i] > cur && named[i] < p.adapters ? named[i] : INT_MAX);
            cur = wave_min(v);
            if (cur == INT_MAX) break;
            float f = 0.0f;
            auto look = [&](const T* at, int64_t n) __attribute__((always_inline)) {
                float w[8];
                load8(at, (int)min(n, (int64_t)8), w);
#pragma unroll
                for (int k = 0; k < 8; ++k) f = __builtin_fmaf(w[k], 0.0f, f);
            };
            if constexpr (WK) {
                const T* at = up + ((int64_t)cur * N + c0) * p.rank;
#pragma unroll 1
                for (int k = 8 * l; k < nc * p.rank; k += 512) look(at + k, nc * p.rank - k);
            } else {
                constexpr int PC = 2 * SH;   // pieces of 8 columns
#pragma unroll 1
                for (int k = l; k < PC * p.rank; k += 64) {
                    const int c = 8 * (k % PC);
                    look(up + ((int64_t)cur * p.rank + k / PC) * N + c0 + c, max(0, nc - c));
                }
            }
            if (__ballot(f != 0.0f)) {
                more = bad >= 0;
                bad = more ? bad : cur;
            }
        }
        if (bad < 0) return;
#pragma unroll 1
        for (int i = 0; i < XF; ++i) {
            const int r = wm * 16 * XF + 16 * i + li;
            const int64_t row = t.row0 + min(r, t.nrows - 1);
            int own = p.ids[row];
            if (own < 0 || own >= p.adapters) own = -1;
            const bool mine = r < t.nrows && (more || own != bad);
            if (!__ballot(mine)) continue;
            v4f (&sum)[WF] = acc[0];   // (the tile's are stored)
#pragma unroll
            for (int j = 0; j < SH; ++j) sum[j] = v4f{};
            // k, and then each adapter that these rows name; 32 values of rows of `ld` at a time, whose lanes `take` them
            const T *xa = xp + row * K, *wa = wp + (WK ? (int64_t)c0 * K : (int64_t)c0);
            int ld = K;
            bool take = true;
#pragma unroll 1
            for (int named = -1;;) {
#pragma unroll 1
                for (int k = 0; k < ld; k += 32) {
                    int q = lane;
                    asm volatile("" : "+v"(q));
                    const int k8 = 8 * (q >> 4), n = ld - k - k8;
                    const v8 b = load_frag8<T>(xa + k + k8, take ? n : 0);
#pragma unroll
                    for (int j = 0; j < SH; ++j) {
                        const uint32_t c = min(16 * j + (q & 15), nc - 1);   // (columns past the last are dropped)
                        v8 a;
                        if constexpr (WK) {
                            a = load_frag8<T>(uni(wa + k) + (c * (uint32_t)ld + k8), n);
                        } else {
                            Loose8<T> e;
#pragma unroll
                            for (int v = 0; v < 8; ++v)
                                e.v[v] = v < n ? uni(wa + (int64_t)k * N)[(uint32_t)(k8 + v) * (uint32_t)N + c] : (T)0.0f;
                            a = __builtin_bit_cast(v8, e);
                        }
                        const v4f s = Elem16<T>::mfma(a, b, sum[j]);
                        sum[j] = take ? s : sum[j];
                    }
                }
                named = wave_min(mine && own > named ? own : INT_MAX);
                if (named == INT_MAX) break;
                take = own == named;
                xa = static_cast<const T*>(p.mid) + row * p.rank;
                wa = up + (int64_t)named * N * p.rank + (WK ? (int64_t)c0 * p.rank : (int64_t)c0);
                ld = p.rank;
            }
            if (!mine) continue;
#pragma unroll
            for (int j = 0; j < SH; ++j) {
#pragma unroll
                for (int v = 0; v < 4; ++v) {
                    const int c = 16 * j + 4 * gg + v;
                    if (c < nc) static_cast<T*>(p.y)[row * N + c0 + c] = (T)sum[j][v];
                }
            }
        }
    };
    // memory instructions of the results at least, where this wave's rows and columns are whole and nothing is asked for
    // that may be left out (pre, z, what is added to): 16 bytes a lane are the most that one of them moves
    constexpr int STORES = XF * (GU ? SH / 2 : KIND == G_SWIGLU_GRAD ? 4 * SH / 2 : (int)sizeof(O) / 2 * SH / 2);
    auto whole = [&](const TileAt& t) __attribute__((always_inline)) {
        return t.nrows >= (wm + 1) * 16 * XF && t.n0 + TN <= N;
    };
    auto clear = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < XF; ++i)
#pragma unroll
            for (int j = 0; j < WF; ++j) acc[i][j] = v4f{};
    };

    // ---- the stream
    TileAt cur = tile_at(jbeg);
    int cj = jbeg, slot = 0;
    int stored = 0;            // steps whose wait comes before the end of a whole tile's stores
    pt = cur;
    make_src();
#pragma unroll
    for (int s = 0; s < NS; ++s) {
        if constexpr (DMA) describe();
        else fetch();
#pragma unroll
        for (int c = 0; c < LPW; ++c) issue(s, c);
        advance(s);
    }
    clear();
    Frags fa, fb;
    if constexpr (DMA) wait_vmcnt<(NS - 1) * LPW>();
    else fetch();
    lds_barrier();
    fa.x[0] = read_x(ring, 0, 0);
#pragma unroll
    for (int j = 0; j < WF; ++j) fa.w[j] = read_w(ring, 0, j);
#pragma unroll
    for (int i = 1; i < XF; ++i) fa.x[i] = read_x(ring, 0, i);
    // What a stage's barrier waits for: this wave's loads of the next stage have landed, then every wave's; and every
    // wave has read this stage (after a whole tile's stores, which are younger, they may be in flight too).
    auto meet = [&]() __attribute__((always_inline)) {
        if constexpr (DMA) {
            if (stored) wait_vmcnt<std::min(60, (NS - 2) * LPW + STORES)>();
            else wait_vmcnt<(NS - 2) * LPW>();
            stored = max(0, stored - 1);
        }
        lds_barrier();
    };
    // The step that reads the next stage's first fragments into `n` and refills this stage's slot; whether this stage
    // was its tile's last.
    auto turn = [&](const Frags& f, Frags& n) __attribute__((always_inline)) {
        const int next = slot == NS - 1 ? 0 : slot + 1;
        mma(f, n, ring + next * STAGE, 0, true, slot);
        const bool done = uni((int)(last >> slot)) & 1;
        advance(slot);
        if constexpr (!DMA) fetch();
        slot = next;
        return done;
    };
    while (true) {
        describe();
        mma(fa, fb, ring + slot * STAGE, 1, false, 0);
        meet();
        if (!turn(fb, fa)) continue;
        bool rescued = false;   // adapters: whether a result of the wave is not finite
        if constexpr (KIND == G_ADAPTER) {
            float f[4] = {};
#pragma unroll
            for (int i = 0; i < XF; ++i)
#pragma unroll
                for (int j = 0; j < WF; ++j)
#pragma unroll
                    for (int v = 0; v < 4; ++v) f[v] = __builtin_fmaf(acc[i][j][v], 0.0f, f[v]);
            rescued = __ballot(f[0] + f[1] + f[2] + f[3] != 0.0f);
        }
        const bool all = whole(cur);
        if (all) results(cur, std::true_type{});
        else results(cur, std::false_type{});
        stored = all ? NS - 1 : 0;
        if (__builtin_expect(rescued, false)) rescue(cur);
        cj += step;
        if (cj >= jend) break;
        cur = tile_at(cj);
        clear();
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
template <int WMC, int WNC, int XF, int WF, int NS, bool DMA, GKind KIND, bool WK, typename T, typename O>
int launch(const GProduct& p, hipStream_t s) {
    constexpr int BM = 16 * XF * WMC, BN = 16 * WF * WNC, TN = KIND == G_SWIGLU ? BN / 2 : BN;
    const int64_t n = (p.N + TN - 1) / TN;
    const int64_t m = KIND == G_WEIGHT_GRAD ? p.groups * ((p.M + BM - 1) / BM)
                      : p.offsets           ? p.rows / BM + std::min((int64_t)p.groups, p.rows)
                                            : (p.rows + BM - 1) / BM;
    if (m * n > INT_MAX / 2) return HM_ERR_OVERFLOW;
    const int64_t slots = (int64_t)cu_count() / kXcds * (NS * 2 * KB * (BM + BN) > 76 * 1024 ? 1 : 2);
    const int64_t grid = kXcds * std::min((m * n + kXcds - 1) / kXcds, slots);
    hipLaunchKernelGGL((g_tile_kernel<WMC, WNC, XF, WF, NS, DMA, KIND, WK, T, O>), dim3((unsigned)grid),
                       dim3(64 * WMC * WNC), 0, s, p);
    HM_LAUNCHED();
    return HM_OK;
}

template <int WMC, int WNC, int XF, int WF, int NS, bool DMA, typename T>
int launch_kind(GKind kind, bool wk, bool f32, const GProduct& p, hipStream_t s) {
    constexpr int BM = 16 * XF * WMC, BN = 16 * WF * WNC;
#define HM_G(KIND, WK, O) launch<WMC, WNC, XF, WF, NS, DMA, KIND, WK, T, O>(p, s)
    switch (kind) {
    case G_SWIGLU:
        if constexpr (BM < 256 && WNC == 2) return HM_G(G_SWIGLU, true, T);
        break;   // (launch_tiles has their own)
    case G_SWIGLU_GRAD:
        if constexpr (BM < 256) return HM_G(G_SWIGLU_GRAD, false, T);
        break;   // (hm_grouped.hip asks for none)
    case G_WEIGHT_GRAD:
        if constexpr (BM == BN) return f32 ? HM_G(G_WEIGHT_GRAD, false, float) : HM_G(G_WEIGHT_GRAD, false, T);
        break;   // (nor for 128 x 256)
    case G_ADAPTER: return wk ? HM_G(G_ADAPTER, true, T) : HM_G(G_ADAPTER, false, T);
    case G_MATMUL:
        if (wk) return f32 ? HM_G(G_MATMUL, true, float) : HM_G(G_MATMUL, true, T);
        return f32 ? HM_G(G_MATMUL, false, float) : HM_G(G_MATMUL, false, T);
    }
    return HM_ERR_UNSUPPORTED;
#undef HM_G
}

template <typename T>
int launch_tiles(int form, GKind kind, bool wk, bool f32, const GProduct& p, hipStream_t s) {
    // (gate and up: waves of twice the columns, whose results then fill lines)
    if (form == 256 && kind == G_SWIGLU) return launch<4, 2, 4, 8, 2, true, G_SWIGLU, true, T, T>(p, s);
    if (form == 128 && kind == G_SWIGLU) return launch<4, 2, 2, 8, 3, true, G_SWIGLU, true, T, T>(p, s);
    if (form == 256) return launch_kind<2, 4, 8, 4, 2, true, T>(kind, wk, f32, p, s);
    if (form == 128) return launch_kind<2, 4, 4, 4, 3, true, T>(kind, wk, f32, p, s);
    if (form == 64) return launch_kind<2, 2, 4, 4, 2, true, T>(kind, wk, f32, p, s);
    return launch_kind<2, 2, 4, 4, 2, false, T>(kind, wk, f32, p, s);
}

}  // namespace
