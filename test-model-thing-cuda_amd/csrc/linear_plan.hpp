// linear_plan.hpp -- the linear layer's products in units, the choice of tiles
// and splits, and the windows that the kernels' loads go through. Host and
// device code, so that a host program can walk what the kernels walk.
#pragma once
#include <algorithm>
#include <cmath>

#include "linear.hpp"

#define TMT_HD __host__ __device__ __forceinline__

namespace tmt {
namespace {

// A window on global memory: loads read zeros past its `bytes`, so that no
// address has to be clamped and a reduction's tail is zero times zero,
// whatever lies behind the operands. Wave-uniform.
struct Window {
    uint64_t at;
    uint32_t bytes;
};
TMT_HD uint64_t address(const void* p) { return reinterpret_cast<uint64_t>(p); }
// The first `rows` of up to 64 rows of row_bytes, without the last one's end.
TMT_HD uint32_t rows_window(int rows, uint32_t row_bytes, uint32_t skip) {
    return rows > 0 ? (uint32_t)min(rows, 64) * row_bytes - skip : 0u;
}
// Back to a scalar register on the GPU: divisions run on the vector unit.
TMT_HD int uniform(int v) {
#ifdef __HIP_DEVICE_COMPILE__
    return __builtin_amdgcn_readfirstlane(v);
#else
    return v;
#endif
}

// ---- units -----------------------------------------------------------------
// tiles_m x tiles_c output tiles. The first `whole` are units of their own;
// the `tail` others, the last round's, are cut into `parts` along the
// reduction, `chunk` (a multiple of 256) each: a launch of its own writes
// their fp32 partial tiles, which linear_fixup_kernel adds in part order.
struct LinearPlan {
    int tile = 256, tiles_m = 0, tiles_c = 0, whole = 0, tail = 0, parts = 1, chunk = 0;
};
struct Unit {
    int m0, c0, kbeg, kend, part;
};
// Consecutive tiles go down 4 rows of tiles (or what 32 tiles leave where
// there are few columns), then to the next column, so that the 32 tiles that
// an XCD works on share operand slices in its L2.
TMT_HD void tile_at(const LinearPlan& pl, int j, int& mt, int& ct) {
    const int rows = pl.tiles_c >= 8 ? 4 : 32 / pl.tiles_c;
    const int blk = j / (rows * pl.tiles_c), rem = j - blk * (rows * pl.tiles_c);
    const int in = min(rows, pl.tiles_m - blk * rows);
    ct = rem / in;
    mt = blk * rows + (rem - ct * in);
}
// Unit of the workgroup's slot vb (blockIdx.x, + gridDim.x, ...). The hardware
// hands workgroup b to XCD b % 8 and the grid is a multiple of 8 where a
// workgroup takes several slots; each XCD takes runs of consecutive units.
template <int TILE, bool SPLIT>
TMT_HD bool unit_at(const LinearPlan& pl, int R, int vb, Unit& u) {
    const int n = SPLIT ? pl.tail * pl.parts : pl.whole, whole = n & ~255, per = (n - whole + 7) / 8;
    int j;
    if (vb < whole) {
        j = (((vb >> 8) << 3) + (vb & 7)) * 32 + ((vb >> 3) & 31);
    } else {
        const int i = (vb - whole) >> 3;
        j = whole + (vb & 7) * per + i;
        if (i >= per || j >= n) return false;
    }
    int mt, ct;
    u.kbeg = 0;
    u.kend = R;
    u.part = j;
    if constexpr (SPLIT) {
        const int q = j / pl.parts;
        u.kbeg = (j - q * pl.parts) * pl.chunk;
        u.kend = min(R, u.kbeg + pl.chunk);
        j = pl.whole + q;
    }
    tile_at(pl, j, mt, ct);
    u.m0 = uniform(mt * TILE);
    u.c0 = uniform(ct * TILE);
    u.kbeg = uniform(u.kbeg);
    u.kend = uniform(u.kend);
    return true;
}

// ---- the loads' cursors ------------------------------------------------------
// What stands behind the kernels' loads: the windows of the next K = 64 step (K
// = 256: both operands MXFP4) and the steps left in its unit. Past the last
// unit the windows are empty and stay so. Every window ends inside its operand.
// grid() is the launch's workgroups, asked for between units only: a scalar load
// in the steps makes every wait for LDS wait for all of it (forward T 777, N
// 4096, K 1024: 13.5 us with it, 12.7 without).

// FORWARD: activations, codes, scales.
template <int TILE, bool SPLIT>
struct FwdCursor {
    Window wa, wq, wsc;
    int left = 0, vl = 0;
    __host__ __device__ void set(const LinearParams& p, const Unit& n) {
        wa = {address(p.x + (int64_t)n.m0 * p.ldx + n.kbeg),
              (uint32_t)(min(p.T - n.m0, TILE) - 1) * (uint32_t)(p.ldx * 2) + (uint32_t)(p.K - n.kbeg) * 2};
        wq = {address(p.w + (int64_t)n.c0 * (p.K / 2) + n.kbeg / 2),
              (uint32_t)(min(p.N - n.c0, TILE) - 1) * (uint32_t)(p.K / 2) + (uint32_t)(p.K - n.kbeg) / 2};
        wsc = {address(p.ws + (int64_t)(n.kbeg / 32) * p.wlds + n.c0), (uint32_t)(2 * p.wlds) - n.c0};
        left = (n.kend - n.kbeg) >> 6;
    }
    template <class Grid>
    __host__ __device__ void next(const LinearParams& p, const LinearPlan& pl, Grid grid) {
        if (left == 0) return;  // no unit left
        if (--left > 0) {
            wa = {wa.at + 128, wa.bytes - 128};
            wq = {wq.at + 32, wq.bytes - 32};
            wsc.at += 2 * p.wlds;
            return;
        }
        Unit n;
        vl += grid();
        if (unit_at<TILE, SPLIT>(pl, p.K, vl, n)) set(p, n);
        else wa.bytes = wq.bytes = wsc.bytes = 0;
    }
};

// DX and DW: the weights' (DW: the checkpoint's) raw codes and scales, K = 64
// steps of 64 reduction rows.
template <int OP, int TILE, bool SPLIT>
struct GradCodesCursor {
    static constexpr bool DW = OP == LINEAR_DW;
    static constexpr int CB = DW ? 8 : 4;  // code bytes of 8 columns
    Window wq, wsc;
    int left = 0, vl = 0;
    int rows = 0;       // reduction rows not loaded yet
    uint32_t skip = 0;  // bytes of a row outside the window behind the last row
    TMT_HD static int64_t row_bytes(const LinearParams& p) { return DW ? p.K : p.K / 2; }
    __host__ __device__ void set(const LinearParams& p, const Unit& n) {
        left = (n.kend - n.kbeg + 63) >> 6;
        rows = n.kend - n.kbeg;
        skip = (uint32_t)n.c0 * CB / 8;
        wq = {address(p.w + n.kbeg * row_bytes(p) + skip), rows_window(rows, (uint32_t)row_bytes(p), skip)};
        const int blocks = min(p.K / 32 - n.c0 / 32, TILE / 32);
        wsc = {address(p.ws + (int64_t)(n.c0 / 32) * p.wlds + n.kbeg), (uint32_t)(blocks * p.wlds) - n.kbeg};
    }
    template <class Grid>
    __host__ __device__ void next(const LinearParams& p, const LinearPlan& pl, Grid grid) {
        if (left == 0) return;
        if (--left > 0) {
            rows -= 64;
            wq = {wq.at + 64 * row_bytes(p), rows_window(rows, (uint32_t)row_bytes(p), skip)};
            wsc = {wsc.at + 64, (uint32_t)max((int)wsc.bytes - 64, 0)};
            return;
        }
        Unit n;
        vl += grid();
        if (unit_at<TILE, SPLIT>(pl, DW ? p.T : p.N, vl, n)) {
            set(p, n);
        } else {
            wq.bytes = wsc.bytes = 0;
            rows = 0;
        }
    }
};

// DX and DW: dY.
template <int OP, int TILE, bool SPLIT>
struct GradRowsCursor {
    static constexpr bool DW = OP == LINEAR_DW;
    Window wa;
    int left = 0, vl = 0;
    int tail = 0;       // DW: rows of the unit's last step
    uint32_t skip = 0;  // DW: as above
    __host__ __device__ uint32_t step_window(uint32_t ldb) const { return (uint32_t)(left > 1 ? 64 : tail) * ldb - skip; }
    __host__ __device__ void set(const LinearParams& p, const Unit& n) {
        const uint32_t ldb = (uint32_t)(p.ldx * 2);
        left = (n.kend - n.kbeg + 63) >> 6;
        if constexpr (DW) {
            skip = ldb - (uint32_t)(p.N - n.m0) * 2;
            tail = n.kend - n.kbeg - 64 * (left - 1);
            wa = {address(p.x + (int64_t)n.kbeg * p.ldx + n.m0), step_window(ldb)};
        } else {
            wa = {address(p.x + (int64_t)n.m0 * p.ldx + n.kbeg),
                  (uint32_t)(min(p.T - n.m0, TILE) - 1) * ldb + (uint32_t)(p.N - n.kbeg) * 2};
        }
    }
    template <class Grid>
    __host__ __device__ void next(const LinearParams& p, const LinearPlan& pl, Grid grid) {
        const uint32_t ldb = (uint32_t)(p.ldx * 2);
        if (left == 0) return;
        if (--left > 0) {
            if constexpr (DW) wa = {wa.at + 64 * (uint64_t)ldb, step_window(ldb)};
            else wa = {wa.at + 128, wa.bytes - 128};
            return;
        }
        Unit n;
        vl += grid();
        if (unit_at<TILE, SPLIT>(pl, DW ? p.T : p.N, vl, n)) set(p, n);
        else wa.bytes = 0;
    }
};

// MATMUL on 128 x 128 tiles: K = 256 steps. Pieces past a row's end are another
// row's: they are not multiplied. A wave loads the scales of one operand, X's
// or (of_w) W's.
template <int TILE, bool SPLIT>
struct MxCursor {
    Window wx, ww, wsc;
    int kn = 0, kend = 0, vl = 0;
    bool left = true, of_w = false;
    __host__ __device__ void set(const LinearParams& p, const Unit& n) {
        kn = n.kbeg;
        kend = n.kend;
        wx = {address(p.xq + (int64_t)n.m0 * (p.K / 2) + kn / 2),
              (uint32_t)(min(p.T - n.m0, TILE) - 1) * (uint32_t)(p.K / 2) + (p.K - kn) / 2};
        ww = {address(p.w + (int64_t)n.c0 * (p.K / 2) + kn / 2),
              (uint32_t)(min(p.N - n.c0, TILE) - 1) * (uint32_t)(p.K / 2) + (p.K - kn) / 2};
        const uint32_t blocks = (uint32_t)min(8, (p.K - kn) / 32);
        const int64_t lds = of_w ? p.wlds : p.xlds;
        const int row = of_w ? n.c0 : n.m0;
        wsc = {address((of_w ? p.ws : p.xs) + (int64_t)(kn / 32) * lds + row), blocks * (uint32_t)lds - row};
    }
    template <class Grid>
    __host__ __device__ void next(const LinearParams& p, const LinearPlan& pl, Grid grid) {  // while left
        kn += 256;
        if (kn < kend) {
            wx = {wx.at + 128, wx.bytes - 128};
            ww = {ww.at + 128, ww.bytes - 128};
            const uint32_t gone = (uint32_t)(8 - min(8, (p.K - kn) / 32));  // blocks past the end in a last step
            const int64_t lds = of_w ? p.wlds : p.xlds;
            wsc = {wsc.at + 8 * lds, wsc.bytes - gone * (uint32_t)lds};
            return;
        }
        Unit n;
        vl += grid();
        left = unit_at<TILE, SPLIT>(pl, p.K, vl, n);
        if (left) set(p, n);
    }
};

// MATMUL on 256 x 256 tiles, K a multiple of 256.
template <int TILE>
struct MxLargeCursor {
    Window wx, ww, wsc;
    int left = 0, vl = 0;
    bool of_w = false;
    __host__ __device__ void set(const LinearParams& p, const Unit& n) {
        wx = {address(p.xq + (int64_t)n.m0 * (p.K / 2)), (uint32_t)min(p.T - n.m0, TILE) * (uint32_t)(p.K / 2)};
        ww = {address(p.w + (int64_t)n.c0 * (p.K / 2)), (uint32_t)min(p.N - n.c0, TILE) * (uint32_t)(p.K / 2)};
        const int row = of_w ? n.c0 : n.m0;
        wsc = {address((of_w ? p.ws : p.xs) + row), 8 * (uint32_t)(of_w ? p.wlds : p.xlds) - row};
        left = p.K / 256;
    }
    template <class Grid>
    __host__ __device__ void next(const LinearParams& p, const LinearPlan& pl, Grid grid) {
        if (left == 0) return;  // no unit left
        if (--left > 0) {
            wx = {wx.at + 128, wx.bytes - 128};
            ww = {ww.at + 128, ww.bytes - 128};
            wsc.at += 8 * (of_w ? p.wlds : p.xlds);
            return;
        }
        Unit n;
        vl += grid();
        if (unit_at<TILE, false>(pl, p.K, vl, n)) set(p, n);
        else wx.bytes = ww.bytes = wsc.bytes = 0;
    }
};

// Bytes of the window on a wave's outputs: `rows` rows `row` bytes apart, `cols`
// elements of `size` bytes in the last one.
TMT_HD uint32_t output_window(int rows, uint32_t row, int cols, int size) {
    return (uint32_t)(rows - 1) * row + (uint32_t)(cols * size);
}

// ---- plan ----------------------------------------------------------------------
struct Sizes {
    int M, C, R;  // output rows and columns, reduction length
};
inline Sizes sizes(LinearOp op, int T, int N, int K) {
    if (op == LINEAR_DX) return {T, K, N};
    if (op == LINEAR_DW) return {N, K, T};
    return {T, N, K};
}

// Workgroups that run at a time.
// (cus: compute units, asked for once a call; each question costs the host 30 ns,
// and a plan of many candidates would ask 100 times.)
inline int64_t tile_slots(int tile, int cus) { return (int64_t)cus * (tile == 256 ? 1 : 2); }
constexpr int kMinSteps = 4;  // K = 64 steps that a part of a split reduction has at least

inline LinearPlan plan_tiles(const Sizes& z, int tile, int64_t parts, int cus) {
    LinearPlan pl;
    pl.tile = tile;
    pl.tiles_m = (z.M + tile - 1) / tile;
    pl.tiles_c = (z.C + tile - 1) / tile;
    const int64_t tiles = (int64_t)pl.tiles_m * pl.tiles_c;
    pl.whole = (int)tiles;
    if (parts >= 2) {
        const int nk = (z.R + 63) / 64;
        pl.whole = (int)(tiles / tile_slots(tile, cus) * tile_slots(tile, cus));
        pl.tail = (int)(tiles - pl.whole);
        pl.chunk = (int)((nk + 4 * parts - 1) / (4 * parts)) * 256;  // whole steps of every kernel
        pl.parts = (nk * 64 + pl.chunk - 1) / pl.chunk;
    }
    return pl;
}

// Workgroups of a launch of `units`: a multiple of 8, one for each XCD.
inline int unit_grid(int tile, int units, int cus) { return std::min((units + 7) & ~7, (int)tile_slots(tile, cus) & ~7); }

// What a launch takes, in us, from its K = 64 steps. Measured on one MI355X
// over 16 .. 512 tiles and 4 .. 512 steps:
//   start  launch, first loads and epilogue of 128 x 128 tiles (256 x 256: 4 more)
//   one    a step of 128 x 128 tiles, one workgroup per CU (bound by latency)
//   two    the same with two
//   large  a step of 256 x 256 tiles (bound by the matrix cores)
struct StepTimes {
    double start, one, two, large;
};
constexpr StepTimes kTimes[4] = {{4.5, 0.62, 1.05, 1.45}, {2.5, 0.28, 0.48, 0.0}, {4.2, 0.82, 1.35, 1.75}, {4.2, 0.82, 1.35, 1.8}};
// A split reduction adds a launch for the sums and its partial tiles' way
// through the last-level cache and back.
constexpr double kSplitStart = 3.5, kSplitPerMiB = 0.25;

inline double round_time(const StepTimes& t, int tile, int64_t units, double steps, int cus) {
    if (tile == 256) return 2.0 + steps * t.large;
    return steps * (units <= cus ? t.one : t.two);
}
inline double plan_time(const StepTimes& t, const Sizes& z, int tile, int64_t parts, int cus) {
    const int64_t slots = tile_slots(tile, cus);
    const int64_t tiles = (int64_t)((z.M + tile - 1) / tile) * ((z.C + tile - 1) / tile);
    const int64_t whole = tiles / slots, rest = tiles - whole * slots;
    const double nk = (z.R + 63) / 64;
    double us = t.start + (tile == 256 ? 4.0 : 0.0) + whole * round_time(t, tile, slots, nk, cus);
    if (rest == 0) return us;
    if (parts < 2) return us + round_time(t, tile, rest, nk, cus);
    const double mib = (double)(rest * parts) * tile * tile * 4 / (1 << 20);
    return us + round_time(t, tile, rest * parts, std::ceil(nk / parts), cus) + (whole > 0 ? t.start : 0.0) + kSplitStart + kSplitPerMiB * mib;
}

// The tile size and split with the shortest estimate. Measured (us, chosen /
// others): forward T 777, N 4096, K 1024 14.9 on whole 128 x 128 tiles / 23.7 in
// two parts, 30.2 on 256 x 256; T 777, N 1024, K 4096 20.7 in four parts / 27.2
// in two, 38.2 whole; dX T 777, N 4096, K 1024 23.9 in four parts / 28.5 in
// three; dW T 32768, N 1024, K 1024 95 on 256 x 256 tiles in 16 parts / 107 on
// 128 x 128 in 8; T 16384, N 256, K 256 16.7 in 32 parts / 32 in 8.
inline LinearPlan linear_plan(LinearOp op, int T, int N, int K, int cus, double* us) {
    const Sizes z = sizes(op, T, N, K);
    const StepTimes& t = kTimes[op];
    int best_tile = 128;
    int64_t best_parts = 1;
    double best = 1e30;
    for (int tile = 128; tile <= (op == LINEAR_MATMUL ? 128 : 256); tile *= 2) {
        const int64_t tiles = (int64_t)((z.M + tile - 1) / tile) * ((z.C + tile - 1) / tile);
        const int64_t rest = tiles % tile_slots(tile, cus);
        const int64_t most = rest > 0 ? std::min<int64_t>(tile_slots(tile, cus) / rest, (z.R + 63) / 64 / kMinSteps) : 1;
        for (int64_t parts = 1; parts <= std::max<int64_t>(most, 1); parts += parts < 8 ? 1 : parts / 4) {
            const double c = plan_time(t, z, tile, parts, cus);
            if (c < best) best = c, best_tile = tile, best_parts = parts;
        }
    }
    *us = best;
    return plan_tiles(z, best_tile, best_parts, cus);
}

// Whether 256 x 256 tiles of MXFP4 x MXFP4 are estimated to be faster: rounds of
// one tile per CU, 5.0 us and 1.9 a step (K = 256), against rounds of 128 x 128
// tiles at two per CU, 1.95 and 1.13, from two of those on. Measured (us, 128 /
// 256): T 65536, N 4096, K 512 134 / 137, K 1024 226 / 206; T 16384, N 4096, K
// 1024 53 / 55, K 2048 87 / 84; T 65536, N 1024, K 4096 152 / 143; T 20011, N
// 2736, K 768 47 / 64.
inline bool mx_large(int T, int N, int K, int cus) {
    const int64_t small = (int64_t)((T + 127) / 128) * ((N + 127) / 128), big = (int64_t)((T + 255) / 256) * ((N + 255) / 256);
    if (K % 256 != 0 || small < 2 * tile_slots(128, cus)) return false;
    const double steps = K / 256, slots2 = (double)tile_slots(128, cus), slots1 = (double)tile_slots(256, cus);
    return 3.0 + std::ceil(big / slots1) * (5.0 + 1.9 * steps) < std::ceil(small / slots2) * (1.95 + 1.13 * steps);
}
// The kernel for few tokens runs where its estimate in us, measured over T 1 ..
// 777, N and K 256 .. 4096, is not above the tiles'. T 777, N 1024, K 1024 10.1
// (tiles 13.6), T 512, N 4096, K 1024 17.7 (tiles 14.2).
// It stays below 2^21 workgroups; a launch holds 2^32 threads.
inline double rows_time(int T, int N, int K) {
    if ((int64_t)T * N >= (int64_t)1 << 30) return 1e30;
    return 3.0 + 7.2e-9 * ((double)T * N * K);
}

// An upper bound over all token counts up to T, so that a workspace for T
// serves fewer: tail tiles times parts fill at most the workgroup slots, and
// neither tiles nor parts fall with T. Both operands in MXFP4 are split on 128 x
// 128 tiles only. A split reduction's estimate is at least its start and end
// and the fewest steps of a part: where the kernel for few tokens is estimated to
// take no longer, no call of up to T tokens is split.
inline size_t workspace_bound(LinearOp op, int T, int N, int K, int cus) {
    const Sizes z = sizes(op, T, N, K);
    const StepTimes& t = kTimes[op];
    if (op == LINEAR_FORWARD && rows_time(T, N, K) <= t.start + kMinSteps * t.one + kSplitStart) return 0;
    size_t most = 0;
    for (int tile = 128; tile <= (op == LINEAR_MATMUL ? 128 : 256); tile *= 2) {
        const int64_t tiles = (int64_t)((z.M + tile - 1) / tile) * ((z.C + tile - 1) / tile);
        const int64_t parts = (z.R + 63) / 64 / kMinSteps;
        if (parts < 2) continue;
        const int64_t units = std::min(tiles * parts, tile_slots(tile, cus));
        most = std::max(most, (size_t)units * tile * tile * 4);
    }
    return most;
}

}  // namespace
}  // namespace tmt

#undef TMT_HD
