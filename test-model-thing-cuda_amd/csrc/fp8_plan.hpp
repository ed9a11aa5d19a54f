// fp8_plan.hpp -- the 8-bit linear layer's products in units, the choice of
// kernels and splits, and the windows that their loads go through. Host and device
// code, so that a host program can walk what the kernels walk.
#pragma once
#include "fp8.hpp"
#include "linear_plan.hpp"

#define TMT_HD __host__ __device__ __forceinline__

namespace tmt {
namespace {

// What stands behind the tiled kernels' loads: the windows of the next step (a
// block of 128 codes of both operands, and its scales) and the steps left in its
// unit. Past the last unit the windows are empty and stay so. Every window ends
// inside its operand: rows past the last one read zeros, and what lies between a
// row's codes and its stride is another matter, which chunks() settles.
template <int TILE, bool TILES, bool SPLIT>
struct Fp8Cursor {
    Window wa, wb, wsa, wsb;
    int left = 0, vl = 0;
    int k = 0;        // of the next step
    int nb = 0;       // tiles: the wave's 128 columns of the unit's
    // Chunks of 16 codes that a row has left: what lies behind them may be anything.
    TMT_HD int chunks(const Fp8Params& p) const { return left > 0 ? (p.K - k + 15) >> 4 : 0; }
    __host__ __device__ void set(const Fp8Params& p, const Unit& n) {
        const int rows = min(p.M - n.m0, TILE), cols = min(p.N - n.c0, TILE), k16 = (p.K - n.kbeg + 15) & ~15;
        k = n.kbeg;
        left = (n.kend - n.kbeg + kFp8Block - 1) / kFp8Block;
        wa = {address(p.a + (int64_t)n.m0 * p.lda + k), (uint32_t)(rows - 1) * (uint32_t)p.lda + (uint32_t)k16};
        wb = {address(p.b + (int64_t)n.c0 * p.ldb + k), (uint32_t)(cols - 1) * (uint32_t)p.ldb + (uint32_t)k16};
        const int64_t kb = k / kFp8Block;
        wsa = {address(p.as + kb * p.ldas + n.m0), (uint32_t)rows * 4u};
        if constexpr (TILES) wsb = {address(p.bs + (int64_t)(n.c0 / kFp8Block + nb) * p.ldbs + kb), kFp8Block * nb < cols ? 4u : 0u};
        else wsb = {address(p.bs + kb * p.ldbs + n.c0), (uint32_t)cols * 4u};
    }
    template <class Grid>
    __host__ __device__ void next(const Fp8Params& p, const LinearPlan& pl, Grid grid) {
        if (left == 0) return;  // no unit left
        if (--left > 0) {
            k += kFp8Block;
            wa = {wa.at + kFp8Block, wa.bytes - kFp8Block};
            wb = {wb.at + kFp8Block, wb.bytes - kFp8Block};
            wsa.at += 4 * p.ldas;
            wsb.at += TILES ? 4 : 4 * p.ldbs;
            return;
        }
        Unit n;
        vl += grid();
        if (unit_at<TILE, SPLIT>(pl, p.K, vl, n)) set(p, n);
        else wa.bytes = wb.bytes = wsa.bytes = wsb.bytes = 0;
    }
};

// ---- plan ----------------------------------------------------------------------
struct Fp8Plan {
    bool rows = false;  // the kernel for few rows
    LinearPlan tiles;
};
constexpr int kFp8MinSteps = 4;  // blocks of 128 that a part of a split reduction has at least

// Tiles of 128 x 128 whole, the rest (fewer tiles than run at a time) in `parts`.
inline LinearPlan fp8_tiles(int M, int N, int K, int tile, int parts, int cus) {
    LinearPlan pl;
    pl.tile = tile;
    pl.tiles_m = (M + tile - 1) / tile;
    pl.tiles_c = (N + tile - 1) / tile;
    const int64_t tiles = (int64_t)pl.tiles_m * pl.tiles_c;
    pl.whole = (int)tiles;
    if (parts >= 2) {
        const int steps = (K + kFp8Block - 1) / kFp8Block;
        pl.whole = (int)(tiles / tile_slots(tile, cus) * tile_slots(tile, cus));
        pl.tail = (int)(tiles - pl.whole);
        pl.chunk = (steps + parts - 1) / parts * kFp8Block;
        pl.parts = (K + pl.chunk - 1) / pl.chunk;
    }
    return pl;
}
inline Fp8Plan fp8_plan(bool f32, int M, int N, int K, int cus) {
    Fp8Plan pl;
    pl.rows = M <= 64 || K == 0;
    if (pl.rows) return pl;
    const int64_t tiles = (int64_t)((M + 127) / 128) * ((N + 127) / 128), slots = tile_slots(128, cus), rest = tiles % slots;
    const int64_t most = rest > 0 ? std::min<int64_t>(slots / rest, (K + kFp8Block - 1) / kFp8Block / kFp8MinSteps) : 1;
    pl.tiles = fp8_tiles(M, N, K, 128, (int)std::max<int64_t>(most, 1), cus);
    return pl;
}
inline bool fp8_large(int M, int N, int K, int cus) {
    const int64_t big = (int64_t)((M + 255) / 256) * ((N + 255) / 256);
    return big >= tile_slots(256, cus);
}
// An upper bound over all row counts up to M: partial tiles fill at most the
// workgroup slots, and neither tiles nor parts fall with M.
inline size_t fp8_workspace_bound(int M, int N, int K, int cus) {
    const int64_t tiles = (int64_t)((M + 127) / 128) * ((N + 127) / 128), parts = (K + kFp8Block - 1) / kFp8Block / kFp8MinSteps;
    if (M <= 64 || parts < 2) return 0;
    return (size_t)std::min(tiles * parts, tile_slots(128, cus)) * 128 * 128 * 4;
}

}  // namespace
}  // namespace tmt

#undef TMT_HD
