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

// The first or second half of a unit's reduction, the first the larger.
TMT_HD Unit half_of(Unit u, int half) {
    const int mid = u.kbeg + ((u.kend - u.kbeg + kFp8Block - 1) / kFp8Block + 1) / 2 * kFp8Block;
    if (half == 0) u.kend = mid;
    else u.kbeg = mid;
    return u;
}

// ---- few rows ------------------------------------------------------------------
// A wave's slot in LDS: 16 RB rows of a's codes and 16 NB of b's, 128 bytes each, and the
// scales of both; DEPTH of them.
template <int RB, int NB, bool ONE>
struct RowSlot {
    static constexpr int SA = (RB + NB) * 2048, SB = SA + 256, BYTES = SB + 256;
    static constexpr int ND = 2 * (RB + NB) + 2;  // loads of a block
    static constexpr int DEPTH = ONE ? 1 : RB * NB == 1 ? 4 : RB * NB == 2 ? 3 : RB * NB == 4 ? 2 : 1;
    static constexpr int WAVE = DEPTH * BYTES;    // bytes of a wave
    static_assert(8 * WAVE <= 160 * 1024 && 1024 * RB * NB <= WAVE && DEPTH * ND < 64, "LDS; a wave's sums; what a wait counts");
};
// A workgroup's outputs and the windows of its loads: rows past the last one, and chunks
// past a row's end, are zeros.
template <bool TILES, int RB, int NB>
struct RowBlock {
    int m0, n0, rows, cols;
    Window wa, wb;
    TMT_HD void set(const Fp8Params& p, unsigned block) {
        const int nb = (p.N + 16 * NB - 1) / (16 * NB);  // blocks of columns, which run fastest
        n0 = (int)(block % nb) * 16 * NB, m0 = (int)(block / nb) * 16 * RB;
        rows = min(p.M - m0, 16 * RB), cols = min(p.N - n0, 16 * NB);
        const uint32_t k16 = (uint32_t)(p.K + 15) & ~15u;
        wa = {address(p.a + (int64_t)m0 * p.lda), (uint32_t)(rows - 1) * (uint32_t)p.lda + k16};
        wb = {address(p.b + (int64_t)n0 * p.ldb), (uint32_t)(cols - 1) * (uint32_t)p.ldb + k16};
    }
    TMT_HD Window a_scales(const Fp8Params& p, int kb) const { return {address(p.as + (int64_t)kb * p.ldas + m0), 4u * (uint32_t)rows}; }
    TMT_HD Window b_scales(const Fp8Params& p, int kb) const {
        if constexpr (TILES) return {address(p.bs + (int64_t)(n0 / kFp8Block) * p.ldbs + kb), 4u};
        else return {address(p.bs + (int64_t)kb * p.ldbs + n0), 4u * (uint32_t)cols};
    }
};
// A load takes 8 rows of 128 codes, a lane 16 codes: chunk (of rows 8 .. 15: ^ 4) of the
// lane's row lane / 8, swizzled as they are read, and where it begins in a row from k on.
TMT_HD int row_chunk(int lane) { return (lane & 7) ^ (lane >> 4); }
TMT_HD uint32_t row_chunk_at(int K, int k, int chunk) { return k + 16 * chunk < K ? (uint32_t)(k + 16 * chunk) : 0x80000000u; }

// ---- plan ----------------------------------------------------------------------
// The kernel for few rows, 64 x 64 or 128 x 128 tiles (whole, or the last round's cut
// along the reduction), or 256 x 256 tiles: the one with the shortest estimate.
enum Fp8Kernel { FP8_ROWS_KERNEL, FP8_TILES_KERNEL, FP8_LARGE_KERNEL };
struct Fp8Plan {
    Fp8Kernel kernel = FP8_ROWS_KERNEL;
    LinearPlan tiles;
};
// Up to these the kernel for few rows, which needs no workspace, so that a decode step has none.
// A long reduction to few outputs would be faster in parts. us, M 64 / 72, whose rest goes
// over 64 x 64 or 128 x 128 tiles: K 32768, N 64 fp32 16.3 / 11.9, bf16 13.6 / 11.2; N 256 16.7 / 14.5,
// 14.1 / 13.1; K 16384, N 1024 bf16 10.1 / 13.7.
constexpr int kFp8FewRows = 64;
constexpr int kFp8MinSteps = 4;  // blocks of 128 that a part of a split reduction has at least

inline int fp8_steps(int K) { return (int)(((int64_t)K + kFp8Block - 1) / kFp8Block); }
inline int64_t fp8_count(int M, int N, int m, int n) { return (((int64_t)M + m - 1) / m) * (((int64_t)N + n - 1) / n); }
// Workgroups of a tile size that run at a time: 128 x 128 tiles of bf16 results and
// 256 x 256 tiles fill a CU.
inline int fp8_slots(int tile, bool f32, int cus) { return tile == 256 || (tile == 128 && !f32) ? cus : 2 * cus; }
// Workgroups of a launch of `units`, a multiple of 8: one for each XCD.
inline int fp8_grid(int tile, bool f32, int units, int cus) { return std::min((units + 7) & ~7, fp8_slots(tile, f32, cus) & ~7); }

// Workgroups of two groups of waves that halve the reduction: 64 x 64 tiles of which each
// has a CU for itself. us with / without: M 777, N 1024, K 4096 12.8 / 15.5, K 1024 6.2 /
// 6.3, K 512 5.2 / 4.8; fp32 2048 x 1024 x 1024 11.4 / 12.7, 777 x 1024 x 1024 8.0 / 7.5.
inline bool fp8_paired(int tile, int units, int K, int cus) { return tile == 64 && units <= cus && fp8_steps(K) >= 8; }

// Tiles whole or, parts >= 2, the rest of the last round's in parts.
inline LinearPlan fp8_tiles(bool f32, int M, int N, int K, int tile, int parts, int cus) {
    LinearPlan pl;
    pl.tile = tile;
    pl.tiles_m = (M + tile - 1) / tile;
    pl.tiles_c = (N + tile - 1) / tile;
    const int64_t tiles = (int64_t)pl.tiles_m * pl.tiles_c;
    pl.whole = (int)tiles;
    if (parts >= 2) {
        const int steps = fp8_steps(K), slots = fp8_slots(tile, f32, cus);
        pl.whole = (int)(tiles / slots * slots);
        pl.tail = (int)(tiles - pl.whole);
        pl.chunk = (steps + parts - 1) / parts * kFp8Block;
        pl.parts = (int)(((int64_t)K + pl.chunk - 1) / pl.chunk);
    }
    return pl;
}

// Outputs of a workgroup of the kernel for few rows: 64 x 64, 32 x 32, 16 x 32 (24)
// or 16 x 16, and not twice as many rows as there are.
inline int fp8_rows_block(int M, int N, int cus) {
    const int64_t enough = 3 * (int64_t)cus / 4;
    return M > 32 && fp8_count(M, N, 64, 64) >= enough ? 64 : M > 16 && fp8_count(M, N, 32, 32) >= enough ? 32 : fp8_count(M, N, 16, 32) >= enough ? 24 : 16;
}
// us, measured on one MI355X over M 1 .. 2304, N and K 256 .. 16000: a block's own time,
// that of a KiB of its operand rows (fp32: widened), and 1 us more where a CU runs a
// second one after the first: with more than one block of 128 a wave, and 64 x 64,
// they fill a CU's LDS.
inline double fp8_rows_time(bool f32, int M, int N, int K, int cus) {
    const int b = fp8_rows_block(M, N, cus), m = b == 24 ? 16 : b, n = b == 24 ? 32 : b;
    const double own = b == 64 ? 3.2 : b == 32 ? 0.8 : 0.1, kib = !f32 ? 0.0145 : b == 64 ? 0.023 : b == 32 ? 0.019 : 0.016;
    const double groups = (double)fp8_count(M, N, m, n) / cus, us = own + kib * (m + n) * (double)K / 1024;
    return b == 64 || fp8_steps(K) > 8 ? 1.6 + std::ceil(groups) * (us + 1.0) : 2.6 + std::max(1.0, groups) * us;
}
// us of tiles: start of a launch, a step with one workgroup per CU and with two.
struct Fp8Times {
    double start, one, two;
};
constexpr Fp8Times kFp8Times[2][2] = {{{3.4, 0.36, 0.53}, {4.2, 0.66, 0.66}},   // bf16 results: 64, 128
                                      {{3.2, 0.53, 0.87}, {4.2, 1.32, 2.35}}};  // fp32
inline double fp8_launch_time(const Fp8Times& t, int64_t units, int slots, double steps, int cus) {
    if (units == 0) return 0.0;
    const int64_t rounds = units / slots, rest = units % slots;
    return t.start + rounds * (steps * t.two + 0.5) + (rest == 0 ? 0.0 : steps * (rest <= cus ? t.one : t.two) + 0.5);
}
// A split reduction adds a launch for the sums and its partial tiles' way through the
// last-level cache and back.
inline double fp8_tiles_time(bool f32, const LinearPlan& pl, int K, int cus) {
    const Fp8Times& t = kFp8Times[f32][pl.tile == 128];
    const int slots = fp8_slots(pl.tile, f32, cus);
    if (pl.tail == 0 && fp8_paired(pl.tile, pl.whole, K, cus)) return t.start + (fp8_steps(K) + 1) / 2 * t.two + 1.0;
    double us = fp8_launch_time(t, pl.whole, slots, fp8_steps(K), cus);
    if (pl.tail > 0) {
        const double mib = (double)pl.tail * pl.parts * pl.tile * pl.tile * 4 / (1 << 20);
        us += fp8_launch_time(t, (int64_t)pl.tail * pl.parts, slots, pl.chunk / kFp8Block, cus) + 2.2 + 0.35 * mib;
    }
    return us;
}
inline double fp8_large_time(int M, int N, int K, int cus) {
    const double tiles = (double)fp8_count(M, N, 256, 256), fill = std::min(1.0, tiles / cus);
    return 6.0 + std::ceil(tiles / cus) * (fp8_steps(K) * (1.25 + 0.35 * fill) + 3.0);
}

// Measured (us, chosen / others): M 256, N 1024, K 4096 7.1 in the kernel for few rows
// / 10.3 on 64 x 64 tiles in four parts; M 777, N 1024, K 1024 6.2 on 64 x 64 / 8.0
// few rows, 9.3 on 128 x 128; M 777, N 1024, K 4096 12.8 on 64 x 64 / 17.4 on 128 x 128
// in four parts; M 777, N 4096, K 1024 10.4 on 128 x 128 / 13.2 on 64 x 64; M = N = 4096,
// K 1024 22.5 on 256 x 256 / 31.4 on 128 x 128. fp32: T 2048, N = K = 1280 17.6 on 64 x
// 64 / 22.3 on 128 x 128 in four parts; T 32768, N = K = 1024 90.6 on 128 x 128 in
// eight parts / 113 on 64 x 64 in two; T 16384, N = K = 256 14.9 on 64 x 64 in eight
// parts / 18.1 few rows.
inline Fp8Plan fp8_plan(bool tiles, bool f32, int M, int N, int K, int cus) {
    Fp8Plan best;
    if (M <= kFp8FewRows) return best;
    // a launch holds 2^32 threads
    double us = fp8_count(M, N, 16, 16) < (1 << 22) ? fp8_rows_time(f32, M, N, K, cus) : 1e30;
    if (tiles && !f32) {
        const double t = fp8_large_time(M, N, K, cus);
        if (t < us) us = t, best = {FP8_LARGE_KERNEL, fp8_tiles(f32, M, N, K, 256, 1, cus)};
    }
    for (int tile = 64; tile <= 128; tile *= 2) {
        const int64_t slots = fp8_slots(tile, f32, cus), rest = fp8_count(M, N, tile, tile) % slots;
        const int64_t most = rest > 0 ? std::min<int64_t>(slots / rest, fp8_steps(K) / kFp8MinSteps) : 1;
        for (int64_t parts = 1; parts <= std::max<int64_t>(most, 1); parts += parts < 8 ? 1 : parts / 4) {
            const LinearPlan pl = fp8_tiles(f32, M, N, K, tile, (int)parts, cus);
            const double t = fp8_tiles_time(f32, pl, K, cus);
            if (t < us) us = t, best = {FP8_TILES_KERNEL, pl};
        }
    }
    return best;
}
// An upper bound over both result types and all row counts up to M: partial tiles
// fill at most the workgroup slots, and neither tiles nor parts fall with M.
inline size_t fp8_workspace_bound(int M, int N, int K, int cus) {
    const int64_t parts = fp8_steps(K) / kFp8MinSteps;
    if (M <= kFp8FewRows || parts < 2) return 0;
    size_t most = 0;
    for (int tile = 64; tile <= 128; tile *= 2)
        most = std::max(most, (size_t)std::min<int64_t>(fp8_count(M, N, tile, tile) * parts, fp8_slots(tile, true, cus)) * tile * tile * 4);
    return most;
}

}  // namespace
}  // namespace tmt

#undef TMT_HD
