"""The tiled products of the 8-bit linear layer walked on the host, from the header that its
kernels and launchers use: every unit once, every step's codes and scales inside its windows,
every window inside its operand, partial tiles inside the workspace. With the compiler's check
of signed overflow, which ends the program."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "test-model-thing-cuda_amd", "csrc")
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")

pytestmark = pytest.mark.skipif(not os.path.exists(HIPCC) and shutil.which("hipcc") is None,
                                reason="hipcc not available")

WALK = r"""
#include <cstdio>
#include <cstdlib>
#include <map>
#include <vector>
#include "fp8_plan.hpp"
using namespace tmt;
#define FAIL(...)                \
    do {                         \
        std::printf(__VA_ARGS__); \
        std::printf(" (M %d N %d K %d lda %lld cus %d tile %d tiles %d)\n", p.M, p.N, p.K, (long long)p.lda, cus, TILE, (int)TILES); \
        std::exit(1);            \
    } while (0)

template <int TILE, bool TILES, bool SPLIT>
void walk(const Fp8Params& p, const LinearPlan& pl, int cus, bool f32) {
    const int units = SPLIT ? pl.tail * pl.parts : pl.whole;
    if (units == 0) return;
    const int grid = fp8_grid(TILE, f32, units, cus), k16 = (p.K + 15) & ~15, nbs = TILES && TILE == 256 ? 2 : 1;
    // operands end behind the last row's last whole chunk, scales behind the last row's
    const uint64_t a_end = address(p.a) + (uint64_t)(p.M - 1) * p.lda + k16, b_end = address(p.b) + (uint64_t)(p.N - 1) * p.ldb + k16;
    const int64_t kb = (p.K + 127) / 128, nb = (p.N + 127) / 128;
    const uint64_t as_end = address(p.as + (kb - 1) * p.ldas + p.M);
    const uint64_t bs_end = TILES ? address(p.bs + (nb - 1) * p.ldbs + kb) : address(p.bs + (kb - 1) * p.ldbs + p.N);
    std::map<std::pair<int, int>, std::vector<std::pair<int, int>>> seen;
    int64_t count = 0;
    const int groups = !SPLIT && fp8_paired(TILE, units, p.K, cus) ? 2 : 1;  // of waves, which halve a unit's reduction
    if (groups == 2 && grid < units) FAIL("%d units on %d workgroups", units, grid);
    for (int block = 0; block < grid; ++block)
        for (int half = 0; half < nbs * groups; ++half) {
            Unit u;
            int vb = block;
            if (!unit_at<TILE, SPLIT>(pl, p.K, vb, u)) continue;
            if (groups == 2) u = half_of(u, half);
            Fp8Cursor<TILE, TILES, SPLIT> at;
            at.nb = groups == 2 ? 0 : half;
            at.vl = vb;
            at.set(p, u);
            auto whole_grid = [&]() { return grid; };
            for (bool more = true; more;) {
                if (half == 0 || groups == 2) {
                    seen[{u.m0, u.c0}].push_back({u.kbeg, u.kend});
                    ++count;
                    if (SPLIT && ((int64_t)u.part + 1) * TILE * TILE * 4 > (int64_t)fp8_workspace_bound(p.M, p.N, p.K, cus))
                        FAIL("part %d is outside the workspace", u.part);
                }
                if (u.m0 >= p.M || u.c0 >= p.N || u.kbeg % 128 || u.kend <= u.kbeg || u.kend > p.K) FAIL("unit %d %d %d %d", u.m0, u.c0, u.kbeg, u.kend);
                const int rows = std::min(TILE, p.M - u.m0), cols = std::min(TILE, p.N - u.c0);
                for (int k = u.kbeg; k < u.kend; k += 128) {
                    const int chunks = std::min(8, at.chunks(p)), want = std::min(8, (p.K - k + 15) / 16);
                    if (chunks != want) FAIL("%d chunks at %d, not %d", chunks, k, want);
                    if (at.wa.at != address(p.a) + (uint64_t)u.m0 * p.lda + k || at.wb.at != address(p.b) + (uint64_t)u.c0 * p.ldb + k) FAIL("codes begin elsewhere");
                    // the last row's last chunk is inside, the next row's first is outside or not asked for
                    if (at.wa.bytes < (uint64_t)(rows - 1) * p.lda + 16 * want || at.wb.bytes < (uint64_t)(cols - 1) * p.ldb + 16 * want) FAIL("codes end early");
                    if (at.wa.bytes > (uint64_t)rows * p.lda || at.wb.bytes > (uint64_t)cols * p.ldb) FAIL("a row too many");
                    if (at.wa.at + at.wa.bytes > a_end || at.wb.at + at.wb.bytes > b_end) FAIL("codes pass their operand");
                    if (at.wsa.at != address(p.as + (int64_t)(k / 128) * p.ldas + u.m0) || at.wsa.bytes != 4u * rows || at.wsa.at + at.wsa.bytes > as_end) FAIL("scales of a");
                    if (TILES) {
                        const bool in = u.c0 + 128 * at.nb < p.N;
                        if (at.wsb.bytes != (in ? 4u : 0u)) FAIL("scale of b: %u bytes", at.wsb.bytes);
                        if (in && (at.wsb.at != address(p.bs + (int64_t)(u.c0 / 128 + at.nb) * p.ldbs + k / 128) || at.wsb.at + 4 > bs_end)) FAIL("scale of b");
                    } else if (at.wsb.at != address(p.bs + (int64_t)(k / 128) * p.ldbs + u.c0) || at.wsb.bytes != 4u * cols || at.wsb.at + at.wsb.bytes > bs_end) {
                        FAIL("scales of b");
                    }
                    at.next(p, pl, whole_grid);
                }
                vb += grid;
                more = unit_at<TILE, SPLIT>(pl, p.K, vb, u);
            }
            for (int n = 0; n < 6; ++n) {  // moves past the last step
                if (at.wa.bytes || at.wb.bytes || at.wsa.bytes || at.wsb.bytes || at.chunks(p) != 0) FAIL("not empty behind the last unit");
                at.next(p, pl, whole_grid);
            }
        }
    if (count != (int64_t)units * groups) FAIL("%lld units, not %d", (long long)count, units);
    for (auto& s : seen) {
        std::vector<std::pair<int, int>> v = s.second;
        std::sort(v.begin(), v.end());
        int k = 0;
        for (auto& r : v) {
            if (r.first != k) FAIL("tile %d %d: reduction from %d, not %d", s.first.first, s.first.second, r.first, k);
            k = r.second;
        }
        if (k != p.K) FAIL("tile %d %d ends at %d", s.first.first, s.first.second, k);
    }
}

template <int TILE, bool TILES>
int64_t tiles(const Fp8Params& p, const LinearPlan& pl, int cus, bool f32) {
    walk<TILE, TILES, false>(p, pl, cus, f32);
    walk<TILE, TILES, true>(p, pl, cus, f32);
    if ((int64_t)pl.tiles_m * pl.tiles_c != pl.whole + pl.tail) FAIL("%d + %d tiles", pl.whole, pl.tail);
    return 1;
}

int walked[2][2][2];
template <bool TILES>
void product(int M, int N, int K, int64_t lda, int64_t ldb, int cus) {
    Fp8Params p{};
    p.M = M, p.N = N, p.K = K, p.lda = lda, p.ldb = ldb;
    p.ldas = M + 3;
    p.ldbs = TILES ? (K + 127) / 128 + 1 : N + 5;
    p.a = reinterpret_cast<const uint8_t*>(0x100000000000ull);
    p.b = reinterpret_cast<const uint8_t*>(0x200000000000ull);
    p.as = reinterpret_cast<const float*>(0x300000000000ull);
    p.bs = reinterpret_cast<const float*>(0x400000000000ull);
    constexpr int TILE = 0;
    size_t last = 0;
    for (int m : {1, M / 3 + 1, M}) {  // a workspace serves fewer rows
        const size_t now = fp8_workspace_bound(m, N, K, cus);
        if (now < last) FAIL("the workspace of %d rows is smaller", m);
        last = now;
    }
    if (TILES) tiles<256, true>(p, fp8_tiles(false, M, N, K, 256, 1, cus), cus, false);
    for (bool f32 : {false, true}) {
        const Fp8Plan pl = fp8_plan(TILES, f32, M, N, K, cus);
        if (pl.kernel != FP8_TILES_KERNEL) continue;
        ++walked[f32][pl.tiles.tile == 128][pl.tiles.tail > 0];
        if (pl.tiles.tile == 64) tiles<64, TILES>(p, pl.tiles, cus, f32);
        else tiles<128, TILES>(p, pl.tiles, cus, f32);
    }
}

int main() {
    const int Ms[] = {1, 64, 65, 129, 301, 400, 777, 1000, 2048, 5003}, Ns[] = {8, 264, 1024, 1280, 4096}, Ks[] = {1, 100, 128, 129, 1024, 2056, 4096, 16500};
    for (int cus : {256, 304, 8})
        for (int M : Ms)
            for (int N : Ns)
                for (int K : Ks) {
                    if ((int64_t)M * N * K > 30ll << 30 && cus != 256) continue;
                    const int64_t k16 = (K + 15) / 16 * 16;
                    product<true>(M, N, K, k16, k16 + 16, cus);
                    product<false>(M, N, K, k16 + 48, k16, cus);
                }
    // the widest strides, and many tokens
    product<true>(700, 1024, 4096, 1 << 22, 1 << 22, 256);
    product<false>(700, 1024, 1 << 22, 1 << 22, 1 << 22, 256);
    product<true>(1 << 20, 512, 256, 256, 256, 256);
    for (int i = 0; i < 8; ++i)
        if (walked[i >> 2][(i >> 1) & 1][i & 1] == 0) {
            std::printf("no case %d\n", i);
            return 1;
        }
    std::printf("ok\n");
    return 0;
}
"""


def test_the_tiled_products(tmp_path):
    src, exe = tmp_path / "walk.hip", tmp_path / "walk"
    src.write_text(WALK)
    r = subprocess.run([HIPCC, "--offload-host-only", "-std=c++17", "-O1", "-I", CSRC,
                        "-Xarch_host", "-fsanitize=signed-integer-overflow",
                        "-Xarch_host", "-fsanitize-trap=signed-integer-overflow",
                        str(src), "-o", str(exe)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout == "ok\n", (r.returncode, r.stdout[-500:])
