"""Launch arithmetic of the microscaled linear layer on the host, from the
header that its kernels and launchers use, with the compiler's check of signed
overflow, which ends the program."""
import ctypes
import os
import shutil
import subprocess

import pytest

import tmt_moe

A, i64 = 0x10000, ctypes.c_int64  # a 16-byte aligned address, never followed

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "test-model-thing-cuda_amd", "csrc")
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")

pytestmark = pytest.mark.skipif(not os.path.exists(HIPCC) and shutil.which("hipcc") is None,
                                reason="hipcc not available")


def _run(tmp_path, program):
    src, exe = tmp_path / "launch.hip", tmp_path / "launch"
    src.write_text(program)
    r = subprocess.run([HIPCC, "--offload-host-only", "-std=c++17", "-O1", "-I", CSRC,
                        "-Xarch_host", "-fsanitize=signed-integer-overflow",
                        "-Xarch_host", "-fsanitize-trap=signed-integer-overflow",
                        str(src), "-o", str(exe)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and r.stdout == "ok\n", (r.returncode, r.stdout)


WIDEST = r"""
#include <cstdio>
#include "linear.hpp"
int main() {
    const int widths[] = {32, 64, 96, 128, 224, 256, 288, 4096, 1 << 22, 2147483392, 2147483424, 2147483616};
    for (int K : widths) {
        const int64_t cols = K >= 256 ? 256 : K >= 128 ? 128 : 64, tiles = ((int64_t)K + cols - 1) / cols;
        if (tmt::mx_tiles_per_row(K) != tiles || tmt::mx_tiles(1, K) != tiles) {
            std::printf("K %d: %d tiles a row\n", K, tmt::mx_tiles_per_row(K));
            return 1;
        }
    }
    std::printf("ok\n");
    return 0;
}
"""


def test_tiles_of_the_widest_rows(tmp_path):
    """Rows of any multiple of 32 columns that 32 bits hold."""
    _run(tmp_path, WIDEST)


@pytest.mark.parametrize("rows,K", [((1 << 28) - 1, 256), ((1 << 28) - 15, 256), ((1 << 28) - 15, 224), ((1 << 24) - 1, 4096),
                                    ((1 << 27) - 1, 512)])
def test_rows_that_fill_a_launch_are_refused(rows, K):
    """A tile is 16 or 32 rows: with those of the last one, 2^24 workgroups of
    256 threads, more than one launch holds."""
    lib = tmt_moe.load_library()
    for rc in (lib.tmt_moe_mx_quantize(None, 0, 0, A, i64(K), rows, K, A, A, i64(rows)),
               lib.tmt_moe_mx_dequantize(None, 1, A, A, i64(rows), rows, K, 1, A, i64(K))):
        assert rc == -1 and "2^36" in tmt_moe.last_error()


LARGEST = r"""
#include <cstdio>
#include "linear.hpp"
int main() {  // accepted: rows and columns, rounded up, under 2^36 values
    for (int64_t K = 32; K < (1ll << 31); K = K < 512 ? K + 32 : K * 2 - 32) {
        const int64_t cols = (K + 255) / 256 * 256, tile = K < 256 ? 32 : 16;
        const int64_t most = ((1ll << 36) - 1) / cols / tile * tile;
        const int rows = (int)(most < (1ll << 31) - 1 ? most : (1ll << 31) - 1);
        for (int r : {rows, rows > 7 ? rows - 7 : rows, rows / 2 + 1})
            if (r > 0 && tmt::mx_tiles(r, (int)K) >= 1 << 24) {
                std::printf("rows %d, K %lld: %lld tiles\n", r, (long long)K, (long long)tmt::mx_tiles(r, (int)K));
                return 1;
            }
    }
    std::printf("ok\n");
    return 0;
}
"""


def test_the_most_rows_fit_a_launch(tmp_path):
    _run(tmp_path, LARGEST)


# The load cursors of the kernels, walked as the kernels walk them. Operands
# are address ranges of exactly their size; nothing is read.
CURSORS = r"""
#include <cstdio>
#include <cstdlib>
#include <type_traits>
#include <vector>
#include "linear_plan.hpp"
using namespace tmt;
struct Span {
    uint64_t beg, end;
};
struct Case {
    LinearOp op;
    LinearParams p;
    Span x, xs, w, ws, y;
    const char* text;
};
#define FAIL(...)                    \
    do {                             \
        std::printf(__VA_ARGS__);    \
        std::printf(" (%s op %d T %d N %d K %d ldx %lld wlds %lld)\n", c.text, c.op, c.p.T, c.p.N, c.p.K, (long long)c.p.ldx, (long long)c.p.wlds); \
        std::exit(1);                \
    } while (0)
// A window begins at `at`, holds what a step needs, up to `need`, and ends
// inside its operand.
void look(const Case& c, const char* what, const Window& w, const Span& s, uint64_t at, uint64_t need) {
    if (w.at != at) FAIL("%s begins at %llx, not %llx", what, (unsigned long long)w.at, (unsigned long long)at);
    if (w.at + w.bytes < need) FAIL("%s ends before the step's data", what);
    if (w.at < s.beg || w.at + w.bytes > s.end) FAIL("%s passes its operand", what);
}
void empty(const Case& c, const char* what, const Window& w) {
    if (w.bytes != 0) FAIL("%s is not empty behind the last unit", what);
}
template <int TILE, bool SPLIT>
std::vector<Unit> units(const LinearPlan& pl, int R, int block, int grid) {
    std::vector<Unit> out;
    Unit u;
    for (int vb = block; unit_at<TILE, SPLIT>(pl, R, vb, u); vb += grid) out.push_back(u);
    return out;
}
constexpr int kBehind = 6;  // moves past the last step

template <int OP, int TILE, bool SPLIT>
void walk(const Case& c, const LinearPlan& pl, int block, int grid, const std::vector<Unit>& us) {
    const LinearParams& p = c.p;
    if constexpr (OP == LINEAR_FORWARD) {
        FwdCursor<TILE, SPLIT> at;
        at.vl = block;
        at.set(p, us[0]);
        for (const Unit& u : us)
            for (int k = u.kbeg; k < u.kend; k += 64) {
                const int rows = std::min(p.T - u.m0, TILE), cols = std::min(p.N - u.c0, TILE);
                const uint64_t a = c.x.beg + ((uint64_t)u.m0 * p.ldx + k) * 2, q = c.w.beg + (uint64_t)u.c0 * (p.K / 2) + k / 2;
                const uint64_t s = c.ws.beg + (uint64_t)(k / 32) * p.wlds + u.c0;
                look(c, "X", at.wa, c.x, a, a + (uint64_t)(rows - 1) * p.ldx * 2 + 128);
                look(c, "codes", at.wq, c.w, q, q + (uint64_t)(cols - 1) * (p.K / 2) + 32);
                look(c, "scales", at.wsc, c.ws, s, s + p.wlds + cols);
                at.next(p, pl, [grid] { return grid; });
            }
        for (int i = 0; i < kBehind; ++i, at.next(p, pl, [grid] { return grid; })) empty(c, "X", at.wa), empty(c, "codes", at.wq), empty(c, "scales", at.wsc);
    } else if constexpr (OP == LINEAR_MATMUL && TILE == 128) {
        for (bool of_w : {false, true}) {
            MxCursor<TILE, SPLIT> at;
            at.vl = block;
            at.of_w = of_w;
            at.set(p, us[0]);
            for (const Unit& u : us)
                for (int k = u.kbeg; k < u.kend; k += 256) {
                    if (!at.left) FAIL("the loads stop early");
                    const int rows = std::min(p.T - u.m0, TILE), cols = std::min(p.N - u.c0, TILE), n = std::min(256, p.K - k);
                    const uint64_t a = c.x.beg + (uint64_t)u.m0 * (p.K / 2) + k / 2, q = c.w.beg + (uint64_t)u.c0 * (p.K / 2) + k / 2;
                    const Span& sp = of_w ? c.ws : c.xs;
                    const uint64_t lds = of_w ? p.wlds : p.xlds, s = sp.beg + (uint64_t)(k / 32) * lds + (of_w ? u.c0 : u.m0);
                    look(c, "X", at.wx, c.x, a, a + (uint64_t)(rows - 1) * (p.K / 2) + n / 2);
                    look(c, "codes", at.ww, c.w, q, q + (uint64_t)(cols - 1) * (p.K / 2) + n / 2);
                    look(c, "scales", at.wsc, sp, s, s + (n / 32 - 1) * lds + (of_w ? cols : rows));
                    at.next(p, pl, [grid] { return grid; });
                }
            if (at.left) FAIL("the loads do not stop");
        }
    } else if constexpr (OP == LINEAR_MATMUL) {
        for (bool of_w : {false, true}) {
            MxLargeCursor<TILE> at;
            at.vl = block;
            at.of_w = of_w;
            at.set(p, us[0]);
            for (const Unit& u : us)
                for (int k = 0; k < p.K; k += 256) {
                    const int rows = std::min(p.T - u.m0, TILE), cols = std::min(p.N - u.c0, TILE);
                    const uint64_t a = c.x.beg + (uint64_t)u.m0 * (p.K / 2) + k / 2, q = c.w.beg + (uint64_t)u.c0 * (p.K / 2) + k / 2;
                    const Span& sp = of_w ? c.ws : c.xs;
                    const uint64_t lds = of_w ? p.wlds : p.xlds, s = sp.beg + (uint64_t)(k / 32) * lds + (of_w ? u.c0 : u.m0);
                    look(c, "X", at.wx, c.x, a, a + (uint64_t)(rows - 1) * (p.K / 2) + 128);
                    look(c, "codes", at.ww, c.w, q, q + (uint64_t)(cols - 1) * (p.K / 2) + 128);
                    look(c, "scales", at.wsc, sp, s, s + 7 * lds + (of_w ? cols : rows));
                    at.next(p, pl, [grid] { return grid; });
                }
            for (int i = 0; i < kBehind; ++i, at.next(p, pl, [grid] { return grid; })) empty(c, "X", at.wx), empty(c, "codes", at.ww), empty(c, "scales", at.wsc);
        }
    } else {
        constexpr bool DW = OP == LINEAR_DW;
        GradCodesCursor<OP, TILE, SPLIT> cq;
        GradRowsCursor<OP, TILE, SPLIT> ca;
        cq.vl = ca.vl = block;
        cq.set(p, us[0]);
        ca.set(p, us[0]);
        const uint64_t rowb = DW ? p.K : p.K / 2, ldb = p.ldx * 2;
        for (const Unit& u : us)
            for (int k = u.kbeg; k < u.kend; k += 64) {
                const int rows = std::min(64, u.kend - k), cols = std::min(p.K - u.c0, TILE);
                const uint64_t q = c.w.beg + (uint64_t)k * rowb + (DW ? u.c0 : u.c0 / 2);
                const uint64_t s = c.ws.beg + (uint64_t)(u.c0 / 32) * p.wlds + k;
                look(c, "codes", cq.wq, c.w, q, q + (uint64_t)(rows - 1) * rowb + (DW ? cols : cols / 2));
                look(c, "scales", cq.wsc, c.ws, s, s + (uint64_t)(cols / 32 - 1) * p.wlds + rows);
                if (cq.wq.at + cq.wq.bytes > c.w.beg + (uint64_t)(k + rows) * rowb) FAIL("codes pass the unit's rows");
                if (cq.rows != u.kend - k) FAIL("%d rows left, not %d", cq.rows, u.kend - k);
                if constexpr (DW) {
                    const uint64_t a = c.x.beg + (uint64_t)k * ldb + u.m0 * 2;
                    look(c, "dY", ca.wa, c.x, a, a + (uint64_t)(rows - 1) * ldb + std::min(p.N - u.m0, TILE) * 2);
                    if (ca.wa.at + ca.wa.bytes > c.x.beg + (uint64_t)(k + rows) * ldb) FAIL("dY passes the unit's rows");
                } else {
                    const uint64_t a = c.x.beg + ((uint64_t)u.m0 * p.ldx + k) * 2;
                    look(c, "dY", ca.wa, c.x, a, a + (uint64_t)(std::min(p.T - u.m0, TILE) - 1) * ldb + std::min(64, p.N - k) * 2);
                }
                cq.next(p, pl, [grid] { return grid; });
                ca.next(p, pl, [grid] { return grid; });
            }
        for (int i = 0; i < kBehind; ++i, cq.next(p, pl, [grid] { return grid; }), ca.next(p, pl, [grid] { return grid; })) {
            empty(c, "dY", ca.wa), empty(c, "codes", cq.wq), empty(c, "scales", cq.wsc);
            if (cq.rows > 0) FAIL("rows behind the last unit");
        }
    }
}

// A launch: every tile (or part) once, its loads, and its waves' outputs.
template <int OP, int TILE, bool SPLIT>
void launch(const Case& c, const LinearPlan& pl, int cus) {
    const Sizes z = sizes(c.op, c.p.T, c.p.N, c.p.K);
    const int n = SPLIT ? pl.tail * pl.parts : pl.whole;
    if (n == 0) return;
    const int grid = unit_grid(TILE, n, cus);
    std::vector<int> seen(n);
    for (int b = 0; b < grid; ++b) {
        const std::vector<Unit> us = units<TILE, SPLIT>(pl, z.R, b, grid);
        if (us.empty()) continue;
        walk<OP, TILE, SPLIT>(c, pl, b, grid, us);
        for (const Unit& u : us) {
            if (u.part < 0 || u.part >= n || seen[u.part]++) FAIL("unit %d twice or none", u.part);
            if (u.m0 >= z.M || u.c0 >= z.C || u.kbeg >= u.kend || u.kend > z.R) FAIL("unit %d is outside", u.part);
            for (int wave = 0; wave < 4; ++wave) {
                const int wrow = (wave >> 1) * (TILE / 2), wcol = (wave & 1) * (TILE / 2);
                const int rows = std::min(z.M - u.m0 - wrow, TILE / 2), cols = std::min(z.C - u.c0 - wcol, TILE / 2);
                if (rows <= 0 || cols <= 0) continue;
                const int size = OP == LINEAR_DW ? 4 : 2;
                const uint64_t o = c.y.beg + ((uint64_t)(u.m0 + wrow) * c.p.ldy + u.c0 + wcol) * size;
                const uint32_t bytes = output_window(rows, (uint32_t)(c.p.ldy * size), cols, size);
                if (o + bytes > c.y.end) FAIL("outputs pass their matrix");
                if (o + bytes < o + (uint64_t)(rows - 1) * c.p.ldy * size + cols * size) FAIL("outputs are cut off");
                if (bytes > 0x80000000u) FAIL("an offset past the columns is inside the window");
            }
        }
    }
    for (int i = 0; i < n; ++i)
        if (!seen[i]) FAIL("unit %d is missing", i);
}
template <int OP, int TILE>
void launches(const Case& c, const LinearPlan& pl, int cus) {
    launch<OP, TILE, false>(c, pl, cus);
    if constexpr (OP != LINEAR_MATMUL || TILE == 128) launch<OP, TILE, true>(c, pl, cus);
}
template <int OP>
void plans(const Case& c, int cus) {
    const LinearParams& p = c.p;
    const Sizes z = sizes(c.op, p.T, p.N, p.K);
    double us;
    const LinearPlan own = linear_plan(c.op, p.T, p.N, p.K, cus, &us);
    if (own.tile == 256) launches<OP, 256>(c, own, cus);
    else launches<OP, 128>(c, own, cus);
    for (int parts : {1, 2, 3, 5, 13}) {  // others
        if (parts > 1 && (z.R + 63) / 64 < parts * kMinSteps) continue;
        launches<OP, 128>(c, plan_tiles(z, 128, parts, cus), cus);
        if (OP != LINEAR_MATMUL) launches<OP, 256>(c, plan_tiles(z, 256, parts, cus), cus);
    }
    if (OP == LINEAR_MATMUL && p.K % 256 == 0) launches<OP, 256>(c, plan_tiles(z, 256, 1, cus), cus);
}
Case make(LinearOp op, int T, int N, int K, int64_t pad, int64_t spad, const char* text) {
    Case c{};
    c.op = op;
    c.text = text;
    LinearParams& p = c.p;
    p.T = T, p.N = N, p.K = K;
    const int cols = op == LINEAR_FORWARD ? K : N, mx = op == LINEAR_DW ? T : N, out = op == LINEAR_FORWARD || op == LINEAR_MATMUL ? N : K;
    const auto up16 = [](int64_t n) { return (n + 15) / 16 * 16; };
    p.ldx = pad < 0 ? kMaxStride : cols + pad;
    p.ldy = pad < 0 ? kMaxStride : out + pad;
    p.wlds = spad < 0 ? kMaxScaleStride : up16(mx) + spad;
    p.xlds = spad < 0 ? kMaxScaleStride : up16(T) + spad;
    c.w = {1ull << 40, (1ull << 40) + (uint64_t)mx * (op == LINEAR_DW ? K : K / 2)};
    c.ws = {2ull << 40, (2ull << 40) + (uint64_t)(K / 32) * p.wlds};
    if (op == LINEAR_MATMUL) {
        c.x = {3ull << 40, (3ull << 40) + (uint64_t)T * (K / 2)};
        c.xs = {4ull << 40, (4ull << 40) + (uint64_t)(K / 32) * p.xlds};
        p.xq = (const uint8_t*)c.x.beg, p.xs = (const uint8_t*)c.xs.beg;
    } else {
        c.x = {3ull << 40, (3ull << 40) + ((uint64_t)(T - 1) * p.ldx + cols) * 2};
        p.x = (const uint16_t*)c.x.beg;
    }
    p.w = (const uint8_t*)c.w.beg, p.ws = (const uint8_t*)c.ws.beg;
    const int rows = op == LINEAR_DW ? N : T, size = op == LINEAR_DW ? 4 : 2;
    c.y = {5ull << 40, (5ull << 40) + ((uint64_t)(rows - 1) * p.ldy + out) * size};
    return c;
}
int main() {
    static const int shapes[][3] = {
        {1, 16, 64}, {1, 4096, 1024}, {15, 272, 64}, {17, 128, 320}, {127, 144, 448}, {128, 128, 128}, {129, 144, 192},
        {255, 272, 320}, {256, 256, 256}, {257, 528, 576}, {300, 16, 4096}, {300, 256, 320}, {777, 1024, 4096}, {777, 4096, 960},
        {1024, 256, 256}, {2048, 1280, 1280}, {2049, 1296, 1344}, {5003, 1008, 960}, {40001, 1024, 256}, {16300, 2000, 2048},
        {70 * 256, 1024, 4096}, {70 * 256, 4096, 1024}, {20011, 2736, 704}, {4096, 4096, 4096}, {256, 65536, 256}, {256, 256, 65536}};
    for (auto& s : shapes)
        for (int pad = 0; pad < 3; ++pad) {
            const int64_t x = pad == 0 ? 0 : pad == 1 ? 8 : -1, sp = pad == 0 ? 0 : pad == 1 ? 16 : -1;
            for (int cus : {256, 80}) {
                plans<LINEAR_FORWARD>(make(LINEAR_FORWARD, s[0], s[1], s[2], x, sp, "Y"), cus);
                plans<LINEAR_MATMUL>(make(LINEAR_MATMUL, s[0], s[1], s[2], x, sp, "both"), cus);
                plans<LINEAR_DX>(make(LINEAR_DX, s[0], s[1], s[2], x, sp, "dX"), cus);
                plans<LINEAR_DW>(make(LINEAR_DW, s[0], s[1], s[2], x, sp, "dW"), cus);
            }
        }
    // a lane's offset inside a window is 32 bits: 256 rows of an operand along
    // the reduction, 64 of one across it, 8 blocks' scales, 128 rows of outputs
    static_assert(255 * 2 * kMaxStride + 2 * 64 < (1ll << 32) && 63 * 2 * kMaxStride + 2 * 256 < (1ll << 32), "rows");
    static_assert(8 * kMaxScaleStride < (1ll << 31), "scales");
    static_assert(127 * 4 * kMaxStride + 4 * 128 <= 0x80000000ll, "outputs");
    std::printf("ok\n");
    return 0;
}
"""


def test_every_window_ends_inside_its_operand(tmp_path):
    """The products' loads and stores: every unit once, every step's data in its
    windows, no window past its operand's last byte, none that is not empty
    behind the last unit."""
    _run(tmp_path, CURSORS)


def test_few_tokens_need_no_workspace():
    """The kernel for few tokens uses none, so none is asked for."""
    for T, N, K in ((1, 4096, 1024), (1, 4096, 4096), (16, 1024, 4096), (64, 1024, 4096), (64, 4096, 1024), (200, 256, 4096)):
        assert tmt_moe.linear_workspace_size(tmt_moe.LINEAR_FORWARD, T, N, K) == 0, (T, N, K)


def test_a_workspace_of_both_operands_in_mxfp4():
    """Split products of two MXFP4 operands are 128 x 128 tiles in fp32, two for
    each of 256 compute units."""
    for T, N, K in ((777, 1024, 4096), (65536, 4096, 4096)):
        assert tmt_moe.linear_workspace_size(tmt_moe.LINEAR_MATMUL, T, N, K) == 512 * 128 * 128 * 4


WORKSPACES = r"""
#include <cstdio>
#include <random>
#include "linear_plan.hpp"
using namespace tmt;
// What launch_linear's choice of kernel writes as partial tiles.
static size_t used(LinearOp op, int T, int N, int K, int cus) {
    if (op == LINEAR_MATMUL && mx_large(T, N, K, cus)) return 0;
    double us;
    const LinearPlan pl = linear_plan(op, T, N, K, cus, &us);
    if (op == LINEAR_FORWARD && rows_time(T, N, K) <= us) return 0;
    return (size_t)pl.tail * pl.parts * pl.tile * pl.tile * 4;
}
int main() {
    std::mt19937 rng(5);
    auto log_uniform = [&](double lo, double hi) { return std::exp2(std::uniform_real_distribution<double>(std::log2(lo), std::log2(hi))(rng)); };
    int none = 0, split = 0;
    for (int i = 0; i < 20000; ++i) {
        const LinearOp op = (LinearOp)(i % 4);
        const int N = 16 * (int)log_uniform(1, 1025), K = 64 * (int)log_uniform(1, 257), T = (int)log_uniform(1, 70000);
        const int cus = i % 3 ? 256 : 80;
        const size_t bound = workspace_bound(op, T, N, K, cus);
        none += bound == 0;
        for (int j = 0; j < 24; ++j) {
            const int t = j == 0 ? T : 1 + (int)(rng() % (unsigned)T);
            const size_t use = used(op, t, N, K, cus);
            split += use > 0;
            if (use > bound) {
                std::printf("op %d T %d of %d N %d K %d: %zu of %zu bytes\n", op, t, T, N, K, use, bound);
                return 1;
            }
            if (workspace_bound(op, t, N, K, cus) > bound) {
                std::printf("op %d T %d N %d K %d: fewer tokens ask for more\n", op, t, N, K);
                return 1;
            }
        }
    }
    if (none < 2000 || split < 20000) {  // both kinds were drawn
        std::printf("%d without, %d split\n", none, split);
        return 1;
    }
    std::printf("ok\n");
    return 0;
}
"""


def test_a_workspace_holds_every_split(tmp_path):
    """The partial tiles of any call of up to T tokens fit a workspace for T."""
    _run(tmp_path, WORKSPACES)
