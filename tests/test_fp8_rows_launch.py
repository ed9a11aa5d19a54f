"""The kernel for few rows of the 8-bit linear layer walked on the host, from the header that it
uses: every lane of every load finds its codes in its operand, or zeros past a window, at the
place in LDS that it is read from. With the compiler's check of signed overflow, which ends
the program."""
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
#include <vector>
#include "fp8_plan.hpp"
using namespace tmt;
#define FAIL(...)                \
    do {                         \
        std::printf(__VA_ARGS__); \
        std::printf(" (M %d N %d K %d lda %lld block %u of %d x %d)\n", p.M, p.N, p.K, (long long)p.lda, block, RB, NB); \
        std::exit(1);            \
    } while (0)

// One operand's loads of the block of the reduction from k on: `rows` of `all` from `first` on.
void codes(const Fp8Params& p, const Window& w, uint64_t base, int64_t ld, int first, int rows, int all, int loads, int k, unsigned block, int RB, int NB) {
    const uint64_t end = base + (uint64_t)(all - 1) * ld + ((p.K + 15) & ~15);
    if (w.at + w.bytes > end) FAIL("the window passes the operand");
    for (int lane = 0; lane < 64; ++lane) {
        const int chunk = row_chunk(lane);
        const uint32_t row = (uint32_t)(lane >> 3) * (uint32_t)ld;
        for (int i = 0; i < loads; ++i) {
            const int r = 8 * i + (lane >> 3), c = (lane & 7) ^ ((r & 15) >> 1);  // of the LDS row; what it is read as
            if ((chunk ^ (4 * (i & 1))) != c) FAIL("lane %d of load %d holds another chunk", lane, i);
            const uint32_t off = row_chunk_at(p.K, k, chunk ^ (4 * (i & 1))) + row + (uint32_t)(8 * i) * (uint32_t)ld;
            const bool in = r < rows && k + 16 * c < p.K;
            if (in != (off < w.bytes) || (in && off + 16 > w.bytes)) FAIL("row %d chunk %d at %d: offset %u of %u", r, c, k, off, w.bytes);
            if (in && w.at + off != base + (uint64_t)(first + r) * ld + k + 16 * c) FAIL("row %d chunk %d at %d lies elsewhere", r, c, k);
        }
    }
}

template <bool TILES, int RB, int NB>
void blocks(const Fp8Params& p) {
    const unsigned grid = (unsigned)((int64_t)((p.N + 16 * NB - 1) / (16 * NB)) * ((p.M + 16 * RB - 1) / (16 * RB)));
    const int kbs = (p.K + 127) / 128, nbs = (p.N + 127) / 128;
    const uint64_t a = address(p.a), b = address(p.b);
    const uint64_t as_end = address(p.as + (int64_t)(kbs - 1) * p.ldas + p.M);
    const uint64_t bs_end = TILES ? address(p.bs + (int64_t)(nbs - 1) * p.ldbs + kbs) : address(p.bs + (int64_t)(kbs - 1) * p.ldbs + p.N);
    std::vector<char> outputs((size_t)p.M * p.N);
    for (unsigned block = 0; block < grid; ++block) {
        RowBlock<TILES, RB, NB> at;
        at.set(p, block);
        if (at.rows < 1 || at.cols < 1 || at.rows > 16 * RB || at.cols > 16 * NB) FAIL("%d rows, %d columns", at.rows, at.cols);
        for (int m = 0; m < at.rows; ++m)
            for (int n = 0; n < at.cols; ++n)
                if (at.m0 + m >= p.M || at.n0 + n >= p.N || outputs[(size_t)(at.m0 + m) * p.N + at.n0 + n]++) FAIL("output %d %d twice", at.m0 + m, at.n0 + n);
        if (TILES && at.n0 / 128 != (at.n0 + at.cols - 1) / 128) FAIL("columns of two tiles");
        int seen = 0;
        for (int wave = 0; wave < 8; ++wave) {
            const int steps = (kbs - wave + 7) / 8;
            for (int n = 0; n < steps; ++n, ++seen) {
                const int kb = wave + n * 8;
                if (kb >= kbs) FAIL("block %d of the reduction", kb);
                codes(p, at.wa, a, p.lda, at.m0, at.rows, p.M, 2 * RB, kb * 128, block, RB, NB);
                codes(p, at.wb, b, p.ldb, at.n0, at.cols, p.N, 2 * NB, kb * 128, block, RB, NB);
                const Window sa = at.a_scales(p, kb), sb = at.b_scales(p, kb);
                if (sa.at != address(p.as + (int64_t)kb * p.ldas + at.m0) || sa.bytes != 4u * at.rows || sa.at + sa.bytes > as_end) FAIL("scales of a");
                const uint64_t want = TILES ? address(p.bs + (int64_t)(at.n0 / 128) * p.ldbs + kb) : address(p.bs + (int64_t)kb * p.ldbs + at.n0);
                if (sb.at != want || sb.bytes != (TILES ? 4u : 4u * at.cols) || sb.at + sb.bytes > bs_end) FAIL("scales of b");
            }
        }
        if (seen != kbs) FAIL("%d blocks of the reduction", seen);
    }
    const unsigned block = grid;
    for (char c : outputs)
        if (c != 1) FAIL("an output is missing");
}

template <bool TILES>
void product(int M, int N, int K, int64_t lda, int64_t ldb) {
    Fp8Params p{};
    p.M = M, p.N = N, p.K = K, p.lda = lda, p.ldb = ldb;
    p.ldas = M + 3;
    p.ldbs = TILES ? (K + 127) / 128 + 1 : N + 5;
    p.a = reinterpret_cast<const uint8_t*>(0x100000000000ull);
    p.b = reinterpret_cast<const uint8_t*>(0x200000000000ull);
    p.as = reinterpret_cast<const float*>(0x300000000000ull);
    p.bs = reinterpret_cast<const float*>(0x400000000000ull);
    blocks<TILES, 1, 1>(p);
    blocks<TILES, 1, 2>(p);
    blocks<TILES, 2, 2>(p);
    blocks<TILES, 4, 4>(p);
}

template <int RB, int NB, bool ONE>
void slot() {
    using S = RowSlot<RB, NB, ONE>;
    // 1 KiB a load of codes, 256 bytes a load of scales, which 16 RB and 16 NB rows fill at most
    static_assert(S::SA == 1024 * (S::ND - 2) && S::SB - S::SA >= 64 * RB && S::BYTES - S::SB >= 64 * NB && S::SB - S::SA >= 256 && S::BYTES - S::SB >= 256, "slot");
}

int main() {
    slot<1, 1, true>(), slot<1, 1, false>(), slot<1, 2, true>(), slot<1, 2, false>(), slot<2, 2, true>(), slot<2, 2, false>(), slot<4, 4, true>();
    for (int M : {1, 2, 16, 17, 33, 64, 130})
        for (int N : {8, 24, 136, 264})
            for (int K : {1, 15, 16, 100, 128, 129, 1000, 2056}) {
                const int64_t k16 = (K + 15) / 16 * 16;
                product<true>(M, N, K, k16, k16 + 16);
                product<false>(M, N, K, k16 + 48, k16);
            }
    // the widest strides and the longest rows
    product<true>(130, 136, 4097, 1 << 22, 1 << 22);
    product<false>(5, 24, 1 << 22, 1 << 22, 1 << 22);
    std::printf("ok\n");
    return 0;
}
"""


def test_the_kernel_for_few_rows(tmp_path):
    src, exe = tmp_path / "walk.hip", tmp_path / "walk"
    src.write_text(WALK)
    r = subprocess.run([HIPCC, "--offload-host-only", "-std=c++17", "-O1", "-I", CSRC,
                        "-Xarch_host", "-fsanitize=signed-integer-overflow",
                        "-Xarch_host", "-fsanitize-trap=signed-integer-overflow",
                        str(src), "-o", str(exe)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout == "ok\n", (r.returncode, r.stdout[-500:])
