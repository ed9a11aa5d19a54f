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
